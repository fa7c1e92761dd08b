// Causal attention over packed sequences of different lengths with grouped heads, forward and backward, head_dim 64 or 128.
//
//   rows [cu[i], cu[i+1]) are sequence i;  key j is visible to query i of the same sequence iff i - window <= j <= i
//   O = softmax(scale Q K^T) V per query head; G = H / KV query heads read one key head
//   dP = dO V^T;  dS = P (dP - rowsum(dO o O));  dQ = scale dS K;  dK = scale dS^T Q;  dV = P^T dO, the last two summed over
//   the G query heads of a key head
//
// A query tile is P = 128 / G positions x the G heads of one key head (row = position * G + head): one K / V tile serves the whole
// group, a short sequence fills more of a tile, and the key-stationary backward sums over the group inside its accumulators, in a
// fixed order and without atomics.  A TMA box {64, G, 1, P} over the [D, G, KV, rows] view of the queries lays that tile out.
//
// Tiles never span two sequences.  Which tiles there are depends on lengths that only the device knows, so a plan kernel writes
// two work lists (query tiles, key tiles), longest first within a span of rows whose K and V stay in L2.  What a tile loads beyond the end of its sequence (another
// sequence's rows, or rows behind the last one, with any values in them) is set to zero in shared memory before a product sums
// over it, so the results of a sequence do not depend on what surrounds it, bit for bit.
//
// The inner pipelines are those of attn_fwd4_sm100.cu (forward: two CTAs per SM) and attn_wide_sm100.cu (backward: ten warps, two-phase
// softmax); what is said there about the MMA order, the TMEM reuse and their bounds holds here too.
#include "attn_common.cuh"

namespace arb {

constexpr long long PACKED_MAX_ROWS = 1ll << 30;
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_LEVELS = 64, PLAN_SPANS = 32, PLAN_BINS = PLAN_LEVELS * PLAN_SPANS;

// One tile: rows [start, start + len) are its sequence and `tile` its number there.  tile < 0: rows that belong to no sequence and
// whose outputs are zero; len = 0: nothing.
struct PackedItem { int start, len, tile, pad; };
static_assert(sizeof(PackedItem) == 16, "read as one 16-byte word");

struct PackedArgs {
  const PackedItem* items_q;
  const PackedItem* items_k;
  int n_q, n_k;                      // capacities of the lists
  int KV, G, P;                      // key heads, query heads per key head, positions per query tile
  int head_span;                     // key heads whose tiles are interleaved
  int window;
  float scale;
  __nv_bfloat16* o;                  // forward: O; backward: dQ.  Row stride in elements, heads D apart
  long long ldo;
  int8_t* o_lo;                      // forward: what the rounding of O to bf16 left over (rest_of), or null
  int* next;                         // backward: [2] next tile of the key and of the query list
  float* lse;                        // [rows, H]
  const float* delta;                // [rows, H]
  __nv_bfloat16* dk;
  __nv_bfloat16* dv;
  long long lddk, lddv;
  int* err;
};

// -----------------------------------------------------------------------------------------------
// plan
// -----------------------------------------------------------------------------------------------
struct PlanArgs {
  const int* cu;                     // [n + 1]
  int n, rows, P;
  int span_rows[2];                  // rows per span of the query and of the key list
  int* bound;                        // [2][n + 3] scratch: first row of each sequence, the rows before and behind them included
  int* first;                        // [2][n + 3] scratch: first tile of each
  PackedItem* items[2];
  int cap[2];
  int* err;
};

// inclusive scan over the block, v in thread order; `shared` holds 32 values
template <typename Op>
__device__ __forceinline__ int block_scan(int v, int* shared, Op op, int neutral) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = op(u, v);
  }
  __syncthreads();
  if (lane == 31) shared[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = shared[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w = op(u, w);
    }
    shared[lane] = w;
  }
  __syncthreads();
  return op(warp ? shared[warp - 1] : neutral, v);
}

// Block 0 writes the query tiles, block 1 the key tiles.  Three passes over the sequences (their bounds, made ascending and kept
// within the rows whatever cu holds; tile counts) and two over the tiles (a counting sort by span of rows, then work).
__global__ void __launch_bounds__(PLAN_THREADS) packed_plan_k(const PlanArgs p) {
  __shared__ int bins[PLAN_BINS];
  __shared__ int shared[32];
  __shared__ int s_carry, s_longest, s_bad;
  const int tid = threadIdx.x, which = blockIdx.x;
  const int step = which ? 128 : p.P;                    // positions per tile
  const int n_seq = p.n + 2;                             // rows before the first sequence, the sequences, rows behind the last
  int* bound = p.bound + (long long)which * (p.n + 3);
  int* first = p.first + (long long)which * (p.n + 3);
  auto add = [](int a, int b) { return a + b; };
  auto most = [](int a, int b) { return max(a, b); };
  grid_enter();
  for (int i = tid; i < PLAN_BINS; i += PLAN_THREADS) bins[i] = 0;
  if (tid == 0) { s_carry = 0; s_longest = 0; s_bad = 0; }
  __syncthreads();
  // bounds: 0, cu[0], ..., cu[n], rows
  for (int base = 0; base < p.n + 3; base += PLAN_THREADS) {
    const int i = base + tid;
    int v = 0;
    if (i >= 1 && i <= p.n + 1) {
      const int c = p.cu[i - 1];
      v = min(max(c, 0), p.rows);
      if (c != v || (i > 1 && c < p.cu[i - 2])) s_bad = 1;
    } else if (i > p.n + 1) {
      v = p.rows;
    }
    const int carry = s_carry;
    const int b = max(carry, block_scan(v, shared, most, 0));
    if (i < p.n + 3) bound[i] = b;
    __syncthreads();
    if (tid == PLAN_THREADS - 1) s_carry = b;
    __syncthreads();
  }
  if (tid == 0) s_carry = 0;
  __syncthreads();
  for (int base = 0; base < n_seq; base += PLAN_THREADS) {
    const int i = base + tid;
    int t = 0;
    if (i < n_seq) {
      const int len = bound[i + 1] - bound[i];
      t = (len + step - 1) / step;
      if (i > 0 && i < n_seq - 1) atomicMax(&s_longest, len);
    }
    const int carry = s_carry;
    const int s = carry + block_scan(t, shared, add, 0);
    if (i < n_seq) first[i + 1] = s;
    __syncthreads();
    if (tid == PLAN_THREADS - 1) s_carry = s;
    __syncthreads();
  }
  if (tid == 0) first[0] = 0;
  __syncthreads();
  const int tiles = min(s_carry, p.cap[which]);
  const int other = which ? p.P : 128;                   // positions per tile of the other side
  const int most_work = s_longest / other + 2;
  auto item_of = [&](int t, PackedItem& it) -> int {     // the tile and its bin
    int lo = 0, hi = n_seq - 1;                          // last sequence whose first tile is <= t; empty ones share theirs with the next
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= t) lo = mid; else hi = mid - 1;
    }
    const bool dead = lo == 0 || lo == n_seq - 1;
    const int start = bound[lo], len = bound[lo + 1] - start, k = t - first[lo];
    it.pad = 0;
    if (dead) {
      it.start = start + k * step; it.len = min(step, len - k * step); it.tile = -1;
      return PLAN_BINS - 1;
    }
    it.start = start; it.len = len; it.tile = k;
    const int work = which ? (len - k * 128 - 1) / other + 1 : min(len - 1, k * step + step - 1) / 128 + 1;
    const int level = min(PLAN_LEVELS - 1, int((long long)work * PLAN_LEVELS / most_work));
    return min(start / p.span_rows[which], PLAN_SPANS - 1) * PLAN_LEVELS + (PLAN_LEVELS - 1 - level);
  };
  for (int t = tid; t < tiles; t += PLAN_THREADS) {
    PackedItem it;
    atomicAdd(&bins[item_of(t, it)], 1);
  }
  __syncthreads();
  if (tid == 0) s_carry = 0;
  __syncthreads();
  for (int base = 0; base < PLAN_BINS; base += PLAN_THREADS) {
    const int v = bins[base + tid];
    const int carry = s_carry;
    const int s = carry + block_scan(v, shared, add, 0);
    bins[base + tid] = s - v;
    __syncthreads();
    if (tid == PLAN_THREADS - 1) s_carry = s;
    __syncthreads();
  }
  for (int t = tid; t < tiles; t += PLAN_THREADS) {
    PackedItem it;
    const int b = item_of(t, it);
    p.items[which][atomicAdd(&bins[b], 1)] = it;          // the order inside a bin decides when a tile runs, not what it computes
  }
  for (int t = tiles + tid; t < p.cap[which]; t += PLAN_THREADS) p.items[which][t] = PackedItem{0, 0, 0, 0};
  if (tid == 0 && which == 0 && s_bad && p.err) atomicExch(p.err, ERR_SEQLENS);
}

// -----------------------------------------------------------------------------------------------
// shared pieces
// -----------------------------------------------------------------------------------------------
// Which tile of which key head a CTA of the flat grid takes: spans of heads one after the other, inside them the head changes
// fastest, so that the list's order (long tiles first) holds across heads.
struct PackedTile { PackedItem it; int kv; };
__device__ __forceinline__ PackedTile packed_tile(const PackedArgs& p, const PackedItem* items, int n, int block) {
  const int per = p.head_span * n, g = block / per, i = block - g * per;
  const int heads = min(p.head_span, p.KV - g * p.head_span);
  PackedTile t;
  const int k = i / heads;
  const int4 v = k < n ? *reinterpret_cast<const int4*>(items + k) : make_int4(0, 0, 0, 0);
  t.it = PackedItem{v.x, v.y, v.z, v.w};
  t.kv = g * p.head_span + i - k * heads;
  return t;
}

// A wait of a whole warp: all of its lanes go on, or none does, so that the warp stays together where a wait runs out.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
}

// Bits of the visible ones of 32 columns, those of [lo, hi] (relative to the first).  A masked score becomes -inf in its register, a
// bit test and a select per element; comparing every column with the row's interval takes three instructions, in both passes over
// the scores.
__device__ __forceinline__ uint32_t visible(int lo, int hi) {
  const int a = max(lo, 0), b = min(hi, 31);
  return b < a ? 0u : ((2u << b) - 1u) & ~((1u << a) - 1u);      // 2 << 31 is 0: all bits from a
}
__device__ __forceinline__ void hide(uint32_t (&s)[32], uint32_t bits) {
#pragma unroll
  for (int j = 0; j < 32; ++j) s[j] = (bits & (1u << j)) ? s[j] : 0xff800000u;
}

// CTAs stay and take tile after tile: barriers, TMEM and the pipeline's start are paid once, and a tile's first loads run under the
// previous tile's last products and epilogue (as one CTA per tile, sequences of 128 rows cost 10 us of an SM per backward tile).
// The loading warp decides which tile is next and hands it to the other roles through two slots.
struct PackedSlot { int start, len, tile, kv; };       // len = 0: no more tiles
struct SlotRing {
  uint64_t* full;                                       // [2] 1 arrival
  uint64_t* empty;                                      // [2] one arrival per consumer
  PackedSlot* slot;                                     // [2]
  volatile int* abort_flag;
  __device__ __forceinline__ void init(int consumers) {
    for (int i = 0; i < 2; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], uint32_t(consumers)); }
  }
  // by one thread
  __device__ __forceinline__ bool put(int n, const PackedTile& t) {
    if (!mbar_wait(&empty[n & 1], (uint32_t(n >> 1) & 1u) ^ 1u, abort_flag)) return false;
    slot[n & 1] = PackedSlot{t.it.start, t.it.len, t.it.tile, t.kv};
    mbar_arrive(&full[n & 1]);
    return true;
  }
  // by one thread
  __device__ __forceinline__ PackedSlot take(int n) {
    if (!mbar_wait(&full[n & 1], uint32_t(n >> 1) & 1u, abort_flag)) return PackedSlot{0, 0, 0, 0};
    const PackedSlot s = slot[n & 1];
    mbar_arrive(&empty[n & 1]);
    return s;
  }
  // by a whole warp
  __device__ __forceinline__ PackedSlot take_warp(int n, int lane) {
    if (!wait_warp(&full[n & 1], uint32_t(n >> 1) & 1u, abort_flag)) return PackedSlot{0, 0, 0, 0};
    const PackedSlot s = slot[n & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[n & 1]);
    return s;
  }
};

// Rows [from, to) of a 128-row tile of D columns, set to zero by the 32 lanes of a warp
template <int D>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from, int to, int lane) {
  const uint32_t base = smem_u32(tile);
  const int n = (to - from) * (D / 8);                    // 16-byte pieces: eight per row and 64-column half
  for (int i = lane; i < n; i += 32) {
    const int r = from + i / (D / 8), c = i % (D / 8);
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + uint32_t(c >> 3) * 16384u + uint32_t(r) * 128u + uint32_t(c & 7) * 16u), "r"(0) : "memory");
  }
}
// ... and made visible to the tensor core before `bar` is arrived on
template <int D>
__device__ __forceinline__ void clean_tile(uint8_t* tile, int from, int to, uint64_t* bar, int lane) {
  zero_rows<D>(tile, from, to, lane);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

template <int D>
__device__ __forceinline__ void load_kv(uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int kv, int row) {
  tma_load_3d(dst, m, bar, 0, kv, row);
  if (D == 128) tma_load_3d(dst + 16384, m, bar, 64, kv, row);
}
template <int D>
__device__ __forceinline__ void load_q(uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int kv, int row) {
  tma_load_4d(dst, m, bar, 0, 0, kv, row);
  if (D == 128) tma_load_4d(dst + 16384, m, bar, 64, 0, kv, row);
}

// What four fp32 values lose when they are rounded to bf16 (as the pairs w01, w23), in steps of 2^-8 of the last bf16 bit: a byte
// each.  In the integers that hold them a value is (bf16 << 16) + what is left; that is kept to 8 of its 16 bits, which leaves
// 2^-16 of the value (2^-15 where the byte would be 128).  0 stands for none.
__device__ __forceinline__ uint32_t rest_of(const uint32_t* v, uint32_t w01, uint32_t w23) {
  const int a = min(int(v[0] - (w01 << 16) + 128u), 32767), b = min(int(v[1] - (w01 & 0xffff0000u) + 128u), 32767);
  const int c = min(int(v[2] - (w23 << 16) + 128u), 32767), d = min(int(v[3] - (w23 & 0xffff0000u) + 128u), 32767);
  return __byte_perm(__byte_perm(uint32_t(a), uint32_t(b), 0x0051), __byte_perm(uint32_t(c), uint32_t(d), 0x0051), 0x5410);
}
// a value from its bf16 bits (upper half of `hi`, lower half zero) and byte k of `rest`
__device__ __forceinline__ float with_rest(uint32_t hi, uint32_t rest, int k) {
  return __uint_as_float(hi + (uint32_t(int(rest << (24 - 8 * k)) >> 24) << 8));
}

// 32 rows of COLS (32 or 64) bf16 columns, a row in each lane, to rows `off` elements from `dst` (off < 0: not written).  Through 64
// bytes a column of shared memory of the warp's own, so that neighbouring lanes write neighbouring bytes and not each 16 bytes of
// another row (32768 rows, window 256, 8 heads on 4: backward 316 -> 291 us; the forward gave 10 us before whole tiles went by TMA,
// which the gradients gain nothing by).
template <int COLS>
__device__ __forceinline__ uint32_t stage_at(uint32_t stage, int row, int piece) {
  constexpr int PIECES = COLS / 8;                       // 16 bytes each
  // pieces of a row change places with its number, so that eight lanes meet no bank twice; as the copy engine's swizzles do
  return stage + uint32_t(row * COLS * 2 + ((piece ^ (PIECES == 8 ? row & 7 : (row >> 1) & 3)) << 4));
}
template <int COLS>
__device__ __forceinline__ void stage_rows(const uint32_t* w, uint32_t stage, int lane) {
#pragma unroll
  for (int j = 0; j < COLS / 8; ++j)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage_at<COLS>(stage, lane, j)), "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3]) : "memory");
}
template <int COLS>
__device__ __forceinline__ void store_rows(__nv_bfloat16* dst, long long off, const uint32_t* w, uint32_t stage, int lane) {
  constexpr int PIECES = COLS / 8;
  __syncwarp();                                          // the previous use has been read
  stage_rows<COLS>(w, stage, lane);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int row = i * (32 / PIECES) + lane / PIECES, piece = lane % PIECES;
    const long long o = __shfl_sync(0xffffffffu, off, row);
    uint4 u;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(stage_at<COLS>(stage, row, piece)) : "memory");
    if (o >= 0) *reinterpret_cast<uint4*>(dst + o + piece * 8) = u;
  }
}
// COLS accumulator columns of the lane's row, times s, as bf16 pairs
template <int COLS>
__device__ __forceinline__ void pack_columns(uint32_t taddr, float s, uint32_t (&w)[COLS / 2]) {
#pragma unroll
  for (int c = 0; c < COLS / 32; ++c) {
    uint32_t v[32];
    tmem_ld32(taddr + uint32_t(c * 32), v);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) w[c * 16 + j] = pack_bf16(__uint_as_float(v[2 * j]) * s, __uint_as_float(v[2 * j + 1]) * s);
  }
}
// `n` rows from `row` of `width` elements each, zero, by a warp
__device__ __forceinline__ void zero_out(__nv_bfloat16* dst, long long ld, int row, int n, int width, int lane) {
  const int per = width / 8;
  for (int i = lane; i < n * per; i += 32)
    *reinterpret_cast<uint4*>(dst + (long long)(row + i / per) * ld + (i % per) * 8) = make_uint4(0, 0, 0, 0);
}

// -----------------------------------------------------------------------------------------------
// forward
// -----------------------------------------------------------------------------------------------
template <int D>
struct PackedFwdSmem {
  static constexpr int TILE = 128 * D * 2;
  static constexpr int Q = 0, K = TILE, V = 2 * TILE;
  static constexpr int OUT = 3 * TILE;                   // 4 KB for each of the four epilogue warps
  static constexpr int BAR = OUT + 16384;
  static constexpr int TOTAL = BAR + 192;
};
static_assert(2 * (PackedFwdSmem<128>::TOTAL + 1024) <= 233472, "two CTAs must fit the 228 KB of an SM");

// positions and key tiles of a query tile
struct QueryTile {
  int m0, m_last, j_lo, n_tiles, live;                   // live: rows of the last key tile that belong to the sequence
  __device__ __forceinline__ QueryTile(const PackedArgs& p, int len, int tile) {
    m0 = tile * p.P;
    m_last = min(m0 + p.P, len) - 1;
    j_lo = max(0, m0 - p.window) / 128;
    n_tiles = m_last / 128 - j_lo + 1;
    live = min(128, len - (j_lo + n_tiles - 1) * 128);
  }
};

template <int D>
__global__ void __launch_bounds__(ATT_THREADS, 2)
attn_packed_fwd_k(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                  const __grid_constant__ CUtensorMap tmR, const PackedArgs p) {
  using L = PackedFwdSmem<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {   // the swizzled tiles need 1 KB alignment; nothing has been allocated yet
    grid_wait();
    if (threadIdx.x == 0 && p.err) atomicExch(p.err, ERR_SMEM_ALIGN);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* q_full = bars;            // Q of the n-th query tile
  uint64_t* k_full = bars + 1;        // below, T counts the key tiles of all query tiles
  uint64_t* v_full = bars + 2;
  uint64_t* s_full = bars + 3;        // S(T) complete: scores readable, K slot free; Q's too behind the last one of a query tile
  uint64_t* p_full = bars + 4;        // [2] P(T) of keys 64..127, then of keys 0..63, written (4 arrivals)
  uint64_t* pv_done = bars + 6;       // P V(T) complete: V slot free, behind the last one O is final
  uint64_t* v_land = bars + 7;        // a V tile that has to be cleaned has landed
  uint64_t* next_full = bars + 12;    // which block to take over has been answered
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 13);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  SlotRing ring{bars + 8, bars + 10, reinterpret_cast<PackedSlot*>(bars + 14), abort_flag};
  uint4* next_block = reinterpret_cast<uint4*>(bars + 18);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1); mbar_init(k_full, 1); mbar_init(v_full, 1);
    mbar_init(s_full, 1); mbar_init(&p_full[0], 4); mbar_init(&p_full[1], 4); mbar_init(pv_done, 1); mbar_init(v_land, 1);
    mbar_init(next_full, 1);
    ring.init(1 + 4);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 256); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_enter();                 // global memory is not touched above
  const uint32_t TM_S = tmem, TM_P = tmem + 64, TM_O = tmem + 128;
  const int H = p.KV * p.G;

  if (warp == 0) {
    if (lane == 0) { tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV); }
    int T = 0, n = 0, cleaned = 0;
    bool ok = true, more = true;
    // the grid has a block for every tile; one that runs takes over those that have not started, longest tiles first
    for (int i = int(blockIdx.x), k = 0; ok && more; ++k) {
      // asked for behind the tile's last loads: whoever asks early takes a second tile while others run out of them
      auto request = [&]() {
        if (lane == 0) {
          mbar_expect_tx(next_full, 16);
          take_block_request(next_block + (k & 1), next_full);
        }
      };
      const PackedTile tile = packed_tile(p, p.items_q, p.n_q, i);
      const int start = tile.it.start, len = tile.it.len, kv = tile.kv;
      if (len <= 0) {
        request();
      } else if (tile.it.tile < 0) {                     // rows of no sequence
        request();
        zero_out(p.o + (long long)kv * p.G * D, p.ldo, start, len, p.G * D, lane);
        if (p.o_lo) zero_out(reinterpret_cast<__nv_bfloat16*>(p.o_lo + (long long)kv * p.G * D), p.ldo / 2, start, len, p.G * D / 2, lane);
        for (int e = lane; e < len * p.G; e += 32) p.lse[(long long)(start + e / p.G) * H + kv * p.G + e % p.G] = -INFINITY;
      } else {
        const QueryTile qt(p, len, tile.it.tile);
        const bool clean = qt.live < 128;
        if (lane == 0) {
          ok = ring.put(n, tile);
          for (int t = 0; ok && t < qt.n_tiles; ++t, ++T) {
            const int row = start + (qt.j_lo + t) * 128;
            if (T > 0 && !mbar_wait(s_full, uint32_t(T - 1) & 1u, abort_flag)) { ok = false; break; }
            if (t == 0) {
              mbar_expect_tx(q_full, uint32_t(p.P * p.G * D * 2));          // rows past the end of the tensor are zero-filled
              load_q<D>(smem + L::Q, &tmQ, q_full, kv, start + qt.m0);
            }
            mbar_expect_tx(k_full, L::TILE);
            load_kv<D>(smem + L::K, &tmK, k_full, kv, row);
            if (T > 0 && !mbar_wait(pv_done, uint32_t(T - 1) & 1u, abort_flag)) { ok = false; break; }
            uint64_t* bar = (clean && t == qt.n_tiles - 1) ? v_land : v_full;
            mbar_expect_tx(bar, L::TILE);
            load_kv<D>(smem + L::V, &tmV, bar, kv, row);
          }
        }
        request();
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (clean && ok) {
          ok = wait_warp(v_land, uint32_t(cleaned) & 1u, abort_flag);
          ++cleaned;
          if (ok) clean_tile<D>(smem + L::V, qt.live, 128, v_full, lane);
        }
        ++n;
      }
      // every request is answered before the block ends
      uint32_t x = 0;
      const bool answered = wait_warp(next_full, uint32_t(k) & 1u, abort_flag);
      for (uint32_t spin = 0; !answered && spin < 65536 && !mbar_try_wait(next_full, uint32_t(k) & 1u); ++spin) {}
      more = answered && take_block_answer(next_block + (k & 1), x);
      i = int(x);
      fence_proxy_async_smem();                          // the answer has been read before the request after the next overwrites it
      __syncwarp();
      ok = ok && answered;
    }
    if (ok && lane == 0) ring.put(n, PackedTile{PackedItem{0, 0, 0, 0}, 0});
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc_bf16(128, 128, false, false);
      constexpr uint32_t idesc_o = make_idesc_bf16(128, D, false, true);
      // descriptor words once; a K slice is a 32-bit add on the low word (start address >> 4)
      const uint32_t hi_k = uint32_t(make_smem_desc(0, 0, 1024) >> 32), hi_v = uint32_t(make_smem_desc(0, 16384, 1024) >> 32);
      const uint32_t q_lo = uint32_t(make_smem_desc(smem_u32(smem + L::Q), 0, 1024));
      const uint32_t k_lo = uint32_t(make_smem_desc(smem_u32(smem + L::K), 0, 1024));
      const uint32_t v_lo = uint32_t(make_smem_desc(smem_u32(smem + L::V), 16384, 1024));
      bool ok = true;
      int T = 0;
      auto issue_s = [&](int tt) {
        if (!mbar_wait(k_full, uint32_t(tt) & 1u, abort_flag)) { ok = false; return; }
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = uint32_t(k >> 2) * 1024u + uint32_t(k & 3) * 2u;     // (16 KB half, 32 B slice) >> 4
          tc_mma_ss_lh(TM_S, q_lo + off, hi_k, k_lo + off, hi_k, idesc_s, k > 0);
        }
        tc_commit(s_full);
      };
      for (int n = 0; ok; ++n) {
        const PackedSlot slot = ring.take(n);
        if (slot.len == 0) break;
        const int n_tiles = QueryTile(p, slot.len, slot.tile).n_tiles;
        ok = mbar_wait(q_full, uint32_t(n) & 1u, abort_flag);
        if (ok) issue_s(T);               // behind the previous query tile's last P V, which reads columns of the tile it overwrites
        for (int t = 0; t < n_tiles && ok; ++t, ++T) {
          if (!mbar_wait(v_full, uint32_t(T) & 1u, abort_flag)) { ok = false; break; }
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {              // the upper keys' products run under the lower keys' exponentials
            // t = 0: the four warps announce P behind their epilogue of the previous query tile, so O may be overwritten
            if (!mbar_wait(&p_full[hf], uint32_t(T) & 1u, abort_flag)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t k = uint32_t(hf ? i : 4 + i);
              tc_mma_ts_lh(TM_O, TM_P + k * 8u, v_lo + k * 128u, hi_v, idesc_o, (t > 0 || hf > 0 || i > 0) ? 1u : 0u);
            }
          }
          if (!ok) break;
          tc_commit(pv_done);
          if (t + 1 < n_tiles) issue_s(T + 1);          // behind P V(T), which reads columns of the tile it overwrites
        }
      }
    }
  } else {
    // ---------------- softmax / epilogue: thread <-> row of the tile = (position, head of the group) ----------------
    const int q = warp & 3;
    const int r = q * 32 + lane;
    const int at = r / p.G;
    const uint32_t lane_addr = uint32_t(q * 32) << 16;
    const float c = p.scale * LOG2E;
    bool ok = true;
    int T = 0;
    for (int n = 0; ok; ++n) {
      const PackedSlot slot = ring.take_warp(n, lane);
      if (slot.len == 0) break;
      const QueryTile qt(p, slot.len, slot.tile);
      const int pos = qt.m0 + at;
      const bool live_row = at < p.P && pos < slot.len;
      float m_used = -INFINITY, l = 0.f;
      for (int t = 0; t < qt.n_tiles; ++t, ++T) {
        const int n0 = (qt.j_lo + t) * 128;
        if (!wait_warp(s_full, uint32_t(T) & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        // in unmasked tiles rows without a query compute results of their own that nothing uses
        const bool need_mask = (n0 + 127 > qt.m0) || (n0 < qt.m_last - p.window);
        // visible keys of this row inside the tile: columns [lo, hi]
        const int lo = live_row ? pos - p.window - n0 : 128, hi = live_row ? pos - n0 : 0;
        uint32_t sc[32], sd[32];                           // columns 64..127 stay in registers
        float mx;
        {
          uint32_t sa[32], sb[32];
          tmem_ld32(TM_S + lane_addr, sa);
          tmem_ld32(TM_S + lane_addr + 32u, sb);
          tmem_wait_ld();
          tmem_ld32(TM_S + lane_addr + 64u, sc);
          tmem_ld32(TM_S + lane_addr + 96u, sd);
          if (need_mask) { hide(sa, visible(lo, hi)); hide(sb, visible(lo - 32, hi - 32)); }
          mx = max32<false>(sb, 32, 0, 0u, max32<false>(sa, 0, 0, 0u, -INFINITY));
          tmem_wait_ld();
        }
        if (need_mask) { hide(sc, visible(lo - 64, hi - 64)); hide(sd, visible(lo - 96, hi - 96)); }
        mx = max32<false>(sd, 96, 0, 0u, max32<false>(sc, 64, 0, 0u, mx));
        const float m_new = fmaxf(m_used, mx);
        bool resc = false;
        if (m_used == -INFINITY) m_used = m_new;            // nothing accumulated for this row yet
        else resc = (m_new - m_used) * c > 8.f;
        if (t > 0 && __any_sync(0xffffffffu, resc)) {
          // S(t) complete implies P V(t-1) complete: O is not in flight
          const float alpha = resc ? fast_exp2((m_used - m_new) * c) : 1.f;
          if (resc) { l *= alpha; m_used = m_new; }
#pragma unroll
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t v[32];
            tmem_ld32(TM_O + lane_addr + uint32_t(cc * 32), v);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha);
            tmem_st32(TM_O + lane_addr + uint32_t(cc * 32), v);
          }
          tmem_wait_st();
        }
        const float mc = (m_used == -INFINITY) ? 0.f : m_used * c;
        const unsigned long long c2 = pk2(c, c), nmc2 = pk2(-mc, -mc);
        unsigned long long rs2 = pk2(0.f, 0.f);
        {
          uint32_t pk[32];
          exp32_mufu<false>(sc, pk, c2, nmc2, 64, 0, 0u, rs2);
          exp32_mufu<false>(sd, pk + 16, c2, nmc2, 96, 0, 0u, rs2);
          tmem_st32(TM_P + lane_addr + 32u, pk);           // over scores that have been read
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[0]);
        {
          uint32_t sa[32], sb[32], pk[32];
          tmem_ld32(TM_S + lane_addr, sa);
          tmem_ld32(TM_S + lane_addr + 32u, sb);
          tmem_wait_ld();
          if (need_mask) { hide(sa, visible(lo, hi)); hide(sb, visible(lo - 32, hi - 32)); }
          exp32_mufu<false>(sa, pk, c2, nmc2, 0, 0, 0u, rs2);
          exp32_mufu<false>(sb, pk + 16, c2, nmc2, 32, 0, 0u, rs2);
          tmem_st32(TM_P + lane_addr, pk);
        }
        float r0, r1;
        unpk2(rs2, r0, r1);
        l += r0 + r1;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[1]);
      }
      if (!ok || !wait_warp(pv_done, uint32_t(T - 1) & 1u, abort_flag)) { ok = false; break; }
      tc_fence_after();
      const float inv_l = (l > 0.f) ? 1.f / l : 0.f;
      const int head = slot.kv * p.G + (r - at * p.G);
      const long long off = live_row ? (long long)(slot.start + pos) * p.ldo + (long long)head * D : -1;
      const uint32_t stage = smem_u32(smem + L::OUT) + uint32_t(q) * 4096u;
      // where the warp's 32 rows all exist, 32 columns at a time go to the copy engine and the next are read and packed meanwhile: where
      // all CTAs write at once the warps' own stores waited 1 to 2 K clk per 64 columns (32768 rows, window 256, 8 heads on 4: 108 -> 98 us;
      // 64 sequences of 512, 4 heads: 60 -> 54 us; long sequences 1 to 2 %)
      const bool whole = 32 % p.G == 0 && __all_sync(0xffffffffu, live_row);
#pragma unroll 1
      for (int cc = 0; cc < D; cc += 32) {
        uint32_t v[32], w[16], rest[8];
        tmem_ld32(TM_O + lane_addr + uint32_t(cc), v);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * inv_l);
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack_bf16(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
#pragma unroll
        for (int j = 0; j < 8; ++j) rest[j] = rest_of(v + 4 * j, w[2 * j], w[2 * j + 1]);
        if (lane == 0) tma_store_wait_read();              // the columns before have left the stage
        if (whole) {
          __syncwarp();
          stage_rows<32>(w, stage, lane);
          if (p.o_lo) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + 2048u + uint32_t(lane * 32 + j * 16)), "r"(rest[4 * j]),
                           "r"(rest[4 * j + 1]), "r"(rest[4 * j + 2]), "r"(rest[4 * j + 3]) : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            const int row = slot.start + qt.m0 + q * (32 / p.G);
            tma_store_4d(&tmO, smem + L::OUT + q * 4096, cc, 0, slot.kv, row);
            if (p.o_lo) tma_store_4d(&tmR, smem + L::OUT + q * 4096 + 2048, cc, 0, slot.kv, row);
            tma_store_commit();
          }
        } else {
          store_rows<32>(p.o + cc, off, w, stage, lane);
          if (p.o_lo && live_row) {
            uint4* dst = reinterpret_cast<uint4*>(p.o_lo + off + cc);
            dst[0] = make_uint4(rest[0], rest[1], rest[2], rest[3]);
            dst[1] = make_uint4(rest[4], rest[5], rest[6], rest[7]);
          }
        }
      }
      if (live_row) p.lse[(long long)(slot.start + pos) * H + head] = (l > 0.f) ? (m_used * p.scale + __logf(l)) : -INFINITY;
    }
    if (lane == 0) tma_store_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag && p.err) atomicExch(p.err, ERR_ATTN_TIMEOUT);
  if (warp == 1) { __syncwarp(); tc_fence_after(); tmem_dealloc(tmem, 256); }
}

// -----------------------------------------------------------------------------------------------
// backward
// -----------------------------------------------------------------------------------------------
// Two resident tiles, a three-slot and a two-slot ring.  A CTA takes key tiles (dK, dV) until there are no more, then query tiles
// (dQ): both lists are handed out by counters, so CTAs that got short tiles take more of them.
template <int D>
struct PackedBwdSmem {
  static constexpr int TILE = 128 * D * 2;
  static constexpr int RES0 = 0, RES1 = TILE;
  static constexpr int RING3 = 2 * TILE;
  static constexpr int RING2 = 5 * TILE;
  static constexpr int STAT = 7 * TILE;                  // lse2[2][128], delta[2][128] (dK/dV)
  static constexpr int BAR = STAT + 4 * 128 * 4;         // dK/dV, dQ, then what both share
  static constexpr int BAR_DQ = BAR + 256, COMMON = BAR_DQ + 256;
  static constexpr int TOTAL = COMMON + 64;
};
static_assert(PackedBwdSmem<128>::TOTAL <= 232448, "exceeds the 227 KB shared memory of one CTA");

struct BwdCta { uint8_t* smem; uint32_t tmem; volatile int* abort_flag; int warp, lane; };

// the next tile of a list that is not empty, to the whole warp; len = 0: none
__device__ __forceinline__ PackedTile next_tile(const PackedArgs& p, const PackedItem* items, int n, int* counter, int lane) {
  const int total = n * p.KV;
  for (;;) {
    int i = 0;
    if (lane == 0) i = atomicAdd(counter, 1);
    i = __shfl_sync(0xffffffffu, i, 0);
    if (i >= total) return PackedTile{PackedItem{0, 0, 0, 0}, 0};
    const PackedTile t = packed_tile(p, items, n, i);
    if (t.it.len > 0) return t;
  }
}

// 128 x 128 product over the D columns of two K-major tiles
template <int D>
__device__ __forceinline__ void mma_scores(uint32_t d_tmem, uint32_t sa, uint32_t sb) {
  constexpr uint32_t idesc = make_idesc_bf16(128, 128, false, false);
  const uint32_t hi = uint32_t(make_smem_desc(0, 0, 1024) >> 32);
  const uint32_t al = uint32_t(make_smem_desc(sa, 0, 1024)), bl = uint32_t(make_smem_desc(sb, 0, 1024));
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    const uint32_t off = uint32_t(k >> 2) * 1024u + uint32_t(k & 3) * 2u;       // (16 KB half, 32 B slice) >> 4
    tc_mma_ss_lh(d_tmem, al + off, hi, bl + off, hi, idesc, k > 0);
  }
}
// 128 x D (+)= A[tmem, 128 x 128 bf16 as two groups of 32 columns] * B[128-row tile, rows are the summed dimension]
template <int D>
__device__ __forceinline__ void mma_sum(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t sb, bool accumulate) {
  constexpr uint32_t idesc = make_idesc_bf16(128, D, false, true);
  const uint32_t hi = uint32_t(make_smem_desc(0, 16384, 1024) >> 32), bl = uint32_t(make_smem_desc(sb, 16384, 1024));
#pragma unroll
  for (int k = 0; k < 8; ++k)
    tc_mma_ts_lh(d_tmem, (k < 4 ? a_lo : a_hi) + uint32_t(k & 3) * 8u, bl + uint32_t(k) * 128u, hi, idesc, (accumulate || k > 0) ? 1u : 0u);
}

// ---- dQ: query tile stationary -----------------------------------------------------------------
// A finished tile leaves through the last ring slot that it used (V's for dQ, dO's for dK and dV), whose next load, two steps on, waits
// for that: the n-th tile's slot is asked for in the second step of the tile behind it, or in the first of the one after where that
// has a single step.  Two barriers in turn: the tile behind may be finished, too, before the loading warp asks for this one.
__device__ __forceinline__ int left_through(int step, int n, bool single) { return step == 1 ? n - 1 : step == 0 && single ? n - 2 : -1; }

template <int D>
struct DqBars {
  uint64_t* b;
  __device__ __forceinline__ uint64_t* q_full() const { return b; }             // Q + dO of the n-th query tile
  __device__ __forceinline__ uint64_t* k_full(int T) const { return b + 1 + T % 3; }
  __device__ __forceinline__ uint64_t* v_full(int T) const { return b + 4 + (T & 1); }
  __device__ __forceinline__ uint64_t* s_full() const { return b + 6; }         // S(T) complete
  __device__ __forceinline__ uint64_t* a_done() const { return b + 7; }         // phase A(T) has read S(T)            (8 arrivals)
  __device__ __forceinline__ uint64_t* dp_full(int T) const { return b + 8 + (T & 1); }    // dP(T) complete; also frees V(T)'s slot
  __device__ __forceinline__ uint64_t* ds_full(int T) const { return b + 10 + (T & 1); }   // phase B(T) wrote dS(T) and has read dP(T) (8)
  __device__ __forceinline__ uint64_t* dq_done(int T) const { return b + 12 + T % 6; }     // dQ(T) complete: K(T)'s slot and dS buffer T & 1 free
  __device__ __forceinline__ uint64_t* done() const { return b + 18; }          // dQ of the n-th query tile complete
  __device__ __forceinline__ uint64_t* land(int i) const { return b + 19 + i; } // K / V tile that has to be cleaned has landed
  __device__ __forceinline__ uint64_t* out_free(int n) const { return b + 21 + (n & 1); }  // dQ of the n-th query tile written (8 arrivals)
  __device__ __forceinline__ uint64_t* ring() const { return b + 23; }          // 4
  static constexpr int COUNT = 27;
  __device__ __forceinline__ void init() const {
    for (int i = 0; i < 23; ++i) mbar_init(b + i, i == 7 || i == 10 || i == 11 || i >= 21 ? 8 : 1);
  }
};
static_assert(DqBars<64>::COUNT * 8 + 2 * sizeof(PackedSlot) <= 256, "barrier space");

template <int D>
__device__ __forceinline__ void packed_bwd_dq(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV,
                                              const CUtensorMap& tmDO, const PackedArgs& p, const BwdCta& cta) {
  using L = PackedBwdSmem<D>;
  uint8_t* smem = cta.smem;
  volatile int* abort_flag = cta.abort_flag;
  const DqBars<D> bar{reinterpret_cast<uint64_t*>(smem + L::BAR_DQ)};
  SlotRing ring{bar.ring(), bar.ring() + 2, reinterpret_cast<PackedSlot*>(smem + L::COMMON + 32), abort_flag};
  const int warp = cta.warp, lane = cta.lane;
  const uint32_t TM_S = cta.tmem, TM_DP = cta.tmem + 128, TM_DQ = cta.tmem + 256, TM_DS = cta.tmem + 384;
  const int H = p.KV * p.G;

  if (warp == 0) {
    const uint32_t q_bytes = uint32_t(p.P * p.G * D * 2);
    int T = 0, cleaned = 0;
    bool ok = true, single = false;                      // whether the tile before had a single step
    auto k_slot = [&](int t) { return smem + L::RING3 + (t % 3) * L::TILE; };
    auto v_slot = [&](int t) { return smem + L::RING2 + (t & 1) * L::TILE; };
    for (int n = 0; ok;) {
      const PackedTile tile = next_tile(p, p.items_q, p.n_q, p.next + 1, lane);
      const int start = tile.it.start, len = tile.it.len, kv = tile.kv;
      if (len == 0) { if (lane == 0) ring.put(n, tile); break; }
      if (tile.it.tile < 0) {                            // rows of no sequence
        zero_out(p.o + (long long)kv * p.G * D, p.ldo, start, len, p.G * D, lane);
        continue;
      }
      const QueryTile qt(p, len, tile.it.tile);
      const bool clean = qt.live < 128;
      const int last = T + qt.n_tiles - 1;
      if (lane == 0) {
        ok = ring.put(n, tile);
        // Q and dO are free behind the last S and dP of the previous query tile (dP of T-3, the phase before on this barrier, was waited
        // for when V's slot was taken for T-1)
        if (ok && T > 0) ok = mbar_wait(bar.dp_full(T - 1), uint32_t((T - 1) >> 1) & 1u, abort_flag);
        if (ok) {
          mbar_expect_tx(bar.q_full(), 2 * q_bytes);
          load_q<D>(smem + L::RES0, &tmQ, bar.q_full(), kv, start + qt.m0);
          load_q<D>(smem + L::RES1, &tmDO, bar.q_full(), kv, start + qt.m0);
        }
        // K(T) is requested when dQ(T-3) has released its slot, V(T) when dP(T-2) has
        for (int t = T; ok && t <= last; ++t) {
          const int row = start + (qt.j_lo + t - T) * 128;
          if (t >= 3 && !mbar_wait(bar.dq_done(t - 3), uint32_t((t - 3) / 6) & 1u, abort_flag)) { ok = false; break; }
          uint64_t* kb = clean && t == last ? bar.land(0) : bar.k_full(t);
          mbar_expect_tx(kb, L::TILE);
          load_kv<D>(k_slot(t), &tmK, kb, kv, row);
          if (t >= 2 && !mbar_wait(bar.dp_full(t), uint32_t((t - 2) >> 1) & 1u, abort_flag)) { ok = false; break; }
          const int left = left_through(t - T, n, single);
          if (left >= 0 && !mbar_wait(bar.out_free(left), uint32_t(left >> 1) & 1u, abort_flag)) { ok = false; break; }
          uint64_t* vb = clean && t == last ? bar.land(1) : bar.v_full(t);
          mbar_expect_tx(vb, L::TILE);
          load_kv<D>(v_slot(t), &tmV, vb, kv, row);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (clean && ok) {
        // both are summed over or multiplied with: rows of other sequences must not leave a NaN behind
        ok = wait_warp(bar.land(0), uint32_t(cleaned) & 1u, abort_flag);
        if (ok) clean_tile<D>(k_slot(last), qt.live, 128, bar.k_full(last), lane);
        ok = ok && wait_warp(bar.land(1), uint32_t(cleaned) & 1u, abort_flag);
        if (ok) clean_tile<D>(v_slot(last), qt.live, 128, bar.v_full(last), lane);
        ++cleaned;
      }
      T = last + 1;
      single = qt.n_tiles == 1;
      ++n;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t sq = smem_u32(smem + L::RES0), sdo = smem_u32(smem + L::RES1);
      const uint32_t sk0 = smem_u32(smem + L::RING3), sv0 = smem_u32(smem + L::RING2);
      bool ok = true;
      auto issue_s = [&](int T) {
        ok = ok && mbar_wait(bar.k_full(T), uint32_t(T / 3) & 1u, abort_flag);
        if (!ok) return;
        tc_fence_after();
        mma_scores<D>(TM_S, sq, sk0 + uint32_t(T % 3) * L::TILE);
        tc_commit(bar.s_full());
      };
      auto issue_dp = [&](int T) {
        ok = ok && mbar_wait(bar.v_full(T), uint32_t(T >> 1) & 1u, abort_flag);
        if (!ok) return;
        tc_fence_after();
        mma_scores<D>(TM_DP, sdo, sv0 + uint32_t(T & 1) * L::TILE);
        tc_commit(bar.dp_full(T));
      };
      int T = 0;
      for (int n = 0; ok; ++n) {
        const PackedSlot slot = ring.take(n);
        if (slot.len == 0) break;
        const int n_tiles = QueryTile(p, slot.len, slot.tile).n_tiles;
        ok = mbar_wait(bar.q_full(), uint32_t(n) & 1u, abort_flag);
        // S and dP of the previous query tile's last key tile have been read: phase B announced its dS behind both
        issue_s(T);
        issue_dp(T);
        for (int t = 0; t < n_tiles && ok; ++t, ++T) {
          const bool more = t + 1 < n_tiles;
          if (more) {
            if (!mbar_wait(bar.a_done(), uint32_t(T) & 1u, abort_flag)) { ok = false; break; }
            issue_s(T + 1);
          }
          if (!ok || !mbar_wait(bar.ds_full(T), uint32_t(T >> 1) & 1u, abort_flag)) { ok = false; break; }
          if (more) issue_dp(T + 1);
          if (!ok) break;
          tc_fence_after();
          // t = 0: the eight warps announce dS behind their epilogue of the previous query tile, so dQ may be overwritten
          const uint32_t ds = TM_DS + uint32_t(T & 1) * 64u;
          mma_sum<D>(TM_DQ, ds, ds + 32, sk0 + uint32_t(T % 3) * L::TILE, t > 0);
          tc_commit(bar.dq_done(T));
          // the last tile's phase A is waited for by nobody else: every phase of a_done is seen here
          if (!more) { tc_commit(bar.done()); ok = mbar_wait(bar.a_done(), uint32_t(T) & 1u, abort_flag); }
        }
      }
    }
  } else {
    const int sw = warp - 2;             // 0..7
    const int q = warp & 3;              // TMEM lane quarter this warp may access
    const int hf = sw >> 2;              // column half of the tile owned by this warp
    const int r = q * 32 + lane;
    const int at = r / p.G;
    const uint32_t lane_addr = uint32_t(q * 32) << 16;
    const float c = p.scale * LOG2E;
    bool ok = true;
    int T = 0;
    float lse2, dlt;
    auto load_stats = [&](const PackedSlot& s) {
      const int pos = s.tile * p.P + at;
      lse2 = INFINITY; dlt = 0.f;
      if (s.len > 0 && at < p.P && pos < s.len) {
        const long long stat = (long long)(s.start + pos) * H + s.kv * p.G + (r - at * p.G);
        lse2 = p.lse[stat] * LOG2E;
        dlt = p.delta[stat];
      }
    };
    PackedSlot slot = ring.take_warp(0, lane);
    load_stats(slot);
    for (int n = 0; ok && slot.len > 0; ++n) {
      const QueryTile qt(p, slot.len, slot.tile);
      const int pos = qt.m0 + at;
      const bool live_row = at < p.P && pos < slot.len;
      for (int t = 0; t < qt.n_tiles; ++t, ++T) {
        const int n0 = (qt.j_lo + t) * 128 + hf * 64;   // first key of this thread's 64 columns
        float pr[64];
        // ---- phase A ----
        if (!wait_warp(bar.s_full(), uint32_t(T) & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        {
          uint32_t s0[32], s1[32];
          tmem_ld64(TM_S + lane_addr + uint32_t(hf * 64), s0, s1);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar.a_done());
          if ((n0 + 63 > qt.m0) || (n0 < qt.m_last - p.window)) {
            // the visible keys of a row are one interval of columns
            const int lo = live_row ? pos - p.window - n0 : 64, hi = live_row ? pos - n0 : 0;
            hide(s0, visible(lo, hi));
            hide(s1, visible(lo - 32, hi - 32));
          }
          exp2_64<true>(s0, s1, c, lse2, nullptr, pr);
        }
        // ---- phase B ----
        if (!wait_warp(bar.dp_full(T), uint32_t(T >> 1) & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        uint32_t pk[32];
        {
          uint32_t d0[32], d1[32];
          tmem_ld64(TM_DP + lane_addr + uint32_t(hf * 64), d0, d1);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            pk[j] = pack_bf16(pr[2 * j] * (__uint_as_float(d0[2 * j]) - dlt), pr[2 * j + 1] * (__uint_as_float(d0[2 * j + 1]) - dlt));
            pk[16 + j] = pack_bf16(pr[32 + 2 * j] * (__uint_as_float(d1[2 * j]) - dlt),
                                   pr[32 + 2 * j + 1] * (__uint_as_float(d1[2 * j + 1]) - dlt));
          }
        }
        // dS buffer T & 1 was last read by the dQ MMAs of tile T-2
        if (T >= 2 && !wait_warp(bar.dq_done(T - 2), uint32_t((T - 2) / 6) & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        tmem_st32(TM_DS + lane_addr + uint32_t((T & 1) * 64 + hf * 32), pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar.ds_full(T));
      }
      if (!ok) break;
      const PackedSlot done = slot;
      slot = ring.take_warp(n + 1, lane);
      load_stats(slot);                    // in flight while this query tile is finished
      if (!wait_warp(bar.done(), uint32_t(n) & 1u, abort_flag)) break;
      tc_fence_after();
      const long long off = live_row ? (long long)(done.start + pos) * p.ldo + (long long)(done.kv * p.G + (r - at * p.G)) * D : -1;
      uint32_t w[D / 4];
      pack_columns<D / 2>(TM_DQ + lane_addr + uint32_t(hf * (D / 2)), p.scale, w);
      store_rows<D / 2>(p.o + hf * (D / 2), off, w, smem_u32(smem + L::RING2 + ((T - 1) & 1) * L::TILE) + uint32_t(sw * (32 * D)), lane);
      fence_proxy_async_smem();            // read before the slot's next load overwrites it
      __syncwarp();
      if (lane == 0) mbar_arrive(bar.out_free(n));
    }
  }
}

// ---- dK / dV: key tile stationary, transposed scores; the query tiles bring all heads of the group -------------------
template <int D>
struct DkvBars {
  uint64_t* b;
  __device__ __forceinline__ uint64_t* kv_full() const { return b; }            // K + V of the n-th key tile
  __device__ __forceinline__ uint64_t* q_full(int T) const { return b + 1 + T % 3; }
  __device__ __forceinline__ uint64_t* q_empty(int T) const { return b + 4 + T % 3; }      // dK(T) complete
  __device__ __forceinline__ uint64_t* do_full(int T) const { return b + 7 + (T & 1); }
  __device__ __forceinline__ uint64_t* do_empty(int T) const { return b + 9 + (T & 1); }   // dV(T) complete
  __device__ __forceinline__ uint64_t* s_full() const { return b + 11; }        // S^T(T) complete
  __device__ __forceinline__ uint64_t* p_full() const { return b + 12; }        // phase A(T) wrote P^T(T)             (8 arrivals)
  __device__ __forceinline__ uint64_t* dp_full() const { return b + 13; }       // dP^T(T) complete
  __device__ __forceinline__ uint64_t* ds_full() const { return b + 14; }       // phase B(T) wrote dS^T(T)            (8 arrivals)
  __device__ __forceinline__ uint64_t* done() const { return b + 15; }          // dK and dV of the n-th key tile complete
  __device__ __forceinline__ uint64_t* land(int i) const { return b + 16 + i; } // Q / dO tile that has to be cleaned has landed
  __device__ __forceinline__ uint64_t* stat() const { return b + 18; }          // statistics of query tile T written (8 arrivals)
  // all S^T and dP^T of the n-th key tile complete.  (dp_full would say so too, but a parity tells a phase only from the one before and
  // the one behind it: who waits for a barrier visits all of its phases, which the loading warp does not with dp_full's.)
  __device__ __forceinline__ uint64_t* kv_free() const { return b + 19; }
  __device__ __forceinline__ uint64_t* out_free(int n) const { return b + 20 + (n & 1); }  // dK and dV of the n-th key tile written (8 arrivals)
  __device__ __forceinline__ uint64_t* ring() const { return b + 22; }          // 4
  static constexpr int COUNT = 26;
  __device__ __forceinline__ void init() const {
    for (int i = 0; i < 22; ++i) mbar_init(b + i, i == 12 || i == 14 || i == 18 || i >= 20 ? 8 : 1);
  }
};
static_assert(DkvBars<64>::COUNT * 8 + 2 * sizeof(PackedSlot) <= 256, "barrier space");

// query tiles of a key tile
struct KeyTile {
  int n0, i_lo, n_tiles, live;                           // live: rows of the last query tile that belong to the sequence
  __device__ __forceinline__ KeyTile(const PackedArgs& p, int len, int tile) {
    n0 = tile * 128;
    const int last_q = min(len - 1, min(n0 + 127, len - 1) + p.window);
    i_lo = n0 / p.P;
    n_tiles = last_q / p.P - i_lo + 1;
    live = min(p.P, len - (i_lo + n_tiles - 1) * p.P) * p.G;
  }
};

template <int D>
__device__ __forceinline__ void packed_bwd_dkv(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV,
                                               const CUtensorMap& tmDO, const PackedArgs& p, const BwdCta& cta) {
  using L = PackedBwdSmem<D>;
  uint8_t* smem = cta.smem;
  volatile int* abort_flag = cta.abort_flag;
  const DkvBars<D> bar{reinterpret_cast<uint64_t*>(smem + L::BAR)};
  SlotRing ring{bar.ring(), bar.ring() + 2, reinterpret_cast<PackedSlot*>(smem + L::BAR + 256 - 2 * sizeof(PackedSlot)), abort_flag};
  float* stat_lse = reinterpret_cast<float*>(smem + L::STAT);   // [2][128]
  float* stat_dl = stat_lse + 256;                               // [2][128]
  const int warp = cta.warp, lane = cta.lane;
  const int used = p.P * p.G;           // rows of a query tile that hold queries
  const uint32_t TM_S = cta.tmem, TM_DP = cta.tmem + 128, TM_DV = cta.tmem + 256, TM_DK = cta.tmem + 384;
  const int H = p.KV * p.G;

  if (warp == 0) {
    const uint32_t q_bytes = uint32_t(used * D * 2);
    int T = 0, cleaned = 0;
    bool ok = true, single = false;                      // whether the tile before had a single step
    auto q_slot = [&](int t) { return smem + L::RING3 + (t % 3) * L::TILE; };
    auto do_slot = [&](int t) { return smem + L::RING2 + (t & 1) * L::TILE; };
    for (int n = 0; ok;) {
      const PackedTile tile = next_tile(p, p.items_k, p.n_k, p.next, lane);
      const int start = tile.it.start, len = tile.it.len, kv = tile.kv;
      if (len == 0) { if (lane == 0) ring.put(n, tile); break; }
      if (tile.it.tile < 0) {                            // rows of no sequence
        zero_out(p.dk + (long long)kv * D, p.lddk, start, len, D, lane);
        zero_out(p.dv + (long long)kv * D, p.lddv, start, len, D, lane);
        continue;
      }
      const KeyTile kt(p, len, tile.it.tile);
      const bool clean = kt.live < used;
      const int last = T + kt.n_tiles - 1;
      if (lane == 0) {
        ok = ring.put(n, tile);
        if (ok && n > 0) ok = mbar_wait(bar.kv_free(), uint32_t(n - 1) & 1u, abort_flag);
        if (ok) {
          mbar_expect_tx(bar.kv_full(), 2 * L::TILE);
          load_kv<D>(smem + L::RES0, &tmK, bar.kv_full(), kv, start + kt.n0);
          load_kv<D>(smem + L::RES1, &tmV, bar.kv_full(), kv, start + kt.n0);
        }
        for (int t = T; ok && t <= last; ++t) {
          const int row = start + (kt.i_lo + t - T) * p.P;
          if (!mbar_wait(bar.q_empty(t), (uint32_t(t / 3) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
          uint64_t* qb = clean && t == last ? bar.land(0) : bar.q_full(t);
          mbar_expect_tx(qb, q_bytes);
          load_q<D>(q_slot(t), &tmQ, qb, kv, row);
          if (!mbar_wait(bar.do_empty(t), (uint32_t(t >> 1) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
          const int left = left_through(t - T, n, single);
          if (left >= 0 && !mbar_wait(bar.out_free(left), uint32_t(left >> 1) & 1u, abort_flag)) { ok = false; break; }
          uint64_t* db = clean && t == last ? bar.land(1) : bar.do_full(t);
          mbar_expect_tx(db, q_bytes);
          load_q<D>(do_slot(t), &tmDO, db, kv, row);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (clean && ok) {
        ok = wait_warp(bar.land(0), uint32_t(cleaned) & 1u, abort_flag);
        if (ok) clean_tile<D>(q_slot(last), kt.live, used, bar.q_full(last), lane);
        ok = ok && wait_warp(bar.land(1), uint32_t(cleaned) & 1u, abort_flag);
        if (ok) clean_tile<D>(do_slot(last), kt.live, used, bar.do_full(last), lane);
        ++cleaned;
      }
      T = last + 1;
      single = kt.n_tiles == 1;
      ++n;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t sk = smem_u32(smem + L::RES0), sv = smem_u32(smem + L::RES1);
      const uint32_t sq0 = smem_u32(smem + L::RING3), sdo0 = smem_u32(smem + L::RING2);
      bool ok = true;
      auto issue_s = [&](int T) {
        ok = ok && mbar_wait(bar.q_full(T), uint32_t(T / 3) & 1u, abort_flag);
        if (!ok) return;
        tc_fence_after();
        mma_scores<D>(TM_S, sk, sq0 + uint32_t(T % 3) * L::TILE);
        tc_commit(bar.s_full());
      };
      auto issue_dp = [&](int T) {
        ok = ok && mbar_wait(bar.do_full(T), uint32_t(T >> 1) & 1u, abort_flag);
        if (!ok) return;
        tc_fence_after();
        mma_scores<D>(TM_DP, sv, sdo0 + uint32_t(T & 1) * L::TILE);
        tc_commit(bar.dp_full());
      };
      int T = 0;
      for (int n = 0; ok; ++n) {
        const PackedSlot slot = ring.take(n);
        if (slot.len == 0) break;
        const int n_tiles = KeyTile(p, slot.len, slot.tile).n_tiles;
        ok = mbar_wait(bar.kv_full(), uint32_t(n) & 1u, abort_flag);
        // behind the previous key tile's last dV and dK, which read columns of the tiles these overwrite
        issue_s(T);
        issue_dp(T);
        if (ok && n_tiles == 1) tc_commit(bar.kv_free());
        for (int t = 0; t < n_tiles && ok; ++t, ++T) {
          const bool more = t + 1 < n_tiles;
          // dV(T) reads P^T(T) from the S^T tile; S^T(T+1) is issued after it and may then overwrite it.  t = 0: the eight warps
          // announce P^T behind their epilogue of the previous key tile, so dV and dK may be overwritten
          if (!mbar_wait(bar.p_full(), uint32_t(T) & 1u, abort_flag)) { ok = false; break; }
          tc_fence_after();
          mma_sum<D>(TM_DV, TM_S, TM_S + 64, sdo0 + uint32_t(T & 1) * L::TILE, t > 0);
          tc_commit(bar.do_empty(T));
          if (more) issue_s(T + 1);
          if (!ok || !mbar_wait(bar.ds_full(), uint32_t(T) & 1u, abort_flag)) { ok = false; break; }
          tc_fence_after();
          mma_sum<D>(TM_DK, TM_DP, TM_DP + 64, sq0 + uint32_t(T % 3) * L::TILE, t > 0);
          tc_commit(bar.q_empty(T));
          if (more) issue_dp(T + 1);
          else tc_commit(bar.done());
          if (ok && t + 2 == n_tiles) tc_commit(bar.kv_free());
        }
      }
    }
  } else {
    const int sw = warp - 2;
    const int q = warp & 3;
    const int hf = sw >> 2;              // query-column half of the tile owned by this warp
    const int r = q * 32 + lane;         // key row inside the tile
    const int tid = threadIdx.x - 64;    // 0..255
    const uint32_t lane_addr = uint32_t(q * 32) << 16;
    const float c = p.scale * LOG2E;
    const int col = tid & 127, col_at = col / p.G, col_g = col - col_at * p.G;
    // tid < 128: lse2 of column tid of the query tile that begins at position q0; else delta of column tid - 128
    auto load_stat = [&](const PackedSlot& s, int q0) -> float {
      const int pos = q0 + col_at;
      if (s.len == 0 || col_at >= p.P || pos >= s.len) return (tid < 128) ? INFINITY : 0.f;
      const long long at = (long long)(s.start + pos) * H + s.kv * p.G + col_g;
      return (tid < 128) ? p.lse[at] * LOG2E : p.delta[at];
    };
    float* stat = tid < 128 ? stat_lse : stat_dl;
    bool ok = true;
    int T = 0;
    PackedSlot slot = ring.take_warp(0, lane);
    if (slot.len > 0) stat[col] = load_stat(slot, KeyTile(p, slot.len, slot.tile).i_lo * p.P);
    for (int n = 0; slot.len > 0; ++n) {
      const KeyTile kt(p, slot.len, slot.tile);
      const int len = slot.len, n0 = kt.n0, key = n0 + r;
      const int last_pos = min(key + min(p.window, len - 1 - n0), len - 1);      // last query that sees this key
      for (int t = 0; t < kt.n_tiles; ++t, ++T) {
        const int q0 = (kt.i_lo + t) * p.P;          // first position of the tile
        const int buf = T & 1;
        // statistics of tile T are visible to all eight warps (an mbarrier, whose wait ends, and no named barrier)
        __syncwarp();
        if (lane == 0) mbar_arrive(bar.stat());
        if (!wait_warp(bar.stat(), uint32_t(T) & 1u, abort_flag)) { ok = false; break; }
        // in flight while this tile is processed; positions past the last tile belong to nobody here
        const float next_stat = t + 1 < kt.n_tiles ? load_stat(slot, q0 + p.P) : 0.f;
        const float4* cl = reinterpret_cast<const float4*>(stat_lse + buf * 128 + hf * 64);
        const float4* cd = reinterpret_cast<const float4*>(stat_dl + buf * 128 + hf * 64);
        float pr[64];
        // ---- phase A: P^T = exp2(S^T * c - lse2[query]) ----
        if (!wait_warp(bar.s_full(), uint32_t(T) & 1u, abort_flag)) { ok = false; break; }
        {
          tc_fence_after();
          uint32_t s0[32], s1[32];
          tmem_ld64(TM_S + lane_addr + uint32_t(hf * 64), s0, s1);
          if (q0 < n0 + 127 || q0 + p.P - 1 > n0 + p.window) {
            // the queries that see a key are one interval of positions, key ... last_pos, and so of columns
            const bool seen = key < len && last_pos >= q0;
            const int lo = seen ? max(key - q0, 0) * p.G - hf * 64 : 64;
            const int hi = seen ? (min(last_pos - q0, p.P - 1) + 1) * p.G - 1 - hf * 64 : 0;
            hide(s0, visible(lo, hi));
            hide(s1, visible(lo - 32, hi - 32));
          }
          exp2_64<false>(s0, s1, c, 0.f, cl, pr);
          uint32_t pk[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) pk[j] = pack_bf16(pr[2 * j], pr[2 * j + 1]);
          tmem_st32(TM_S + lane_addr + uint32_t(hf * 64), pk);   // over this thread's own, already read, S^T columns
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar.p_full());
        }
        // ---- phase B: dS^T = P^T * (dP^T - delta[query]) ----
        if (!wait_warp(bar.dp_full(), uint32_t(T) & 1u, abort_flag)) { ok = false; break; }
        {
          tc_fence_after();
          uint32_t d0[32], d1[32];
          tmem_ld64(TM_DP + lane_addr + uint32_t(hf * 64), d0, d1);
          uint32_t pk[32];
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const float4 e0 = cd[g], e1 = cd[8 + g];
            pk[2 * g] = pack_bf16(pr[4 * g] * (__uint_as_float(d0[4 * g]) - e0.x), pr[4 * g + 1] * (__uint_as_float(d0[4 * g + 1]) - e0.y));
            pk[2 * g + 1] = pack_bf16(pr[4 * g + 2] * (__uint_as_float(d0[4 * g + 2]) - e0.z),
                                      pr[4 * g + 3] * (__uint_as_float(d0[4 * g + 3]) - e0.w));
            pk[16 + 2 * g] = pack_bf16(pr[32 + 4 * g] * (__uint_as_float(d1[4 * g]) - e1.x),
                                       pr[32 + 4 * g + 1] * (__uint_as_float(d1[4 * g + 1]) - e1.y));
            pk[16 + 2 * g + 1] = pack_bf16(pr[32 + 4 * g + 2] * (__uint_as_float(d1[4 * g + 2]) - e1.z),
                                           pr[32 + 4 * g + 3] * (__uint_as_float(d1[4 * g + 3]) - e1.w));
          }
          tmem_st32(TM_DP + lane_addr + uint32_t(hf * 64), pk);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar.ds_full());
        }
        if (t + 1 < kt.n_tiles) stat[((T + 1) & 1) * 128 + col] = next_stat;
      }
      if (!ok) break;
      const PackedSlot done = slot;
      slot = ring.take_warp(n + 1, lane);
      const float first_stat = slot.len > 0 ? load_stat(slot, KeyTile(p, slot.len, slot.tile).i_lo * p.P) : 0.f;
      if (!wait_warp(bar.done(), uint32_t(n) & 1u, abort_flag)) break;
      {
        tc_fence_after();
        const uint32_t stage = smem_u32(smem + L::RING2 + ((T - 1) & 1) * L::TILE) + uint32_t(sw * (32 * D));
        const long long at = (long long)done.kv * D + hf * (D / 2);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          const long long off = key < len ? (long long)(done.start + key) * (which ? p.lddk : p.lddv) + at : -1;
          uint32_t w[D / 4];
          pack_columns<D / 2>((which ? TM_DK : TM_DV) + lane_addr + uint32_t(hf * (D / 2)), which ? p.scale : 1.f, w);
          store_rows<D / 2>(which ? p.dk : p.dv, off, w, stage, lane);
        }
        // rows of the slot that no load of dO fills are zero again
        constexpr int OWN = D / 4;                         // rows of 128 bytes that this warp has used
        const int first = (sw * OWN) & 127;
        __syncwarp();
        for (int e = lane; e < OWN * 8; e += 32) {
          if (first + (e >> 3) >= used) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(stage + uint32_t(e) * 16u), "r"(0) : "memory");
        }
        fence_proxy_async_smem();                          // before the slot's next load overwrites it
        __syncwarp();
        if (lane == 0) mbar_arrive(bar.out_free(n));
      }
      if (slot.len > 0) stat[(T & 1) * 128 + col] = first_stat;
    }
  }
}

template <int D>
__global__ void __launch_bounds__(ATT_WIDE_THREADS, 1)
attn_packed_bwd_k(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO, const __grid_constant__ PackedArgs p) {
  using L = PackedBwdSmem<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {   // the swizzled tiles need 1 KB alignment; nothing has been allocated yet
    grid_wait();
    if (threadIdx.x == 0 && p.err) atomicExch(p.err, ERR_SMEM_ALIGN);
    return;
  }
  BwdCta cta;
  cta.smem = smem;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::COMMON);
  cta.abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  cta.warp = threadIdx.x >> 5;
  cta.lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    const DkvBars<D> kb{reinterpret_cast<uint64_t*>(smem + L::BAR)};
    const DqBars<D> qb{reinterpret_cast<uint64_t*>(smem + L::BAR_DQ)};
    kb.init();
    qb.init();
    for (int i = 0; i < 2; ++i) {
      mbar_init(kb.ring() + i, 1); mbar_init(kb.ring() + 2 + i, 1 + 8);
      mbar_init(qb.ring() + i, 1); mbar_init(qb.ring() + 2 + i, 1 + 8);
    }
    *cta.abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV); tma_prefetch_desc(&tmDO);
  }
  if (cta.warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  const int used = p.P * p.G;
  if (used < 128 && cta.warp >= 2 && cta.warp < 7) {      // rows that no copy fills, in the five slots: they are summed over as well
    zero_rows<D>(smem + L::RING3 + (cta.warp - 2) * L::TILE, used, 128, cta.lane);
    fence_proxy_async_smem();
  }
  static_assert(L::RING2 == L::RING3 + 3 * L::TILE, "the rings follow one another");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cta.tmem = *tmem_slot;
  grid_enter();                 // global memory is not touched above
  packed_bwd_dkv<D>(tmQ, tmK, tmV, tmDO, p, cta);
  __syncwarp();
  tc_fence_before();
  __syncthreads();              // every role has left the key tiles: their shared memory and TMEM are free
  tc_fence_after();
  if (!*cta.abort_flag) packed_bwd_dq<D>(tmQ, tmK, tmV, tmDO, p, cta);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *cta.abort_flag && p.err) atomicExch(p.err, ERR_ATTN_TIMEOUT);
  if (cta.warp == 1) { __syncwarp(); tc_fence_after(); tmem_dealloc(cta.tmem, 512); }
}

// delta[row, head] = sum_d dO * O in fp32, with the part of O that its rounding left over: dS = P (dP - delta) cancels, and the error
// of delta would add as much to dQ and dK as the rounding of dS itself.  D / 16 lanes per (row, head).  Also starts the two lists of
// the kernel behind it.
template <int D>
__global__ void __launch_bounds__(256) attn_packed_delta_k(const __nv_bfloat16* o, const int8_t* o_lo, long long ldo,
                                                           const __nv_bfloat16* d_o, long long row_do, long long head_do, float* delta, int* next,
                                                           long long n, int H) {
  constexpr int LANES = D / 16;
  grid_enter();
  if (blockIdx.x == 0 && threadIdx.x < 2) next[threadIdx.x] = 0;
  const long long i = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int l = threadIdx.x % LANES;
  float acc = 0.f;
  if (i < n) {
    const long long row = n >> 32 ? i / H : (long long)(uint32_t(i) / uint32_t(H)), head = i - row * H;
    const long long at = row * ldo + head * D + l * 16;
    const uint4* a = reinterpret_cast<const uint4*>(o + at);
    const uint4* b = reinterpret_cast<const uint4*>(d_o + row * row_do + head * head_do + l * 16);
    const uint4 a0 = a[0], a1 = a[1], b0 = b[0], b1 = b[1], c = *reinterpret_cast<const uint4*>(o_lo + at);
    const uint32_t aw[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w}, bw[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
    const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 y = unpack_bf16(bw[e]);
      acc += with_rest(aw[e] << 16, cw[e / 2], 2 * (e & 1)) * y.x + with_rest(aw[e] & 0xffff0000u, cw[e / 2], 2 * (e & 1) + 1) * y.y;
    }
  }
#pragma unroll
  for (int s = LANES / 2; s > 0; s >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, s);
  if (l == 0 && i < n) delta[i] = acc;
}

// -----------------------------------------------------------------------------------------------
// [D, G, KV, rows] view of the queries; one box is a query tile's 64-column half
static int make_group_tmap(CUtensorMap* m, const void* base, const ArbPacked& a, long long row, long long head) {
  const uint32_t P = 128 / uint32_t(a.G);
  uint64_t dims[4] = {uint64_t(a.D), uint64_t(a.G), uint64_t(a.KV), uint64_t(a.rows)};
  uint64_t str[3] = {uint64_t(head) * 2, uint64_t(head) * uint64_t(a.G) * 2, uint64_t(row) * 2};
  uint32_t box[4] = {64, uint32_t(a.G), 1, P};
  return make_tmap_bf16(m, base, 4, dims, str, box);
}
// the same of O (two bytes an element) or its rest (one), as they are written; one box is 32 columns of the 32 rows of a warp
// (G divides 32)
static int make_out_tmap(CUtensorMap* m, const void* base, const ArbPacked& a, int bytes) {
  uint64_t dims[4] = {uint64_t(a.D), uint64_t(a.G), uint64_t(a.KV), uint64_t(a.rows)};
  uint64_t str[3] = {uint64_t(a.D) * bytes, uint64_t(a.D) * uint64_t(a.G) * bytes, uint64_t(a.o_row) * bytes};
  uint32_t box[4] = {32, uint32_t(a.G), 1, 32 / uint32_t(a.G)};
  return make_tmap_typed(m, base, 4, dims, str, box, bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8,
                         bytes == 2 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE);
}
static int make_key_tmap(CUtensorMap* m, const void* base, const ArbPacked& a, long long row, long long head) {
  uint64_t dims[3] = {uint64_t(a.D), uint64_t(a.KV), uint64_t(a.rows)};
  uint64_t str[2] = {uint64_t(head) * 2, uint64_t(row) * 2};
  uint32_t box[3] = {64, 1, 128};
  return make_tmap_bf16(m, base, 3, dims, str, box);
}

static int check_packed(const ArbPacked& a) {
  // masked scores are -inf, rows take the largest score; in fp32 neither the scale nor its reciprocal nears the ends of the range
  constexpr double TOP = 18446744073709551616.0;         // 2^64
  if (!(a.scale >= 1.0 / TOP && a.scale <= TOP)) return -3;
  // positions plus a window stay within 31 bits
  if (a.rows <= 0 || a.rows > PACKED_MAX_ROWS || a.KV <= 0 || a.KV > 65535 || a.G <= 0 || a.G > 128 || (a.D != 64 && a.D != 128) || a.window < 0) return -3;
  if (!a.items || bad_ptr(a.items) || a.cap_q <= 0 || a.cap_k <= 0 || (a.cap_q + a.cap_k) * a.KV > 0x7fffffffll) return -3;
  const void* ptrs[] = {a.q, a.k, a.v, a.o, a.o_lo, a.d_o, a.dq, a.dk, a.dv};
  const long long strides[] = {a.q_row, a.q_head, a.k_row, a.k_head, a.v_row, a.v_head, a.o_row, a.do_row, a.do_head, a.dq_row, a.dk_row, a.dv_row};
  for (const void* p : ptrs) if (bad_ptr(p)) return -4;
  for (long long s : strides) if (s < 0 || (s & 7)) return -4;
  if (a.o_lo && (a.o_row & 15)) return -4;               // a byte an element
  return 0;
}

static int packed_sms() {
  static int n = 0;
  if (!n) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  }
  return n;
}

static PackedArgs packed_args(const ArbPacked& a, int* err) {
  PackedArgs r{};
  r.KV = int(a.KV); r.G = int(a.G); r.P = 128 / r.G;
  r.items_q = reinterpret_cast<const PackedItem*>(a.items);
  r.items_k = r.items_q + a.cap_q;
  r.n_q = int(a.cap_q); r.n_k = int(a.cap_k);
  r.head_span = r.KV < 8 ? r.KV : 8;
  r.window = int(a.window < a.rows ? a.window : a.rows);
  r.scale = float(a.scale);
  r.lse = a.lse; r.delta = a.delta; r.err = err;
  return r;
}

template <int D>
static int packed_fwd(const ArbPacked& a, int* err, cudaStream_t stream) {
  static PerDeviceOnce cfg;
  if (cfg.first()) { if (int r = set_smem(attn_packed_fwd_k<D>, PackedFwdSmem<D>::TOTAL)) return r; }
  CUtensorMap tq, tk, tv, to{}, tr{};
  int r;
  if ((r = make_group_tmap(&tq, a.q, a, a.q_row, a.q_head))) return 1000 + r;
  if ((r = make_key_tmap(&tk, a.k, a, a.k_row, a.k_head))) return 1000 + r;
  if ((r = make_key_tmap(&tv, a.v, a, a.v_row, a.v_head))) return 1000 + r;
  if (32 % a.G == 0) {
    if ((r = make_out_tmap(&to, a.o, a, 2))) return 1000 + r;
    if (a.o_lo && (r = make_out_tmap(&tr, a.o_lo, a, 1))) return 1000 + r;
  }
  PackedArgs p = packed_args(a, err);
  p.o = reinterpret_cast<__nv_bfloat16*>(a.o); p.ldo = a.o_row;
  p.o_lo = reinterpret_cast<int8_t*>(a.o_lo);
  return launch_dependent(true, attn_packed_fwd_k<D>, unsigned(a.cap_q * a.KV), ATT_THREADS, PackedFwdSmem<D>::TOTAL, stream, tq, tk, tv, to, tr, p);
}

template <int D>
static int packed_bwd(const ArbPacked& a, int* err, cudaStream_t stream) {
  static PerDeviceOnce cfg;
  if (cfg.first()) { if (int r = set_smem(attn_packed_bwd_k<D>, PackedBwdSmem<D>::TOTAL)) return r; }
  CUtensorMap tq, tk, tv, tdo;
  int r;
  if ((r = make_group_tmap(&tq, a.q, a, a.q_row, a.q_head))) return 1000 + r;
  if ((r = make_key_tmap(&tk, a.k, a, a.k_row, a.k_head))) return 1000 + r;
  if ((r = make_key_tmap(&tv, a.v, a, a.v_row, a.v_head))) return 1000 + r;
  if ((r = make_group_tmap(&tdo, a.d_o, a, a.do_row, a.do_head))) return 1000 + r;
  const int H = int(a.KV * a.G);
  const long long n = a.rows * H, blocks = (n * (D / 16) + 255) / 256;
  if (blocks > 0x7fffffffll) return -3;
  int* next = reinterpret_cast<int*>(a.delta + n);
  if ((r = launch_dependent(n * D * 2 <= EARLY_BYTES, attn_packed_delta_k<D>, unsigned(blocks), 256, 0, stream,
                            reinterpret_cast<const __nv_bfloat16*>(a.o), reinterpret_cast<const int8_t*>(a.o_lo), a.o_row,
                            reinterpret_cast<const __nv_bfloat16*>(a.d_o), a.do_row, a.do_head, a.delta, next, n, H)))
    return r;
  PackedArgs p = packed_args(a, err);
  p.o = reinterpret_cast<__nv_bfloat16*>(a.dq); p.ldo = a.dq_row;
  p.dk = reinterpret_cast<__nv_bfloat16*>(a.dk); p.lddk = a.dk_row;
  p.dv = reinterpret_cast<__nv_bfloat16*>(a.dv); p.lddv = a.dv_row;
  p.next = next;
  const long long most = (a.cap_q > a.cap_k ? a.cap_q : a.cap_k) * a.KV, ctas = packed_sms();
  return launch_dependent(true, attn_packed_bwd_k<D>, unsigned(most < ctas ? most : ctas), ATT_WIDE_THREADS, PackedBwdSmem<D>::TOTAL, stream, tq, tk,
                          tv, tdo, p);
}

}  // namespace arb

using namespace arb;

extern "C" int arb_packed_plan(const int* cu, int n_seq, int rows, int G, int span_rows, void* items, int cap_q, int cap_k, int* scratch,
                               int* err_flag, cudaStream_t stream) {
  if (!cu || !items || !scratch || n_seq < 0 || rows <= 0 || rows > PACKED_MAX_ROWS || G <= 0 || G > 128 || span_rows <= 0 || bad_ptr(items)) return -3;
  PlanArgs p{};
  p.cu = cu; p.n = n_seq; p.rows = rows; p.P = 128 / G;
  // every sequence and the rows before and behind them end in at most one tile that is not full
  const long long most_q = (long long)rows / p.P + n_seq + 2, most_k = (long long)rows / 128 + n_seq + 2;
  if (cap_q < most_q || cap_k < most_k) return -6;
  const long long n = (long long)n_seq + 3;
  p.bound = scratch; p.first = scratch + 2 * n;
  p.items[0] = reinterpret_cast<PackedItem*>(items); p.items[1] = p.items[0] + cap_q;
  p.cap[0] = cap_q; p.cap[1] = cap_k;
  p.span_rows[0] = p.span_rows[1] = span_rows;
  p.err = err_flag;
  return launch_dependent(true, packed_plan_k, 2, PLAN_THREADS, 0, stream, p);
}

extern "C" int arb_packed_attn_fwd(const ArbPacked* a, int* err_flag, cudaStream_t stream) {
  if (!a || !a->q || !a->k || !a->v || !a->o || !a->lse) return -3;
  if (int r = check_packed(*a)) return r;
  return a->D == 64 ? packed_fwd<64>(*a, err_flag, stream) : packed_fwd<128>(*a, err_flag, stream);
}

extern "C" int arb_packed_attn_bwd(const ArbPacked* a, int* err_flag, cudaStream_t stream) {
  if (!a || !a->q || !a->k || !a->v || !a->o || !a->o_lo || !a->lse || !a->d_o || !a->delta || !a->dq || !a->dk || !a->dv) return -3;
  if (int r = check_packed(*a)) return r;
  return a->D == 64 ? packed_bwd<64>(*a, err_flag, stream) : packed_bwd<128>(*a, err_flag, stream);
}
