// Global gradient norm over a list of tensors, and clipping by it.
//
//   norm = sqrt(sum over all tensors and elements g^2);   out = g * min(1, max_norm / norm)
//
// Two launches, both bound by memory: one pass that leaves a sum per block, one that joins them (every block by itself, in one
// fixed order) and scales, from the last item to the first: what the first pass read last is still in L2.  The list travels as
// a kernel argument, so nothing is copied to the device and a captured graph holds it.  Work items are 16384 elements of one
// tensor; a thread has four loads of 16 bytes in flight and few enough registers for five blocks an SM (with all of an item's
// loads in flight at once, 120 and 242 registers a thread: 2.9 TB/s).
//
// Sums: a thread squares and adds up to 32 elements in fp32, then adds to a 64-bit sum.  Where the 32 leave the range in which
// fp32 squares are exact enough (elements around 1e-15 and below or 1e15 and above), they are squared again in 64 bits, from
// registers: the norm of any finite gradients is right.
#include "api.h"
#include "ptx.cuh"

#include <cuda_fp16.h>

namespace arb {

constexpr int CLIP_THREADS = 256;
constexpr int CLIP_ITEM = 16384;                 // elements: 64 per thread
constexpr int CLIP_SMALL = 128, CLIP_LARGE = 1024;

template <int CAP>
struct GradTable {
  const void* in[CAP];
  void* out[CAP];
  long long n[CAP];
  int first[CAP + 1];                            // first work item of each tensor
  unsigned char type[CAP];                       // input type + 4 x output type
  int count;
};
static_assert(sizeof(GradTable<CLIP_LARGE>) <= 32000, "kernel arguments end at 32764 bytes");

enum { GRAD_F32 = 0, GRAD_BF16 = 1, GRAD_F16 = 2 };

template <int TYPE> struct GradType;
template <> struct GradType<GRAD_F32> { using T = float; };
template <> struct GradType<GRAD_BF16> { using T = __nv_bfloat16; };
template <> struct GradType<GRAD_F16> { using T = __half; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f32(float x, float& y) { y = x; }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16& y) { y = __float2bfloat16(x); }
__device__ __forceinline__ void from_f32(float x, __half& y) { y = __float2half(x); }

// conversions that keep subnormal numbers (fast math flushes them)
__device__ __forceinline__ double widen(float x) {
  double y;
  asm("cvt.f64.f32 %0, %1;" : "=d"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float narrow(double x) {
  float y;
  asm("cvt.rn.f32.f64 %0, %1;" : "=f"(y) : "d"(x));
  return y;
}

// W elements as one access where they have at most 16 bytes, else as several
template <typename T, int W>
struct alignas(sizeof(T) * W < 16 ? sizeof(T) * W : 16) Vec { T v[W]; };

// elements from `p` on that one access of at most 16 bytes may take
template <typename T>
__device__ __forceinline__ int grad_width(const void* p) {
  const unsigned a = unsigned(reinterpret_cast<uintptr_t>(p));
  if (sizeof(T) == 2 && (a & 15u) == 0) return 8;
  if ((a & (4u * sizeof(T) - 1)) == 0) return 4;
  return (a & (2u * sizeof(T) - 1)) == 0 ? 2 : 1;
}

// the tensor that work item `i` belongs to
template <int CAP>
__device__ __forceinline__ int grad_tensor(const GradTable<CAP>& t, int i) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < CLIP_THREADS / 32; ++w) v += sh[w];
  return v;
}

// squares of N values, in 64 bits where fp32 would lose them
template <int N, typename T, int W>
__device__ __forceinline__ double batch_squares(const Vec<T, W> (&v)[N]) {
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const float x = to_f32(v[k].v[e]);
      float& a = s[(k * W + e) & 3];
      a = fmaf(x, x, a);
    }
  const float sum = (s[0] + s[1]) + (s[2] + s[3]);
  if (sum > 1e-28f && sum < 1e30f) return double(sum);
  double d = 0.0;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const double x = widen(to_f32(v[k].v[e]));
      d = fma(x, x, d);
    }
  return d;
}

// sum of squares of the thread's share of `n` <= CLIP_ITEM elements: four accesses at a time, then what is left one by one
template <typename T, int W>
__device__ __forceinline__ double item_squares(const T* p, int n) {
  double acc = 0.0;
  constexpr int STEP = CLIP_THREADS * W * 4;
  int at = 0;
#pragma unroll 1
  for (; at + STEP <= n; at += STEP) {
    Vec<T, W> v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const Vec<T, W>*>(p + at + (k * CLIP_THREADS + int(threadIdx.x)) * W);
    acc += batch_squares<4>(v);
  }
#pragma unroll 1
  for (int i = at + int(threadIdx.x); i < n; i += CLIP_THREADS) {
    Vec<T, 1> v[1];
    v[0].v[0] = p[i];
    acc += batch_squares<1>(v);
  }
  return acc;
}

template <typename T>
__device__ __forceinline__ double tensor_squares(const void* p, long long from, int n) {
  const T* q = reinterpret_cast<const T*>(p) + from;
  switch (grad_width<T>(q)) {
    case 8: if constexpr (sizeof(T) == 2) return item_squares<T, 8>(q, n);
    case 4: return item_squares<T, 4>(q, n);
    case 2: return item_squares<T, 2>(q, n);
    default: return item_squares<T, 1>(q, n);
  }
}

template <int CAP>
__global__ void __launch_bounds__(CLIP_THREADS, 5) grad_squares_k(const __grid_constant__ GradTable<CAP> t, double* partial) {
  __shared__ double sh[CLIP_THREADS / 32];
  grid_enter();
  double acc = 0.0;
  for (int i = blockIdx.x; i < t.first[t.count]; i += gridDim.x) {
    const int k = grad_tensor(t, i);
    const long long from = (long long)(i - t.first[k]) * CLIP_ITEM, left = t.n[k] - from;
    const int n = left < CLIP_ITEM ? int(left) : CLIP_ITEM;
    switch (t.type[k] & 3) {
      case GRAD_F32: acc += tensor_squares<float>(t.in[k], from, n); break;
      case GRAD_BF16: acc += tensor_squares<__nv_bfloat16>(t.in[k], from, n); break;
      default: acc += tensor_squares<__half>(t.in[k], from, n); break;
    }
  }
  acc = block_sum(acc, sh);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// min(1, max_norm / norm) as a product of two fp32 numbers: by itself it may be smaller than the normal numbers, and fast math takes those
// for zero.  (The first factor is normal down to 2^-252; below that no element comes out above 2^-124.)  1 is no multiplication at all,
// so that copies keep subnormal elements as they are.
struct GradFactor {
  float a, b;
  __device__ __forceinline__ explicit GradFactor(double c) : a(float(c)), b(1.f) {
    if (c < 0x1p-126) { a = float(c * 0x1p126); b = 0x1p-126f; }
  }
  __device__ __forceinline__ float operator()(float x) const { return a == 1.f ? x : x * a * b; }
};

template <typename TI, typename TO, int W>
__device__ __forceinline__ void item_scale(const TI* p, TO* q, int n, GradFactor c) {
  constexpr int STEP = CLIP_THREADS * W * 4;
  int at = 0;
#pragma unroll 1
  for (; at + STEP <= n; at += STEP) {
    Vec<TI, W> v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const Vec<TI, W>*>(p + at + (k * CLIP_THREADS + int(threadIdx.x)) * W);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      Vec<TO, W> o;
#pragma unroll
      for (int e = 0; e < W; ++e) from_f32(c(to_f32(v[k].v[e])), o.v[e]);
      *reinterpret_cast<Vec<TO, W>*>(q + at + (k * CLIP_THREADS + int(threadIdx.x)) * W) = o;
    }
  }
#pragma unroll 1
  for (int i = at + int(threadIdx.x); i < n; i += CLIP_THREADS) from_f32(c(to_f32(p[i])), q[i]);
}

template <typename TI, typename TO>
__device__ __forceinline__ void tensor_scale(const void* in, void* out, long long from, int n, GradFactor c) {
  const TI* p = reinterpret_cast<const TI*>(in) + from;
  TO* q = reinterpret_cast<TO*>(out) + from;
  switch (min(grad_width<TI>(p), grad_width<TO>(q))) {
    case 8: if constexpr (sizeof(TI) == 2 && sizeof(TO) == 2) { item_scale<TI, TO, 8>(p, q, n, c); break; }
    case 4: item_scale<TI, TO, 4>(p, q, n, c); break;
    case 2: item_scale<TI, TO, 2>(p, q, n, c); break;
    default: item_scale<TI, TO, 1>(p, q, n, c); break;
  }
}
template <typename TI>
__device__ __forceinline__ void tensor_scale_to(int to, const void* in, void* out, long long from, int n, GradFactor c) {
  switch (to) {
    case GRAD_F32: tensor_scale<TI, float>(in, out, from, n, c); break;
    case GRAD_BF16: tensor_scale<TI, __nv_bfloat16>(in, out, from, n, c); break;
    default: tensor_scale<TI, __half>(in, out, from, n, c); break;
  }
}

// max_norm < 0: the norm alone.  A norm that is not finite scales nothing (in 64 bits that of finite elements always is, also where it is
// infinite as the fp32 number that is handed out).
template <int CAP>
__global__ void __launch_bounds__(CLIP_THREADS, 5) grad_scale_k(const __grid_constant__ GradTable<CAP> t, const double* partial, int partials,
                                                             double max_norm, float* norm_out) {
  __shared__ double sh[CLIP_THREADS / 32];
  grid_enter();
  double acc = 0.0;
  for (int i = threadIdx.x; i < partials; i += CLIP_THREADS) acc += partial[i];
  const double norm = sqrt(block_sum(acc, sh));
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) *norm_out = narrow(norm);
  if (max_norm < 0.f) return;
  const GradFactor c(norm > double(max_norm) && norm <= 1.7976931348623157e308 ? double(max_norm) / norm : 1.0);
  for (int i = t.first[t.count] - 1 - int(blockIdx.x); i >= 0; i -= gridDim.x) {
    const int k = grad_tensor(t, i);
    if (c.a == 1.f && t.out[k] == t.in[k]) continue;          // in place and nothing to do
    const long long from = (long long)(i - t.first[k]) * CLIP_ITEM, left = t.n[k] - from;
    const int n = left < CLIP_ITEM ? int(left) : CLIP_ITEM;
    const int to = t.type[k] >> 2;
    switch (t.type[k] & 3) {
      case GRAD_F32: tensor_scale_to<float>(to, t.in[k], t.out[k], from, n, c); break;
      case GRAD_BF16: tensor_scale_to<__nv_bfloat16>(to, t.in[k], t.out[k], from, n, c); break;
      default: tensor_scale_to<__half>(to, t.in[k], t.out[k], from, n, c); break;
    }
  }
}

template <int CAP>
static int fill_table(GradTable<CAP>& t, const ArbGrad* g, int n) {
  long long items = 0;
  for (int k = 0; k < n; ++k) {
    if (g[k].n <= 0 || !g[k].in || g[k].type < 0 || g[k].type > 2 || g[k].out_type < 0 || g[k].out_type > 2) return -3;
    const uintptr_t in_size = g[k].type == GRAD_F32 ? 4 : 2, out_size = g[k].out_type == GRAD_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(g[k].in) % in_size) || (reinterpret_cast<uintptr_t>(g[k].out) % out_size)) return -4;
    t.in[k] = g[k].in; t.out[k] = g[k].out; t.n[k] = g[k].n;
    t.type[k] = (unsigned char)(g[k].type + 4 * g[k].out_type);
    t.first[k] = int(items);
    items += (g[k].n + CLIP_ITEM - 1) / CLIP_ITEM;
    if (items > 0x3fffffffll) return -3;
  }
  t.first[n] = int(items);
  t.count = n;
  return 0;
}

template <int CAP>
static int squares(const ArbGrad* g, int n, double* partial, int blocks, cudaStream_t stream) {
  GradTable<CAP> t;
  if (int r = fill_table(t, g, n)) return r;
  return launch_dependent(true, grad_squares_k<CAP>, unsigned(blocks), CLIP_THREADS, 0, stream, t, partial);
}
template <int CAP>
static int scale(const ArbGrad* g, int n, const double* partial, int partials, float max_norm, float* norm, int blocks, cudaStream_t stream) {
  GradTable<CAP> t;
  if (int r = fill_table(t, g, n)) return r;
  for (int k = 0; k < n && max_norm >= 0.f; ++k) if (!g[k].out) return -3;
  const int items = t.first[n];
  const int grid = max_norm < 0.f ? 1 : (items < blocks ? (items > 0 ? items : 1) : blocks);
  return launch_dependent(true, grad_scale_k<CAP>, unsigned(grid), CLIP_THREADS, 0, stream, t, partial, partials, max_norm, norm);
}

}  // namespace arb

using namespace arb;

extern "C" int arb_grad_squares(const ArbGrad* g, int n, double* partial, int blocks, cudaStream_t stream) {
  if (!g || n <= 0 || n > CLIP_LARGE || !partial || blocks <= 0) return -3;
  return n <= CLIP_SMALL ? squares<CLIP_SMALL>(g, n, partial, blocks, stream) : squares<CLIP_LARGE>(g, n, partial, blocks, stream);
}

extern "C" int arb_grad_scale(const ArbGrad* g, int n, const double* partial, int partials, float max_norm, float* norm, int blocks,
                              cudaStream_t stream) {
  if (!g || n <= 0 || n > CLIP_LARGE || !partial || partials <= 0 || blocks <= 0 || max_norm != max_norm) return -3;
  return n <= CLIP_SMALL ? scale<CLIP_SMALL>(g, n, partial, partials, max_norm, norm, blocks, stream)
                         : scale<CLIP_LARGE>(g, n, partial, partials, max_norm, norm, blocks, stream);
}
