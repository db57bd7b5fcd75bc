// Global gradient norm over many tensors and clipping:
//   norm = sqrt(sum over all tensors of g^2),   g *= min(1, max_norm / (norm + 1e-6)).
//
// Two kernels.  The first gives each CTA a fixed list of chunks and writes one partial sum per CTA; the second adds the partials
// (every CTA the same ones in the same order, so all get the same bits and nothing depends on the order in which CTAs ran), and
// scales its chunks unless the factor is 1.  There are no atomics and no state between calls.  The tensor table travels in the
// kernel's parameters: no copy to the device, and a captured call keeps its own.
//
// Bound by memory: N values read, and when the norm is above the bound N read and written again.  The second kernel takes its
// chunks from the last to the first, since the end of what the first one read is what L2 still holds.  2^30 fp32 values: norm 610 us
// (7.0 TB/s), with scaling 2038 (three passes at 0.97 of a copy's rate); bf16 305 and 1040.  Chunks of 4 K to 64 K values, four CTAs
// an SM and streaming stores all measured within 2 %.
//
// Sums: 16 squares in fp32, those sums in fp64.  Sixteen squares that leave fp32's range (|g| beyond 1e19 or below 1e-15) are
// redone in fp64.
#include "gated.cuh"

namespace sb {

constexpr int CLIP_TENSORS = 512;
constexpr int CLIP_THREADS = 256;

struct ClipTable {
  void* ptr[CLIP_TENSORS];
  long long numel[CLIP_TENSORS];
  int chunk_end[CLIP_TENSORS];     // chunks of this launch up to and including tensor i
  unsigned char dtype[CLIP_TENSORS];
  int n, chunks;
  long long chunk;                 // elements per chunk, a multiple of 16 * CLIP_THREADS
};

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < CLIP_THREADS / 32; ++w) s += red[w];
  __syncthreads();
  return s;
}

// Sum of the squares of up to 16 values in registers.
__device__ __forceinline__ double squares16(const float (&v)[16]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s = fmaf(v[i], v[i], s);
  if (s > 1e-28f && s < 1e37f) return static_cast<double>(s);
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    // fast math flushes subnormal fp32 values: the conversion reads their bits instead
    const unsigned bits = __float_as_uint(v[i]);
    const double x = (bits & 0x7f800000u) ? static_cast<double>(v[i]) : static_cast<double>(bits & 0x7fffffu) * 1.401298464324817e-45;
    d += x * x;
  }
  return d;
}

template <typename T>
struct alignas(16) Vec16 {
  T v[16 / sizeof(T)];
};

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, long long len) {
  constexpr int W = 16 / sizeof(T), LOADS = 16 / W;
  double acc = 0.0;
  long long done = 0;
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const Vec16<T>* v = reinterpret_cast<const Vec16<T>*>(p);
    const long long step = 16LL * CLIP_THREADS;
    for (; done + step <= len; done += step) {
      float f[16];
#pragma unroll
      for (int l = 0; l < LOADS; ++l) {
        const Vec16<T> x = v[done / W + l * CLIP_THREADS + threadIdx.x];
#pragma unroll
        for (int i = 0; i < W; ++i) f[l * W + i] = to_f32(x.v[i]);
      }
      acc += squares16(f);
    }
  }
  for (; done < len; done += 16LL * CLIP_THREADS) {
    float f[16];
#pragma unroll
    for (int l = 0; l < 16; ++l) {
      const long long at = done + l * CLIP_THREADS + threadIdx.x;
      f[l] = at < len ? to_f32(p[at]) : 0.f;
    }
    acc += squares16(f);
  }
  return acc;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(T* p, long long len, float by) {
  constexpr int W = 16 / sizeof(T);
  long long done = 0;
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    Vec16<T>* v = reinterpret_cast<Vec16<T>*>(p);
    const long long nv = len / W;
#pragma unroll 4
    for (long long i = threadIdx.x; i < nv; i += CLIP_THREADS) {
      Vec16<T> x = v[i];
#pragma unroll
      for (int j = 0; j < W; ++j) x.v[j] = from_f32<T>(to_f32(x.v[j]) * by);
      v[i] = x;
    }
    done = nv * W;
  }
  for (long long i = done + threadIdx.x; i < len; i += CLIP_THREADS) p[i] = from_f32<T>(to_f32(p[i]) * by);
}

// tensor of chunk c, and where in it the chunk starts and how long it is
__device__ __forceinline__ int locate(const ClipTable& t, int c, long long& start, long long& len) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (c < t.chunk_end[mid]) hi = mid; else lo = mid + 1;
  }
  start = static_cast<long long>(c - (lo ? t.chunk_end[lo - 1] : 0)) * t.chunk;
  len = t.numel[lo] - start < t.chunk ? t.numel[lo] - start : t.chunk;
  return lo;
}

__global__ void __launch_bounds__(CLIP_THREADS) grad_squares_kernel(const __grid_constant__ ClipTable t, double* __restrict__ partial) {
  __shared__ double red[CLIP_THREADS / 32];
  double acc = 0.0;
  after_predecessors();
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    long long start, len;
    const int i = locate(t, c, start, len);
    if (t.dtype[i] == DT_FP32) acc += chunk_squares(static_cast<const float*>(t.ptr[i]) + start, len);
    else if (t.dtype[i] == DT_BF16) acc += chunk_squares(static_cast<const __nv_bfloat16*>(t.ptr[i]) + start, len);
    else acc += chunk_squares(static_cast<const __half*>(t.ptr[i]) + start, len);
  }
  acc = block_sum(acc, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// scale = 0: only the norm (one CTA)
__global__ void __launch_bounds__(CLIP_THREADS) grad_scale_kernel(const __grid_constant__ ClipTable t, const double* __restrict__ partial, int n_partial,
                                                                  double max_norm, int scale, float* __restrict__ norm_out) {
  __shared__ double red[CLIP_THREADS / 32];
  double acc = 0.0;
  after_predecessors();
  for (int i = threadIdx.x; i < n_partial; i += CLIP_THREADS) acc += partial[i];
  const double norm = sqrt(block_sum(acc, red));
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = static_cast<float>(norm);
  if (!scale) return;
  const double factor = max_norm / (norm + 1e-6);
  if (factor >= 1.0) return;      // a NaN norm scales: every gradient becomes NaN, as a finite factor would leave it unnoticed
  const float by = static_cast<float>(factor);
  for (int c = t.chunks - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
    long long start, len;
    const int i = locate(t, c, start, len);
    if (t.dtype[i] == DT_FP32) chunk_scale(static_cast<float*>(t.ptr[i]) + start, len, by);
    else if (t.dtype[i] == DT_BF16) chunk_scale(static_cast<__nv_bfloat16*>(t.ptr[i]) + start, len, by);
    else chunk_scale(static_cast<__half*>(t.ptr[i]) + start, len, by);
  }
}

// Elements per chunk: enough chunks for every CTA of a small job, 16 K elements for a large one.
static long long clip_chunk(const long long* numel, int n, int ctas) {
  long long total = 0;
  for (int i = 0; i < n; ++i) total += numel[i];
  const long long quantum = 16LL * CLIP_THREADS;
  long long c = (total / ctas + quantum - 1) / quantum * quantum;
  return c < quantum ? quantum : c > 4 * quantum ? 4 * quantum : c;
}

static bool fill_table(ClipTable& t, void* const* ptrs, const long long* numel, const unsigned char* dtype, int n, long long chunk) {
  t.n = n;
  t.chunk = chunk;
  long long end = 0;
  for (int i = 0; i < n; ++i) {
    t.ptr[i] = ptrs[i];
    t.numel[i] = numel[i];
    t.dtype[i] = dtype[i];
    end += (numel[i] + chunk - 1) / chunk;
    if (end > 0x7fffffffLL) return false;
    t.chunk_end[i] = static_cast<int>(end);
  }
  t.chunks = static_cast<int>(end);
  return true;
}

}  // namespace sb

extern "C" int sb_clip_tensors_per_launch() { return sb::CLIP_TENSORS; }

// Doubles that `partial` of sb_grad_clip has to hold for n tensors.
extern "C" int sb_clip_partials(int n, int sms) { return ((n + sb::CLIP_TENSORS - 1) / sb::CLIP_TENSORS) * sms * 8; }

// Norm of n tensors (dtype 0 bf16, 1 fp16, 2 fp32; none empty, none overlapping) into *norm_out, and with scale != 0 their clipping
// to max_norm in place.
extern "C" int sb_grad_clip(void* const* ptrs, const long long* numel, const unsigned char* dtype, int n, double* partial, float* norm_out,
                            double max_norm, int scale, int sms, void* stream) {
  using namespace sb;
  if (n <= 0) return -2;
  for (int i = 0; i < n; ++i)
    if (numel[i] <= 0 || dtype[i] > DT_FP32) return -2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int ctas = sms * 8;
  const long long chunk = clip_chunk(numel, n, ctas);
  ClipTable t;
  int parts = 0;
  for (int lo = 0; lo < n; lo += CLIP_TENSORS) {
    const int m = n - lo < CLIP_TENSORS ? n - lo : CLIP_TENSORS;
    if (!fill_table(t, ptrs + lo, numel + lo, dtype + lo, m, chunk)) return -2;
    const int grid = t.chunks < ctas ? t.chunks : ctas;
    const int rc = launch_early(grad_squares_kernel, dim3(grid), dim3(CLIP_THREADS), 0, st, t, partial + parts);
    if (rc) return rc;
    parts += grid;
  }
  // the groups in reverse: the last one's table is still in t, and its end is what L2 holds
  for (int lo = (n - 1) / CLIP_TENSORS * CLIP_TENSORS; lo >= 0; lo -= CLIP_TENSORS) {
    const int m = n - lo < CLIP_TENSORS ? n - lo : CLIP_TENSORS;
    fill_table(t, ptrs + lo, numel + lo, dtype + lo, m, chunk);
    const int grid = !scale ? 1 : t.chunks < ctas ? t.chunks : ctas;
    const int rc = launch_early(grad_scale_kernel, dim3(grid), dim3(CLIP_THREADS), 0, st, t, partial, parts, max_norm, scale, norm_out);
    if (rc) return rc;
    if (!scale) break;
  }
  return 0;
}
