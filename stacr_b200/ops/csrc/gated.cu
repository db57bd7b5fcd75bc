// Gated activation: out = act(gate) * up, and its two gradients
//   dgate = dout * up * act'(gate),   dup = dout * act(gate)
// for bf16, fp16 and fp32 matrices whose rows may be strided (the two halves of one fused projection are read in place).
// All arithmetic is fp32 and a result is rounded once, to the type of the tensors.
//
// Bound by memory: 3 values per element forward, 5 backward.  A thread moves 16 bytes per operand, the widest vector that
// widths, strides and addresses allow; with the threads of a full SM about 100 KB are in flight, which hides the DRAM latency.
// 8192 x 8192 in bf16, silu: 62.8 us forward, 100.4 backward (6.4 and 6.7 TB/s, a copy's rate); two vectors a thread took
// 63.0 and 117, four 67 and 183 (fewer threads fit).
#include "gated.cuh"

namespace sb {

struct GatedArgs {
  const void *gate, *up, *dout;
  void *out, *dgate, *dup;
  long long ld_gate, ld_up, ld_dout, rows, n;  // results are contiguous, n per row
};

// One vector of every operand: its loads, and what is made of them.
template <typename T, int VEC, int ACT, bool BWD>
struct GatedItem {
  using P = Pack<T, VEC>;
  P g, u, d;
  __device__ __forceinline__ void load(const T* gate, const T* up, const T* dout, long long c) {
    g = load_once<P>(gate + c * VEC);
    u = load_once<P>(up + c * VEC);
    if (BWD) d = load_once<P>(dout + c * VEC);
  }
  __device__ __forceinline__ void finish(T* out, T* dgate, T* dup, long long c) const {
    float gv[VEC], uv[VEC], o1[VEC];
    unpack(g, gv);
    unpack(u, uv);
    if (BWD) {
      float dv[VEC], o2[VEC];
      unpack(d, dv);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float act, der;
        act_and_derivative<ACT, sizeof(T) == 2>(gv[i], act, der);
        o1[i] = dv[i] * uv[i] * der;
        o2[i] = dv[i] * act;
      }
      if (dgate) reinterpret_cast<P*>(dgate)[c] = pack<T, VEC>(o1);
      if (dup) reinterpret_cast<P*>(dup)[c] = pack<T, VEC>(o2);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) o1[i] = activation<ACT, sizeof(T) == 2>(gv[i]) * uv[i];
      reinterpret_cast<P*>(out)[c] = pack<T, VEC>(o1);
    }
  }
};

template <typename T, int VEC, int ACT, bool BWD>
__global__ void __launch_bounds__(256) gated_product_kernel(const GatedArgs a) {
  after_predecessors();
  const long long nv = a.n / VEC, step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long r = blockIdx.y * static_cast<long long>(blockDim.y) + threadIdx.y; r < a.rows; r += static_cast<long long>(gridDim.y) * blockDim.y) {
    const T* gate = static_cast<const T*>(a.gate) + r * a.ld_gate;
    const T* up = static_cast<const T*>(a.up) + r * a.ld_up;
    const T* dout = BWD ? static_cast<const T*>(a.dout) + r * a.ld_dout : nullptr;
    T* out = BWD ? nullptr : static_cast<T*>(a.out) + r * a.n;
    T* dgate = BWD && a.dgate ? static_cast<T*>(a.dgate) + r * a.n : nullptr;
    T* dup = BWD && a.dup ? static_cast<T*>(a.dup) + r * a.n : nullptr;
    for (long long c = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; c < nv; c += step) {
      GatedItem<T, VEC, ACT, BWD> item;
      item.load(gate, up, dout, c);
      item.finish(out, dgate, dup, c);
    }
    // values behind the last whole vector: only where there is one row
    if (VEC > 1 && blockIdx.x == 0 && nv * VEC + threadIdx.x < a.n) {
      GatedItem<T, 1, ACT, BWD> item;
      item.load(gate, up, dout, nv * VEC + threadIdx.x);
      item.finish(out, dgate, dup, nv * VEC + threadIdx.x);
    }
  }
}

template <typename T, int VEC, bool BWD>
static int gated_launch(const GatedArgs& a, int act, int sms, cudaStream_t st) {
  const long long nv = a.n / VEC;
  int tx = 32;
  while (tx < 256 && tx < nv) tx <<= 1;
  const dim3 block(tx, 256 / tx);
  // columns first, then as many row blocks as fill the GPU a few times over; longer inputs are strided over
  const long long bx = nv ? (nv + tx - 1) / tx : 1, want = static_cast<long long>(sms) * 32;
  const unsigned gx = static_cast<unsigned>(bx < want ? bx : want);
  long long by = (a.rows + block.y - 1) / block.y;
  const long long cap = (want + gx - 1) / gx;
  if (by > cap) by = cap;
  if (by > 65535) by = 65535;
  const dim3 grid(gx, static_cast<unsigned>(by));
  if (act == ACT_SILU) return launch_early(gated_product_kernel<T, VEC, ACT_SILU, BWD>, grid, block, 0, st, a);
  if (act == ACT_GELU) return launch_early(gated_product_kernel<T, VEC, ACT_GELU, BWD>, grid, block, 0, st, a);
  return launch_early(gated_product_kernel<T, VEC, ACT_GELU_TANH, BWD>, grid, block, 0, st, a);
}

// The widest power-of-two vector (in elements) that every operand's address and row stride allow, at most 16 bytes.  Of one row, the
// width does not matter: what is left behind the last vector is done by itself.
static int gated_width(const GatedArgs& a, int size) {
  unsigned long long bits = 16 / size;
  if (a.rows > 1)
    bits |= static_cast<unsigned long long>(a.n) | static_cast<unsigned long long>(a.ld_gate) | static_cast<unsigned long long>(a.ld_up) |
            static_cast<unsigned long long>(a.ld_dout);
  const void* ptrs[] = {a.gate, a.up, a.dout, a.out, a.dgate, a.dup};
  for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p) / size;
  return static_cast<int>(bits & (~bits + 1));
}

template <typename T, bool BWD>
static int gated_typed(const GatedArgs& a, int act, int sms, cudaStream_t st) {
  switch (gated_width(a, sizeof(T))) {
    case 8: if constexpr (sizeof(T) == 2) return gated_launch<T, 8, BWD>(a, act, sms, st);
    case 4: return gated_launch<T, 4, BWD>(a, act, sms, st);
    case 2: return gated_launch<T, 2, BWD>(a, act, sms, st);
    default: return gated_launch<T, 1, BWD>(a, act, sms, st);
  }
}

template <bool BWD>
static int gated_dispatch(GatedArgs a, int dtype, int act, int sms, cudaStream_t st) {
  if (a.rows <= 0 || a.n <= 0) return 0;
  if (act < 0 || act > 2) return -2;
  switch (dtype) {
    case DT_BF16: return gated_typed<__nv_bfloat16, BWD>(a, act, sms, st);
    case DT_FP16: return gated_typed<__half, BWD>(a, act, sms, st);
    case DT_FP32: return gated_typed<float, BWD>(a, act, sms, st);
  }
  return -2;
}

}  // namespace sb

// out[rows, n] = act(gate) * up; row strides in elements; dtype 0 bf16, 1 fp16, 2 fp32; act 0 silu, 1 gelu (erf), 2 gelu (tanh).
extern "C" int sb_gated_product_fwd(const void* gate, const void* up, void* out, long long ld_gate, long long ld_up, long long rows, long long n,
                                    int dtype, int act, int sms, void* stream) {
  sb::GatedArgs a{gate, up, nullptr, out, nullptr, nullptr, ld_gate, ld_up, 0, rows, n};
  return sb::gated_dispatch<false>(a, dtype, act, sms, static_cast<cudaStream_t>(stream));
}

// Gradients of the above, contiguous; either may be null.
extern "C" int sb_gated_product_bwd(const void* dout, const void* gate, const void* up, void* dgate, void* dup, long long ld_dout, long long ld_gate,
                                    long long ld_up, long long rows, long long n, int dtype, int act, int sms, void* stream) {
  sb::GatedArgs a{gate, up, dout, nullptr, dgate, dup, ld_gate, ld_up, ld_dout, rows, n};
  return sb::gated_dispatch<true>(a, dtype, act, sms, static_cast<cudaStream_t>(stream));
}
