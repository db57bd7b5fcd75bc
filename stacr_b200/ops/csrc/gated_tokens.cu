// Gated projections of single tokens: h[M, F] = act(x Wg^T + bg) * (x Wu^T + bu) for M <= 64 (see sb_gated_forward for when).
//
// Bound by the weights, 4 K F bytes that are read once (one token, K 4096, F 14336: 38.3 us, 6.1 TB/s, 0.94 of a copy's rate);
// everything here serves that stream.  A CTA owns 16 features (16 rows of
// each weight) and its eight warps share the reduction: warp w takes every eighth block of 32 values, so that the CTA reads 512
// contiguous bytes of a row at a time.  Weights go from memory straight into the A fragments of mma.m16n8k16 (features are the
// 16 rows, tokens the 8 columns): a reduction does not care which k sits where as long as both operands agree, so a thread's 16
// contiguous bytes are its share of two instructions, and no shared memory, barrier or transpose stands between the
// loads.  The tokens' B fragments are read the same way and hit L1 / L2.  Few tokens keep the tensor work far below
// the stream's time on these instructions; tcgen05 would need its weights staged in shared memory and gains nothing here.
// The eight partial sums meet in shared memory, in one order always.
#include "gated.cuh"

namespace sb {
namespace gt {

constexpr int WARPS = 8, FT = 16, KB = 32;

struct Args {
  const __nv_bfloat16 *x, *wg, *wu;
  const float *bg, *bu;
  __nv_bfloat16* h;
  unsigned short *a_hi, *b_hi;     // the backward's factors in 24 bits (see gated_gemm.cu), null: not kept
  unsigned char *a_lo, *b_lo;
  long long ld_lo;
  int M, K, F;
};

// weights pass through once: they are kept out of L1, where the tokens are
__device__ __forceinline__ uint4 load_stream(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: groups of 8 tokens.  U: blocks of 32 values whose weights are in flight together.
template <int NT, int U, int ACT>
__global__ void __launch_bounds__(WARPS * 32, NT == 8 ? 1 : 2) gated_tokens_kernel(const Args a) {
  extern __shared__ float part[];                       // [WARPS][2][NT][FT * 8]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int f0 = blockIdx.x * FT;
  // rows beyond F are read as row F - 1: their sums are never stored
  const int r0 = f0 + g < a.F ? f0 + g : a.F - 1, r1 = f0 + g + 8 < a.F ? f0 + g + 8 : a.F - 1;
  const __nv_bfloat16* w[4] = {a.wg + static_cast<size_t>(r0) * a.K, a.wg + static_cast<size_t>(r1) * a.K, a.wu + static_cast<size_t>(r0) * a.K,
                               a.wu + static_cast<size_t>(r1) * a.K};
  float cg[NT][4] = {}, cu[NT][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
  after_predecessors();
  for (int k0 = warp * KB; k0 < a.K; k0 += WARPS * KB * U) {
    uint4 v[U][4], bx[U][NT];
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int k = k0 + s * WARPS * KB + t * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[s][i] = k < a.K ? load_stream(w[i] + k) : zero;
    }
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int k = k0 + s * WARPS * KB + t * 8;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int m = n * 8 + g;
        bx[s][n] = (m < a.M && k < a.K) ? __ldg(reinterpret_cast<const uint4*>(a.x + static_cast<size_t>(m) * a.K + k)) : zero;
      }
    }
#pragma unroll
    for (int s = 0; s < U; ++s)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 b = bx[s][n];
        mma16816(cg[n], v[s][0].x, v[s][1].x, v[s][0].y, v[s][1].y, b.x, b.y);
        mma16816(cg[n], v[s][0].z, v[s][1].z, v[s][0].w, v[s][1].w, b.z, b.w);
        mma16816(cu[n], v[s][2].x, v[s][3].x, v[s][2].y, v[s][3].y, b.x, b.y);
        mma16816(cu[n], v[s][2].z, v[s][3].z, v[s][2].w, v[s][3].w, b.z, b.w);
      }
  }
  // partial sums, feature fastest: [warp][gate or up][token][feature]
  float* mine = part + warp * (2 * NT * FT * 8);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (n * 8 + 2 * t + (i & 1)) * FT + g + (i >> 1) * 8;
      mine[at] = cg[n][i];
      mine[NT * FT * 8 + at] = cu[n][i];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < NT * FT * 8; i += WARPS * 32) {
    const int f = f0 + i % FT, m = i / FT;
    if (f >= a.F || m >= a.M) continue;
    float gate = 0.f, up = 0.f;
#pragma unroll
    for (int q = 0; q < WARPS; ++q) {
      gate += part[q * (2 * NT * FT * 8) + i];
      up += part[q * (2 * NT * FT * 8) + NT * FT * 8 + i];
    }
    if (a.bg) gate += a.bg[f];
    if (a.bu) up += a.bu[f];
    float act, der;
    act_and_derivative<ACT, true>(gate, act, der);
    const size_t at = static_cast<size_t>(m) * a.F + f;
    a.h[at] = __float2bfloat16_rn(act * up);
    if (a.a_hi) {
      const unsigned fa = __float_as_uint(up * der), fb = __float_as_uint(act);
      a.a_hi[at] = static_cast<unsigned short>(fa >> 16);
      a.b_hi[at] = static_cast<unsigned short>(fb >> 16);
      a.a_lo[m * a.ld_lo + f] = static_cast<unsigned char>(fa >> 8);
      a.b_lo[m * a.ld_lo + f] = static_cast<unsigned char>(fb >> 8);
    }
  }
}

template <int NT, int U, int ACT>
static int launch(const Args& a, cudaStream_t st) {
  static PerDeviceOnce once;
  bool* configured = once.slot();
  if (configured == nullptr) return -8;
  constexpr int bytes = WARPS * 2 * NT * FT * 8 * 4;
  if (!*configured) {
    const cudaError_t e = cudaFuncSetAttribute(gated_tokens_kernel<NT, U, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    *configured = true;
  }
  return launch_early(gated_tokens_kernel<NT, U, ACT>, dim3((a.F + FT - 1) / FT), dim3(WARPS * 32), bytes, st, a);
}

template <int ACT>
static int launch_tokens(const Args& a, cudaStream_t st) {
  // as many blocks in flight as two CTAs per SM have registers for (one with 64 tokens)
  if (a.M <= 8) return launch<1, 4, ACT>(a, st);
  if (a.M <= 16) return launch<2, 3, ACT>(a, st);
  if (a.M <= 32) return launch<4, 2, ACT>(a, st);
  return launch<8, 2, ACT>(a, st);
}

int forward(const void* x, const void* wg, const void* wu, const float* bg, const float* bu, void* h, unsigned short* hi, unsigned char* lo, int M, int K, int F,
            int act, cudaStream_t st) {
  const long long ld_lo = (F + 15) / 16 * 16;
  const Args a{static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(wg), static_cast<const __nv_bfloat16*>(wu), bg, bu,
               static_cast<__nv_bfloat16*>(h), hi, hi ? hi + static_cast<size_t>(M) * F : nullptr, lo, lo ? lo + M * ld_lo : nullptr, ld_lo, M, K, F};
  switch (act) {
    case ACT_SILU: return launch_tokens<ACT_SILU>(a, st);
    case ACT_GELU: return launch_tokens<ACT_GELU>(a, st);
    case ACT_GELU_TANH: return launch_tokens<ACT_GELU_TANH>(a, st);
  }
  return -2;
}

}  // namespace gt
}  // namespace sb
