// Gated projections of some tokens, h[M, F] = act(x Wg^T + bg) * (x Wu^T + bu) for M <= 128, where the weights' bytes are still the
// bound but there are too many tokens for the fragments of gated_tokens.cu.
//
// The operands change places: 64 rows of Wg and the same 64 of Wu are the 128 rows (tensor memory lanes) of a tcgen05.mma, the
// tokens, padded to N = 16, 32, 64 or 128, its columns.  So a CTA streams 64 features' weights once, 16 KB a k-block, and no row
// of the tensor memory is spent on tokens that are not there.  Where there are more CTAs than SMs two share one, with 110 KB of
// stages each, so that all F / 64 CTAs of a usual width are resident at once.  64 tokens, K 4096, F 14336 (235 MB): 41.8 us, 5.6
// TB/s or 0.86 of a copy's rate, against 54 for the 256-token tiles; K 2048, F 8192: 15.0 against 19.3.
// Lanes 0..63 end up with gate, 64..127 with up: the halves trade the tokens they do not finish through shared memory, gate lanes
// finish the first half of the tokens, up lanes the second.
#include "gated.cuh"

namespace sb {

int make_tensor_map_bf16(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t outer, uint64_t ld, uint32_t box_outer);

namespace gf {

constexpr int BK = 64, UMMA_K = 16, FT = 64, EPI_WARPS = 8, THREADS = 64 + 32 * EPI_WARPS;
constexpr int W_BYTES = 2 * FT * BK * 2;

// ALONE: a CTA has an SM to itself and takes all its shared memory for stages; else two share it.
template <int N, bool ALONE>
struct Layout {
  static constexpr int STAGE = W_BYTES + N * BK * 2;
  static constexpr int STAGES = (ALONE ? 224 : 110) * 1024 / STAGE;
  static constexpr int BYTES = STAGES * STAGE + 1024 + 256;
  static constexpr int COLS = N < 32 ? 32 : N;
  static_assert(FT * N * 4 <= STAGES * STAGE, "the trade takes the stages' place");
  static_assert((ALONE ? 1 : 2) * (BYTES + 1024) <= 233472, "of the SM's 228 KB");
};

struct Args {
  const float *bg, *bu;
  __nv_bfloat16* h;
  unsigned short *a_hi, *b_hi;     // the backward's factors in 24 bits (see gated_gemm.cu), null: not kept
  unsigned char *a_lo, *b_lo;
  long long ld_lo;
  int M, K, F;
  int* status;
};

__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI_WARPS) : "memory"); }

template <int N, bool ALONE, int ACT>
__global__ void __launch_bounds__(THREADS) gated_few_kernel(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_u,
                                                            const __grid_constant__ CUtensorMap map_x, const Args a) {
  using L = Layout<N, ALONE>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::STAGES * L::STAGE);
  uint64_t* empty_bar = full_bar + L::STAGES;
  uint64_t* done_bar = empty_bar + L::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int f0 = blockIdx.x * FT, num_kb = (a.K + BK - 1) / BK;

  auto load = [&](int kb, int s) {
    uint8_t* at = smem + s * L::STAGE;
    mbar_expect_tx(&full_bar[s], L::STAGE);
    tma_load_2d(at, &map_g, &full_bar[s], kb * BK, f0);
    tma_load_2d(at + W_BYTES / 2, &map_u, &full_bar[s], kb * BK, f0);
    tma_load_2d(at + W_BYTES, &map_x, &full_bar[s], kb * BK, 0);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
    after_predecessors();
    // the producer has its barriers: the first stages are under way while the others wait for the tensor memory
    for (int kb = 0; kb < L::STAGES && kb < num_kb; ++kb) load(kb, kb);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::COLS);
    tmem_relinquish();
  }
  after_predecessors();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;                                  // parity of the phase in which a stage's first contents are released
      for (int kb = L::STAGES; kb < num_kb; ++kb) {
        if (!mbar_wait(&empty_bar[s], ph, abort_flag, a.status, ST_TIMEOUT_SMEM_EMPTY)) break;
        load(kb, s);
        if (++s == L::STAGES) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_bf16(128, N, false, false);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&full_bar[s], ph, abort_flag, a.status, ST_TIMEOUT_SMEM_FULL)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sw = smem_u32(smem + s * L::STAGE);
#pragma unroll
        for (int j = 0; j < BK / UMMA_K; ++j)
          umma_bf16(tmem, make_smem_desc_sw128(sw + j * 32, 16, 1024), make_smem_desc_sw128(sw + W_BYTES + j * 32, 16, 1024), idesc, (kb > 0 || j > 0) ? 1u : 0u);
        umma_commit(&empty_bar[s]);
        if (++s == L::STAGES) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (ok) umma_commit(done_bar);
    }
  } else {
    // two warps for each quarter of the lanes, which take the chunks of 16 tokens in turn
    const int quad = warp & 3, sub = (warp - 2) >> 2;
    const bool is_gate = quad < 2;
    const int fl = (quad & 1) * 32 + lane, f = f0 + fl;
    const float* bias_of = is_gate ? a.bg : a.bu;
    const float bias = bias_of != nullptr && f < a.F ? bias_of[f] : 0.f;
    // when every product is done every copy has landed and been read: the stages' memory is free
    // (the whole warp goes on or gives up together: the tensor memory loads are warp-wide instructions)
    const bool ok = __all_sync(0xffffffffu, mbar_wait(done_bar, 0, abort_flag, a.status, ST_TIMEOUT_TMEM_FULL));
    tc_fence_after();
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    float* trade = reinterpret_cast<float*>(smem) + fl;   // [token][feature]: up of the first half of the tokens, gate of the second
    constexpr int HALF = N / 2, CHUNKS = (HALF + 15) / 16;           // N = 16: one chunk holds both halves
    const int mine = is_gate ? 0 : HALF, theirs = is_gate ? HALF : 0;
    if (ok) {
#pragma unroll
      for (int c = sub; c < CHUNKS; c += 2) {
        const int col = N == 16 ? 0 : theirs + c * 16;
        if (col >= a.M) break;                                       // the same for the whole warp
        uint32_t v[16];
        tmem_ld_x16(t_row + col, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (col + i >= theirs && col + i < theirs + HALF) trade[(col + i) * FT] = __uint_as_float(v[i]) + bias;
      }
    }
    epilogue_sync();
    if (ok) {
#pragma unroll
      for (int c = sub; c < CHUNKS; c += 2) {
        const int col = N == 16 ? 0 : mine + c * 16;
        if (col >= a.M) break;
        uint32_t v[16];
        tmem_ld_x16(t_row + col, v);
        float other[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) other[i] = col + i >= mine && col + i < mine + HALF ? trade[(col + i) * FT] : 0.f;
        tmem_ld_wait();
        __nv_bfloat16* h = a.h + static_cast<size_t>(col) * a.F + f;
#pragma unroll
        for (int i = 0; i < 16; ++i, h += a.F) {
          const int m = col + i;
          const float own = __uint_as_float(v[i]) + bias;
          const float gate = is_gate ? own : other[i], up = is_gate ? other[i] : own;
          float act, der;
          act_and_derivative<ACT, true>(gate, act, der);
          if (m >= mine && m < mine + HALF && m < a.M && f < a.F) {
            *h = __float2bfloat16_rn(act * up);
            if (a.a_hi) {
              const size_t at = static_cast<size_t>(m) * a.F + f;
              const unsigned fa = __float_as_uint(up * der), fb = __float_as_uint(act);
              a.a_hi[at] = static_cast<unsigned short>(fa >> 16);
              a.b_hi[at] = static_cast<unsigned short>(fb >> 16);
              a.a_lo[m * a.ld_lo + f] = static_cast<unsigned char>(fa >> 8);
              a.b_lo[m * a.ld_lo + f] = static_cast<unsigned char>(fb >> 8);
            }
          }
        }
      }
    }
  }

  // Common exit.  After an abandoned wait, give copies that may still be in flight time to land.
  __syncwarp();
  if (*abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::COLS);
  }
}

template <int N, bool ALONE, int ACT>
static int launch(const void* x, const void* wg, const void* wu, const Args& a, cudaStream_t st) {
  using L = Layout<N, ALONE>;
  static PerDeviceOnce once;
  bool* configured = once.slot();
  if (configured == nullptr) return -8;
  if (!*configured) {
    const cudaError_t e = cudaFuncSetAttribute(gated_few_kernel<N, ALONE, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::BYTES);
    if (e != cudaSuccess) return static_cast<int>(e);
    *configured = true;
  }
  CUtensorMap mg, mu, mx;
  int rc = make_tensor_map_bf16(&mg, wg, a.K, a.F, a.K, FT);
  if (!rc) rc = make_tensor_map_bf16(&mu, wu, a.K, a.F, a.K, FT);
  if (!rc) rc = make_tensor_map_bf16(&mx, x, a.K, a.M, a.K, N);
  if (rc) return rc;
  return launch_early(gated_few_kernel<N, ALONE, ACT>, dim3((a.F + FT - 1) / FT), dim3(THREADS), L::BYTES, st, mg, mu, mx, a);
}

template <bool ALONE, int ACT>
static int launch_few(const void* x, const void* wg, const void* wu, const Args& a, cudaStream_t st) {
  if (a.M <= 16) return launch<16, ALONE, ACT>(x, wg, wu, a, st);
  if (a.M <= 32) return launch<32, ALONE, ACT>(x, wg, wu, a, st);
  if (a.M <= 64) return launch<64, ALONE, ACT>(x, wg, wu, a, st);
  return launch<128, ALONE, ACT>(x, wg, wu, a, st);
}
template <int ACT>
static int launch_act(const void* x, const void* wg, const void* wu, const Args& a, int sms, cudaStream_t st) {
  return (a.F + FT - 1) / FT <= sms ? launch_few<true, ACT>(x, wg, wu, a, st) : launch_few<false, ACT>(x, wg, wu, a, st);
}

int forward(const void* x, const void* wg, const void* wu, const float* bg, const float* bu, void* h, unsigned short* hi, unsigned char* lo, int M, int K, int F,
            int act, int sms, int* status, cudaStream_t st) {
  const long long ld_lo = (F + 15) / 16 * 16;
  const Args a{bg, bu, static_cast<__nv_bfloat16*>(h), hi, hi ? hi + static_cast<size_t>(M) * F : nullptr, lo, lo ? lo + M * ld_lo : nullptr, ld_lo, M, K, F, status};
  switch (act) {
    case ACT_SILU: return launch_act<ACT_SILU>(x, wg, wu, a, sms, st);
    case ACT_GELU: return launch_act<ACT_GELU>(x, wg, wu, a, sms, st);
    case ACT_GELU_TANH: return launch_act<ACT_GELU_TANH>(x, wg, wu, a, sms, st);
  }
  return -2;
}

}  // namespace gf
}  // namespace sb
