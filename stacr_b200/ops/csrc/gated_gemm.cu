// The matrix products of a gated feed-forward block on CTA pairs (tcgen05.mma.cta_group::2, 256 x 256 accumulators):
//
//   forward       G = x Wg^T + bg,  U = x Wu^T + bu,  h = act(G) U       one kernel, G and U exist in tensor memory only
//   recomputing   the same G and U again, and from them and dh:  dG = dh U act'(G),  dU = dh act(G)
//   input grad    dx = dG Wg + dU Wu                                     one accumulator over both products, see share()
//   weight grads  dWg = dG^T x,  dWu = dU^T x                            one launch over the tiles of both
//
// Forward and recomputation work on tiles of 256 tokens x 128 features.  Each CTA stages its own 128 tokens of x; the even CTA
// stages 128 rows of Wg, the odd one 128 rows of Wu, and the pair's MMA sees them as one 256-row operand: accumulator columns
// 0..127 are G, 128..255 are U of the same features, so the epilogue finds both in its own tensor memory lanes.  This costs the
// main loop nothing: per k-block and CTA the same 32 KB as a plain 256 x 256 GEMM tile.
//
// What backward needs of G and U are two factors, dG = dh A and dU = dh B with A = U act'(G), B = act(G).  When they are kept, the
// forward epilogue writes each as the upper 24 bits of its fp32 value (cut, off by at most 2^-15; rounding them took as many
// instructions as forming them), 16 in one matrix and 8 in another: kept in bf16 they
// would add as much error to the weight gradients as the bf16 rounding of dG itself does (relative error 3.0e-3 against 2.3e-3),
// and the three bytes are the two factors' share of what separate layers keep (gate, act(gate), up in bf16: six bytes a feature).
//
// Pipeline, barriers and bounded waits are those of gemm_tc2.cu: a producer warp per CTA (TMA), one MMA thread in the even CTA,
// eight epilogue warps per CTA, five 32 KB stages, two accumulators so that a tile's epilogue runs under the next tile's main loop.
#include "cta_pair.cuh"
#include "gated.cuh"

namespace sb {

int make_tensor_map_bf16(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t outer, uint64_t ld, uint32_t box_outer);

namespace gt {
int forward(const void* x, const void* wg, const void* wu, const float* bg, const float* bu, void* h, unsigned short* hi, unsigned char* lo, int M, int K, int F,
            int act, cudaStream_t st);
}
namespace gf {
int forward(const void* x, const void* wg, const void* wu, const float* bg, const float* bu, void* h, unsigned short* hi, unsigned char* lo, int M, int K, int F,
            int act, int sms, int* status, cudaStream_t st);
}

namespace gg {

using namespace g2;

constexpr int TM = 256, TN = 256, TF = 128;  // accumulator of a CTA pair; features of a forward tile
constexpr int HM = 128, BK = 64, UMMA_K = 16;
constexpr int EPI_WARPS = 8;                 // two per quarter of the tensor memory lanes, each with one half of the columns
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int A_BYTES = HM * BK * 2, STAGE_BYTES = 2 * A_BYTES;
constexpr int STAGES = 5;
constexpr int WARP_EPI = 8192;               // staging of one epilogue warp
constexpr int EPI_BYTES = EPI_WARPS * WARP_EPI;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_BYTES + 1024 + 256;
constexpr int TMEM_COLS = 512;

enum : int { FORWARD = 0, RECOMPUTE = 1, INPUT_GRAD = 2, WEIGHT_GRAD = 3 };

struct Params {
  int M, N, K;              // tokens, columns of the result (features in the first two modes), length of one reduction
  int problems;             // WEIGHT_GRAD: 1 or 2 results
  int out_fp32[2];
  long long ld_hi, ld_lo;   // rows of the results in elements; rows of the 8-bit matrices
  void* out[2];             // h / dG, dU / dx / dWg, dWu
  const float* bias[2];
  const __nv_bfloat16* dh;
  unsigned short *a_hi, *b_hi;   // kept factors, null: not kept
  unsigned char *a_lo, *b_lo;
  int* status;
  int whole, splits;        // INPUT_GRAD, WEIGHT_GRAD: tiles [0, whole) are reduced by one pair each, the others in `splits` parts
  float4* partial;          // one 256 x 256 fp32 tile a part, [part][64 groups of 4 columns][256 rows]
};

// What a pair does at a time: a tile, and the k-blocks of its reduction.  A part of a split tile leaves its fp32 sums in slot `part`.
struct Unit {
  int tile, kb0, kb1, part;
};
__device__ __forceinline__ Unit unit_at(const Params& p, int u, int num_kb) {
  if (u < p.whole) return {u, 0, num_kb, -1};
  const int v = u - p.whole, tile = v / p.splits, k = v - tile * p.splits, per = (num_kb + p.splits - 1) / p.splits;
  return {p.whole + tile, k * per, (k + 1) * per < num_kb ? (k + 1) * per : num_kb, v};
}

// Tiles side by side: ROWS rows of them at a time, column by column, so that what a round reads of both operands stays in L2.  Under
// the power cap, 8192 tokens of K 2048, F 8192: forward 462 us with 4 rows, 444 with 8, 430 with 16 or 32 (4095 of K 4096, F 14336:
// 794, 752, 731; 16384 of K 4096, F 4096: 843 with 16, 916 with 32); input and weight gradients change by less than 3 %, 4 is best.
template <int MODE>
constexpr int ROWS = MODE <= RECOMPUTE ? 16 : 4;

template <int G>
__device__ __forceinline__ void decode(int tile, int num_m, int num_n, int& m_blk, int& n_blk) {
  const int group = G * num_n;
  const int g = tile / group;
  const int first_m = g * G;
  const int gm = (num_m - first_m) < G ? (num_m - first_m) : G;
  const int r = tile - g * group;
  m_blk = first_m + r % gm;
  n_blk = r / gm;
}

// Staging of 32 rows x 32 two-byte columns: 64-byte rows of four 16-byte units, the unit index twisted so that eight rows of one
// unit, and the four units of eight rows, fall into different banks.
__device__ __forceinline__ uint4* stage2(uint8_t* base, int row, int unit) {
  return reinterpret_cast<uint4*>(base) + row * 4 + (unit ^ ((row >> 1) & 3));
}
// The same for one-byte columns: 32-byte rows of two units.
__device__ __forceinline__ uint4* stage1(uint8_t* base, int row, int unit) {
  return reinterpret_cast<uint4*>(base) + row * 2 + (unit ^ ((row >> 2) & 1));
}

__device__ __forceinline__ void put16(uint8_t* base, int row, int unit, const float (&f)[16]) {
  *stage2(base, row, unit) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  *stage2(base, row, unit + 1) = make_uint4(pack_bf16x2(f[8], f[9]), pack_bf16x2(f[10], f[11]), pack_bf16x2(f[12], f[13]), pack_bf16x2(f[14], f[15]));
}
// 16 values as their upper 16 and next 8 bits; the last 8 are cut off (a NaN that arithmetic made keeps bits above them)
__device__ __forceinline__ void put24(uint8_t* hi, uint8_t* lo, int row, int unit, const float (&f)[16]) {
  uint32_t h[8], l[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = __byte_perm(__float_as_uint(f[2 * i]), __float_as_uint(f[2 * i + 1]), 0x7632);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t p = __byte_perm(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), 0x0051);
    const uint32_t q = __byte_perm(__float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]), 0x0051);
    l[i] = __byte_perm(p, q, 0x5410);
  }
  *stage2(hi, row, unit) = make_uint4(h[0], h[1], h[2], h[3]);
  *stage2(hi, row, unit + 1) = make_uint4(h[4], h[5], h[6], h[7]);
  *stage1(lo, row, unit >> 1) = make_uint4(l[0], l[1], l[2], l[3]);
}

// Copy a staged 32 x 32 block to rows row0.. and columns col0.. of a matrix (a unit of 8 columns is inside or outside as a whole).
__device__ __forceinline__ void flush2(uint8_t* base, int lane, void* out, long long ld, int row0, int rows, int col0, int cols) {
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int idx = it * 32 + lane, r = idx >> 2, u = idx & 3;
    if (row0 + r < rows && col0 + u * 8 < cols)
      *reinterpret_cast<uint4*>(static_cast<unsigned short*>(out) + static_cast<size_t>(row0 + r) * ld + col0 + u * 8) = *stage2(base, r, u);
  }
}
// One-byte rows are padded to 16 columns, so a unit that starts inside may be stored whole.
__device__ __forceinline__ void flush1(uint8_t* base, int lane, unsigned char* out, long long ld, int row0, int rows, int col0, int cols) {
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    const int idx = it * 32 + lane, r = idx >> 1, u = idx & 1;
    if (row0 + r < rows && col0 + u * 16 < cols)
      *reinterpret_cast<uint4*>(out + static_cast<size_t>(row0 + r) * ld + col0 + u * 16) = *stage1(base, r, u);
  }
}

__device__ __forceinline__ void add_bias(float (&f)[16], const float* bias, int col0, int cols) {
  if (bias == nullptr) return;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (col0 + i < cols) f[i] += __ldg(bias + col0 + i);
}

// One 16-feature chunk of a token row: gate and up projections in, results staged at unit `unit`.
template <int MODE, int ACT>
__device__ __forceinline__ void gated_chunk(const Params& p, const uint32_t (&vg)[16], const uint32_t (&vu)[16], const uint4 (&dh)[2], int col0, int lane,
                                            uint8_t* st, int unit) {
  float g[16], u[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    g[i] = __uint_as_float(vg[i]);
    u[i] = __uint_as_float(vu[i]);
  }
  add_bias(g, p.bias[0], col0, p.N);
  add_bias(u, p.bias[1], col0, p.N);
  float a[16], b[16];        // the two factors
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float der;
    act_and_derivative<ACT, true>(g[i], b[i], der);
    a[i] = u[i] * der;
  }
  float o[16];
  if (MODE == FORWARD) {
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = b[i] * u[i];
    put16(st, lane, unit, o);
    if (p.a_hi != nullptr) {
      put24(st + 2048, st + 6144, lane, unit, a);
      put24(st + 4096, st + 7168, lane, unit, b);
    }
  } else {
    const uint32_t d[8] = {dh[0].x, dh[0].y, dh[0].z, dh[0].w, dh[1].x, dh[1].y, dh[1].z, dh[1].w};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float dv = __uint_as_float(i & 1 ? d[i >> 1] & 0xffff0000u : d[i >> 1] << 16);
      o[i] = dv * a[i];
      b[i] *= dv;
    }
    put16(st, lane, unit, o);
    put16(st + 2048, lane, unit, b);
  }
}

template <int MODE, int ACT>
__global__ void __launch_bounds__(THREADS, 1)
gated_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a0, const __grid_constant__ CUtensorMap tmap_a1, const __grid_constant__ CUtensorMap tmap_b0,
                  const __grid_constant__ CUtensorMap tmap_b1, const __grid_constant__ Params p) {
  constexpr bool PROJECT = MODE == FORWARD || MODE == RECOMPUTE;
  constexpr bool A_MN = MODE == WEIGHT_GRAD, B_MN = MODE == INPUT_GRAD || MODE == WEIGHT_GRAD;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi_stage = smem + STAGES * STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi_stage + EPI_BYTES);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + STAGES;
  uint64_t* tmem_full = bars + 2 * STAGES;
  uint64_t* tmem_empty = bars + 2 * STAGES + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const bool leader = crank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  constexpr int STEP_N = PROJECT ? TF : TN;
  const int num_m = (p.M + TM - 1) / TM, num_n = (p.N + STEP_N - 1) / STEP_N;
  const int kb_one = (p.K + BK - 1) / BK;                            // k-blocks of one product
  const int num_kb = MODE == INPUT_GRAD ? 2 * kb_one : kb_one;       // both products fall into one accumulator
  const int tiles_one = num_m * num_n;
  const int total_tiles = MODE == WEIGHT_GRAD ? tiles_one * p.problems : tiles_one;
  const int total_units = p.whole + (total_tiles - p.whole) * p.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 2 * EPI_WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  after_predecessors();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (one per CTA)
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int u = pair; u < total_units && ok; u += npairs) {
        const Unit unit = unit_at(p, u, num_kb);
        const int tile = unit.tile, problem = MODE == WEIGHT_GRAD && tile >= tiles_one ? 1 : 0;
        int m_blk, n_blk;
        decode<ROWS<MODE>>(tile - problem * tiles_one, num_m, num_n, m_blk, n_blk);
        const int m0 = m_blk * TM + static_cast<int>(crank) * HM;
        const int n0 = PROJECT ? n_blk * TF : n_blk * TN + static_cast<int>(crank) * HM;
        for (int kb = unit.kb0; kb < unit.kb1; ++kb) {
          if (!mbar_wait(&empty_bar[s], ph ^ 1u, abort_flag, p.status, ST_TIMEOUT_SMEM_EMPTY)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + s * STAGE_BYTES;
          uint8_t* sb_ = sa + A_BYTES;
          const bool second = MODE == INPUT_GRAD ? kb >= kb_one : problem == 1;
          const CUtensorMap* ta = second ? &tmap_a1 : &tmap_a0;
          const CUtensorMap* tb = PROJECT ? (leader ? &tmap_b0 : &tmap_b1) : (MODE == INPUT_GRAD && second) ? &tmap_b1 : &tmap_b0;
          const int k0 = (MODE == INPUT_GRAD && second ? kb - kb_one : kb) * BK;
          if (leader) mbar_expect_tx(&full_bar[s], 2 * STAGE_BYTES);
          if (A_MN) {
#pragma unroll
            for (int h = 0; h < HM / 64; ++h) tma_load_2d_pair(sa + h * 8192, ta, &full_bar[s], m0 + h * 64, k0);
          } else {
            tma_load_2d_pair(sa, ta, &full_bar[s], k0, m0);
          }
          if (B_MN) {
#pragma unroll
            for (int h = 0; h < HM / 64; ++h) tma_load_2d_pair(sb_ + h * 8192, tb, &full_bar[s], n0 + h * 64, k0);
          } else {
            tma_load_2d_pair(sb_, tb, &full_bar[s], k0, n0);
          }
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA only)
    if (leader && lane == 0) {
      constexpr uint32_t idesc = make_idesc_bf16(TM, TN, A_MN, B_MN);
      int s = 0;
      uint32_t ph = 0;
      int local = 0;
      bool ok = true;
      for (int u = pair; u < total_units && ok; u += npairs, ++local) {
        const Unit unit = unit_at(p, u, num_kb);
        const int acc = local & 1;
        const uint32_t acc_ph = (local >> 1) & 1;
        if (!mbar_wait(&tmem_empty[acc], acc_ph ^ 1u, abort_flag, p.status, ST_TIMEOUT_TMEM_EMPTY)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * TN;
        for (int kb = unit.kb0; kb < unit.kb1; ++kb) {
          if (!mbar_wait(&full_bar[s], ph, abort_flag, p.status, ST_TIMEOUT_SMEM_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * STAGE_BYTES);
          const uint32_t sb_ = sa + A_BYTES;
#pragma unroll
          for (int j = 0; j < BK / UMMA_K; ++j) {
            const uint64_t adesc = A_MN ? make_smem_desc_sw128(sa + j * 2048, 8192, 1024) : make_smem_desc_sw128(sa + j * 32, 16, 1024);
            const uint64_t bdesc = B_MN ? make_smem_desc_sw128(sb_ + j * 2048, 8192, 1024) : make_smem_desc_sw128(sb_ + j * 32, 16, 1024);
            umma_bf16_pair(d_tmem, adesc, bdesc, idesc, (kb > unit.kb0 || j > 0) ? 1u : 0u);
          }
          umma_commit_pair(&empty_bar[s]);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok) umma_commit_pair(&tmem_full[acc]);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue warps of both CTAs
    const int quad = warp & 3, half = (warp - 2) >> 2;
    uint8_t* st = epi_stage + (warp - 2) * WARP_EPI;
    int local = 0;
    bool ok = true;
    for (int u = pair; u < total_units && ok; u += npairs, ++local) {
      const Unit unit = unit_at(p, u, num_kb);
      const int tile = unit.tile, problem = MODE == WEIGHT_GRAD && tile >= tiles_one ? 1 : 0;
      int m_blk, n_blk;
      decode<ROWS<MODE>>(tile - problem * tiles_one, num_m, num_n, m_blk, n_blk);
      const int acc = local & 1;
      const uint32_t acc_ph = (local >> 1) & 1;
      const int row_base = m_blk * TM + static_cast<int>(crank) * HM + quad * 32;
      const int row = row_base + lane;
      constexpr int CHUNKS = (PROJECT ? TF : TN) / 32;            // chunks of 16 columns in this warp's half
      const int col_first = n_blk * STEP_N + half * CHUNKS * 16;
      // the whole warp goes on or gives up together: the tensor memory loads below are warp-wide instructions
      if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], acc_ph, abort_flag, p.status, ST_TIMEOUT_TMEM_FULL))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * TN + half * CHUNKS * 16;
      if (row_base < p.M && col_first < p.N) {                     // the same for the whole warp
        if (PROJECT) {
          // 32 features at a time: two 16-column chunks of both projections, staged and stored as row segments of 64 (32) bytes.
          // The next chunk is on its way from tensor memory while one is worked on.
          uint32_t vg[2][16], vu[2][16];
          tmem_ld_x16(t_row, vg[0]);
          tmem_ld_x16(t_row + TF, vu[0]);
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            const int col0 = col_first + c * 16;
            uint4 dh[2] = {};
            if (MODE == RECOMPUTE && row < p.M) {
#pragma unroll
              for (int q = 0; q < 2; ++q)
                if (col0 + q * 8 < p.N) dh[q] = __ldg(reinterpret_cast<const uint4*>(p.dh + static_cast<size_t>(row) * p.ld_hi + col0 + q * 8));
            }
            tmem_ld_wait();
            if (c + 1 < CHUNKS) {
              tmem_ld_x16(t_row + (c + 1) * 16, vg[(c + 1) & 1]);
              tmem_ld_x16(t_row + TF + (c + 1) * 16, vu[(c + 1) & 1]);
            }
            gated_chunk<MODE, ACT>(p, vg[c & 1], vu[c & 1], dh, col0, lane, st, (c & 1) * 2);
            if (c & 1) {
              __syncwarp();
              const int g0 = col0 - 16;
              flush2(st, lane, p.out[0], p.ld_hi, row_base, p.M, g0, p.N);
              if (MODE == RECOMPUTE) {
                flush2(st + 2048, lane, p.out[1], p.ld_hi, row_base, p.M, g0, p.N);
              } else if (p.a_hi != nullptr) {
                flush2(st + 2048, lane, p.a_hi, p.ld_hi, row_base, p.M, g0, p.N);
                flush2(st + 4096, lane, p.b_hi, p.ld_hi, row_base, p.M, g0, p.N);
                flush1(st + 6144, lane, p.a_lo, p.ld_lo, row_base, p.M, g0, p.N);
                flush1(st + 7168, lane, p.b_lo, p.ld_lo, row_base, p.M, g0, p.N);
              }
              __syncwarp();
            }
          }
        } else {
          const bool fp32 = p.out_fp32[problem] != 0;
          void* out = p.out[problem];
          uint32_t v[2][16];
          tmem_ld_x16(t_row, v[0]);
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            const int col0 = col_first + c * 16;
            tmem_ld_wait();
            if (c + 1 < CHUNKS) tmem_ld_x16(t_row + (c + 1) * 16, v[(c + 1) & 1]);
            const uint32_t(&w)[16] = v[c & 1];
            if (unit.part >= 0) {       // neighbouring lanes are neighbouring rows: whole lines
              float4* part = p.partial + (static_cast<size_t>(unit.part) * 64 + (half * CHUNKS + c) * 4) * TM + static_cast<int>(crank) * HM + quad * 32 + lane;
#pragma unroll
              for (int q = 0; q < 4; ++q)
                part[q * TM] = make_float4(__uint_as_float(w[4 * q]), __uint_as_float(w[4 * q + 1]), __uint_as_float(w[4 * q + 2]), __uint_as_float(w[4 * q + 3]));
            } else if (fp32) {
              if (row < p.M) {
                float* o = static_cast<float*>(out) + static_cast<size_t>(row) * p.ld_hi + col0;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  if (col0 + q * 4 < p.N)
                    reinterpret_cast<float4*>(o)[q] = make_float4(__uint_as_float(w[4 * q]), __uint_as_float(w[4 * q + 1]), __uint_as_float(w[4 * q + 2]),
                                                                 __uint_as_float(w[4 * q + 3]));
              }
            } else {
              float f[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(w[i]);
              put16(st, lane, (c & 1) * 2, f);
              if (c & 1) {
                __syncwarp();
                flush2(st, lane, out, p.ld_hi, row_base, p.M, col0 - 16, p.N);
                __syncwarp();
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(&tmem_empty[acc]);
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
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// Sums of the parts of the split tiles, in the order of the parts.  A block has 16 columns of a tile, a thread one row of them.
template <int MODE>
__global__ void __launch_bounds__(TM) gated_join_kernel(const __grid_constant__ Params p) {
  after_predecessors();
  const int num_m = (p.M + TM - 1) / TM, num_n = (p.N + TN - 1) / TN, tiles_one = num_m * num_n;
  const int split_tile = blockIdx.x >> 4, c = blockIdx.x & 15;
  const int tile = p.whole + split_tile, problem = MODE == WEIGHT_GRAD && tile >= tiles_one ? 1 : 0;
  int m_blk, n_blk;
  decode<ROWS<MODE>>(tile - problem * tiles_one, num_m, num_n, m_blk, n_blk);
  const int row = m_blk * TM + threadIdx.x, col0 = n_blk * TN + c * 16;
  if (row >= p.M || col0 >= p.N) return;
  float f[16] = {};
  const float4* part = p.partial + (static_cast<size_t>(split_tile) * p.splits * 64 + c * 4) * TM + threadIdx.x;
  for (int k = 0; k < p.splits; ++k, part += 64 * TM)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 v = part[q * TM];
      f[4 * q] += v.x, f[4 * q + 1] += v.y, f[4 * q + 2] += v.z, f[4 * q + 3] += v.w;
    }
  const size_t at = static_cast<size_t>(row) * p.ld_hi + col0;
  if (p.out_fp32[problem]) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (col0 + q * 4 < p.N) reinterpret_cast<float4*>(static_cast<float*>(p.out[problem]) + at)[q] = make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (col0 + q * 8 < p.N)
        reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out[problem]) + at)[q] =
            make_uint4(pack_bf16x2(f[8 * q], f[8 * q + 1]), pack_bf16x2(f[8 * q + 2], f[8 * q + 3]), pack_bf16x2(f[8 * q + 4], f[8 * q + 5]),
                       pack_bf16x2(f[8 * q + 6], f[8 * q + 7]));
  }
}

// How the reductions of `tiles` tiles of num_kb k-blocks are shared among the pairs.  Tiles are dealt out in rounds; the last
// round, or the only one, rarely has a tile for every pair, and the idle ones take parts of its reductions instead.  Joining the
// parts costs a second kernel of about 4 us, 14 k-blocks' time (0.28 us each), so a split has to shorten the round by more: 24.
// 512 tokens of K 2048, F 8192: dx has 16 tiles for 74 pairs, 103 us whole, 51 in four parts; 8192 tokens: 3.5 rounds of tiles
// instead of four.
struct Shares {
  int whole, splits;
};
static Shares share(long long tiles, int num_kb, int sms) {
  const int pairs = sms / 2 < 1 ? 1 : sms / 2;
  const int last = static_cast<int>(tiles % pairs);
  if (last == 0) return {static_cast<int>(tiles), 1};
  int splits = pairs / last;
  if (splits > num_kb / 8) splits = num_kb / 8;
  if (splits < 2) return {static_cast<int>(tiles), 1};
  const int per = (num_kb + splits - 1) / splits;
  splits = (num_kb + per - 1) / per;        // no part is empty
  if (num_kb - per < 24) return {static_cast<int>(tiles), 1};
  return {static_cast<int>(tiles) - last, splits};
}
static long long tiles_of(int rows, int cols) { return static_cast<long long>((rows + TM - 1) / TM) * ((cols + TN - 1) / TN); }
static int blocks_of(int k) { return (k + BK - 1) / BK; }
static size_t partial_bytes(long long tiles, int num_kb, int sms) {
  const Shares s = share(tiles, num_kb, sms);
  return static_cast<size_t>(tiles - s.whole) * s.splits * TM * TN * 4;
}

template <int MODE, int ACT>
static int launch(const CUtensorMap& a0, const CUtensorMap& a1, const CUtensorMap& b0, const CUtensorMap& b1, const Params& p, int sms, cudaStream_t stream) {
  static PerDeviceOnce once;
  bool* configured = once.slot();
  if (configured == nullptr) return -8;
  auto kern = gated_gemm_kernel<MODE, ACT>;
  if (!*configured) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return static_cast<int>(e);
    *configured = true;
  }
  constexpr int STEP_N = MODE <= RECOMPUTE ? TF : TN;
  const long long tiles = static_cast<long long>((p.M + TM - 1) / TM) * ((p.N + STEP_N - 1) / STEP_N) * (MODE == WEIGHT_GRAD ? p.problems : 1);
  if (tiles > 0x3fffffff) return -2;
  const long long units = p.whole + (tiles - p.whole) * p.splits;
  int pairs = sms / 2;
  if (pairs > units) pairs = static_cast<int>(units);
  if (pairs < 1) pairs = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs, 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // see launch_early
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a0, a1, b0, b1, p);
  if (e != cudaSuccess) return static_cast<int>(e);
  if constexpr (MODE == INPUT_GRAD || MODE == WEIGHT_GRAD) {
    if (tiles > p.whole) {
      return launch_early(gated_join_kernel<MODE>, dim3(static_cast<unsigned>((tiles - p.whole) * 16)), dim3(TM), 0, stream, p);
    }
  }
  return 0;
}

template <int MODE>
static int launch_act(int act, const CUtensorMap& a0, const CUtensorMap& a1, const CUtensorMap& b0, const CUtensorMap& b1, const Params& p, int sms, cudaStream_t st) {
  switch (act) {
    case ACT_SILU: return launch<MODE, ACT_SILU>(a0, a1, b0, b1, p, sms, st);
    case ACT_GELU: return launch<MODE, ACT_GELU>(a0, a1, b0, b1, p, sms, st);
    case ACT_GELU_TANH: return launch<MODE, ACT_GELU_TANH>(a0, a1, b0, b1, p, sms, st);
  }
  return -2;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ------------------------------------------------------------------ dG = dh A, dU = dh B from kept factors
__device__ __forceinline__ float join24(unsigned hi, unsigned lo) { return __uint_as_float((hi << 16) | (lo << 8)); }

__global__ void __launch_bounds__(256) gated_factors_kernel(const uint4* __restrict__ dh, const uint4* __restrict__ a_hi, const unsigned char* __restrict__ a_lo,
                                                            const uint4* __restrict__ b_hi, const unsigned char* __restrict__ b_lo, uint4* __restrict__ dg,
                                                            uint4* __restrict__ du, int rows, int nv, long long ld_lo) {
  after_predecessors();
  for (int r = blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += gridDim.y * blockDim.y)
    for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < nv; c += gridDim.x * blockDim.x) {
      const size_t i = static_cast<size_t>(r) * nv + c;
      const uint4 d = __ldg(dh + i), ah = __ldg(a_hi + i), bh = __ldg(b_hi + i);
      const uint2 al = __ldg(reinterpret_cast<const uint2*>(a_lo + r * ld_lo) + c), bl = __ldg(reinterpret_cast<const uint2*>(b_lo + r * ld_lo) + c);
      const uint32_t dw[4] = {d.x, d.y, d.z, d.w}, aw[4] = {ah.x, ah.y, ah.z, ah.w}, bw[4] = {bh.x, bh.y, bh.z, bh.w};
      const uint32_t av[2] = {al.x, al.y}, bv[2] = {bl.x, bl.y};
      uint32_t og[4], ou[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned la = av[j >> 1] >> ((j & 1) * 16), lb = bv[j >> 1] >> ((j & 1) * 16);
        const float d0 = __uint_as_float(dw[j] << 16), d1 = __uint_as_float(dw[j] & 0xffff0000u);
        og[j] = pack_bf16x2(d0 * join24(aw[j] & 0xffffu, la & 0xffu), d1 * join24(aw[j] >> 16, (la >> 8) & 0xffu));
        ou[j] = pack_bf16x2(d0 * join24(bw[j] & 0xffffu, lb & 0xffu), d1 * join24(bw[j] >> 16, (lb >> 8) & 0xffu));
      }
      dg[i] = make_uint4(og[0], og[1], og[2], og[3]);
      du[i] = make_uint4(ou[0], ou[1], ou[2], ou[3]);
    }
}

}  // namespace gg
}  // namespace sb

namespace sb {
namespace gg {

// what every entry asks for: operands on 16 bytes, K and F multiples of 8 (rows of 16 bytes, as TMA and the vector stores need them)
static bool proper(int M, int K, int F) { return M > 0 && K > 0 && F > 0 && K % 8 == 0 && F % 8 == 0; }

template <int MODE>
static int project(const void* x, const void* wg, const void* wu, Params& p, int act, int sms, cudaStream_t st) {
  p.whole = static_cast<int>(static_cast<long long>((p.M + TM - 1) / TM) * ((p.N + TF - 1) / TF));
  p.splits = 1;
  CUtensorMap ta, tg, tu;
  int rc = make_tensor_map_bf16(&ta, x, p.K, p.M, p.K, HM);
  if (!rc) rc = make_tensor_map_bf16(&tg, wg, p.K, p.N, p.K, HM);
  if (!rc) rc = make_tensor_map_bf16(&tu, wu, p.K, p.N, p.K, HM);
  return rc ? rc : launch_act<MODE>(act, ta, ta, tg, tu, p, sms, st);
}

// dG, dU [M, F] from dh and the kept factors
static int factors(const void* dh, const unsigned short* hi, const unsigned char* lo, __nv_bfloat16* d, int M, int F, int sms, cudaStream_t st) {
  const int nv = F / 8;
  const size_t mf = static_cast<size_t>(M) * F;
  const long long ld_lo = (F + 15) / 16 * 16;
  int tx = 32;
  while (tx < 256 && tx < nv) tx <<= 1;
  const dim3 block(tx, 256 / tx);
  const unsigned gx = (nv + tx - 1) / tx;
  const long long cap = (sms * 32ll + gx - 1) / gx, by = (M + static_cast<int>(block.y) - 1) / static_cast<int>(block.y);
  const long long lim = cap < 65535 ? cap : 65535;
  const dim3 grid(gx, static_cast<unsigned>(by < lim ? by : lim));
  return launch_early(gated_factors_kernel, grid, block, 0, st, static_cast<const uint4*>(dh), reinterpret_cast<const uint4*>(hi), lo,
                      reinterpret_cast<const uint4*>(hi + mf), lo + M * ld_lo, reinterpret_cast<uint4*>(d), reinterpret_cast<uint4*>(d + mf), M, nv, ld_lo);
}

// dx[M, K] = dG Wg + dU Wu
static int input_grad(const __nv_bfloat16* dg, const __nv_bfloat16* du, const void* wg, const void* wu, void* dx, int M, int K, int F, int sms, int* status,
                      float4* partial, cudaStream_t st) {
  CUtensorMap a0, a1, b0, b1;
  int rc = make_tensor_map_bf16(&a0, dg, F, M, F, HM);
  if (!rc) rc = make_tensor_map_bf16(&a1, du, F, M, F, HM);
  if (!rc) rc = make_tensor_map_bf16(&b0, wg, K, F, K, 64);
  if (!rc) rc = make_tensor_map_bf16(&b1, wu, K, F, K, 64);
  if (rc) return rc;
  const Shares sh = share(tiles_of(M, K), 2 * blocks_of(F), sms);
  Params p{M, K, F, 1, {0, 0}, K, 0, {dx, nullptr}, {nullptr, nullptr}, nullptr, nullptr, nullptr, nullptr, nullptr, status, sh.whole, sh.splits, partial};
  return launch<INPUT_GRAD, ACT_SILU>(a0, a1, b0, b1, p, sms, st);
}

// dWg = dG^T x and dWu = dU^T x [F, K], each fp32 or bf16; a null result is left out
static int weight_grads(const __nv_bfloat16* dg, const __nv_bfloat16* du, const void* x, void* dwg, void* dwu, int fp32_g, int fp32_u, int M, int K, int F,
                        int sms, int* status, float4* partial, cudaStream_t st) {
  if (!dwg) {
    dg = du;
    dwg = dwu;
    fp32_g = fp32_u;
    dwu = nullptr;
  }
  CUtensorMap a0, a1, b;
  int rc = make_tensor_map_bf16(&a0, dg, F, M, F, 64);
  if (!rc) rc = make_tensor_map_bf16(&a1, dwu ? du : dg, F, M, F, 64);
  if (!rc) rc = make_tensor_map_bf16(&b, x, K, M, K, 64);
  if (rc) return rc;
  const Shares sh = share(tiles_of(F, K) * (dwu ? 2 : 1), blocks_of(M), sms);
  Params p{F, K, M, dwu ? 2 : 1, {fp32_g, fp32_u}, K, 0, {dwg, dwu}, {nullptr, nullptr}, nullptr, nullptr, nullptr, nullptr, nullptr, status, sh.whole, sh.splits,
           partial};
  return launch<WEIGHT_GRAD, ACT_SILU>(a0, a1, b, b, p, sms, st);
}

}  // namespace gg
}  // namespace sb

namespace sb {
namespace gg {

// Which forward kernel: for at most 128 tokens one that streams the weights, whichever of the two the following lines, fitted to
// measurements at weights of 0.7 to 272 MB, expect to be done first; above, the 256-token tiles of this file.
//   gated_tokens.cu (to 64 tokens): 2 us and the weights at 6, 4.9, 3.2 and 1.7 TB/s for 8, 16, 32 and 64 tokens.  Measured at
//     67 MB (K 2048, F 8192): 12.5, 15.3, 20.6, 40.8 us, at 4 MB (K 512, F 2048): 2.3, 2.7, 3.3, 4.7.
//   gated_few.cu: 4.4 us and 0.27 for each k-block, or 3.5 and the weights at 5.9 TB/s, and more for more columns to finish.
//     Measured at the same: 15.2 us to 32 tokens, 15.5, and 17.0 for 128; 5.9 to 32 tokens, 6.7, 8.5.
//   tiles, 128 tokens: 19.8 and 9.3.
static bool streams_fragments(int M, int K, int F) {
  if (M > 64) return false;
  const double mb = 4e-6 * K * F, chain = 4.4 + 0.27 * (K / 64.0), stream = 3.5 + mb / 5.9;
  const double tokens = 2.0 + mb / (M <= 8 ? 6.0 : M <= 16 ? 4.9 : M <= 32 ? 3.2 : 1.7);
  return tokens <= (chain > stream ? chain : stream) + (M > 32 ? 0.8 : 0.0);
}

}  // namespace gg
}  // namespace sb

// h[M, F] = act(x Wg^T + bg) * (x Wu^T + bu) in bf16; x [M, K], weights [F, K] contiguous; K and F multiples of 8.
// hi [2, M, F] 16-bit and lo [2, M, ceil16(F)] 8-bit receive the backward's factors; both null: not kept.
extern "C" int sb_gated_forward(const void* x, const void* wg, const void* wu, const float* bg, const float* bu, void* h, void* hi, void* lo, int M, int K, int F,
                                int act, int sms, int* status, void* stream) {
  using namespace sb;
  if (!gg::proper(M, K, F)) return -2;
  if (!gg::aligned16(x) || !gg::aligned16(wg) || !gg::aligned16(wu) || !gg::aligned16(h) || !gg::aligned16(hi) || !gg::aligned16(lo)) return -3;
  const long long ld_lo = (F + 15) / 16 * 16;
  unsigned short* ah = static_cast<unsigned short*>(hi);
  unsigned char* al = static_cast<unsigned char*>(lo);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (gg::streams_fragments(M, K, F)) return gt::forward(x, wg, wu, bg, bu, h, ah, al, M, K, F, act, st);
  if (M <= 128) return gf::forward(x, wg, wu, bg, bu, h, ah, al, M, K, F, act, sms, status, st);
  gg::Params p{M, F, K, 1, {0, 0}, F, ld_lo, {h, nullptr}, {bg, bu}, nullptr, ah, ah ? ah + static_cast<size_t>(M) * F : nullptr, al, al ? al + M * ld_lo : nullptr,
               status};
  return gg::project<gg::FORWARD>(x, wg, wu, p, act, sms, st);
}

// Bytes that `partial` of sb_gated_backward has to hold; 0: it may be null.
extern "C" long long sb_gated_partial_bytes(int M, int K, int F, int need_dx, int weights, int sms) {
  using namespace sb::gg;
  if (!proper(M, K, F)) return 0;
  size_t most = need_dx ? partial_bytes(tiles_of(M, K), 2 * blocks_of(F), sms) : 0;
  if (weights > 0) {
    const size_t w = partial_bytes(tiles_of(F, K) * weights, blocks_of(M), sms);
    if (w > most) most = w;
  }
  return static_cast<long long>(most);
}

// d [2, M, F] = dG and dU, from the kept factors or (hi null) from the projections formed again; dx [M, K] unless null; the weight
// gradients [F, K], each fp32 or bf16, unless null.
extern "C" int sb_gated_backward(const void* dh, const void* x, const void* wg, const void* wu, const float* bg, const float* bu, const void* hi, const void* lo,
                                 void* d, void* dx, void* dwg, void* dwu, void* partial, long long partial_size, int fp32_g, int fp32_u, int M, int K, int F,
                                 int act, int sms, int* status, void* stream) {
  using namespace sb;
  if (!gg::proper(M, K, F) || partial_size < sb_gated_partial_bytes(M, K, F, dx != nullptr, (dwg != nullptr) + (dwu != nullptr), sms)) return -2;
  if (!gg::aligned16(dh) || !gg::aligned16(x) || !gg::aligned16(wg) || !gg::aligned16(wu) || !gg::aligned16(hi) || !gg::aligned16(lo) || !gg::aligned16(d) ||
      !gg::aligned16(dx) || !gg::aligned16(dwg) || !gg::aligned16(dwu) || !gg::aligned16(partial))
    return -3;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  __nv_bfloat16* dg = static_cast<__nv_bfloat16*>(d);
  __nv_bfloat16* du = dg + static_cast<size_t>(M) * F;
  int rc;
  if (hi) {
    rc = gg::factors(dh, static_cast<const unsigned short*>(hi), static_cast<const unsigned char*>(lo), dg, M, F, sms, st);
  } else {
    gg::Params p{M, F, K, 1, {0, 0}, F, 0, {dg, du}, {bg, bu}, static_cast<const __nv_bfloat16*>(dh), nullptr, nullptr, nullptr, nullptr, status};
    rc = gg::project<gg::RECOMPUTE>(x, wg, wu, p, act, sms, st);
  }
  if (!rc && dx) rc = gg::input_grad(dg, du, wg, wu, dx, M, K, F, sms, status, static_cast<float4*>(partial), st);
  if (!rc && (dwg || dwu)) rc = gg::weight_grads(dg, du, x, dwg, dwu, fp32_g, fp32_u, M, K, F, sms, status, static_cast<float4*>(partial), st);
  return rc;
}
