// Rotary positions for query and key heads of any layout, one launch for both.
//
// A head's first `rot` values are rot/2 pairs, (i, i + rot/2) in the half layout or (2i, 2i+1) interleaved; pair i of a token
// at position p is turned by the angle p f_i and multiplied by `scale`:
//   y1 = s (x1 cos - x2 sin),  y2 = s (x2 cos + x1 sin);   the rest of the head is copied.
// The gradient is the same map with the opposite angle (the transpose of a rotation), so one kernel serves both directions.
//
// Angles are formed here from the positions: p f_i / 2 pi in 64 bits, reduced to a fraction of a turn, then sine and cosine of
// that fraction in fp32.  A table would be as large as a sequence is long and, built in fp32, wrong by 2^-24 p radians; here
// an angle is good to 1e-7 at any position.
//
// Bound by memory: each value is read once and written once.  A block takes a few consecutive tokens and as many heads as it has
// threads for: it forms the tokens' sines once in shared memory, and then a thread walks with one vector of one head over the
// tokens, so that addresses advance by constants.  What is left to save is instructions: at a copy's rate an SM has 75 issue slots
// for each warp's 16 bytes in and out.  Threads whose vectors are turned come before those whose vectors are copied, so that
// few warps do both.  4 x 2048 tokens of 40 heads of 128 in bf16: 30.7 us (5.5 TB/s, 0.83 of a copy's rate; interleaved 35.4); 64
// heads of 64 in fp32, 16384 tokens: 81 us (6.6 TB/s); a quarter of 64 heads of 80, 30011 tokens: 117 us interleaved, 140 in halves
// (5.3, 4.4 TB/s).  Sines in the registers of threads that walk over the heads took 37.6, 99, 149 and 169; 320 threads and 48
// registers measured better than 256 to 640 threads and 40 to 80 registers, 4 tokens better than 2 and 8.
//
// Vectors are as wide as extents, strides and addresses allow.  Where the rotary part does not divide into whole vectors but the
// head does (a quarter of an 80-value head: 20), a thread owns one vector of the head whatever lies in it (MIXED): pairs of the
// interleaved layout never cross a vector; in the half layout the partners are loaded one by one, from L1, where a neighbour's
// vector brings them.
#include "gated.cuh"

namespace sb {
namespace rot {

struct RotaryArgs {
  const void *q, *k;
  void *oq, *ok;                          // contiguous [B, S, heads, D]
  long long qb, qs, qh, kb, ks, kh;       // strides of the inputs in elements; the last dimension is contiguous
  const double* inv_freq;                 // [rot / 2]
  const void* positions;                  // int32 or int64, or null: position = first + s
  long long pb, ps, first;
  long long B;
  int S, hq, hk, D, rot, pos64, step;     // step: positions from one token to the next where there is no tensor
  float scale, sign;
};

constexpr int ROT_THREADS = 320;   // threads of a block at most
constexpr int ROT_TOKENS = 4;      // tokens of a block

template <typename T, int VEC, bool INTER, bool MIXED>
__global__ void __launch_bounds__(VEC == 1 ? 512 : ROT_THREADS, VEC == 1 ? 2 : 4) rotary_kernel(const RotaryArgs a, int heads_side, int tokens_most) {
  using P = Pack<T, VEC>;
  constexpr bool SINGLE = INTER && VEC > 1;                              // both values of a pair lie in one vector
  constexpr int PAIRS = MIXED ? VEC : SINGLE ? VEC / 2 : INTER ? 1 : VEC;   // sines of a turning slot; MIXED: one for each value
  constexpr int SPAN = INTER && VEC == 1 ? 2 : VEC;                      // values from one turning slot to the next
  extern __shared__ float2 turn[];                                       // [tokens of the block][turning * PAIRS]: scale * (cos, sin)
  const int half = a.rot / 2;
  const int turning = MIXED ? (a.rot + VEC - 1) / VEC : INTER ? a.rot / SPAN : half / VEC;
  const int copied = MIXED ? a.D / VEC - turning : (a.D - a.rot) / VEC;
  const int row = turning * PAIRS;
  // threads [0, turning * heads_side) turn, the others copy
  const bool turns = threadIdx.x < turning * heads_side;
  const int i = turns ? threadIdx.x : threadIdx.x - turning * heads_side, per = turns ? turning : copied;
  const int hl = i / per, slot = i - hl * per;
  const int h = blockIdx.z * heads_side + hl;
  const int d = turns ? slot * SPAN : MIXED ? (turning + slot) * VEC : a.rot + slot * VEC;
  const int other = INTER ? 1 : half;                                    // where the partners of a turning slot lie
  const int s0 = blockIdx.x * tokens_most;
  const int tokens = a.S - s0 < tokens_most ? a.S - s0 : tokens_most;
  const bool isq = h < a.hq, works = h < a.hq + a.hk;
  const long long sstep = isq ? a.qs : a.ks, dstep = static_cast<long long>(isq ? a.hq : a.hk) * a.D;

  after_predecessors();
  for (long long b = blockIdx.y; b < a.B; b += gridDim.y) {
    const T* src = nullptr;
    T* dst = nullptr;
    P xa, xb;
    if (works) {
      src = (isq ? static_cast<const T*>(a.q) + b * a.qb + h * a.qh : static_cast<const T*>(a.k) + b * a.kb + (h - a.hq) * a.kh) + s0 * sstep + d;
      dst = (isq ? static_cast<T*>(a.oq) : static_cast<T*>(a.ok)) + (b * a.S + s0) * dstep + static_cast<long long>(isq ? h : h - a.hq) * a.D + d;
      xa = load_once<P>(src);
      if (!MIXED && !SINGLE && turns) xb = load_once<P>(src + other);
    }

    for (int n = threadIdx.x; n < tokens * half; n += blockDim.x) {
      const int t = n / half, pair = n - t * half, s = s0 + t;
      long long pos = a.first + static_cast<long long>(s) * a.step;
      if (a.positions) {
        const long long at = b * a.pb + s * a.ps;
        pos = a.pos64 ? static_cast<const long long*>(a.positions)[at] : static_cast<const int*>(a.positions)[at];
      }
      const double turns64 = static_cast<double>(pos) * (__ldg(a.inv_freq + pair) * 0.15915494309189535);
      float c, sn;
      sincospif(2.f * static_cast<float>(turns64 - rint(turns64)), &sn, &c);
      c *= a.scale;
      sn *= a.scale * a.sign;
      // neighbouring slots read 16 bytes (two entries) each: laid side by side these fall into different banks
      auto put = [&](int e, float sine) {
        const int own = e / PAIRS, j = e % PAIRS;
        turn[t * row + (PAIRS == 1 ? e : ((j >> 1) * turning + own) * 2 + (j & 1))] = make_float2(c, sine);
      };
      if (MIXED) {                                                       // y = x cos + partner * (-sin for the first, sin for the second)
        put(INTER ? 2 * pair : pair, -sn);
        put(INTER ? 2 * pair + 1 : pair + half, sn);
      } else {
        put(pair, sn);
      }
    }
    __syncthreads();

    if (works && !turns) {
#pragma unroll 4
      for (int t = 0; t < tokens; ++t) *reinterpret_cast<P*>(dst + t * dstep) = t ? load_once<P>(src + t * sstep) : xa;
    } else if (works) {
#pragma unroll 2
      for (int t = 0; t < tokens; ++t) {
        if (t) {
          src += sstep;
          dst += dstep;
          xa = load_once<P>(src);
          if (!MIXED && !SINGLE) xb = load_once<P>(src + other);
        }
        const float2* tab = turn + t * row;
        float2 cs[PAIRS];
        if constexpr (PAIRS > 1) {
#pragma unroll
          for (int j = 0; j < PAIRS; j += 2) {
            const float4 two = *reinterpret_cast<const float4*>(tab + ((j >> 1) * turning + slot) * 2);
            cs[j] = make_float2(two.x, two.y);
            cs[j + 1] = make_float2(two.z, two.w);
          }
        } else {
          cs[0] = tab[slot];
        }
        float x[VEC], y[VEC];
        unpack(xa, x);
        if (MIXED) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float o = x[j ^ 1];
            if (!INTER) o = d + j < a.rot ? to_f32(load_once<Pack<T, 1>>(src + (d + j < half ? j + half : j - half)).v[0]) : 0.f;
            y[j] = x[j] * cs[j].x + o * cs[j].y;
          }
          P out = pack<T, VEC>(y);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (d + j >= a.rot) out.v[j] = xa.v[j];
          *reinterpret_cast<P*>(dst) = out;
        } else if (SINGLE) {
#pragma unroll
          for (int j = 0; j < PAIRS; ++j) {
            y[(2 * j) % VEC] = x[(2 * j) % VEC] * cs[j].x - x[(2 * j + 1) % VEC] * cs[j].y;
            y[(2 * j + 1) % VEC] = x[(2 * j + 1) % VEC] * cs[j].x + x[(2 * j) % VEC] * cs[j].y;
          }
          *reinterpret_cast<P*>(dst) = pack<T, VEC>(y);
        } else {
          float x2[VEC], y2[VEC];
          unpack(xb, x2);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            y[j] = x[j] * cs[j % PAIRS].x - x2[j] * cs[j % PAIRS].y;
            y2[j] = x2[j] * cs[j % PAIRS].x + x[j] * cs[j % PAIRS].y;
          }
          *reinterpret_cast<P*>(dst) = pack<T, VEC>(y);
          *reinterpret_cast<P*>(dst + other) = pack<T, VEC>(y2);
        }
      }
    }
    if (b + gridDim.y < a.B) __syncthreads();     // the table is written again
  }
}

template <typename T, int VEC, bool INTER, bool MIXED>
static int rotary_launch(const RotaryArgs& a, int sms, cudaStream_t st) {
  const int turning = MIXED ? (a.rot + VEC - 1) / VEC : INTER ? a.rot / (VEC > 1 ? VEC : 2) : (a.rot / 2) / VEC;
  const int copied = MIXED ? a.D / VEC - turning : (a.D - a.rot) / VEC, slots = turning + copied;
  const int heads = a.hq + a.hk, most = VEC == 1 ? 512 : ROT_THREADS;
  if (slots > most) return -2;
  // as many heads as the block has threads for, evened out over the blocks that takes
  const int rounds = (heads + most / slots - 1) / (most / slots), side = (heads + rounds - 1) / rounds;
  // few tokens: a block each, so that all SMs have one
  int tokens = a.B * a.S * rounds >= static_cast<long long>(sms) * 4 * ROT_TOKENS ? ROT_TOKENS : 1;
  const size_t row = static_cast<size_t>(turning) * (MIXED ? VEC : INTER && VEC > 1 ? VEC / 2 : INTER ? 1 : VEC) * sizeof(float2);
  if (tokens * row > 48 * 1024) tokens = 1;
  const long long by = a.B < 65535 ? a.B : 65535;
  const dim3 grid((a.S + tokens - 1) / tokens, static_cast<unsigned>(by), rounds);
  return launch_early(rotary_kernel<T, VEC, INTER, MIXED>, grid, dim3(slots * side), tokens * row, st, a, side, tokens);
}

// The widest power-of-two vector that divides every extent, stride and address, at most 16 bytes; `parts`: the rotary part too.
static int rotary_width(const RotaryArgs& a, int size, bool inter, bool parts) {
  unsigned long long bits = static_cast<unsigned long long>(a.D) | (16 / size);
  if (parts) bits |= static_cast<unsigned long long>(inter ? a.rot : a.rot / 2) | static_cast<unsigned long long>(a.D - a.rot);
  const long long strides[] = {a.qb, a.qs, a.qh, a.kb, a.ks, a.kh};
  for (long long v : strides) bits |= static_cast<unsigned long long>(v);
  const void* ptrs[] = {a.q, a.k, a.oq, a.ok};
  for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p) / size;
  return static_cast<int>(bits & (~bits + 1));
}

template <typename T, bool INTER>
static int rotary_typed(const RotaryArgs& a, int sms, cudaStream_t st) {
  const int whole = rotary_width(a, sizeof(T), INTER, true), any = rotary_width(a, sizeof(T), INTER, false);
  if (any > whole) {      // wider accesses to all values outweigh the single loads of the partners
    switch (any) {
      case 8: if constexpr (sizeof(T) == 2) return rotary_launch<T, 8, INTER, true>(a, sms, st);
      case 4: return rotary_launch<T, 4, INTER, true>(a, sms, st);
      default: return rotary_launch<T, 2, INTER, true>(a, sms, st);
    }
  }
  switch (whole) {
    case 8: if constexpr (sizeof(T) == 2) return rotary_launch<T, 8, INTER, false>(a, sms, st);
    case 4: return rotary_launch<T, 4, INTER, false>(a, sms, st);
    case 2: return rotary_launch<T, 2, INTER, false>(a, sms, st);
    default: return rotary_launch<T, 1, INTER, false>(a, sms, st);
  }
}

}  // namespace rot
}  // namespace sb

// q [B, S, hq, D] and k [B, S, hk, D] (null with hk = 0) with the strides given, into contiguous oq, ok; dtype 0 bf16, 1 fp16, 2 fp32.
// rot is even, 2 <= rot <= D <= 512 (a head's vectors are the threads of one block).  sign +1 forward, -1 backward.
extern "C" int sb_rotary(const void* q, const void* k, void* oq, void* ok, long long qb, long long qs, long long qh, long long kb, long long ks, long long kh,
                         const double* inv_freq, const void* positions, int pos64, long long pb, long long ps, long long first, long long B, int S, int hq,
                         int hk, int D, int rot, int interleaved, int dtype, float scale, float sign, int sms, void* stream) {
  using namespace sb;
  using namespace sb::rot;
  if (B <= 0 || S <= 0 || hq + hk <= 0) return 0;
  if (rot < 2 || rot % 2 || rot > D || D > 512 || hq < 0 || hk < 0) return -2;
  RotaryArgs a{q, k, oq, ok, qb, qs, qh, kb, ks, kh, inv_freq, positions, pb, ps, first, B, S, hq, hk, D, rot, pos64, 1, scale, sign};
  if (S == 1 && B <= 0x7fffffffLL) {     // one token a sequence: the batch takes the sequence's place, all at the first position
    a.qs = qb, a.ks = kb, a.ps = pb;
    a.S = static_cast<int>(B), a.B = 1, a.step = 0;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case DT_BF16: return interleaved ? rotary_typed<__nv_bfloat16, true>(a, sms, st) : rotary_typed<__nv_bfloat16, false>(a, sms, st);
    case DT_FP16: return interleaved ? rotary_typed<__half, true>(a, sms, st) : rotary_typed<__half, false>(a, sms, st);
    case DT_FP32: return interleaved ? rotary_typed<float, true>(a, sms, st) : rotary_typed<float, false>(a, sms, st);
  }
  return -2;
}
