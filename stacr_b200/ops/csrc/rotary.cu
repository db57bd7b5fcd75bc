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
// Bound by memory: each value is read once and written once.  A thread owns one vector position of one token (its pairs' sines
// are computed once) and walks over a group of heads; how many heads a group has follows from how many threads the tokens
// alone give (see rotary_launch).
#include "gated.cuh"

namespace sb {

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RotPack {
  T v[VEC];
};

struct RotaryArgs {
  const void *q, *k;
  void *oq, *ok;                          // contiguous [B, S, heads, D]
  long long qb, qs, qh, kb, ks, kh;       // strides of the inputs in elements; the last dimension is contiguous
  const double* inv_freq;                 // [rot / 2]
  const void* positions;                  // int32 or int64, or null: position = first + s
  long long pb, ps, first;
  long long tokens;                       // B * S
  int S, hq, hk, D, rot, pos64, heads_per_group;
  float scale, sign;
};

template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  using P = RotPack<T, VEC>;
  constexpr int PAIRS = INTER ? (VEC > 1 ? VEC / 2 : 1) : VEC;   // pairs a thread turns
  constexpr int SPAN = INTER ? (VEC > 1 ? VEC : 2) : VEC;        // values from the start of one turning slot to the next
  const int turning = INTER ? a.rot / SPAN : (a.rot / 2) / VEC;
  const int slots = turning + (a.D - a.rot) / VEC;
  const long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
  if (i >= a.tokens * slots) return;
  const long long tok = i / slots;
  const int slot = static_cast<int>(i - tok * slots);
  const long long b = tok / a.S, s = tok - b * a.S;
  const int h0 = blockIdx.y * a.heads_per_group, total = a.hq + a.hk;
  const int h1 = h0 + a.heads_per_group < total ? h0 + a.heads_per_group : total;
  const T* q = static_cast<const T*>(a.q) + b * a.qb + s * a.qs;
  const T* k = static_cast<const T*>(a.k) + b * a.kb + s * a.ks;
  T* oq = static_cast<T*>(a.oq) + tok * a.hq * a.D;
  T* ok = static_cast<T*>(a.ok) + tok * a.hk * a.D;

  if (slot >= turning) {
    const int d = a.rot + (slot - turning) * VEC;
#pragma unroll 4
    for (int h = h0; h < h1; ++h) {
      const bool isq = h < a.hq;
      const T* src = isq ? q + h * a.qh : k + (h - a.hq) * a.kh;
      T* dst = isq ? oq + static_cast<long long>(h) * a.D : ok + static_cast<long long>(h - a.hq) * a.D;
      *reinterpret_cast<P*>(dst + d) = *reinterpret_cast<const P*>(src + d);
    }
    return;
  }

  long long pos = a.first + s;
  if (a.positions) {
    const long long at = b * a.pb + s * a.ps;
    pos = a.pos64 ? static_cast<const long long*>(a.positions)[at] : static_cast<const int*>(a.positions)[at];
  }
  float c[PAIRS], sn[PAIRS];
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) {
    const double turns = static_cast<double>(pos) * (__ldg(a.inv_freq + slot * PAIRS + j) * 0.15915494309189535);
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &sn[j], &c[j]);
    c[j] *= a.scale;
    sn[j] *= a.scale * a.sign;
  }
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const bool isq = h < a.hq;
    const T* src = (isq ? q + h * a.qh : k + (h - a.hq) * a.kh) + slot * SPAN;
    T* dst = (isq ? oq + static_cast<long long>(h) * a.D : ok + static_cast<long long>(h - a.hq) * a.D) + slot * SPAN;
    if (INTER && VEC > 1) {
      const P x = *reinterpret_cast<const P*>(src);
      P y;
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const float x1 = to_f32(x.v[(2 * j) % VEC]), x2 = to_f32(x.v[(2 * j + 1) % VEC]);
        y.v[(2 * j) % VEC] = from_f32<T>(x1 * c[j] - x2 * sn[j]);
        y.v[(2 * j + 1) % VEC] = from_f32<T>(x2 * c[j] + x1 * sn[j]);
      }
      *reinterpret_cast<P*>(dst) = y;
    } else {
      const int other = INTER ? 1 : a.rot / 2;
      const P xa = *reinterpret_cast<const P*>(src), xb = *reinterpret_cast<const P*>(src + other);
      P ya, yb;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float x1 = to_f32(xa.v[j]), x2 = to_f32(xb.v[j]);
        ya.v[j] = from_f32<T>(x1 * c[j % PAIRS] - x2 * sn[j % PAIRS]);
        yb.v[j] = from_f32<T>(x2 * c[j % PAIRS] + x1 * sn[j % PAIRS]);
      }
      *reinterpret_cast<P*>(dst) = ya;
      *reinterpret_cast<P*>(dst + other) = yb;
    }
  }
}

template <typename T, int VEC, bool INTER>
static int rotary_launch(RotaryArgs a, int sms, cudaStream_t st) {
  const int turning = INTER ? a.rot / (VEC > 1 ? VEC : 2) : (a.rot / 2) / VEC;
  const long long threads = a.tokens * (turning + (a.D - a.rot) / VEC);
  const int heads = a.hq + a.hk;
  // a thousand threads per SM keep enough loads in flight; the heads are split only as far as that takes
  long long groups = (static_cast<long long>(sms) * 1024 + threads - 1) / threads;
  if (groups > heads) groups = heads;
  a.heads_per_group = static_cast<int>((heads + groups - 1) / groups);
  const long long blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffLL) return -2;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((heads + a.heads_per_group - 1) / a.heads_per_group));
  rotary_kernel<T, VEC, INTER><<<grid, 256, 0, st>>>(a);
  return static_cast<int>(cudaGetLastError());
}

// The widest power-of-two vector that divides every extent, stride and address, at most 16 bytes.
static int rotary_width(const RotaryArgs& a, int size, bool inter) {
  unsigned long long bits = static_cast<unsigned long long>(inter ? a.rot : a.rot / 2) | static_cast<unsigned long long>(a.D) |
                            static_cast<unsigned long long>(a.D - a.rot) | (16 / size);
  const long long strides[] = {a.qb, a.qs, a.qh, a.kb, a.ks, a.kh};
  for (long long v : strides) bits |= static_cast<unsigned long long>(v);
  const void* ptrs[] = {a.q, a.k, a.oq, a.ok};
  for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p) / size;
  return static_cast<int>(bits & (~bits + 1));
}

template <typename T, bool INTER>
static int rotary_typed(const RotaryArgs& a, int sms, cudaStream_t st) {
  switch (rotary_width(a, sizeof(T), INTER)) {
    case 8: if constexpr (sizeof(T) == 2) return rotary_launch<T, 8, INTER>(a, sms, st);
    case 4: return rotary_launch<T, 4, INTER>(a, sms, st);
    case 2: return rotary_launch<T, 2, INTER>(a, sms, st);
    default: return rotary_launch<T, 1, INTER>(a, sms, st);
  }
}

}  // namespace sb

// q [B, S, hq, D] and k [B, S, hk, D] (null with hk = 0) with the strides given, into contiguous oq, ok; dtype 0 bf16, 1 fp16, 2 fp32.
// rot is even, 2 <= rot <= D.  sign +1 forward, -1 backward.
extern "C" int sb_rotary(const void* q, const void* k, void* oq, void* ok, long long qb, long long qs, long long qh, long long kb, long long ks, long long kh,
                         const double* inv_freq, const void* positions, int pos64, long long pb, long long ps, long long first, long long B, int S, int hq,
                         int hk, int D, int rot, int interleaved, int dtype, float scale, float sign, int sms, void* stream) {
  using namespace sb;
  if (B <= 0 || S <= 0 || hq + hk <= 0) return 0;
  if (rot < 2 || rot % 2 || rot > D || hq < 0 || hk < 0) return -2;
  RotaryArgs a{q, k, oq, ok, qb, qs, qh, kb, ks, kh, inv_freq, positions, pb, ps, first,
               B * S, S, hq, hk, D, rot, pos64, 0, scale, sign};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case DT_BF16: return interleaved ? rotary_typed<__nv_bfloat16, true>(a, sms, st) : rotary_typed<__nv_bfloat16, false>(a, sms, st);
    case DT_FP16: return interleaved ? rotary_typed<__half, true>(a, sms, st) : rotary_typed<__half, false>(a, sms, st);
    case DT_FP32: return interleaved ? rotary_typed<float, true>(a, sms, st) : rotary_typed<float, false>(a, sms, st);
  }
  return -2;
}
