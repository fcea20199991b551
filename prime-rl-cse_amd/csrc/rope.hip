// Rotary position embedding from position ids, query and key in one launch.
//
// Pair j of a head (j < r / 2, r = rotary_dim) turns by the angle p f_j, p the token's position and f_j the given
// inverse frequency, with amplitude a:
//     u' = a (u cos - v sin),   v' = a (v cos + u sin),        inverse: u = a (u' cos + v' sin), v = a (v' cos - u' sin)
// The pair is (x_j, x_{j + r/2}) in the half layout and (x_2j, x_2j+1) in the interleaved one; x_i for i >= r passes
// through.  Stands beside k_rope (norm.hip), which takes cos / sin tables, whole heads and the half layout only; the
// reference's switch for such kernels is `model.impl = "liger_kernel"` (src/prime_rl/trainer/model.py:74-75).
//
// The angle of a far position does not fit fp32: at p = 10^6 one unit in the last place of the product is 0.06 rad.
// It is formed in fp64 in turns, p f / (2 pi), and only its fraction of a turn goes to fp32, where sincospi is good to
// fp32 rounding.
//
// Bound by HBM: every element read and written once.  A workgroup takes a few tokens, forms their cos / sin once in
// LDS (r / 2 pairs per token) and uses them for all heads of query and key.
#include "logprob_dev.h"

namespace prl {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxPairs = 4096;  // r / 2 at most: 32 KB of LDS per token

// n / d for n < 2^31 without a division: (mulhi(n, mul) + n) >> shift, exact for every such n.
struct FastDiv {
  uint32_t d, mul, shift;
};
static FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}
__device__ __forceinline__ uint32_t quotient(uint32_t n, const FastDiv& f) { return (__umulhi(n, f.mul) + n) >> f.shift; }

// The fraction of a turn that p f radians are, in [-1/2, 1/2].  p f / (2 pi) is carried as a sum of two doubles (1 / (2 pi)
// to twice their length, the products' remainders by fma), so that what is left after the whole turns is good to fp32
// for every position a double holds.
__device__ __forceinline__ float turn_fraction(double p, double f) {
  constexpr double kHi = 0x1.45f306dc9c883p-3, kLo = -0x1.6b01ec5417056p-57;  // 1 / (2 pi)
  const double g = f * kHi, gl = fma(f, kHi, -g) + f * kLo;
  const double t = p * g, tl = fma(p, g, -t) + p * gl;
  return (float)((t - rint(t)) + tl);
}

struct RopeSide {
  const char* x;
  char* out;
  int64_t xb, xh, xt, ob, oh, ot;  // strides in bytes
};

// 16 bytes at an address that is only aligned to an element
typedef unsigned int u32x4_e2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x4_e4 __attribute__((ext_vector_type(4), aligned(4)));

// `n` of the VE elements from p on (n < VE: the rest is 0 and not read)
template <int DT, bool AL>
__device__ __forceinline__ void rope_load(const char* p, int n, float* y) {
  constexpr int VE = DT == PRL_F32 ? 4 : 8;
  if (n >= VE) {
    u32x4 v;
    if constexpr (AL) v = *reinterpret_cast<const u32x4*>(p);
    else if constexpr (DT == PRL_F32) v = *reinterpret_cast<const u32x4_e4*>(p);
    else v = *reinterpret_cast<const u32x4_e2*>(p);
    decode16_raw<DT>(v, y);
    return;
  }
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    y[i] = 0.0f;
    if (i < n) y[i] = DT == PRL_F32 ? reinterpret_cast<const float*>(p)[i] : bf16_one(reinterpret_cast<const uint16_t*>(p)[i]);
  }
}
template <int DT, bool AL>
__device__ __forceinline__ void rope_store(char* p, int n, const float* y) {
  constexpr int VE = DT == PRL_F32 ? 4 : 8;
  if (n >= VE) {
    u32x4 v;
    if constexpr (DT == PRL_F32) {
      v.x = __float_as_uint(y[0]), v.y = __float_as_uint(y[1]), v.z = __float_as_uint(y[2]), v.w = __float_as_uint(y[3]);
    } else {
      v.x = pack_bf16(y[0], y[1]), v.y = pack_bf16(y[2], y[3]), v.z = pack_bf16(y[4], y[5]), v.w = pack_bf16(y[6], y[7]);
    }
    if constexpr (AL) *reinterpret_cast<u32x4*>(p) = v;
    else if constexpr (DT == PRL_F32) *reinterpret_cast<u32x4_e4*>(p) = v;
    else *reinterpret_cast<u32x4_e2*>(p) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < VE; ++i)
    if (i < n) store_elem<DT>(p, i, y[i]);
}

// One row of a head is `rot` units of rotation (VE pairs of the half layout, VE / 2 of the interleaved one) and then
// the units of VE elements that pass through; a unit at the end of either part may be shorter.
template <int DT, bool IL, bool AL>
__global__ __launch_bounds__(kRopeThreads) void k_rope_positions(
    RopeSide q, RopeSide k, int q_heads, FastDiv heads, FastDiv units, FastDiv per_batch, int rot,
    const char* __restrict__ pos, int pos64, int64_t pos_b, int64_t pos_t, const char* __restrict__ inv_freq, int freq64,
    int r, int D, float amplitude, int inverse, int n_tokens, int tok_per_wg) {
  constexpr int ES = DT == PRL_F32 ? 4 : 2;
  constexpr int VE = 16 / ES;
  extern __shared__ float2 cs[];  // [token of the workgroup][pair]
  const int half = r >> 1;
  const int tok0 = blockIdx.x * tok_per_wg;
  const int ntok = min(tok_per_wg, n_tokens - tok0);
  for (int i = threadIdx.x; i < ntok * half; i += kRopeThreads) {
    const int tok = i / half, j = i - tok * half;
    const uint32_t n = tok0 + tok, b = quotient(n, per_batch), t = n - b * per_batch.d;
    const char* pp = pos + b * pos_b + t * pos_t;
    const double p = pos64 ? (double)*reinterpret_cast<const int64_t*>(pp) : (double)*reinterpret_cast<const int32_t*>(pp);
    const double f = freq64 ? reinterpret_cast<const double*>(inv_freq)[j] : (double)reinterpret_cast<const float*>(inv_freq)[j];
    float s, c;
    sincospif(2.0f * turn_fraction(p, f), &s, &c);
    cs[i] = make_float2(c * amplitude, (inverse ? -s : s) * amplitude);
  }
  __syncthreads();
  const uint32_t per_tok = heads.d * units.d;
  for (uint32_t i = threadIdx.x; i < ntok * per_tok; i += kRopeThreads) {
    const uint32_t row = quotient(i, units), u = i - row * units.d;
    const uint32_t tok = quotient(row, heads), h = row - tok * heads.d;
    const uint32_t n = tok0 + tok, b = quotient(n, per_batch), t = n - b * per_batch.d;
    const RopeSide& a = (int)h < q_heads ? q : k;
    const int64_t hh = (int)h < q_heads ? h : h - q_heads;
    const char* xp = a.x + b * a.xb + hh * a.xh + t * a.xt;
    char* op = a.out + b * a.ob + hh * a.oh + t * a.ot;
    float x1[VE], x2[VE], o1[VE], o2[VE];
    if ((int)u >= rot) {  // the part of the head that passes through
      const int at = r + ((int)u - rot) * VE, left = D - at;
      rope_load<DT, AL>(xp + (int64_t)at * ES, left, x1);
      rope_store<DT, AL>(op + (int64_t)at * ES, left, x1);
    } else if (IL) {
      const int at = (int)u * VE, left = r - at;
      const float2* w = cs + tok * half + at / 2;
      rope_load<DT, AL>(xp + at * ES, left, x1);
#pragma unroll
      for (int e = 0; e < VE; e += 2) {
        const float2 z = e < left ? w[e / 2] : make_float2(0.0f, 0.0f);
        o1[e] = fmaf(x1[e], z.x, -(x1[e + 1] * z.y));
        o1[e + 1] = fmaf(x1[e + 1], z.x, x1[e] * z.y);
      }
      rope_store<DT, AL>(op + at * ES, left, o1);
    } else {
      const int at = (int)u * VE, left = half - at;
      const float2* w = cs + tok * half + at;
      rope_load<DT, AL>(xp + at * ES, left, x1);
      rope_load<DT, AL>(xp + (at + half) * ES, left, x2);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float2 z = e < left ? w[e] : make_float2(0.0f, 0.0f);
        o1[e] = fmaf(x1[e], z.x, -(x2[e] * z.y));
        o2[e] = fmaf(x2[e], z.x, x1[e] * z.y);
      }
      rope_store<DT, AL>(op + at * ES, left, o1);
      rope_store<DT, AL>(op + (at + half) * ES, left, o2);
    }
  }
}

}  // namespace prl

using namespace prl;

extern "C" int prl_rope_positions_supported(int dtype, int64_t D, int64_t rotary_dim) {
  return (dtype == PRL_F32 || dtype == PRL_BF16) && rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= D &&
                 rotary_dim <= 2 * kRopeMaxPairs && D <= (1 << 20)
             ? 1
             : 0;
}

extern "C" int prl_rope_positions(const void* q, void* q_out, const int64_t* q_strides, int64_t q_heads, const void* k,
                                  void* k_out, const int64_t* k_strides, int64_t k_heads, const void* positions,
                                  int positions_64, int64_t pos_batch_stride, int64_t pos_token_stride,
                                  const void* inv_freq, int inv_freq_64, int64_t rotary_dim, int interleaved,
                                  float amplitude, int dtype, int64_t B, int64_t T, int64_t D, int inverse, void* stream) {
  clear_error();
  PRL_REQUIRE(B >= 0 && T >= 0 && q_heads >= 0 && k_heads >= 0, "rope_positions: sizes must be >= 0");
  PRL_REQUIRE(prl_rope_positions_supported(dtype, D, rotary_dim),
              "rope_positions: dtype %d, head size %lld or rotary_dim %lld is not supported (rotary_dim even, 2 .. %d and "
              "at most the head size)", dtype, (long long)D, (long long)rotary_dim, 2 * kRopeMaxPairs);
  if (B == 0 || T == 0 || q_heads + k_heads == 0) return PRL_OK;
  const int es = dtype == PRL_F32 ? 4 : 2, ve = 16 / es;
  PRL_REQUIRE(positions && inv_freq, "rope_positions: positions and inv_freq must not be NULL");
  PRL_REQUIRE(q_heads == 0 || (q && q_out && q_strides), "rope_positions: q, q_out and q_strides must not be NULL");
  PRL_REQUIRE(k_heads == 0 || (k && k_out && k_strides), "rope_positions: k, k_out and k_strides must not be NULL");
  const int64_t half = rotary_dim / 2;
  const int64_t rot = interleaved ? (rotary_dim + ve - 1) / ve : (half + ve - 1) / ve;
  const int64_t units = rot + (D - rotary_dim + ve - 1) / ve;
  const int64_t heads = q_heads + k_heads;
  PRL_REQUIRE(B < (1ll << 31) && T < (1ll << 31) && B * T < (1ll << 31) - 64, "rope_positions: B * T must be below 2^31");
  PRL_REQUIRE(heads < (1ll << 20) && units * heads < (1ll << 26), "rope_positions: too many heads");
  uintptr_t bits = 0, elem = 0;
  RopeSide side[2] = {};
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t* st[2] = {q_strides, k_strides};
  for (int i = 0; i < 2; ++i) {
    if ((i ? k_heads : q_heads) == 0) continue;
    side[i] = {(const char*)in[i], (char*)out[i], st[i][0] * es, st[i][1] * es, st[i][2] * es,
               st[i][3] * es,      st[i][4] * es, st[i][5] * es};
    const uintptr_t p = reinterpret_cast<uintptr_t>(in[i]) | reinterpret_cast<uintptr_t>(out[i]);
    elem |= p;
    bits |= p;
    for (int j = 0; j < 6; ++j) bits |= (uintptr_t)(st[i][j] * es);
  }
  PRL_REQUIRE((elem & (es - 1)) == 0, "rope_positions: pointers must be aligned to an element");
  // every 16-byte access of a row starts a multiple of 16 bytes from the row's start
  const bool al = ((bits | (uintptr_t)(rotary_dim * es) | (uintptr_t)(interleaved ? 0 : half * es)) & 15) == 0;
  const int64_t tokens = B * T;
  int tok = 1;
  const int64_t grid = (tokens + tok - 1) / tok;
  const size_t lds = (size_t)tok * half * sizeof(float2);
#define PRL_ROPE(DT, IL, AL)                                                                                         \
  hipLaunchKernelGGL((k_rope_positions<DT, IL, AL>), dim3((unsigned)grid), dim3(kRopeThreads), lds, (hipStream_t)stream, \
                     side[0], side[1], (int)q_heads, fast_div((uint32_t)heads), fast_div((uint32_t)units),           \
                     fast_div((uint32_t)T), (int)rot, (const char*)positions, positions_64 ? 1 : 0,                  \
                     pos_batch_stride * (positions_64 ? 8 : 4), pos_token_stride * (positions_64 ? 8 : 4),           \
                     (const char*)inv_freq, inv_freq_64 ? 1 : 0, (int)rotary_dim, (int)D, amplitude, inverse ? 1 : 0, \
                     (int)tokens, tok)
#define PRL_ROPE_AL(DT, IL) \
  if (al) PRL_ROPE(DT, IL, true); else PRL_ROPE(DT, IL, false)
  if (dtype == PRL_BF16) {
    if (interleaved) { PRL_ROPE_AL(PRL_BF16, true); } else { PRL_ROPE_AL(PRL_BF16, false); }
  } else {
    if (interleaved) { PRL_ROPE_AL(PRL_F32, true); } else { PRL_ROPE_AL(PRL_F32, false); }
  }
#undef PRL_ROPE_AL
#undef PRL_ROPE
  PRL_CHECK_LAUNCH("rope_positions");
  return PRL_OK;
}
