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
// Bound by HBM: every element read and written once, 201 MB in 39.5 us (5.1 TB/s).  A workgroup takes a few tokens and
// forms their cos / sin once in LDS (r / 2 pairs per token).  A thread then owns one place in the head, two 16-byte
// vectors of it, keeps its cos / sin in registers and walks over the heads of query and key, two at a time.
#include "logprob_dev.h"

namespace prl {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxPairs = 4096;  // r / 2 at most: 32 KB of LDS per token

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

// VEC: a thread's two pieces of a head are 16-byte vectors (rows aligned, the pairs of the half layout in whole vectors);
// otherwise single elements, side by side over the lanes (r = 34 of 128 in the half layout: 49.2 us; 16-byte accesses at
// places aligned to an element only took 107).  NT: the loads go past the caches.
template <int DT, bool VEC, bool NT>
struct RopeUnit {
  static constexpr int kEs = DT == PRL_F32 ? 4 : 2;
  static constexpr int kN = VEC ? 16 / kEs : 1;  // elements of a piece
  u32x4 z;
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (VEC && NT) z = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    else if constexpr (VEC) z = *reinterpret_cast<const u32x4*>(p);
    else if constexpr (DT == PRL_F32) z.x = *reinterpret_cast<const uint32_t*>(p);
    else z.x = *reinterpret_cast<const uint16_t*>(p);
  }
  __device__ __forceinline__ void get(float* y) const {
    if constexpr (VEC) decode16_raw<DT>(z, y);
    else y[0] = DT == PRL_F32 ? __uint_as_float(z.x) : bf16_lo(z.x);
  }
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (VEC) *reinterpret_cast<u32x4*>(p) = z;
    else if constexpr (DT == PRL_F32) *reinterpret_cast<uint32_t*>(p) = z.x;
    else *reinterpret_cast<uint16_t*>(p) = (uint16_t)z.x;
  }
  __device__ __forceinline__ void put(const float* y) {
    if constexpr (!VEC) z.x = DT == PRL_F32 ? __float_as_uint(y[0]) : one_bf16(y[0]);
    else if constexpr (DT == PRL_F32)
      z.x = __float_as_uint(y[0]), z.y = __float_as_uint(y[1]), z.z = __float_as_uint(y[2]), z.w = __float_as_uint(y[3]);
    else
      z.x = pack_bf16(y[0], y[1]), z.y = pack_bf16(y[2], y[3]), z.z = pack_bf16(y[4], y[5]), z.w = pack_bf16(y[6], y[7]);
  }
};

struct RopeShape {
  int r, D;         // rotated dimensions, head size
  int units;        // places in a head: pairs of pieces
  int per_row;      // threads side by side on a row: min(units, threads)
  int slots, toks;  // heads and tokens a workgroup has in flight
};

// Turns the two pieces of one head in place; `turn` bit e: pair e belongs to the rotated part.
template <int DT, bool IL, bool VEC, bool NT>
__device__ __forceinline__ void rope_turn(RopeUnit<DT, VEC, NT>& p1, RopeUnit<DT, VEC, NT>& p2, const float* c, const float* s,
                                          uint32_t turn) {
  constexpr int N = RopeUnit<DT, VEC, NT>::kN;
  if (!turn) return;
  float x[2 * N], y[2 * N];
  p1.get(x), p2.get(x + N);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int i = IL ? 2 * e : e, j = IL ? 2 * e + 1 : e + N;
    const bool on = !IL || (turn >> e & 1);
    y[i] = on ? fmaf(x[i], c[e], -(x[j] * s[e])) : x[i];
    y[j] = on ? fmaf(x[j], c[e], x[i] * s[e]) : x[j];
  }
  p1.put(y), p2.put(y + N);
}

template <int DT, bool IL, bool VEC, bool NT>
__global__ __launch_bounds__(kRopeThreads) void k_rope_positions(RopeSide q, RopeSide k, int q_heads, int heads,
                                                                 RopeShape sh, const char* __restrict__ pos, int pos64,
                                                                 int64_t pos_b, int64_t pos_t,
                                                                 const char* __restrict__ inv_freq, int freq64,
                                                                 float amplitude, int inverse, int first, int n_tokens, int T) {
  using P = RopeUnit<DT, VEC, NT>;
  constexpr int N = P::kN, ES = P::kEs;
  extern __shared__ float2 cs[];  // [token of the workgroup][pair]
  const int half = sh.r >> 1;
  const int tok0 = first + blockIdx.x * sh.toks;
  const int ntok = min(sh.toks, n_tokens - tok0);
  for (int i = threadIdx.x; i < ntok * half; i += kRopeThreads) {
    const int tk = i / half, j = i - tk * half;
    const int n = tok0 + tk, b = n / T, t = n - b * T;
    const char* pp = pos + b * pos_b + t * pos_t;
    const double p = pos64 ? (double)*reinterpret_cast<const int64_t*>(pp) : (double)*reinterpret_cast<const int32_t*>(pp);
    const double f = freq64 ? reinterpret_cast<const double*>(inv_freq)[j] : (double)reinterpret_cast<const float*>(inv_freq)[j];
    float s, c;
    sincospif(2.0f * turn_fraction(p, f), &s, &c);
    cs[i] = make_float2(c * amplitude, (inverse ? -s : s) * amplitude);
  }
  __syncthreads();
  const int g = threadIdx.x / sh.per_row, u0 = threadIdx.x - g * sh.per_row;
  const int tok = g / sh.slots, h0 = g - tok * sh.slots;
  if (tok >= ntok) return;
  const int n = tok0 + tok;
  const int64_t b = n / T, t = n - b * T;
  for (int u = u0; u < sh.units; u += sh.per_row) {
    // The two pieces' first elements, and which of their pairs turn.  Neighbouring lanes take neighbouring pieces.
    int e1, e2, pair1, pair2;
    uint32_t turn;
    if (IL && VEC) {  // half of a unit's pairs in either piece
      e1 = N * u, e2 = N * (u + sh.units), pair1 = e1 / 2, pair2 = e2 / 2;
      const int on1 = min(max(half - pair1, 0), N / 2), on2 = min(max(half - pair2, 0), N / 2);
      turn = ((1u << on1) - 1) | ((1u << on2) - 1) << (N / 2);
    } else if (IL) {
      e1 = 2 * u, e2 = e1 + 1, pair1 = pair2 = u;
      turn = u < half;
    } else {
      const int rot = half / N;
      pair1 = pair2 = N * u;
      turn = u < rot;
      e1 = turn ? pair1 : sh.r + N * (u - rot), e2 = turn ? half + pair1 : e1 + N * (sh.units - rot);
    }
    const bool two = e2 < sh.D;
    float c[N], s[N];
    if (turn) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int j = IL && VEC ? min(e < N / 2 ? pair1 + e : pair2 + e - N / 2, half - 1) : pair1 + e;
        const float2 z = cs[tok * half + j];
        c[e] = z.x, s[e] = z.y;
      }
    }
    const char* xq = q.x + b * q.xb + t * q.xt + (int64_t)e1 * ES;
    const char* xk = k.x + b * k.xb + t * k.xt + (int64_t)e1 * ES;
    char* oq = q.out + b * q.ob + t * q.ot + (int64_t)e1 * ES;
    char* ok = k.out + b * k.ob + t * k.ot + (int64_t)e1 * ES;
    const int64_t gap = (int64_t)(two ? e2 - e1 : 0) * ES;  // (a last piece alone is loaded twice and stored once)
    for (int h = h0; h < heads; h += 2 * sh.slots) {
      const int g2 = h + sh.slots;
      const bool also = g2 < heads;
      const char *xa = h < q_heads ? xq + h * q.xh : xk + (h - q_heads) * k.xh, *xb = xa;
      char *oa = h < q_heads ? oq + h * q.oh : ok + (h - q_heads) * k.oh, *ob = oa;
      if (also) {
        xb = g2 < q_heads ? xq + g2 * q.xh : xk + (g2 - q_heads) * k.xh;
        ob = g2 < q_heads ? oq + g2 * q.oh : ok + (g2 - q_heads) * k.oh;
      }
      P a1, a2, b1, b2;
      a1.load(xa), a2.load(xa + gap);
      if (also) b1.load(xb), b2.load(xb + gap);
      rope_turn<DT, IL, VEC, NT>(a1, a2, c, s, turn);
      a1.store(oa);
      if (two) a2.store(oa + gap);
      if (also) {
        rope_turn<DT, IL, VEC, NT>(b1, b2, c, s, turn);
        b1.store(ob);
        if (two) b2.store(ob + gap);
      }
    }
  }
}

// Threads of a workgroup: `units` side by side on a row as far as they go, the rest over two tokens and as many heads of
// each as fit (24 heads of 128 bf16, 16384 tokens: 39.5 us with two tokens, 50.5 with one, 39.7 with four; 2048 tokens:
// 7.2, 8.4, 8.3; 48 single tokens: 4.2 with any).
static RopeShape rope_shape(int64_t r, int64_t D, int64_t heads, int ve, bool il, bool vec) {
  RopeShape s;
  s.r = (int)r, s.D = (int)D;
  const int64_t n = vec ? ve : 1;
  s.units = (int)(il ? (D + 2 * n - 1) / (2 * n) : r / 2 / n + (D - r + 2 * n - 1) / (2 * n));
  s.per_row = s.units < kRopeThreads ? s.units : kRopeThreads;
  const int groups = kRopeThreads / s.per_row;
  int toks = groups < 2 || r / 2 > kRopeMaxPairs / 2 ? 1 : 2;
  s.slots = groups / toks < heads ? groups / toks : (int)heads;
  s.toks = groups / s.slots < toks ? groups / s.slots : toks;
  return s;
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
  const int64_t half = rotary_dim / 2, heads = q_heads + k_heads;
  PRL_REQUIRE(B < (1ll << 31) && T < (1ll << 31) && B * T < (1ll << 31) - 64, "rope_positions: B * T must be below 2^31");
  PRL_REQUIRE(heads < (1ll << 20), "rope_positions: too many heads");
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
  const bool vec = ((bits | (uintptr_t)(D * es) | (uintptr_t)(interleaved ? 0 : half * es)) & 15) == 0;
  const int64_t tokens = B * T;
  // Loads go past the caches where a wave's accesses are whole lines (half of 128 dimensions turned in halves, 167 MB:
  // 83.8 us against 81.0 through them), stores stay in them for the attention that reads them.  Cold, one side just
  // written and read behind; neither past the caches, loads only, both: 25 MB 20.8, 20.4, 20.8 us; 167 MB 81.2, 80.3,
  // 82.4; 402 MB 213, 208, 202; by itself 402 MB 75.3, 74.7, 69.0.
  const bool nt = interleaved || rotary_dim == D;
  const RopeShape sh = rope_shape(rotary_dim, D, heads, ve, interleaved, vec);
  const size_t lds = (size_t)sh.toks * half * sizeof(float2);
#define PRL_ROPE(DT, IL, VEC, NT)                                                                                       \
  hipLaunchKernelGGL((k_rope_positions<DT, IL, VEC, NT>), dim3(grid), dim3(kRopeThreads), lds, (hipStream_t)stream, \
                     side[0], side[1], (int)q_heads, (int)heads, sh, (const char*)positions, positions_64 ? 1 : 0,   \
                     pos_batch_stride * (positions_64 ? 8 : 4), pos_token_stride * (positions_64 ? 8 : 4),           \
                     (const char*)inv_freq, inv_freq_64 ? 1 : 0, amplitude, inverse ? 1 : 0, (int)first, (int)tokens, (int)T)
#define PRL_ROPE_VEC(DT, IL) \
  if (vec && nt) PRL_ROPE(DT, IL, true, true); else if (vec) PRL_ROPE(DT, IL, true, false); else PRL_ROPE(DT, IL, false, false)
  const int64_t most = (int64_t)sh.toks << 22;  // tokens of a launch, which holds fewer than 2^32 threads
  for (int64_t first = 0; first < tokens; first += most) {
    const unsigned grid = (unsigned)(((tokens - first < most ? tokens - first : most) + sh.toks - 1) / sh.toks);
    if (dtype == PRL_BF16) {
      if (interleaved) { PRL_ROPE_VEC(PRL_BF16, true); } else { PRL_ROPE_VEC(PRL_BF16, false); }
    } else {
      if (interleaved) { PRL_ROPE_VEC(PRL_F32, true); } else { PRL_ROPE_VEC(PRL_F32, false); }
    }
  }
#undef PRL_ROPE_VEC
#undef PRL_ROPE
  PRL_CHECK_LAUNCH("rope_positions");
  return PRL_OK;
}
