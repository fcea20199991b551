// The global norm of many gradient tensors, and their clipping, as torch.nn.utils.clip_grad_norm_ does it for the
// reference (src/prime_rl/trainer/rl/train.py:336-338):
//     N = sqrt(sum g^2)  or  max |g|,    c = min(1, max_norm / (N + 1e-6)),    g <- g c
// Two passes over the gradients; where c is exactly 1 the second touches none.  Bound by HBM: 1.8 GB of fp32 in 310
// tensors take 874 us when they are clipped (6.1 TB/s over two reads and a write), 325 when there is nothing to clip
// (5.5).  Both passes go past the caches (non-temporal: 1029 -> 875 us); keeping the end of the first in the last-level
// cache for the second gained nothing.
//
// The tensors' addresses and lengths travel in the launch itself, up to kClipPieces of them each: nothing is copied to
// the device, the calls are legal under stream capture, and no table outlives them.  Pieces are cut into chunks; a
// workgroup takes every so-manieth of them.  Squares are formed and added in fp64: no overflow for any fp32
// gradient.  The order of the sums is fixed by the tensors' sizes and places in memory (which of them touch, where each
// starts within 16 bytes): the same buffers give the same bits, others may differ in the last of 64.
#include "prl_common.h"

namespace prl {

constexpr int kClipThreads = 256;
constexpr int kClipPieces = 160;   // 24 bytes each: a launch's arguments stay below 4 KB
constexpr int kClipChunk = 8192;   // elements
constexpr int kClipNormBlocks = 1024;  // and partial values of a launch, few enough for every workgroup to add up
constexpr int kClipScaleBlocks = 1 << 22;  // one chunk a workgroup (1.8 GB: 623 us; 2048 workgroups in a loop 665)
constexpr int kClipAhead = 4;  // 16-byte vectors a thread has in flight

struct ClipTable {
  char* x[kClipPieces];
  int64_t n[kClipPieces];             // elements
  uint32_t end[kClipPieces];          // chunks up to and including this piece
  uint8_t f32[kClipPieces];
  int32_t pieces;
};
static_assert(sizeof(ClipTable) <= 3600, "the launch's arguments have to stay below 4 KB");

// Calls f(address, elements, is fp32) for every gridDim.x-th chunk of the table: all workgroups move through memory
// together (a run of chunks each: 1064 us for the norm and the scaling of 1.8 GB, this way 1028).
template <typename F>
__device__ __forceinline__ void clip_walk(const ClipTable& t, F f) {
  const uint32_t chunks = t.end[t.pieces - 1];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    int lo = 0, hi = t.pieces - 1;  // the piece that chunk c lies in: the first whose end is beyond it
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (t.end[mid] > c) hi = mid; else lo = mid + 1;
    }
    const int64_t at = (int64_t)(c - (lo ? t.end[lo - 1] : 0)) * kClipChunk;
    const int64_t left = t.n[lo] - at;
    const bool f32 = t.f32[lo] != 0;
    f(t.x[lo] + at * (f32 ? 4 : 2), (int)(left < kClipChunk ? left : kClipChunk), f32);
  }
}

template <bool MAX>
__device__ __forceinline__ double clip_take(double s, float v) {
  const double d = (double)v;
  if (!MAX) return fma(d, d, s);
  const double a = fabs(d);
  return a > s || a != a ? a : s;  // a NaN stays: nothing compares greater than it
}
template <bool MAX>
__device__ __forceinline__ double clip_join(double a, double b) {
  if (!MAX) return a + b;
  return b > a || b != b ? b : a;
}

// Elements of a chunk: singles up to the first 16-byte boundary, 16-byte vectors, singles behind them.
template <bool F32, bool MAX>
__device__ __forceinline__ double clip_chunk_sum(const char* x, int n, double s) {
  constexpr int ES = F32 ? 4 : 2, VE = 16 / ES;
  int head = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / ES);
  if (head > n) head = n;
  const int nvec = (n - head) / VE;
  const u32x4* v = reinterpret_cast<const u32x4*>(x + head * ES);
  auto take = [&](const u32x4& z) {
    const uint32_t w[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (F32) {
        s = clip_take<MAX>(s, __uint_as_float(w[j]));
      } else {
        s = clip_take<MAX>(s, bf16_lo(w[j]));
        s = clip_take<MAX>(s, bf16_hi(w[j]));
      }
    }
  };
  int i = threadIdx.x;
  for (; i + (kClipAhead - 1) * kClipThreads < nvec; i += kClipAhead * kClipThreads) {
    u32x4 z[kClipAhead];
#pragma unroll
    for (int j = 0; j < kClipAhead; ++j) z[j] = __builtin_nontemporal_load(v + i + j * kClipThreads);
#pragma unroll
    for (int j = 0; j < kClipAhead; ++j) take(z[j]);
  }
  for (; i < nvec; i += kClipThreads) take(v[i]);
  const int rest = n - nvec * VE;  // head + tail: fewer than 2 VE
  if ((int)threadIdx.x < rest) {
    const int e = (int)threadIdx.x < head ? threadIdx.x : threadIdx.x + nvec * VE;
    s = clip_take<MAX>(s, F32 ? reinterpret_cast<const float*>(x)[e] : bf16_one(reinterpret_cast<const uint16_t*>(x)[e]));
  }
  return s;
}

template <bool MAX>
__device__ __forceinline__ double clip_block_join(double s, double* slots) {
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) s = clip_join<MAX>(s, __shfl_xor(s, o, kWave));
  if ((threadIdx.x & (kWave - 1)) == 0) slots[threadIdx.x / kWave] = s;
  __syncthreads();
  s = slots[0];
  for (int i = 1; i < (int)blockDim.x / kWave; ++i) s = clip_join<MAX>(s, slots[i]);
  return s;
}

template <bool MAX>
__global__ __launch_bounds__(kClipThreads) void k_grad_norm(const ClipTable t, double* __restrict__ part) {
  __shared__ double slots[kClipThreads / kWave];
  double s = 0.0;
  clip_walk(t, [&](const char* x, int n, bool f32) {
    s = f32 ? clip_chunk_sum<true, MAX>(x, n, s) : clip_chunk_sum<false, MAX>(x, n, s);
  });
  s = clip_block_join<MAX>(s, slots);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// From the joined partial values (sum of squares, or largest magnitude): the norm and the factor, min(1, .) that lets a
// NaN through: with a norm that is not a number every gradient becomes one, as torch's clamp makes it; with an infinite
// norm the factor is 0.
template <bool MAX>
__device__ __forceinline__ float clip_factor(double total, float max_norm, float& norm) {
  norm = (float)(MAX ? total : sqrt(total));
  const float c = max_norm / (norm + 1e-6f);
  return c > 1.0f ? 1.0f : c;
}
template <bool MAX>
__device__ __forceinline__ double clip_total(const double* part, int nparts, double* slots) {
  double s = 0.0;
  for (int i = threadIdx.x; i < nparts; i += kClipThreads) s = clip_join<MAX>(s, part[i]);
  return clip_block_join<MAX>(s, slots);
}

template <bool MAX>
__global__ __launch_bounds__(kClipThreads) void k_grad_norm_finish(const double* part, int nparts, double* total,
                                                                   float max_norm, float* norm, float* coef) {
  __shared__ double slots[kClipThreads / kWave];
  const double s = clip_total<MAX>(part, nparts, slots);
  if (threadIdx.x != 0) return;
  float n;
  const float c = clip_factor<MAX>(s, max_norm, n);
  if (total) *total = s;
  if (norm) *norm = n;
  if (coef) *coef = c;
}

template <bool F32>
__device__ __forceinline__ void clip_chunk_scale(char* x, int n, float c) {
  constexpr int ES = F32 ? 4 : 2, VE = 16 / ES;
  int head = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / ES);
  if (head > n) head = n;
  const int nvec = (n - head) / VE;
  u32x4* v = reinterpret_cast<u32x4*>(x + head * ES);
  auto scaled = [&](u32x4 z) {
    uint32_t w[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = F32 ? __float_as_uint(__uint_as_float(w[j]) * c) : pack_bf16(bf16_lo(w[j]) * c, bf16_hi(w[j]) * c);
    z.x = w[0], z.y = w[1], z.z = w[2], z.w = w[3];
    return z;
  };
  int i = threadIdx.x;
  for (; i + (kClipAhead - 1) * kClipThreads < nvec; i += kClipAhead * kClipThreads) {
    u32x4 z[kClipAhead];
#pragma unroll
    for (int j = 0; j < kClipAhead; ++j) z[j] = __builtin_nontemporal_load(v + i + j * kClipThreads);
#pragma unroll
    for (int j = 0; j < kClipAhead; ++j) __builtin_nontemporal_store(scaled(z[j]), v + i + j * kClipThreads);
  }
  for (; i < nvec; i += kClipThreads) v[i] = scaled(v[i]);
  const int rest = n - nvec * VE;
  if ((int)threadIdx.x < rest) {
    const int e = (int)threadIdx.x < head ? threadIdx.x : threadIdx.x + nvec * VE;
    if (F32) reinterpret_cast<float*>(x)[e] *= c;
    else reinterpret_cast<uint16_t*>(x)[e] = one_bf16(bf16_one(reinterpret_cast<const uint16_t*>(x)[e]) * c);
  }
}

__device__ __forceinline__ void clip_scale(const ClipTable& t, float c) {
  if (c == 1.0f) return;
  clip_walk(t, [&](char* x, int n, bool f32) {
    if (f32) clip_chunk_scale<true>(x, n, c);
    else clip_chunk_scale<false>(x, n, c);
  });
}
__global__ __launch_bounds__(kClipThreads) void k_grad_scale(const ClipTable t, const float* __restrict__ coef) {
  clip_scale(t, *coef);
}
// The scaling with the finish in it: every workgroup joins the partial values itself, in the same order, which is
// cheaper than a launch between the two (2 us against 4.5 with nothing to clip) for few launches' partial values.  With
// many tensors the joining shows: 706 of bf16, 1.9 GB, five launches of partial values, take 624 us with nothing to clip,
// about twice the time of their read.  There is no other form for that yet.
template <bool MAX>
__global__ __launch_bounds__(kClipThreads) void k_grad_clip(const ClipTable t, const double* __restrict__ part, int nparts,
                                                            float max_norm, float* __restrict__ norm) {
  __shared__ double slots[kClipThreads / kWave];
  float n;
  const float c = clip_factor<MAX>(clip_total<MAX>(part, nparts, slots), max_norm, n);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  clip_scale(t, c);
}

static int64_t clip_chunks(int64_t n) { return (n + kClipChunk - 1) / kClipChunk; }
static int clip_blocks(int64_t chunks, int most) { return (int)(chunks < most ? chunks : most); }

static int clip_check(const char* who, const prl_grad_piece* pieces, int64_t n_pieces) {
  PRL_REQUIRE(n_pieces >= 0, "%s: n_pieces must be >= 0", who);
  PRL_REQUIRE(n_pieces == 0 || pieces, "%s: pieces must not be NULL", who);
  for (int64_t i = 0; i < n_pieces; ++i) {
    const prl_grad_piece& p = pieces[i];
    PRL_REQUIRE(p.dtype == PRL_F32 || p.dtype == PRL_BF16, "%s: piece %lld has unsupported dtype %d", who, (long long)i,
                p.dtype);
    // chunk numbers of a launch are 32-bit
    PRL_REQUIRE(p.n >= 0 && p.n <= (int64_t)1 << 42, "%s: piece %lld has %lld elements", who, (long long)i, (long long)p.n);
    PRL_REQUIRE(p.n == 0 || (p.x && (reinterpret_cast<uintptr_t>(p.x) & (p.dtype == PRL_F32 ? 3 : 1)) == 0),
                "%s: piece %lld is NULL or not aligned to an element", who, (long long)i);
  }
  return PRL_OK;
}

// The next launch's table from piece `at` on; returns its number of chunks (0: no pieces left) and moves `at`.
static int64_t clip_fill(ClipTable& t, const prl_grad_piece* pieces, int64_t n_pieces, int64_t& at) {
  int64_t chunks = 0;
  t.pieces = 0;
  for (; at < n_pieces && t.pieces < kClipPieces; ++at) {
    const int64_t c = clip_chunks(pieces[at].n);
    if (c == 0) continue;
    if (chunks + c > 0x7fffffff) break;
    chunks += c;
    t.x[t.pieces] = (char*)pieces[at].x;
    t.n[t.pieces] = pieces[at].n;
    t.end[t.pieces] = (uint32_t)chunks;
    t.f32[t.pieces] = pieces[at].dtype == PRL_F32;
    ++t.pieces;
  }
  return chunks;
}

static int64_t clip_partials(const prl_grad_piece* pieces, int64_t n_pieces) {
  int64_t at = 0, total = 0, c;
  ClipTable t;
  while ((c = clip_fill(t, pieces, n_pieces, at)) > 0) total += clip_blocks(c, kClipNormBlocks);
  return total;
}

}  // namespace prl

using namespace prl;

extern "C" size_t prl_grad_norm_workspace_bytes(const prl_grad_piece* pieces, int64_t n_pieces) {
  if (clip_check("grad_norm_workspace_bytes", pieces, n_pieces) != PRL_OK) return 0;
  const int64_t n = clip_partials(pieces, n_pieces);
  return (size_t)(n > 0 ? n : 1) * sizeof(double);
}

// Launches the partial values of all pieces into `part`; `done` becomes their number.
static int clip_norm_launches(const char* who, const prl_grad_piece* pieces, int64_t n_pieces, int kind, void* workspace,
                              size_t workspace_bytes, int64_t& done, hipStream_t st) {
  int rc = clip_check(who, pieces, n_pieces);
  if (rc != PRL_OK) return rc;
  PRL_REQUIRE(kind == PRL_NORM_L2 || kind == PRL_NORM_MAX, "%s: unknown norm kind %d", who, kind);
  const int64_t need = clip_partials(pieces, n_pieces);
  PRL_REQUIRE(need == 0 || (workspace && workspace_bytes >= (size_t)need * sizeof(double) &&
                            (reinterpret_cast<uintptr_t>(workspace) & 7) == 0),
              "%s: 8-byte aligned workspace of %lld bytes needed (prl_grad_norm_workspace_bytes)", who, (long long)need * 8);
  PRL_REQUIRE(need <= 0x7fffffff, "%s: too many pieces", who);
  int64_t at = 0, chunks;
  done = 0;
  ClipTable t;
  while ((chunks = clip_fill(t, pieces, n_pieces, at)) > 0) {
    const dim3 grid((unsigned)clip_blocks(chunks, kClipNormBlocks)), block(kClipThreads);
    double* part = (double*)workspace + done;
    if (kind == PRL_NORM_MAX) hipLaunchKernelGGL((k_grad_norm<true>), grid, block, 0, st, t, part);
    else hipLaunchKernelGGL((k_grad_norm<false>), grid, block, 0, st, t, part);
    PRL_CHECK_LAUNCH(who);
    done += grid.x;
  }
  return PRL_OK;
}

extern "C" int prl_grad_norm(const prl_grad_piece* pieces, int64_t n_pieces, int kind, float max_norm, double* total,
                             float* norm, float* coef, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  PRL_REQUIRE(total || norm || coef, "grad_norm: nothing asked for");
  int64_t done;
  int rc = clip_norm_launches("grad_norm", pieces, n_pieces, kind, workspace, workspace_bytes, done, (hipStream_t)stream);
  if (rc != PRL_OK) return rc;
  return prl_grad_norm_finish((const double*)workspace, done, kind, max_norm, total, norm, coef, stream);
}

extern "C" int prl_grad_clip(const prl_grad_piece* pieces, int64_t n_pieces, int kind, float max_norm, float* norm,
                             void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  PRL_REQUIRE(norm, "grad_clip: norm must not be NULL");
  int64_t done;
  hipStream_t st = (hipStream_t)stream;
  int rc = clip_norm_launches("grad_clip", pieces, n_pieces, kind, workspace, workspace_bytes, done, st);
  if (rc != PRL_OK) return rc;
  if (done == 0) return prl_grad_norm_finish(nullptr, 0, kind, max_norm, nullptr, norm, nullptr, stream);
  int64_t at = 0, chunks;
  ClipTable t;
  while ((chunks = clip_fill(t, pieces, n_pieces, at)) > 0) {
    const dim3 grid((unsigned)clip_blocks(chunks, kClipScaleBlocks)), block(kClipThreads);
    const double* part = (const double*)workspace;
    if (kind == PRL_NORM_MAX) hipLaunchKernelGGL((k_grad_clip<true>), grid, block, 0, st, t, part, (int)done, max_norm, norm);
    else hipLaunchKernelGGL((k_grad_clip<false>), grid, block, 0, st, t, part, (int)done, max_norm, norm);
    PRL_CHECK_LAUNCH("grad_clip");
  }
  return PRL_OK;
}

extern "C" int prl_grad_norm_finish(const double* parts, int64_t n_parts, int kind, float max_norm, double* total,
                                    float* norm, float* coef, void* stream) {
  clear_error();
  PRL_REQUIRE(n_parts >= 0 && n_parts <= 0x7fffffff && (n_parts == 0 || parts), "grad_norm_finish: bad partial values");
  PRL_REQUIRE(kind == PRL_NORM_L2 || kind == PRL_NORM_MAX, "grad_norm_finish: unknown norm kind %d", kind);
  const dim3 block(kClipThreads);
  hipStream_t st = (hipStream_t)stream;
  if (kind == PRL_NORM_MAX)
    hipLaunchKernelGGL((k_grad_norm_finish<true>), dim3(1), block, 0, st, parts, (int)n_parts, total, max_norm, norm, coef);
  else
    hipLaunchKernelGGL((k_grad_norm_finish<false>), dim3(1), block, 0, st, parts, (int)n_parts, total, max_norm, norm, coef);
  PRL_CHECK_LAUNCH("grad_norm_finish");
  return PRL_OK;
}

extern "C" int prl_grad_scale(const prl_grad_piece* pieces, int64_t n_pieces, const float* coef, void* stream) {
  clear_error();
  int rc = clip_check("grad_scale", pieces, n_pieces);
  if (rc != PRL_OK) return rc;
  if (n_pieces == 0) return PRL_OK;
  PRL_REQUIRE(coef, "grad_scale: coef must not be NULL");
  int64_t at = 0, chunks;
  ClipTable t;
  while ((chunks = clip_fill(t, pieces, n_pieces, at)) > 0) {
    hipLaunchKernelGGL(k_grad_scale, dim3((unsigned)clip_blocks(chunks, kClipScaleBlocks)),
                       dim3(kClipThreads), 0, (hipStream_t)stream, t, coef);
    PRL_CHECK_LAUNCH("grad_scale");
  }
  return PRL_OK;
}
