// The global norm of many gradient tensors, and their clipping, as torch.nn.utils.clip_grad_norm_ does it for the
// reference (src/prime_rl/trainer/rl/train.py:336-338):
//     N = sqrt(sum g^2)  or  max |g|,    c = min(1, max_norm / (N + 1e-6)),    g <- g c
// Two passes over the gradients with a small finish between them; where c is exactly 1 the second returns at once.
//
// The tensors' addresses and lengths travel in the launch itself, up to kClipPieces of them each: nothing is copied to
// the device, the calls are legal under stream capture, and no table outlives them.  Pieces are cut into chunks; a
// workgroup takes a run of consecutive chunks.  Squares are formed and added in fp64: no overflow for any fp32
// gradient, and the order of the sums is fixed by the sizes alone.
#include "prl_common.h"

namespace prl {

constexpr int kClipThreads = 256;
constexpr int kClipPieces = 160;   // 24 bytes each: a launch's arguments stay below 4 KB
constexpr int kClipChunk = 8192;   // elements
constexpr int kClipMaxBlocks = 2048;

struct ClipTable {
  char* x[kClipPieces];
  int64_t n[kClipPieces];             // elements
  uint32_t end[kClipPieces];          // chunks up to and including this piece
  uint8_t f32[kClipPieces];
  int32_t pieces;
};
static_assert(sizeof(ClipTable) <= 3600, "the launch's arguments have to stay below 4 KB");

// Calls f(address, elements, is fp32) for the chunks [c0, c1) of the table, in order.
template <typename F>
__device__ __forceinline__ void clip_walk(const ClipTable& t, uint32_t c0, uint32_t c1, F f) {
  int lo = 0, hi = t.pieces - 1;  // the piece that chunk c0 lies in: the first whose end is beyond it
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (t.end[mid] > c0) hi = mid; else lo = mid + 1;
  }
  int p = lo;
  for (uint32_t c = c0; c < c1; ++c) {
    while (t.end[p] <= c) ++p;
    const uint32_t first = p ? t.end[p - 1] : 0;
    const int64_t at = (int64_t)(c - first) * kClipChunk;
    const int64_t left = t.n[p] - at;
    const int es = t.f32[p] ? 4 : 2;
    f(t.x[p] + at * es, (int)(left < kClipChunk ? left : kClipChunk), t.f32[p] != 0);
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
  for (int i = threadIdx.x; i < nvec; i += kClipThreads) {
    const u32x4 z = v[i];
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
  }
  const int rest = n - nvec * VE;  // head + tail: fewer than 2 VE
  if ((int)threadIdx.x < rest) {
    const int i = (int)threadIdx.x < head ? threadIdx.x : threadIdx.x + nvec * VE;
    s = clip_take<MAX>(s, F32 ? reinterpret_cast<const float*>(x)[i] : bf16_one(reinterpret_cast<const uint16_t*>(x)[i]));
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
  const uint64_t chunks = t.end[t.pieces - 1];
  const uint32_t c0 = (uint32_t)(chunks * blockIdx.x / gridDim.x), c1 = (uint32_t)(chunks * (blockIdx.x + 1) / gridDim.x);
  double s = 0.0;
  clip_walk(t, c0, c1, [&](const char* x, int n, bool f32) {
    s = f32 ? clip_chunk_sum<true, MAX>(x, n, s) : clip_chunk_sum<false, MAX>(x, n, s);
  });
  s = clip_block_join<MAX>(s, slots);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// total = the joined partial values (sum of squares, or largest magnitude), and from it the norm and the factor.
template <bool MAX>
__global__ __launch_bounds__(1024) void k_grad_norm_finish(const double* part, int nparts, double* total, float max_norm,
                                                           float* norm, float* coef) {
  __shared__ double slots[16];
  double s = 0.0;
  for (int i = threadIdx.x; i < nparts; i += blockDim.x) s = clip_join<MAX>(s, part[i]);
  s = clip_block_join<MAX>(s, slots);
  if (threadIdx.x != 0) return;
  if (total) *total = s;
  const float n = (float)(MAX ? s : sqrt(s));
  if (norm) *norm = n;
  // min(1, .) that lets a NaN through: with a norm that is not a number every gradient becomes one, as torch's
  // clamp makes it; with an infinite norm the factor is 0
  const float c = max_norm / (n + 1e-6f);
  if (coef) *coef = c > 1.0f ? 1.0f : c;
}

template <bool F32>
__device__ __forceinline__ void clip_chunk_scale(char* x, int n, float c) {
  constexpr int ES = F32 ? 4 : 2, VE = 16 / ES;
  int head = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / ES);
  if (head > n) head = n;
  const int nvec = (n - head) / VE;
  u32x4* v = reinterpret_cast<u32x4*>(x + head * ES);
  for (int i = threadIdx.x; i < nvec; i += kClipThreads) {
    u32x4 z = v[i];
    uint32_t w[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = F32 ? __float_as_uint(__uint_as_float(w[j]) * c) : pack_bf16(bf16_lo(w[j]) * c, bf16_hi(w[j]) * c);
    z.x = w[0], z.y = w[1], z.z = w[2], z.w = w[3];
    v[i] = z;
  }
  const int rest = n - nvec * VE;
  if ((int)threadIdx.x < rest) {
    const int i = (int)threadIdx.x < head ? threadIdx.x : threadIdx.x + nvec * VE;
    if (F32) reinterpret_cast<float*>(x)[i] *= c;
    else reinterpret_cast<uint16_t*>(x)[i] = one_bf16(bf16_one(reinterpret_cast<const uint16_t*>(x)[i]) * c);
  }
}

__global__ __launch_bounds__(kClipThreads) void k_grad_scale(const ClipTable t, const float* __restrict__ coef) {
  const float c = *coef;
  if (c == 1.0f) return;
  const uint64_t chunks = t.end[t.pieces - 1];
  const uint32_t c0 = (uint32_t)(chunks * blockIdx.x / gridDim.x), c1 = (uint32_t)(chunks * (blockIdx.x + 1) / gridDim.x);
  clip_walk(t, c0, c1, [&](char* x, int n, bool f32) {
    if (f32) clip_chunk_scale<true>(x, n, c);
    else clip_chunk_scale<false>(x, n, c);
  });
}

static int64_t clip_chunks(int64_t n) { return (n + kClipChunk - 1) / kClipChunk; }
static int clip_blocks(int64_t chunks) { return (int)(chunks < kClipMaxBlocks ? chunks : kClipMaxBlocks); }

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
  while ((c = clip_fill(t, pieces, n_pieces, at)) > 0) total += clip_blocks(c);
  return total;
}

}  // namespace prl

using namespace prl;

extern "C" size_t prl_grad_norm_workspace_bytes(const prl_grad_piece* pieces, int64_t n_pieces) {
  if (clip_check("grad_norm_workspace_bytes", pieces, n_pieces) != PRL_OK) return 0;
  const int64_t n = clip_partials(pieces, n_pieces);
  return (size_t)(n > 0 ? n : 1) * sizeof(double);
}

extern "C" int prl_grad_norm(const prl_grad_piece* pieces, int64_t n_pieces, int kind, float max_norm, double* total,
                             float* norm, float* coef, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  int rc = clip_check("grad_norm", pieces, n_pieces);
  if (rc != PRL_OK) return rc;
  PRL_REQUIRE(kind == PRL_NORM_L2 || kind == PRL_NORM_MAX, "grad_norm: unknown norm kind %d", kind);
  PRL_REQUIRE(total || norm || coef, "grad_norm: nothing asked for");
  const int64_t need = clip_partials(pieces, n_pieces);
  PRL_REQUIRE(need == 0 || (workspace && workspace_bytes >= (size_t)need * sizeof(double) &&
                            (reinterpret_cast<uintptr_t>(workspace) & 7) == 0),
              "grad_norm: 8-byte aligned workspace of %lld bytes needed (prl_grad_norm_workspace_bytes)",
              (long long)need * 8);
  PRL_REQUIRE(need <= 0x7fffffff, "grad_norm: too many pieces");
  hipStream_t st = (hipStream_t)stream;
  double* part = (double*)workspace;
  int64_t at = 0, chunks, done = 0;
  ClipTable t;
  while ((chunks = clip_fill(t, pieces, n_pieces, at)) > 0) {
    const dim3 grid((unsigned)clip_blocks(chunks)), block(kClipThreads);
    if (kind == PRL_NORM_MAX) hipLaunchKernelGGL((k_grad_norm<true>), grid, block, 0, st, t, part + done);
    else hipLaunchKernelGGL((k_grad_norm<false>), grid, block, 0, st, t, part + done);
    PRL_CHECK_LAUNCH("grad_norm");
    done += grid.x;
  }
  return prl_grad_norm_finish(part, done, kind, max_norm, total, norm, coef, stream);
}

extern "C" int prl_grad_norm_finish(const double* parts, int64_t n_parts, int kind, float max_norm, double* total,
                                    float* norm, float* coef, void* stream) {
  clear_error();
  PRL_REQUIRE(n_parts >= 0 && n_parts <= 0x7fffffff && (n_parts == 0 || parts), "grad_norm_finish: bad partial values");
  PRL_REQUIRE(kind == PRL_NORM_L2 || kind == PRL_NORM_MAX, "grad_norm_finish: unknown norm kind %d", kind);
  const dim3 block(n_parts <= 256 ? 256 : 1024);
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
    hipLaunchKernelGGL(k_grad_scale, dim3((unsigned)clip_blocks(chunks)), dim3(kClipThreads), 0, (hipStream_t)stream, t, coef);
    PRL_CHECK_LAUNCH("grad_scale");
  }
  return PRL_OK;
}
