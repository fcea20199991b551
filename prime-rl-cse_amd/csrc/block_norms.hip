// The norm behind a block's branch, its gate and residual scale, the addition and the norm before the next block,
// forward and backward, over the rows of [rows, H] activations:
//     n = b r1 (w1 + o),    r1 = rsqrt(mean(b^2) + e1)        (w1 absent: n = b)
//     h = x + s g n                                            (gate g absent: 1; one value, per channel, per token, per element)
//     y = h r2 (w2 + o),    r2 = rsqrt(mean(h^2) + e2)         (w2 absent: y is not formed)
// and, with gh and gy the gradients of h and y, hh = h r2, bh = b r1:
//     G  = gh + r2 (gy (w2 + o) - hh mean(gy (w2 + o) hh))     gx = G
//     u  = s g G,    gb = r1 (u (w1 + o) - bh mean(u (w1 + o) bh))
//     gw1 = sum_rows u bh,    gw2 = sum_rows gy hh,    gg = s G n (summed over what the gate is broadcast over)
// Transformer layers with a norm on either side of a block spell this as some fifteen kernels forward and forty
// backward, twice per layer; layers with a plain addition run on k_rmsnorm_* (norm.hip), the counterpart of the
// reference's `model.impl = "liger_kernel"` (src/prime_rl/trainer/model.py:74-75).
//
// Everything between the loads and the stores is fp32; each output is rounded once.  y is formed from the unrounded
// h, and the backward forms h again from x and b rather than reading the rounded one: the same bytes, and no gradient
// sees that rounding.
//
// Bound by HBM.  A row stays in registers, EPT elements a thread, between the two sums it needs; the column sums of
// the weight gradients stay in registers over all rows a workgroup takes and leave it once.
#include <initializer_list>

#include "logprob_dev.h"

namespace prl {

constexpr int kBnMaxH = 8192;
constexpr int kBnMaxBlocks = 1024;  // backward: also the number of partial rows the finish adds up

typedef unsigned int bn_v_e2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int bn_v_e4 __attribute__((ext_vector_type(4), aligned(4)));

// The VE elements of unit v of a row of H; with AL every unit is whole and 16-byte aligned, otherwise the address is
// aligned to an element only and the last unit may be short (the rest reads as 0).
template <int DT, bool AL>
__device__ __forceinline__ void bn_load(const char* row, int v, int H, float* y) {
  constexpr int ES = DT == PRL_F32 ? 4 : 2, VE = 16 / ES;
  const char* p = row + (int64_t)v * 16;
  const int left = H - v * VE;
  if (AL || left >= VE) {
    u32x4 z;
    if constexpr (AL) z = *reinterpret_cast<const u32x4*>(p);
    else if constexpr (DT == PRL_F32) z = *reinterpret_cast<const bn_v_e4*>(p);
    else z = *reinterpret_cast<const bn_v_e2*>(p);
    decode16_raw<DT>(z, y);
    return;
  }
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    y[i] = 0.0f;
    if (i < left) y[i] = DT == PRL_F32 ? reinterpret_cast<const float*>(p)[i] : bf16_one(reinterpret_cast<const uint16_t*>(p)[i]);
  }
}
template <int DT, bool AL>
__device__ __forceinline__ void bn_store(char* row, int v, int H, const float* y) {
  constexpr int ES = DT == PRL_F32 ? 4 : 2, VE = 16 / ES;
  char* p = row + (int64_t)v * 16;
  const int left = H - v * VE;
  if (AL || left >= VE) {
    u32x4 z;
    if constexpr (DT == PRL_F32) {
      z.x = __float_as_uint(y[0]), z.y = __float_as_uint(y[1]), z.z = __float_as_uint(y[2]), z.w = __float_as_uint(y[3]);
    } else {
      z.x = pack_bf16(y[0], y[1]), z.y = pack_bf16(y[2], y[3]), z.z = pack_bf16(y[4], y[5]), z.w = pack_bf16(y[6], y[7]);
    }
    if constexpr (AL) *reinterpret_cast<u32x4*>(p) = z;
    else if constexpr (DT == PRL_F32) *reinterpret_cast<bn_v_e4*>(p) = z;
    else *reinterpret_cast<bn_v_e2*>(p) = z;
    return;
  }
#pragma unroll
  for (int i = 0; i < VE; ++i)
    if (i < left) store_elem<DT>(p, i, y[i]);
}

// Sum over the threads of a row: one wave, or the whole workgroup through `slots` (16 floats).  Two calls in turn
// with two sets of slots need one barrier each: a set is written again only after the other set's barrier, which
// every thread passes after its reads of the first.
template <bool ONEWAVE>
__device__ __forceinline__ float bn_row_sum(float v, float* slots) {
  v = wave_sum(v);
  if (ONEWAVE) return v;
  const int wid = threadIdx.x >> 6, nw = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) slots[wid] = v;
  __syncthreads();
  float r = slots[0];
  for (int i = 1; i < nw; ++i) r += slots[i];
  return r;
}

struct BnRows {  // base address and row pitch in bytes
  const char* p;
  int64_t pitch;
  __device__ __forceinline__ const char* row(int64_t r) const { return p + r * pitch; }
};
struct BnRowsOut {
  char* p;
  int64_t pitch;
  __device__ __forceinline__ char* row(int64_t r) const { return p + r * pitch; }
};

template <int DT>
__device__ __forceinline__ float bn_elem(const char* p) {
  return DT == PRL_F32 ? *reinterpret_cast<const float*>(p) : bf16_one(*reinterpret_cast<const uint16_t*>(p));
}

// ONEWAVE: a wave per row, blockDim / 64 rows at a time; otherwise a workgroup per row.
template <int DT, int NV, bool ONEWAVE, bool AL>
__global__ __launch_bounds__(ONEWAVE ? 256 : 1024) void k_block_norms_fwd(BnRows x, BnRows b, const char* __restrict__ w1,
                                                          const char* __restrict__ w2, int gate_kind, BnRows gate,
                                                          float scale, float offset, float eps1, float eps2,
                                                          BnRowsOut h, BnRowsOut y, float* __restrict__ rstd1,
                                                          float* __restrict__ rstd2, int64_t rows, int H) {
  constexpr int VE = DT == PRL_F32 ? 4 : 8;
  __shared__ float slots[2][16];
  const int tpr = ONEWAVE ? 64 : blockDim.x;
  const int li = ONEWAVE ? threadIdx.x & 63 : threadIdx.x;
  const int rpb = ONEWAVE ? blockDim.x >> 6 : 1;
  const int nvec = (H + VE - 1) / VE;
  const float inv_h = 1.0f / (float)H;
  for (int64_t row = (int64_t)blockIdx.x * rpb + (ONEWAVE ? threadIdx.x >> 6 : 0); row < rows;
       row += (int64_t)gridDim.x * rpb) {
    float bv[NV][VE], hv[NV][VE];
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = li + k * tpr;
#pragma unroll
      for (int i = 0; i < VE; ++i) bv[k][i] = hv[k][i] = 0.0f;
      if (v < nvec) {
        bn_load<DT, AL>(b.row(row), v, H, bv[k]);
        bn_load<DT, AL>(x.row(row), v, H, hv[k]);
      }
#pragma unroll
      for (int i = 0; i < VE; ++i) ss = fmaf(bv[k][i], bv[k][i], ss);
    }
    float r1 = 1.0f;
    if (w1) {
      r1 = rsqrtf(bn_row_sum<ONEWAVE>(ss, slots[0]) * inv_h + eps1);
      if (rstd1 && li == 0) rstd1[row] = r1;
    }
    float gs = scale;
    if (gate_kind == PRL_GATE_TOKEN || gate_kind == PRL_GATE_ONE) gs *= bn_elem<DT>(gate.row(row));
    ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = li + k * tpr;
      if (v < nvec) {
        float f[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) f[i] = gs * r1;
        if (w1) {
          float w[VE];
          bn_load<DT, AL>(w1, v, H, w);
#pragma unroll
          for (int i = 0; i < VE; ++i) f[i] *= w[i] + offset;
        }
        if (gate_kind == PRL_GATE_CHANNEL || gate_kind == PRL_GATE_FULL) {
          float g[VE];
          bn_load<DT, AL>(gate_kind == PRL_GATE_FULL ? gate.row(row) : gate.p, v, H, g);
#pragma unroll
          for (int i = 0; i < VE; ++i) f[i] *= g[i];
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) hv[k][i] = fmaf(f[i], bv[k][i], hv[k][i]);
        bn_store<DT, AL>(h.row(row), v, H, hv[k]);
      }
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (AL || v * VE + i < H) ss = fmaf(hv[k][i], hv[k][i], ss);
    }
    if (w2) {
      const float r2 = rsqrtf(bn_row_sum<ONEWAVE>(ss, slots[1]) * inv_h + eps2);
      if (rstd2 && li == 0) rstd2[row] = r2;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int v = li + k * tpr;
        if (v < nvec) {
          float w[VE];
          bn_load<DT, AL>(w2, v, H, w);
#pragma unroll
          for (int i = 0; i < VE; ++i) w[i] = (w[i] + offset) * (hv[k][i] * r2);
          bn_store<DT, AL>(y.row(row), v, H, w);
        }
      }
    }
    if (!ONEWAVE && !(w1 && w2)) __syncthreads();  // one set of slots only: it is written again by the next row
  }
}

// part[array][blockIdx.x][H]: arrays 0 gw1, 1 gw2, 2 a channel gate's gradient (for a gate of one value: [blockIdx.x]),
// each there only when asked for
template <int DT, int NV, bool ONEWAVE, bool AL>
__global__ __launch_bounds__(ONEWAVE ? 256 : 1024) void k_block_norms_bwd(
    BnRows x, BnRows b, const char* __restrict__ w1, const char* __restrict__ w2, int gate_kind, BnRows gate, float scale,
    float offset, const float* __restrict__ rstd1, const float* __restrict__ rstd2, BnRows gh, BnRows gy, BnRowsOut gx,
    BnRowsOut gb, float* __restrict__ part1, float* __restrict__ part2, float* __restrict__ partg, BnRowsOut gg,
    int64_t rows, int H) {
  constexpr int VE = DT == PRL_F32 ? 4 : 8;
  __shared__ float slots[3][16];
  extern __shared__ float lds[];  // ONEWAVE: rows of the workgroup x H
  const int tpr = ONEWAVE ? 64 : blockDim.x;
  const int li = ONEWAVE ? threadIdx.x & 63 : threadIdx.x;
  const int slot = ONEWAVE ? threadIdx.x >> 6 : 0;
  const int rpb = ONEWAVE ? blockDim.x >> 6 : 1;
  const int nvec = (H + VE - 1) / VE;
  const float inv_h = 1.0f / (float)H;
  float a1[NV][VE], a2[NV][VE], ag[NV][VE], aone = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VE; ++i) a1[k][i] = a2[k][i] = ag[k][i] = 0.0f;
  for (int64_t row = (int64_t)blockIdx.x * rpb + slot; row < rows; row += (int64_t)gridDim.x * rpb) {
    const float r1 = w1 ? rstd1[row] : 1.0f;
    const float r2 = w2 ? rstd2[row] : 0.0f;
    const float gt = gate_kind == PRL_GATE_TOKEN || gate_kind == PRL_GATE_ONE ? bn_elem<DT>(gate.row(row)) : 1.0f;
    float bh[NV][VE], hh[NV][VE], G[NV][VE], q[NV][VE];  // q: gy (w2 + o), later u (w1 + o)
    float dot = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = li + k * tpr;
#pragma unroll
      for (int i = 0; i < VE; ++i) bh[k][i] = hh[k][i] = G[k][i] = q[k][i] = 0.0f;
      if (v < nvec) {
        float t[VE], w[VE];
        bn_load<DT, AL>(b.row(row), v, H, bh[k]);
        if (w2) {
          bn_load<DT, AL>(x.row(row), v, H, hh[k]);
          bn_load<DT, AL>(gy.row(row), v, H, t);
#pragma unroll
          for (int i = 0; i < VE; ++i) w[i] = scale * gt * r1;
          if (w1) {
            float z[VE];
            bn_load<DT, AL>(w1, v, H, z);
#pragma unroll
            for (int i = 0; i < VE; ++i) w[i] *= z[i] + offset;
          }
          if (gate_kind == PRL_GATE_CHANNEL || gate_kind == PRL_GATE_FULL) {
            float z[VE];
            bn_load<DT, AL>(gate_kind == PRL_GATE_FULL ? gate.row(row) : gate.p, v, H, z);
#pragma unroll
            for (int i = 0; i < VE; ++i) w[i] *= z[i];
          }
#pragma unroll
          for (int i = 0; i < VE; ++i) hh[k][i] = fmaf(w[i], bh[k][i], hh[k][i]) * r2;
          bn_load<DT, AL>(w2, v, H, w);
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            if (part2) a2[k][i] = fmaf(t[i], hh[k][i], a2[k][i]);
            q[k][i] = t[i] * (w[i] + offset);
            if (AL || v * VE + i < H) dot = fmaf(q[k][i], hh[k][i], dot);
          }
        }
        if (gh.p) bn_load<DT, AL>(gh.row(row), v, H, G[k]);
#pragma unroll
        for (int i = 0; i < VE; ++i) bh[k][i] *= r1;
      }
    }
    if (w2) {
      dot = bn_row_sum<ONEWAVE>(dot, slots[0]) * inv_h;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) G[k][i] = fmaf(r2, q[k][i] - hh[k][i] * dot, G[k][i]);
    }
    dot = 0.0f;
    float gdot = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = li + k * tpr;
      if (v < nvec) {
        float w[VE], g[VE];
        bn_store<DT, AL>(gx.row(row), v, H, G[k]);
#pragma unroll
        for (int i = 0; i < VE; ++i) w[i] = 1.0f, g[i] = gt;
        if (w1) {
          bn_load<DT, AL>(w1, v, H, w);
#pragma unroll
          for (int i = 0; i < VE; ++i) w[i] += offset;
        }
        if (gate_kind == PRL_GATE_CHANNEL || gate_kind == PRL_GATE_FULL)
          bn_load<DT, AL>(gate_kind == PRL_GATE_FULL ? gate.row(row) : gate.p, v, H, g);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const bool in = AL || v * VE + i < H;
          const float gn = scale * G[k][i] * bh[k][i] * w[i];  // the gate's gradient
          const float u = scale * g[i] * G[k][i];
          if (part1) a1[k][i] = fmaf(u, bh[k][i], a1[k][i]);
          if (partg && gate_kind == PRL_GATE_CHANNEL) ag[k][i] += gn;
          if (in) gdot += gn;
          q[k][i] = u * w[i];
          if (in) dot = fmaf(q[k][i], bh[k][i], dot);
          w[i] = gn;
        }
        if (gate_kind == PRL_GATE_FULL && gg.p) bn_store<DT, AL>(gg.row(row), v, H, w);
      }
    }
    aone += gdot;
    if (gate_kind == PRL_GATE_TOKEN && gg.p) {
      gdot = bn_row_sum<ONEWAVE>(gdot, slots[2]);
      if (li == 0) store_elem<DT>(gg.row(row), 0, gdot);
    }
    dot = w1 ? bn_row_sum<ONEWAVE>(dot, slots[1]) * inv_h : 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = li + k * tpr;
      if (v < nvec) {
#pragma unroll
        for (int i = 0; i < VE; ++i) q[k][i] = r1 * (q[k][i] - bh[k][i] * dot);
        bn_store<DT, AL>(gb.row(row), v, H, q[k]);
      }
    }
    if (!ONEWAVE) __syncthreads();  // slots are written again by the next row
  }
  if (gate_kind == PRL_GATE_ONE && partg) {
    __syncthreads();
    aone = bn_row_sum<false>(aone, slots[2]);
    if (threadIdx.x == 0) partg[blockIdx.x] = aone;
  }
  float* const part[3] = {part1, part2, gate_kind == PRL_GATE_ONE ? nullptr : partg};
#pragma unroll
  for (int a = 0; a < 3; ++a) {
    if (!part[a]) continue;
    float(&acc)[NV][VE] = a == 0 ? a1 : a == 1 ? a2 : ag;
    float* out = part[a] + (int64_t)blockIdx.x * H;
    if (ONEWAVE) __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int c = (li + k * tpr) * VE + i;
        if (c < H) (ONEWAVE ? lds + slot * H : out)[c] = acc[k][i];
      }
    if (ONEWAVE) {
      __syncthreads();
      for (int c = threadIdx.x; c < H; c += blockDim.x) {
        float s = lds[c];
        for (int r = 1; r < rpb; ++r) s += lds[r * H + c];
        out[c] = s;
      }
    }
  }
}

// out[a][c] = sum over the partial rows of part[a][p][c], in a fixed order; 32 columns a workgroup, 32 groups of
// threads over the rows.
template <int DT>
__global__ __launch_bounds__(1024) void k_block_norms_finish(const float* p0, const float* p1, const float* p2, char* o0,
                                                             char* o1, char* o2, int nparts, int H, int Hg) {
  const float* part = blockIdx.y == 0 ? p0 : blockIdx.y == 1 ? p1 : p2;
  char* out = blockIdx.y == 0 ? o0 : blockIdx.y == 1 ? o1 : o2;
  if (blockIdx.y == 2) H = Hg;  // a gate of one value has one column
  if (!part || (int)blockIdx.x * 32 >= H) return;
  __shared__ float lds[32][33];
  const int lc = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lc;
  float s = 0.0f;
  if (c < H)
    for (int p = g; p < nparts; p += 32) s += part[(int64_t)p * H + c];
  lds[g][lc] = s;
  __syncthreads();
  if (g == 0 && c < H) {
    float t = lds[0][lc];
#pragma unroll
    for (int k = 1; k < 32; ++k) t += lds[k][lc];
    store_elem<DT>(out, c, t);
  }
}

// Threads of a row and units a thread: one wave while a row has at most 128 units, else as many waves as give each
// thread one unit of bf16 or two of fp32 (8 elements).
struct BnShape {
  bool onewave;
  int nv, threads, rpb;
};
static BnShape bn_shape(int dtype, int64_t H) {
  const int ve = dtype == PRL_F32 ? 4 : 8;
  const int64_t nvec = (H + ve - 1) / ve;
  if (nvec <= 64) return {true, 1, 256, 4};
  if (nvec <= 128) return {true, 2, 256, 4};
  const int nv = dtype == PRL_F32 ? 2 : 1;
  return {false, nv, (int)(((nvec + nv - 1) / nv + 63) / 64 * 64), 1};
}
static int bn_blocks(int64_t rows, int rpb, int cap) {
  const int64_t want = (rows + rpb - 1) / rpb;
  return (int)(want < cap ? (want > 0 ? want : 1) : cap);
}

}  // namespace prl

using namespace prl;

extern "C" int prl_block_norms_supported(int dtype, int64_t H) {
  return (dtype == PRL_F32 || dtype == PRL_BF16) && H >= 1 && H <= kBnMaxH ? 1 : 0;
}

extern "C" size_t prl_block_norms_bwd_workspace_bytes(int dtype, int64_t rows, int64_t H) {
  if (!prl_block_norms_supported(dtype, H) || rows < 0) return 0;
  return (size_t)3 * bn_blocks(rows, bn_shape(dtype, H).rpb, kBnMaxBlocks) * (size_t)H * sizeof(float);
}

static bool bn_aligned(int es, int64_t H, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
  uintptr_t bits = (uintptr_t)(H * es);
  for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p);
  for (int64_t s : strides) bits |= (uintptr_t)(s * es);
  return (bits & 15) == 0;
}

static int bn_check(const char* who, int dtype, int64_t rows, int64_t H, int gate_kind, const void* gate,
                    std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> out_strides) {
  PRL_REQUIRE(rows >= 0, "%s: rows must be >= 0", who);
  PRL_REQUIRE(prl_block_norms_supported(dtype, H), "%s: unsupported dtype %d or row length %lld (1 .. %d)", who, dtype,
              (long long)H, kBnMaxH);
  PRL_REQUIRE(gate_kind >= PRL_GATE_NONE && gate_kind <= PRL_GATE_ONE, "%s: unknown gate kind %d", who, gate_kind);
  PRL_REQUIRE(rows == 0 || gate_kind == PRL_GATE_NONE || gate, "%s: gate must not be NULL", who);
  const uintptr_t es = dtype == PRL_F32 ? 4 : 2;
  for (const void* p : ptrs)
    PRL_REQUIRE((reinterpret_cast<uintptr_t>(p) & (es - 1)) == 0, "%s: pointers must be aligned to an element", who);
  for (int64_t s : out_strides) PRL_REQUIRE(s >= H, "%s: output row strides must be >= H", who);
  return PRL_OK;
}

#define PRL_BN_DISPATCH(KERNEL)                                                   \
  do {                                                                            \
    if (dtype == PRL_BF16) {                                                      \
      if (!sh.onewave) { if (al) KERNEL(PRL_BF16, 1, false, true); else KERNEL(PRL_BF16, 1, false, false); }   \
      else if (sh.nv == 1) { if (al) KERNEL(PRL_BF16, 1, true, true); else KERNEL(PRL_BF16, 1, true, false); } \
      else { if (al) KERNEL(PRL_BF16, 2, true, true); else KERNEL(PRL_BF16, 2, true, false); }                 \
    } else {                                                                      \
      if (!sh.onewave) { if (al) KERNEL(PRL_F32, 2, false, true); else KERNEL(PRL_F32, 2, false, false); }     \
      else if (sh.nv == 1) { if (al) KERNEL(PRL_F32, 1, true, true); else KERNEL(PRL_F32, 1, true, false); }   \
      else { if (al) KERNEL(PRL_F32, 2, true, true); else KERNEL(PRL_F32, 2, true, false); }                   \
    }                                                                             \
  } while (0)

extern "C" int prl_block_norms_fwd(const void* x, int64_t x_stride, const void* branch, int64_t branch_stride,
                                   const void* w_post, const void* w_pre, int gate_kind, const void* gate,
                                   int64_t gate_stride, float scale, float weight_offset, float eps_post, float eps_pre,
                                   void* hidden, int64_t hidden_stride, void* normed, int64_t normed_stride,
                                   float* rstd_post, float* rstd_pre, int dtype, int64_t rows, int64_t H, void* stream) {
  clear_error();
  const int64_t n_stride = w_pre ? normed_stride : H;
  int rc = bn_check("block_norms_fwd", dtype, rows, H, gate_kind, gate, {x, branch, w_post, w_pre, gate, hidden, normed},
                    {hidden_stride, n_stride});
  if (rc != PRL_OK) return rc;
  if (rows == 0) return PRL_OK;
  PRL_REQUIRE(x && branch && hidden && (!w_pre || normed),
              "block_norms_fwd: x, branch, hidden (and normed, with w_pre) must not be NULL");
  const int64_t es = dtype == PRL_F32 ? 4 : 2;
  const bool narrow = gate_kind == PRL_GATE_TOKEN || gate_kind == PRL_GATE_ONE;
  const int64_t gate_pitch = gate_kind == PRL_GATE_ONE ? 0 : gate_stride * es;
  const bool al = bn_aligned((int)es, H, {x, branch, w_post, w_pre, hidden, w_pre ? normed : nullptr,
                                          narrow ? nullptr : gate},
                             {x_stride, branch_stride, hidden_stride, n_stride,
                              gate_kind == PRL_GATE_FULL ? gate_stride : 0});
  const BnShape sh = bn_shape(dtype, H);
  const dim3 grid((unsigned)bn_blocks(rows, sh.rpb, 1 << 20)), block((unsigned)sh.threads);
#define PRL_BN_FWD(DT, NV, OW, AL)                                                                                   \
  hipLaunchKernelGGL((k_block_norms_fwd<DT, NV, OW, AL>), grid, block, 0, (hipStream_t)stream,                       \
                     (BnRows{(const char*)x, x_stride * es}), (BnRows{(const char*)branch, branch_stride * es}),      \
                     (const char*)w_post, (const char*)w_pre, gate_kind, (BnRows{(const char*)gate, gate_pitch}), \
                     scale, weight_offset, eps_post, eps_pre, (BnRowsOut{(char*)hidden, hidden_stride * es}),         \
                     (BnRowsOut{(char*)normed, n_stride * es}), rstd_post, rstd_pre, rows, (int)H)
  PRL_BN_DISPATCH(PRL_BN_FWD);
#undef PRL_BN_FWD
  PRL_CHECK_LAUNCH("block_norms_fwd");
  return PRL_OK;
}

extern "C" int prl_block_norms_bwd(const void* x, int64_t x_stride, const void* branch, int64_t branch_stride,
                                   const void* w_post, const void* w_pre, int gate_kind, const void* gate,
                                   int64_t gate_stride, float scale, float weight_offset, const float* rstd_post,
                                   const float* rstd_pre, const void* g_hidden, int64_t g_hidden_stride,
                                   const void* g_normed, int64_t g_normed_stride, void* gx, int64_t gx_stride,
                                   void* g_branch, int64_t g_branch_stride, void* g_w_post, void* g_w_pre, void* g_gate,
                                   int64_t g_gate_stride, int dtype, int64_t rows, int64_t H, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  clear_error();
  int rc = bn_check("block_norms_bwd", dtype, rows, H, gate_kind, gate,
                    {x, branch, w_post, w_pre, gate, g_hidden, g_normed, gx, g_branch, g_w_post, g_w_pre, g_gate},
                    {gx_stride, g_branch_stride, gate_kind == PRL_GATE_FULL && g_gate ? g_gate_stride : H});
  if (rc != PRL_OK) return rc;
  PRL_REQUIRE(gate_kind != PRL_GATE_TOKEN || !g_gate || g_gate_stride >= 1,
              "block_norms_bwd: the row stride of a token gate's gradient must be >= 1");
  PRL_REQUIRE(!g_w_post || w_post, "block_norms_bwd: g_w_post without w_post");
  PRL_REQUIRE(!g_w_pre || w_pre, "block_norms_bwd: g_w_pre without w_pre");
  PRL_REQUIRE(!g_gate || gate_kind != PRL_GATE_NONE, "block_norms_bwd: g_gate without a gate");
  PRL_REQUIRE(rows == 0 || (x && branch && gx && g_branch && (!w_post || rstd_post) && (!w_pre || rstd_pre) &&
                            (!w_pre == !g_normed)),
              "block_norms_bwd: x, branch, gx, g_branch and (with their weights) rstd_post, rstd_pre, g_normed must not be "
              "NULL; g_normed goes with w_pre");
  const BnShape sh = bn_shape(dtype, H);
  const int nblk = bn_blocks(rows, sh.rpb, kBnMaxBlocks);
  const size_t one = (size_t)nblk * H, need = 3 * one * sizeof(float);
  const bool channel = (gate_kind == PRL_GATE_CHANNEL || gate_kind == PRL_GATE_ONE) && g_gate;
  const bool sums = g_w_post || g_w_pre || channel;
  PRL_REQUIRE(!sums || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
              "block_norms_bwd: 16-byte aligned workspace of %zu bytes needed (prl_block_norms_bwd_workspace_bytes)", need);
  float* ws = (float*)workspace;
  float *p1 = g_w_post ? ws : nullptr, *p2 = g_w_pre ? ws + one : nullptr, *pg = channel ? ws + 2 * one : nullptr;
  const int64_t es = dtype == PRL_F32 ? 4 : 2;
  hipStream_t st = (hipStream_t)stream;
  // rows == 0: the kernel runs with no row and leaves sums of zero
  const bool full = gate_kind == PRL_GATE_FULL, narrow = gate_kind == PRL_GATE_TOKEN || gate_kind == PRL_GATE_ONE;
  const bool al = bn_aligned((int)es, H,
                             {x, branch, w_post, w_pre, g_hidden, g_normed, gx, g_branch,
                              narrow ? nullptr : gate, full ? g_gate : nullptr},
                             {x_stride, branch_stride, g_hidden ? g_hidden_stride : 0, g_normed ? g_normed_stride : 0,
                              gx_stride, g_branch_stride, full ? gate_stride : 0, full && g_gate ? g_gate_stride : 0});
  const int64_t gate_pitch = gate_kind == PRL_GATE_ONE ? 0 : gate_stride * es;
  const dim3 grid((unsigned)nblk), block((unsigned)sh.threads);
  const size_t lds = sh.onewave ? (size_t)sh.rpb * H * sizeof(float) : 0;
  char* gg = channel || !g_gate ? nullptr : (char*)g_gate;
#define PRL_BN_BWD(DT, NV, OW, AL)                                                                                    \
  hipLaunchKernelGGL((k_block_norms_bwd<DT, NV, OW, AL>), grid, block, lds, st, (BnRows{(const char*)x, x_stride * es}), \
                     (BnRows{(const char*)branch, branch_stride * es}), (const char*)w_post, (const char*)w_pre, gate_kind, \
                     (BnRows{(const char*)gate, gate_pitch}), scale, weight_offset, rstd_post, rstd_pre,         \
                     (BnRows{(const char*)g_hidden, g_hidden_stride * es}),                                           \
                     (BnRows{(const char*)g_normed, g_normed_stride * es}), (BnRowsOut{(char*)gx, gx_stride * es}),    \
                     (BnRowsOut{(char*)g_branch, g_branch_stride * es}), p1, p2, pg, (BnRowsOut{gg, g_gate_stride * es}), \
                     rows, (int)H)
  PRL_BN_DISPATCH(PRL_BN_BWD);
#undef PRL_BN_BWD
  PRL_CHECK_LAUNCH("block_norms_bwd");
  if (!sums) return PRL_OK;
  const dim3 fgrid((unsigned)((H + 31) / 32), 3);
  if (dtype == PRL_BF16)
    hipLaunchKernelGGL((k_block_norms_finish<PRL_BF16>), fgrid, dim3(1024), 0, st, p1, p2, pg, (char*)g_w_post,
                       (char*)g_w_pre, (char*)g_gate, nblk, (int)H, gate_kind == PRL_GATE_ONE ? 1 : (int)H);
  else
    hipLaunchKernelGGL((k_block_norms_finish<PRL_F32>), fgrid, dim3(1024), 0, st, p1, p2, pg, (char*)g_w_post,
                       (char*)g_w_pre, (char*)g_gate, nblk, (int)H, gate_kind == PRL_GATE_ONE ? 1 : (int)H);
  PRL_CHECK_LAUNCH("block_norms_bwd");
  return PRL_OK;
}
