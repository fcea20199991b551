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
// Bound by HBM: 8192 rows of 5120 bf16 with a gate per channel take 62 us forward (336 MB, 5.4 TB/s) and 103 backward
// with its finish (503 MB, 4.9 TB/s), 16384 rows of 1024 without a gate 26 and 44 us.  A row stays in registers, four to
// sixteen elements a thread, between the two sums it needs; the column sums of the weight gradients stay in registers
// over all rows a workgroup takes and leave it once.
#include <initializer_list>

#include "logprob_dev.h"

namespace prl {

constexpr int kBnMaxH = 8192;
constexpr int kBnStream = 2;              // non-temporal
constexpr int kBnNoLoads = 0x0f70;        // s_waitcnt vmcnt(0), the other counters free
constexpr int kBnRsrcFlags = 0x00020000;  // raw buffer, 32-bit data format (gfx9 family descriptor word 3)

// A thread reads its share of a row in units of four registers.  VEC: a unit is 16 consecutive bytes, unit v at
// 16 v, for rows whose every unit is whole and aligned.  Otherwise it is four single elements, `tpr` apart, so that a
// wave's accesses lie side by side whatever the row's alignment: 16-byte accesses at odd places ran at half the
// rate (8192 rows of 1531 bf16, a gate per element: forward 45.0 us against 31.8, backward 82.6 against 53.4).
// Vector loads go past the caches and stores stay in them, for the kernel that reads them next.  Cold inputs and outputs,
// no gate; neither past the caches, loads only, both:
//     8192 rows of 5120 bf16, forward alone   63.7   63.0   57.3 us      its backward alone          101.2   97.0   89.8
//     one input just written, result read      132.9  113.5  116.6                                   173.4  145.2  148.4
//     16384 rows of 1024, the same forward     50.6   50.1   52.4        backward                     67.9   65.9   69.4
//     2051 rows of 1536                        15.2   15.1   14.6                                     23.1   23.0   23.4
// Single elements are read through the caches (8192 rows of 1531, a gate per element: 31.4 us against 34.0 past them).
// Rows are read through descriptors of exactly their bytes: lanes beyond the end, and every lane of a tensor that is
// not there, read 0 and store nothing, without a branch.
template <int DT, bool VEC>
struct BnUnit {
  static constexpr int kEs = DT == PRL_F32 ? 4 : 2;
  static constexpr int kN = VEC ? 16 / kEs : 4;  // elements
  // column of element i of unit k of thread li
  static __device__ __forceinline__ int column(int k, int i, int li, int tpr) {
    return VEC ? (li + k * tpr) * kN + i : li + (k * kN + i) * tpr;
  }
  template <int AUX = VEC ? kBnStream : 0>
  static __device__ __forceinline__ u32x4 load(const char* row, int bytes, int k, int li, int tpr) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(row), 0, bytes, kBnRsrcFlags);
    if constexpr (VEC) return __builtin_amdgcn_raw_buffer_load_b128(rsrc, (li + k * tpr) * 16, 0, AUX);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = column(k, i, li, tpr) * kEs;
      if constexpr (DT == PRL_F32) w[i] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, at, 0, 0);
      else w[i] = __builtin_amdgcn_raw_buffer_load_b16(rsrc, at, 0, 0);
    }
    u32x4 z;
    z.x = w[0], z.y = w[1], z.z = w[2], z.w = w[3];
    return z;
  }
  static __device__ __forceinline__ void decode(const u32x4& z, float* y) {
    if constexpr (VEC || DT == PRL_F32) {
      decode16_raw<DT>(z, y);
    } else {
      y[0] = bf16_lo(z.x), y[1] = bf16_lo(z.y), y[2] = bf16_lo(z.z), y[3] = bf16_lo(z.w);
    }
  }
  static __device__ __forceinline__ void store(char* row, int k, int li, int tpr, int H, const float* y) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(row, 0, H * kEs, kBnRsrcFlags);
    if constexpr (VEC) {
      u32x4 z;
      if constexpr (DT == PRL_F32) {
        z.x = __float_as_uint(y[0]), z.y = __float_as_uint(y[1]), z.z = __float_as_uint(y[2]), z.w = __float_as_uint(y[3]);
      } else {
        z.x = pack_bf16(y[0], y[1]), z.y = pack_bf16(y[2], y[3]), z.z = pack_bf16(y[4], y[5]), z.w = pack_bf16(y[6], y[7]);
      }
      __builtin_amdgcn_raw_buffer_store_b128(z, rsrc, (li + k * tpr) * 16, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = column(k, i, li, tpr) * kEs;
        if constexpr (DT == PRL_F32) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y[i]), rsrc, at, 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b16(one_bf16(y[i]), rsrc, at, 0, 0);
      }
    }
  }
};

// Sum over a wave in six vector adds whose second operand comes from another lane (no trip through LDS): neighbours,
// pairs, halves of a row of 16 lanes, the row's mirror, then each row's last lane on to the next rows.  Lane 63 has
// the total; it is read back as a scalar.
template <int CTRL, int ROWS>
__device__ __forceinline__ float bn_lane_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ float bn_wave_sum(float v) {
  v = bn_lane_add<0xb1, 0xf>(v);   // quad_perm [1, 0, 3, 2]
  v = bn_lane_add<0x4e, 0xf>(v);   // quad_perm [2, 3, 0, 1]
  v = bn_lane_add<0x141, 0xf>(v);  // row_half_mirror
  v = bn_lane_add<0x140, 0xf>(v);  // row_mirror
  v = bn_lane_add<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  v = bn_lane_add<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// A barrier that orders LDS only: loads of the next row stay in flight across it.
__device__ __forceinline__ void bn_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Sum over the threads of a row: one wave, or the whole workgroup through `slots` (16 floats).  Two calls in turn
// with two sets of slots need one barrier each: a set is written again only after the other set's barrier, which
// every thread passes after its reads of the first.
template <bool ONEWAVE>
__device__ __forceinline__ float bn_row_sum(float v, float* slots) {
  v = bn_wave_sum(v);
  if (ONEWAVE) return v;
  const int wid = threadIdx.x >> 6, nw = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) slots[wid] = v;
  bn_barrier();
  float r = slots[0];
  for (int i = 1; i < nw; ++i) r += slots[i];
  return r;
}

// Floats from one partial row to the next: whole cache lines.
__host__ __device__ __forceinline__ int64_t bn_part_pitch(int64_t H) { return (H + 31) / 32 * 32; }

struct BnRows {  // base address, row pitch and bytes of a row (0 for a tensor that is not there)
  const char* p;
  int64_t pitch;
  int bytes;
  __device__ __forceinline__ const char* row(int64_t r) const { return p + r * pitch; }
};
static BnRows bn_rows(const void* p, int64_t stride, int64_t H, int64_t es) {
  return {(const char*)p, p ? stride * es : 0, p ? (int)(H * es) : 0};
}
struct BnRowsOut {
  char* p;
  int64_t pitch;
  __device__ __forceinline__ char* row(int64_t r) const { return p + r * pitch; }
};

template <int DT>
__device__ __forceinline__ float bn_elem(const char* p) {
  return DT == PRL_F32 ? *reinterpret_cast<const float*>(p) : bf16_one(*reinterpret_cast<const uint16_t*>(p));
}

// How the gate comes: not at all, as one value or one per row (GATE 0), one per channel (1, kept over the rows), one
// per element (2).
template <int NV, bool BWD, int GATE>
struct BnRow {  // what a thread reads of one row, as it lies in memory
  u32x4 x[NV], b[NV], gy[BWD ? NV : 1], gh[BWD ? NV : 1], g[GATE == 2 ? NV : 1];
  float r1, r2, gt;
};
struct BnIn {
  BnRows x, b, gy, gh, gate;
  const float *rstd1, *rstd2;
  const char *w1, *w2;
  int gate_kind;
};

template <int DT, int NV, bool BWD, int GATE, bool VEC>
__device__ __forceinline__ void bn_fetch(BnRow<NV, BWD, GATE>& r, const BnIn& in, int64_t row, int li, int tpr) {
  using U = BnUnit<DT, VEC>;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    r.b[k] = U::load(in.b.row(row), in.b.bytes, k, li, tpr);
    r.x[k] = U::load(in.x.row(row), in.x.bytes, k, li, tpr);
    if (BWD) r.gy[k] = U::load(in.gy.row(row), in.gy.bytes, k, li, tpr);
    if (BWD) r.gh[k] = U::load(in.gh.row(row), in.gh.bytes, k, li, tpr);
    if (GATE == 2) r.g[k] = U::load(in.gate.row(row), in.gate.bytes, k, li, tpr);
  }
  r.r1 = BWD && in.rstd1 ? in.rstd1[row] : 1.0f;
  r.r2 = BWD && in.rstd2 ? in.rstd2[row] : 0.0f;
  r.gt = GATE == 0 && in.gate_kind != PRL_GATE_NONE ? bn_elem<DT>(in.gate.row(row)) : 1.0f;
}

// What a thread reads once: its columns of the weights and of a gate per channel.
template <int DT, int NV, int GATE, bool VEC>
struct BnCols {
  using U = BnUnit<DT, VEC>;
  u32x4 w1[NV], w2[NV], g[GATE ? NV : 1];
  __device__ __forceinline__ void load(const BnIn& in, int li, int tpr, int H) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      w1[k] = U::template load<0>(in.w1, in.w1 ? H * U::kEs : 0, k, li, tpr);
      w2[k] = U::template load<0>(in.w2, in.w2 ? H * U::kEs : 0, k, li, tpr);
      if (GATE == 1) g[k] = U::template load<0>(in.gate.p, H * U::kEs, k, li, tpr);
    }
  }
  // Keeps them packed through the loop over rows: the compiler would unpack what does not change in front of it, into
  // twice the registers.
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      asm volatile("" : "+v"(w1[k]), "+v"(w2[k]));
      if (GATE == 1) asm volatile("" : "+v"(g[GATE ? k : 0]));
    }
  }
};

// Places beyond a row's end read as 0 and add 0 to every sum: they are not masked.  (Only a factor that is not finite
// makes them something else, and then the row's own values are not numbers either.)

// ONEWAVE: a wave per row, blockDim / 64 rows at a time; otherwise a workgroup per row.  The next row's loads go out
// as soon as this one's are unpacked and stay in flight while it is worked on.  BOTH: both weights are there.
template <int DT, int NV, bool ONEWAVE, int GATE, bool VEC, bool BOTH>
__global__ __launch_bounds__(ONEWAVE ? 256 : 1024) void k_block_norms_fwd(BnIn in, float scale, float offset, float eps1,
                                                                          float eps2, BnRowsOut h, BnRowsOut y,
                                                                          float* __restrict__ rstd1,
                                                                          float* __restrict__ rstd2, int64_t rows, int H) {
  using U = BnUnit<DT, VEC>;
  constexpr int VE = U::kN;
  const bool has1 = BOTH || in.w1 != nullptr, has2 = BOTH || in.w2 != nullptr;
  __shared__ float slots[2][16];
  const int tpr = ONEWAVE ? 64 : blockDim.x;
  const int li = ONEWAVE ? threadIdx.x & 63 : threadIdx.x;
  const float inv_h = 1.0f / (float)H;
  const int64_t step = (int64_t)gridDim.x * (ONEWAVE ? blockDim.x >> 6 : 1);
  int64_t row = (int64_t)blockIdx.x * (ONEWAVE ? blockDim.x >> 6 : 1) +
                (ONEWAVE ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  if (row >= rows) return;
  BnCols<DT, NV, GATE, VEC> w;
  BnRow<NV, false, GATE> cur;
  bn_fetch<DT, NV, false, GATE, VEC>(cur, in, row, li, tpr);
  w.load(in, li, tpr, H);
  __builtin_amdgcn_s_waitcnt(kBnNoLoads);  // (see k_block_norms_bwd)
  for (;;) {
    const int64_t next = row + step;
    w.keep();
    float hv[NV][VE], bv[NV][VE];
    float ss = 0.0f;
    if (GATE == 2) {
#pragma unroll
      for (int k = 0; k < NV; ++k) w.g[GATE ? k : 0] = cur.g[GATE == 2 ? k : 0];
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      U::decode(cur.b[k], bv[k]);
      U::decode(cur.x[k], hv[k]);
#pragma unroll
      for (int i = 0; i < VE; ++i) ss = fmaf(bv[k][i], bv[k][i], ss);
    }
    const float gt = cur.gt;
    if (next < rows) bn_fetch<DT, NV, false, GATE, VEC>(cur, in, next, li, tpr);
    float r1 = 1.0f;
    if (has1) {
      r1 = rsqrtf(bn_row_sum<ONEWAVE>(ss, slots[0]) * inv_h + eps1);
      if (rstd1 && li == 0) rstd1[row] = r1;
    }
    const float gs = scale * gt * r1;
    ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[VE], t[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) f[i] = gs;
      if (has1) {
        U::decode(w.w1[k], t);
#pragma unroll
        for (int i = 0; i < VE; ++i) f[i] *= t[i] + offset;
      }
      if (GATE) {
        U::decode(w.g[GATE ? k : 0], t);
#pragma unroll
        for (int i = 0; i < VE; ++i) f[i] *= t[i];
      }
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        hv[k][i] = fmaf(f[i], bv[k][i], hv[k][i]);
        ss = fmaf(hv[k][i], hv[k][i], ss);
      }
      U::store(h.row(row), k, li, tpr, H, hv[k]);
    }
    if (has2) {
      const float r2 = rsqrtf(bn_row_sum<ONEWAVE>(ss, slots[1]) * inv_h + eps2);
      if (rstd2 && li == 0) rstd2[row] = r2;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float t[VE];
        U::decode(w.w2[k], t);
#pragma unroll
        for (int i = 0; i < VE; ++i) t[i] = (t[i] + offset) * (hv[k][i] * r2);
        U::store(y.row(row), k, li, tpr, H, t);
      }
    }
    if (next >= rows) break;
    if (!ONEWAVE && !(has1 && has2)) bn_barrier();  // one set of slots only: it is written again by the next row
    row = next;
  }
}

// part[array][blockIdx.x][H]: arrays 0 gw1, 1 gw2, 2 a channel gate's gradient (for a gate of one value: [blockIdx.x]),
// each there only when asked for
template <int DT, int NV, bool ONEWAVE, int GATE, bool VEC, bool BOTH>
__global__ __launch_bounds__(ONEWAVE ? 256 : 1024) void k_block_norms_bwd(BnIn in, float scale, float offset, BnRowsOut gx,
                                                                          BnRowsOut gb, float* __restrict__ part1,
                                                                          float* __restrict__ part2,
                                                                          float* __restrict__ partg, BnRowsOut gg,
                                                                          int64_t rows, int H) {
  using U = BnUnit<DT, VEC>;
  constexpr int VE = U::kN;
  const bool has1 = BOTH || in.w1 != nullptr, has2 = BOTH || in.w2 != nullptr;
  __shared__ float slots[3][16];
  extern __shared__ float lds[];  // ONEWAVE: rows of the workgroup x H
  const int tpr = ONEWAVE ? 64 : blockDim.x;
  const int li = ONEWAVE ? threadIdx.x & 63 : threadIdx.x;
  const int slot = ONEWAVE ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int rpb = ONEWAVE ? blockDim.x >> 6 : 1;
  const float inv_h = 1.0f / (float)H;
  const int64_t step = (int64_t)gridDim.x * rpb;
  float a1[NV][VE], a2[NV][VE], ag[GATE == 1 ? NV : 1][VE], aone = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VE; ++i) a1[k][i] = a2[k][i] = ag[GATE == 1 ? k : 0][i] = 0.0f;
  int64_t row = (int64_t)blockIdx.x * rpb + slot;
  BnCols<DT, NV, GATE, VEC> w;
  BnRow<NV, true, GATE> cur;
  if (row < rows) bn_fetch<DT, NV, true, GATE, VEC>(cur, in, row, li, tpr);
  w.load(in, li, tpr, H);
  // Nothing outstanding on entry: the loop then waits for its own loads by their number and never for the stores
  // behind them.
  __builtin_amdgcn_s_waitcnt(kBnNoLoads);
  while (row < rows) {
    const int64_t next = row + step;
    w.keep();
    const float r1 = cur.r1, r2 = cur.r2, gt = cur.gt;
    float bh[NV][VE], hh[NV][VE], q[NV][VE];  // q: gy (w2 + o), then G, then G's share of the branch
    u32x4 ghr[NV];
    float dot = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      ghr[k] = cur.gh[k];
      if (GATE == 2) w.g[GATE ? k : 0] = cur.g[GATE == 2 ? k : 0];
      U::decode(cur.b[k], bh[k]);
#pragma unroll
      for (int i = 0; i < VE; ++i) bh[k][i] *= r1;
      if (has2) {
        float f[VE], t[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) f[i] = scale * gt;
        if (has1) {
          U::decode(w.w1[k], t);
#pragma unroll
          for (int i = 0; i < VE; ++i) f[i] *= t[i] + offset;
        }
        if (GATE) {
          U::decode(w.g[GATE ? k : 0], t);
#pragma unroll
          for (int i = 0; i < VE; ++i) f[i] *= t[i];
        }
        U::decode(cur.x[k], hh[k]);
        U::decode(cur.gy[k], t);
        U::decode(w.w2[k], q[k]);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          hh[k][i] = fmaf(f[i], bh[k][i], hh[k][i]) * r2;
          q[k][i] = t[i] * (q[k][i] + offset);
          a2[k][i] = fmaf(t[i], hh[k][i], a2[k][i]);
          dot = fmaf(q[k][i], hh[k][i], dot);
        }
      }
    }
    if (next < rows) bn_fetch<DT, NV, true, GATE, VEC>(cur, in, next, li, tpr);
    if (has2) dot = bn_row_sum<ONEWAVE>(dot, slots[0]) * inv_h;
    float dot1 = 0.0f, gdot = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float t[VE], v[VE];
      U::decode(ghr[k], t);
#pragma unroll
      for (int i = 0; i < VE; ++i) q[k][i] = has2 ? fmaf(r2, q[k][i] - hh[k][i] * dot, t[i]) : t[i];
      U::store(gx.row(row), k, li, tpr, H, q[k]);
#pragma unroll
      for (int i = 0; i < VE; ++i) v[i] = 1.0f, t[i] = gt;
      if (has1) {
        U::decode(w.w1[k], v);
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] += offset;
      }
      if (GATE) U::decode(w.g[GATE ? k : 0], t);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float s = scale * q[k][i];
        const float gn = s * bh[k][i] * v[i];  // the gate's gradient
        const float u = s * t[i];
        q[k][i] = u * v[i];
        a1[k][i] = fmaf(u, bh[k][i], a1[k][i]);
        if (GATE == 0) gdot += gn;
        if (GATE == 1) ag[GATE == 1 ? k : 0][i] += gn;
        dot1 = fmaf(q[k][i], bh[k][i], dot1);
        v[i] = gn;
      }
      if (GATE == 2 && gg.p) U::store(gg.row(row), k, li, tpr, H, v);
    }
    if (GATE == 0) {
      aone += gdot;
      if (gg.p) {
        gdot = bn_row_sum<ONEWAVE>(gdot, slots[2]);
        if (li == 0) store_elem<DT>(gg.row(row), 0, gdot);
      }
    }
    if (has1) dot1 = bn_row_sum<ONEWAVE>(dot1, slots[1]) * inv_h;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int i = 0; i < VE; ++i) q[k][i] = has1 ? r1 * (q[k][i] - bh[k][i] * dot1) : q[k][i];
      U::store(gb.row(row), k, li, tpr, H, q[k]);
    }
    if (!ONEWAVE && !(has1 && has2)) bn_barrier();  // a set of slots would be written again with no barrier between
    row = next;
  }
  if (GATE == 0 && partg) {
    __syncthreads();
    aone = bn_row_sum<false>(aone, slots[2]);
    if (threadIdx.x == 0) partg[blockIdx.x] = aone;
  }
  float* const part[3] = {part1, part2, GATE == 1 ? partg : nullptr};
#pragma unroll
  for (int a = 0; a < (GATE == 1 ? 3 : 2); ++a) {
    if (!part[a]) continue;
    float* out = part[a] + (int64_t)blockIdx.x * bn_part_pitch(H);
    if (ONEWAVE) __syncthreads();
    float* mine = ONEWAVE ? lds + slot * bn_part_pitch(H) : out;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const float* z = a == 0 ? a1[k] : a == 1 ? a2[k] : ag[GATE == 1 ? k : 0];
#pragma unroll
      for (int i = 0; i < VE; i += VEC ? 4 : 1) {
        const int c = U::column(k, i, li, tpr);
        if (c >= H) continue;
        if (VEC) *reinterpret_cast<float4*>(mine + c) = make_float4(z[i], z[i + 1], z[i + 2], z[i + 3]);
        else mine[c] = z[i];
      }
    }
    if (ONEWAVE) {
      __syncthreads();
      for (int c = threadIdx.x; c < H; c += blockDim.x) {
        float s = lds[c];
        for (int r = 1; r < rpb; ++r) s += lds[r * bn_part_pitch(H) + c];
        out[c] = s;
      }
    }
  }
}

// out[a][c] = sum over the partial rows of part[a][p][c], in a fixed order.  A workgroup owns 32 columns (whole cache
// lines); 32 groups of 8 threads take every 32nd row, four columns a thread, eight rows in flight.
template <int DT>
__global__ __launch_bounds__(256) void k_block_norms_finish(const float* p0, const float* p1, const float* p2, char* o0,
                                                            char* o1, char* o2, int nparts, int H, int gate_one) {
  const float* part = blockIdx.y == 0 ? p0 : blockIdx.y == 1 ? p1 : p2;
  char* out = blockIdx.y == 0 ? o0 : blockIdx.y == 1 ? o1 : o2;
  if (!part) return;
  __shared__ float lds[32][33];
  if (gate_one && blockIdx.y == 2) {  // one value from every workgroup
    if (blockIdx.x) return;
    float s = 0.0f;
    for (int i = threadIdx.x; i < nparts; i += 256) s += part[i];
    s = block_sum<4>(s, lds[0]);
    if (threadIdx.x == 0) store_elem<DT>(out, 0, s);
    return;
  }
  const int q = threadIdx.x & 7, g = threadIdx.x >> 3;
  const int64_t pitch = bn_part_pitch(H) / 4;
  const float4* at = reinterpret_cast<const float4*>(part) + blockIdx.x * 8 + q;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int p = g; p < nparts; p += 256) {
    float4 z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = p + 32 * j < nparts ? at[(p + 32 * j) * pitch] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < 8; ++j) s.x += z[j].x, s.y += z[j].y, s.z += z[j].z, s.w += z[j].w;
  }
  lds[g][4 * q] = s.x, lds[g][4 * q + 1] = s.y, lds[g][4 * q + 2] = s.z, lds[g][4 * q + 3] = s.w;
  __syncthreads();
  const int c = blockIdx.x * 32 + threadIdx.x;
  if (threadIdx.x < 32 && c < H) {
    float t = lds[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < 32; ++k) t += lds[k][threadIdx.x];
    store_elem<DT>(out, c, t);
  }
}

// Threads of a row and units a thread: one wave while a row has at most 128 units, else as many waves as give each
// thread one unit (two where that would be over 16 waves: fp32 and single elements beyond 4096).  The backward with two
// units does not fit 128 registers and spills in 17 of its forms, up to 74 registers: 4096 rows of 8192 fp32 take 149 us
// (5.4 TB/s; 8192 rows of 4096, without spills, 128 us, 6.3), 4096 rows of 8191 bf16 149 us (2.7).
struct BnShape {
  bool onewave;
  int nv, threads, rpb;
};
static BnShape bn_shape(int dtype, int64_t H, bool vec) {
  const int n = !vec || dtype == PRL_F32 ? 4 : 8;
  const int64_t units = (H + n - 1) / n;
  if (units <= 64) return {true, 1, 256, 4};
  if (units <= 128) return {true, 2, 256, 4};
  const int nv = units > 1024 ? 2 : 1;
  return {false, nv, (int)(((units + nv - 1) / nv + 63) / 64 * 64), 1};
}
static int bn_blocks(int64_t rows, int rpb, int cap) {
  const int64_t want = (rows + rpb - 1) / rpb;
  return (int)(want < cap ? (want > 0 ? want : 1) : cap);
}

// Forward: rows of one wave each have their own; of wider rows few workgroups take many, and fetch the next row while
// they wait for this one's sums (8192 rows of 5120 bf16: 62.1 us with 256 workgroups, 74.6 with one per row; 8192 rows of
// 1531: 30.7 against 33.4; 16384 rows of 2048: 53.3 against 52.8).
static int bn_fwd_blocks(int64_t rows, const BnShape& sh) {
  const int waves = sh.threads / 64;
  return bn_blocks(rows, sh.rpb, sh.onewave ? 1 << 20 : 256 * (waves < 16 ? 16 / waves : 1));
}
// Backward: every workgroup leaves a partial row per weight, so as few as keep 8 waves on each compute unit (16 where
// the accesses are single elements): 16384 rows of 2048 bf16 79.3 us with 512 workgroups, 86.4 with 1024; 8192 rows of
// 1531 52.9 with 16 waves, 79.5 with 8.
static int bn_bwd_blocks(int64_t rows, const BnShape& sh, bool vec) {
  const int waves = sh.threads / 64, want = vec ? 8 : 16;
  return bn_blocks(rows, sh.rpb, 256 * (want > waves ? want / waves : 1));
}

}  // namespace prl

using namespace prl;

extern "C" int prl_block_norms_supported(int dtype, int64_t H) {
  return (dtype == PRL_F32 || dtype == PRL_BF16) && H >= 1 && H <= kBnMaxH ? 1 : 0;
}

extern "C" size_t prl_block_norms_bwd_workspace_bytes(int dtype, int64_t rows, int64_t H) {
  if (!prl_block_norms_supported(dtype, H) || rows < 0) return 0;
  const int a = bn_bwd_blocks(rows, bn_shape(dtype, H, true), true), b = bn_bwd_blocks(rows, bn_shape(dtype, H, false), false);
  return (size_t)3 * (a > b ? a : b) * bn_part_pitch(H) * sizeof(float);
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

#define PRL_BN_GATE(KERNEL, DT, NV, OW, VEC, BOTH)                                      \
  do {                                                                                  \
    if (gate_kind == PRL_GATE_FULL) KERNEL(DT, NV, OW, 2, VEC, BOTH);                   \
    else if (gate_kind == PRL_GATE_CHANNEL) KERNEL(DT, NV, OW, 1, VEC, BOTH);           \
    else KERNEL(DT, NV, OW, 0, VEC, BOTH);                                              \
  } while (0)
#define PRL_BN_VEC(KERNEL, DT, NV, OW, VEC)                            \
  do {                                                                 \
    if (w_post && w_pre) PRL_BN_GATE(KERNEL, DT, NV, OW, VEC, true);   \
    else PRL_BN_GATE(KERNEL, DT, NV, OW, VEC, false);                  \
  } while (0)
#define PRL_BN_SHAPE(KERNEL, DT, VEC)                                   \
  do {                                                                  \
    if (sh.onewave && sh.nv == 1) PRL_BN_VEC(KERNEL, DT, 1, true, VEC); \
    else if (sh.onewave) PRL_BN_VEC(KERNEL, DT, 2, true, VEC);          \
    else PRL_BN_VEC(KERNEL, DT, 1, false, VEC);                         \
  } while (0)
#define PRL_BN_DISPATCH(KERNEL)                                                           \
  do { /* (two units a thread of a workgroup: rows of more than 4096 fp32 or single elements) */ \
    const bool wide = !sh.onewave && sh.nv == 2;                                          \
    if (dtype == PRL_F32 && vec && wide) PRL_BN_VEC(KERNEL, PRL_F32, 2, false, true);     \
    else if (dtype == PRL_F32 && vec) PRL_BN_SHAPE(KERNEL, PRL_F32, true);                \
    else if (dtype == PRL_F32 && wide) PRL_BN_VEC(KERNEL, PRL_F32, 2, false, false);      \
    else if (dtype == PRL_F32) PRL_BN_SHAPE(KERNEL, PRL_F32, false);                      \
    else if (vec) PRL_BN_SHAPE(KERNEL, PRL_BF16, true);                                   \
    else if (wide) PRL_BN_VEC(KERNEL, PRL_BF16, 2, false, false);                         \
    else PRL_BN_SHAPE(KERNEL, PRL_BF16, false);                                           \
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
  const bool vec = bn_aligned((int)es, H, {x, branch, w_post, w_pre, hidden, w_pre ? normed : nullptr,
                                          narrow ? nullptr : gate},
                             {x_stride, branch_stride, hidden_stride, n_stride,
                              gate_kind == PRL_GATE_FULL ? gate_stride : 0});
  const BnShape sh = bn_shape(dtype, H, vec);
  const dim3 grid((unsigned)bn_fwd_blocks(rows, sh)), block((unsigned)sh.threads);
  const BnIn in = {bn_rows(x, x_stride, H, es), bn_rows(branch, branch_stride, H, es), {}, {},
                   {(const char*)gate, gate_pitch, (int)(H * es)}, nullptr, nullptr, (const char*)w_post,
                   (const char*)w_pre, gate_kind};
#define PRL_BN_FWD(DT, NV, OW, GATE, VEC, BOTH)                                                                       \
  hipLaunchKernelGGL((k_block_norms_fwd<DT, NV, OW, GATE, VEC, BOTH>), grid, block, 0, (hipStream_t)stream, in, scale, \
                     weight_offset, eps_post, eps_pre, (BnRowsOut{(char*)hidden, hidden_stride * es}),                \
                     (BnRowsOut{(char*)normed, n_stride * es}), w_post ? rstd_post : nullptr,                         \
                     w_pre ? rstd_pre : nullptr, rows, (int)H)
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
  // (also without a row: the launch that leaves sums of zero reads it)
  PRL_REQUIRE(gate_kind != PRL_GATE_CHANNEL || gate, "block_norms_bwd: a gate per channel must not be NULL");
  PRL_REQUIRE(gate_kind != PRL_GATE_TOKEN || !g_gate || g_gate_stride >= 1,
              "block_norms_bwd: the row stride of a token gate's gradient must be >= 1");
  PRL_REQUIRE(!g_w_post || w_post, "block_norms_bwd: g_w_post without w_post");
  PRL_REQUIRE(!g_w_pre || w_pre, "block_norms_bwd: g_w_pre without w_pre");
  PRL_REQUIRE(!g_gate || gate_kind != PRL_GATE_NONE, "block_norms_bwd: g_gate without a gate");
  PRL_REQUIRE(rows == 0 || (x && branch && gx && g_branch && (!w_post || rstd_post) && (!w_pre || rstd_pre) &&
                            (!w_pre == !g_normed)),
              "block_norms_bwd: x, branch, gx, g_branch and (with their weights) rstd_post, rstd_pre, g_normed must not be "
              "NULL; g_normed goes with w_pre");
  const int64_t es = dtype == PRL_F32 ? 4 : 2;
  const bool full = gate_kind == PRL_GATE_FULL, narrow = gate_kind == PRL_GATE_TOKEN || gate_kind == PRL_GATE_ONE;
  const bool vec = bn_aligned((int)es, H,
                             {x, branch, w_post, w_pre, g_hidden, g_normed, gx, g_branch,
                              narrow ? nullptr : gate, full ? g_gate : nullptr},
                             {x_stride, branch_stride, g_hidden ? g_hidden_stride : 0, g_normed ? g_normed_stride : 0,
                              gx_stride, g_branch_stride, full ? gate_stride : 0, full && g_gate ? g_gate_stride : 0});
  const BnShape sh = bn_shape(dtype, H, vec);
  const int nblk = bn_bwd_blocks(rows, sh, vec);
  const size_t one = (size_t)nblk * bn_part_pitch(H), need = 3 * one * sizeof(float);
  const bool channel = (gate_kind == PRL_GATE_CHANNEL || gate_kind == PRL_GATE_ONE) && g_gate;
  const bool sums = g_w_post || g_w_pre || channel;
  PRL_REQUIRE(!sums || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
              "block_norms_bwd: 16-byte aligned workspace of %zu bytes needed (prl_block_norms_bwd_workspace_bytes)", need);
  float* ws = (float*)workspace;
  float *p1 = g_w_post ? ws : nullptr, *p2 = g_w_pre ? ws + one : nullptr, *pg = channel ? ws + 2 * one : nullptr;
  hipStream_t st = (hipStream_t)stream;
  // rows == 0: the kernel runs with no row and leaves sums of zero
  const int64_t gate_pitch = gate_kind == PRL_GATE_ONE ? 0 : gate_stride * es;
  const dim3 grid((unsigned)nblk), block((unsigned)sh.threads);
  const size_t lds = sh.onewave ? (size_t)sh.rpb * bn_part_pitch(H) * sizeof(float) : 0;
  char* gg = channel || !g_gate ? nullptr : (char*)g_gate;
  const BnIn in = {bn_rows(x, x_stride, H, es),
                   bn_rows(branch, branch_stride, H, es),
                   bn_rows(g_normed, g_normed_stride, H, es),
                   bn_rows(g_hidden, g_hidden_stride, H, es),
                   {(const char*)gate, gate_pitch, (int)(H * es)},
                   w_post ? rstd_post : nullptr,
                   w_pre ? rstd_pre : nullptr,
                   (const char*)w_post,
                   (const char*)w_pre,
                   gate_kind};
#define PRL_BN_BWD(DT, NV, OW, GATE, VEC, BOTH)                                                                       \
  hipLaunchKernelGGL((k_block_norms_bwd<DT, NV, OW, GATE, VEC, BOTH>), grid, block, lds, st, in, scale, weight_offset, \
                     (BnRowsOut{(char*)gx, gx_stride * es}), (BnRowsOut{(char*)g_branch, g_branch_stride * es}), p1, p2, \
                     pg, (BnRowsOut{gg, g_gate_stride * es}), rows, (int)H)
  PRL_BN_DISPATCH(PRL_BN_BWD);
#undef PRL_BN_BWD
  PRL_CHECK_LAUNCH("block_norms_bwd");
  if (!sums) return PRL_OK;
  const dim3 fgrid((unsigned)((H + 31) / 32), 3);
  if (dtype == PRL_BF16)
    hipLaunchKernelGGL((k_block_norms_finish<PRL_BF16>), fgrid, dim3(256), 0, st, p1, p2, pg, (char*)g_w_post,
                       (char*)g_w_pre, (char*)g_gate, nblk, (int)H, gate_kind == PRL_GATE_ONE);
  else
    hipLaunchKernelGGL((k_block_norms_finish<PRL_F32>), fgrid, dim3(256), 0, st, p1, p2, pg, (char*)g_w_post,
                       (char*)g_w_pre, (char*)g_gate, nblk, (int)H, gate_kind == PRL_GATE_ONE);
  PRL_CHECK_LAUNCH("block_norms_bwd");
  return PRL_OK;
}
