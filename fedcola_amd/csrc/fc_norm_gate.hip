// Between two branches of a block, in one pass over the rows:
//
//   n = norm(y) wp + bp;   r = alpha x + s_b gate n;   h = norm(r) wn + bn
//
// y the branch's output, x the residual stream, gate one vector for all rows or one for each sample, s_b a sample's drop-path multiplier;
// norm: LayerNorm or RMSNorm.  Each part may be absent.  A multiplier of 0 drops the branch: y and the gate are not used and their gradients are 0,
// whatever they hold (the loads are in range all the same).  h comes from r before r is rounded.
// Backward: r and both norms' statistics are formed again from y and x, so nothing is kept and dwn, dwp are those of the unrounded r.
// Bound: HBM, 4 T D elements forward (y, x in; r, h out), 6 T D backward (y, x, dr, dh in; dy, dx out).
// A row is held in registers by 8, 16 or 32 lanes (D <= 64, 128, 256), a wave (<= 1024), 4 waves (<= 2048, backward <= 4096) or 8 (<= 8192): 8 or 16
// values a lane.  A workgroup walks several
// rows with the weight vectors in registers (forward) or LDS (backward): read per row they would be 20 bytes an element from L2 beside the 8
// from HBM.  The next row is loaded while this one is summed.  Measured at the rate of a large copy (4.9 TB/s) for 65536 x 4096 bf16: 417 us
// forward (5.1 TB/s), 667 us backward (4.8 TB/s); fp32, 32768 x 4096: 418 (5.1) and 662 (4.9), 65536 x 1024: 223 and 328; 12608 x 384: 13 and 27 us, where
// filling and draining the chip is most of the time.  Rows that are no whole eights wide are read value by value, and above 512 values a lane's
// 16 of them spill in the backward (144 to 240 bytes; fp32 of whole eights above 2048, 16): 65536 x 1001 bf16 133 and 592 us, 65536 x 1024 112 and 181.
// dwp, dbp, dwn, dbn, dgate: each workgroup's sums over its rows (fp32) are one row of partial sums, added in fp64 in a fixed order by a
// second launch.  A workgroup's rows share one gate vector.
#include "../../include/fedcola_hip.h"
#include "fc_tiles.h"

struct NgArgs {
  const void *y, *x, *dr, *dh;
  long ldy, ldx, lddr, lddh;
  void *r, *h, *dy, *dx;                       // rows D apart
  const float *wp, *bp, *gate, *scale, *wn, *bn;
  float alpha, eps;
  int rms, post, pre, D;
  long T, gate_rows, scale_rows;               // rows of one gate vector / one multiplier
  long per, blocks;                            // rows of a workgroup, workgroups of a gate vector
  float* part;                                 // [workgroups][5][D]: dwp, dbp, dwn, dbn, dgate
};
enum { NG_DWP = 0, NG_DBP, NG_DWN, NG_DBN, NG_DGATE, NG_SUMS };

// E values of a row for lane l of NTH: VEC 8: chunks l, l + NTH, ... of 8; VEC 1: values l, l + NTH, ...
template <int VEC, int NTH, int E, class F> __device__ __forceinline__ void ng_each(int l, int D, F f) {
  if (VEC == 8) {
#pragma unroll
    for (int t = 0; t < E / 8; ++t)
      if ((l + NTH * t) * 8 < D) f(t * 8, (l + NTH * t) * 8);
  } else {
#pragma unroll
    for (int t = 0; t < E; ++t)
      if (l + NTH * t < D) f(t, l + NTH * t);
  }
}
__device__ __forceinline__ void ng_ld8(const bf16_t* p, float* v) {
  const uint4 u = *(const uint4*)p;
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void ng_ld8(const float* p, float* v) {
  const ft_f4 a = *(const ft_f4*)p, b = *(const ft_f4*)(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
__device__ __forceinline__ void ng_st8(bf16_t* p, const float* v) { *(uint4*)p = make_uint4(f2bf2(v[0], v[1]), f2bf2(v[2], v[3]), f2bf2(v[4], v[5]), f2bf2(v[6], v[7])); }
__device__ __forceinline__ void ng_st8(float* p, const float* v) {
  *(ft_f4*)p = ft_f4{v[0], v[1], v[2], v[3]};
  *(ft_f4*)(p + 4) = ft_f4{v[4], v[5], v[6], v[7]};
}
template <typename T, int VEC, int NTH, int E> __device__ __forceinline__ void ng_load(const T* p, int l, int D, float (&v)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = 0.f;
  if (!p) return;
  ng_each<VEC, NTH, E>(l, D, [&](int k, int c) {
    if constexpr (VEC == 8) ng_ld8(p + c, v + k); else v[k] = Io<T>::ld(p, c);
  });
}
template <typename T, int VEC, int NTH, int E> __device__ __forceinline__ void ng_store(T* p, int l, int D, const float (&v)[E]) {
  ng_each<VEC, NTH, E>(l, D, [&](int k, int c) {
    if constexpr (VEC == 8) ng_st8(p + c, v + k); else Io<T>::st(p, c, v[k]);
  });
}
// a row as it lies in memory, so that the next row's loads can be in flight under this row's sums.  Every lane loads, from inside the row;
// lanes past its end, and rows that are not there, become zeros in get(), whose asm keeps the conversion in front of the next row's loads.
template <typename T, int VEC, int NTH, int E> struct NgRaw {
  T v[E] __attribute__((aligned(16)));
  __device__ __forceinline__ void load(const T* p, int l, int D) {
    if (VEC == 8) {
#pragma unroll
      for (int t = 0; t < E / 8; ++t) {
        const int c = (l + NTH * t) * 8;
        const uint4* q = (const uint4*)(p + (c < D ? c : 0));
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) *(uint4*)&v[t * 8 + i * 16 / sizeof(T)] = q[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = p[l + NTH * i < D ? l + NTH * i : 0];
    }
  }
  __device__ __forceinline__ void get(float (&f)[E], int l, int D, bool there) const {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = VEC == 8 ? (l + NTH * (i / 8)) * 8 : l + NTH * i;
      const float u = Io<T>::ld(v, i);
      f[i] = there && c < D ? u : 0.f;
      asm volatile("" : "+v"(f[i]));
    }
  }
};
// the sum of each G lanes of a wave in all of them, by DPP: pairs, quads, eights, sixteens, then the rows of sixteen (shuffles through LDS cost six
// round trips instead; the rows' sums stand in the way of every row's loads)
template <int G> __device__ __forceinline__ float ng_lane_sum(float v) {
#define NG_DPP(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, false))
  NG_DPP(0xb1);     // quad_perm 1 0 3 2
  NG_DPP(0x4e);     // quad_perm 2 3 0 1
  NG_DPP(0x141);    // row_half_mirror
  if (G > 8) NG_DPP(0x140);    // row_mirror
#undef NG_DPP
  if (G <= 16) return v;
  if (G == 32) return v + __shfl_xor(v, 16, 64);
  const int i = __float_as_int(v);
  return (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16))) +
         (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
}
// sums over a row's lanes.  W waves: through LDS, one barrier, two buffers in turn (a wave is never two sums ahead of another)
template <int W, int G> struct NgSum {
  float2* red;     // [2][W]
  int turn = 0;
  __device__ __forceinline__ float2 operator()(float a, float b) {
    a = ng_lane_sum<G>(a);
    b = ng_lane_sum<G>(b);
    return join(a, b);
  }
  __device__ __forceinline__ float operator()(float a) { return join(ng_lane_sum<G>(a), 0.f).x; }
  __device__ __forceinline__ float2 join(float a, float b) {
    if (W == 1) return make_float2(a, b);
    float2* q = red + turn * W;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) q[threadIdx.x >> 6] = make_float2(a, b);
    ft_barrier();
    float2 s = q[0];
#pragma unroll
    for (int i = 1; i < W; ++i) { s.x += q[i].x; s.y += q[i].y; }
    return s;
  }
};
// v -> normalised v; lanes past D keep 0.  Returns 1 / deviation
template <int VEC, int NTH, int E, class SUM> __device__ __forceinline__ float ng_norm(float (&v)[E], int l, int D, int rms, float eps, SUM& sum) {
  const float inv = 1.f / (float)D;
  float a = 0.f;
  if (!rms) {
#pragma unroll
    for (int i = 0; i < E; ++i) a += v[i];
    const float mu = sum(a) * inv;
    constexpr int STEP = VEC == 8 ? 8 : 1;
    ng_each<VEC, NTH, E>(l, D, [&](int k, int c) {
#pragma unroll
      for (int i = 0; i < STEP; ++i) v[k + i] -= mu;
    });
    a = 0.f;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) a += v[i] * v[i];
  const float rs = 1.f / sqrtf(sum(a) * inv + eps);
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] *= rs;
  return rs;
}

__device__ __forceinline__ float ng_uniform(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }
// the multiplier of a workgroup's rows, which come in order: one division in all
struct NgSample {
  long q, rem;
  __device__ __forceinline__ NgSample(const NgArgs& a, long row) {
    q = rem = 0;
    if (a.scale) { q = row / a.scale_rows; rem = row - q * a.scale_rows; }
  }
  __device__ __forceinline__ float scale(const NgArgs& a, int step) {     // of the row; then `step` rows on
    if (!a.scale) return 1.f;
    const float s = a.scale[q];
    for (rem += step; rem >= a.scale_rows; rem -= a.scale_rows) ++q;
    return s;
  }
};

template <typename T, int VEC, int W, int E, int G>
__global__ void __launch_bounds__(W == 8 ? 512 : 256) k_ng_fwd(NgArgs a) {
  constexpr int NTH = W == 1 ? G : W * 64, RB = W == 1 ? 256 / G : 1;       // lanes of a row, rows at once
  __shared__ float2 red[2 * W];
  NgSum<W, G> sum{red};
  const int l = W == 1 ? threadIdx.x % G : threadIdx.x, sub = W > 1 ? 0 : G == 64 ? ft_wave() : threadIdx.x / G, D = a.D;
  const unsigned grp = blockIdx.x / (unsigned)a.blocks;
  const long b0 = (long)(blockIdx.x - grp * (unsigned)a.blocks) * a.per, first = (long)grp * a.gate_rows + b0, left = a.gate_rows - b0;
  const int n = (int)(left < a.per ? left : a.per);
  NgSample smp(a, first + sub);
  NgRaw<T, VEC, NTH, E> ry, rx;
  float s = 1.f, snext = 1.f;
  auto fetch = [&](int i) {
    const long row = first + (i < n ? i : n - 1);
    snext = i < n ? smp.scale(a, RB) : 0.f;
    ry.load((const T*)a.y + row * a.ldy, l, D);
    rx.load((const T*)a.x + row * a.ldx, l, D);
  };
  if (sub < n) fetch(sub);
  float wp[E], bp[E], gt[E], wn[E], bn[E];
  ng_load<float, VEC, NTH, E>(a.wp, l, D, wp);
  ng_load<float, VEC, NTH, E>(a.bp, l, D, bp);
  ng_load<float, VEC, NTH, E>(a.gate ? a.gate + (long)grp * D : nullptr, l, D, gt);
  ng_load<float, VEC, NTH, E>(a.wn, l, D, wn);
  ng_load<float, VEC, NTH, E>(a.bn, l, D, bn);
  for (int i = sub; i < n; i += RB) {
    const long row = first + i;
    float y[E], x[E];
    s = G == 64 ? ng_uniform(snext) : snext;
    ry.get(y, l, D, s != 0.f);
    rx.get(x, l, D, true);
    fetch(i + RB);
    if (a.post) {
      ng_norm<VEC, NTH, E>(y, l, D, a.rms, a.eps, sum);
#pragma unroll
      for (int k = 0; k < E; ++k) y[k] = y[k] * wp[k] + bp[k];
    }
#pragma unroll
    for (int k = 0; k < E; ++k) x[k] = a.alpha * x[k] + (s != 0.f ? s * (a.gate ? gt[k] * y[k] : y[k]) : 0.f);      // (a dropped sample's gate may hold anything)
    ng_store<T, VEC, NTH, E>((T*)a.r + row * D, l, D, x);
    if (a.pre) {
      ng_norm<VEC, NTH, E>(x, l, D, a.rms, a.eps, sum);
#pragma unroll
      for (int k = 0; k < E; ++k) x[k] = x[k] * wn[k] + bn[k];
      ng_store<T, VEC, NTH, E>((T*)a.h + row * D, l, D, x);
    }
  }
}

// The weight vectors stand in LDS here: with the five running sums and the next row's loads they do not fit the registers.
enum { NG_WP = 0, NG_BP, NG_GT, NG_WN, NG_VECS };
template <typename T, int VEC, int W, int E, int G>
__global__ void __launch_bounds__(W == 8 ? 512 : 256, E == 8 ? (sizeof(T) == 2 && VEC == 8 && G == 64 ? 4 : 3) : 2) k_ng_bwd(NgArgs a) {
  constexpr int NTH = W == 1 ? G : W * 64, RB = W == 1 ? 256 / G : 1;
  extern __shared__ __attribute__((aligned(16))) float vec[];   // [NG_VECS][Dp], then for W = 1 [4][NG_SUMS][Dp] over them
  __shared__ float2 red[2 * W];
  NgSum<W, G> sum{red};
  const int l = W == 1 ? threadIdx.x % G : threadIdx.x, sub = W > 1 ? 0 : G == 64 ? ft_wave() : threadIdx.x / G, D = a.D, Dp = (D + 7) & ~7;
  const float inv = 1.f / (float)D;
  const unsigned grp = blockIdx.x / (unsigned)a.blocks;
  const long b0 = (long)(blockIdx.x - grp * (unsigned)a.blocks) * a.per, first = (long)grp * a.gate_rows + b0, left = a.gate_rows - b0;
  const int n = (int)(left < a.per ? left : a.per);
  NgSample smp(a, first + sub);
  NgRaw<T, VEC, NTH, E> ry, rx, rr, rh;
  float s = 1.f, snext = 1.f;
  auto fetch = [&](int i) {
    const long row = first + (i < n ? i : n - 1);
    snext = i < n ? smp.scale(a, RB) : 0.f;
    ry.load((const T*)a.y + row * a.ldy, l, D);
    rx.load((const T*)a.x + row * a.ldx, l, D);
    rr.load(a.dr ? (const T*)a.dr + row * a.lddr : (const T*)a.x + row * a.ldx, l, D);
    rh.load(a.dh ? (const T*)a.dh + row * a.lddh : (const T*)a.x + row * a.ldx, l, D);
  };
  if (sub < n) fetch(sub);
  for (int c = threadIdx.x; c < Dp; c += W == 8 ? 512 : 256) {
    const bool in = c < D;
    vec[NG_WP * Dp + c] = in && a.wp ? a.wp[c] : 0.f;
    vec[NG_BP * Dp + c] = in && a.bp ? a.bp[c] : 0.f;
    vec[NG_GT * Dp + c] = in ? (a.gate ? a.gate[(long)grp * D + c] : 1.f) : 0.f;
    vec[NG_WN * Dp + c] = in && a.wn ? a.wn[c] : 0.f;
  }
  float sums[NG_SUMS][E];
#pragma unroll
  for (int q = 0; q < NG_SUMS; ++q)
#pragma unroll
    for (int k = 0; k < E; ++k) sums[q][k] = 0.f;
  __syncthreads();
  auto get = [&](int q, float (&w)[E]) {
    asm volatile("" ::: "memory");                       // read again for every row: hoisted out of the loop they take the registers they are to save
    ng_load<float, VEC, NTH, E>(vec + q * Dp, l, D, w);
  };
  for (int i = sub; i < n; i += RB) {
    const long row = first + i;
    float y[E], x[E], d[E], dn[E], w[E], v[E];
    s = G == 64 ? ng_uniform(snext) : snext;
    ry.get(y, l, D, s != 0.f);
    rx.get(x, l, D, true);
    rr.get(d, l, D, a.dr != nullptr);
    rh.get(dn, l, D, a.dh != nullptr);
    fetch(i + RB);       // here alone: in two branches the loads' registers would be copied, and so waited for, where these meet
    const float rs1 = a.post ? ng_norm<VEC, NTH, E>(y, l, D, a.rms, a.eps, sum) : 1.f;      // y: its normalised row from here on
    auto branch = [&](float (&p)[E]) {                                                      // the branch as the gate sees it
#pragma unroll
      for (int k = 0; k < E; ++k) p[k] = y[k];
      if (!a.post) return;
      get(NG_WP, w);
#pragma unroll
      for (int k = 0; k < E; ++k) p[k] *= w[k];
      get(NG_BP, w);
#pragma unroll
      for (int k = 0; k < E; ++k) p[k] += w[k];
    };
    if (a.pre) {
      branch(v);
      get(NG_GT, w);
#pragma unroll
      for (int k = 0; k < E; ++k) x[k] = a.alpha * x[k] + (s != 0.f ? s * (w[k] * v[k]) : 0.f);
      const float rs2 = ng_norm<VEC, NTH, E>(x, l, D, a.rms, a.eps, sum);
      get(NG_WN, w);
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        sums[NG_DWN][k] += dn[k] * x[k];
        sums[NG_DBN][k] += dn[k];
        dn[k] *= w[k];
        s1 += dn[k];
        s2 += dn[k] * x[k];
      }
      const float2 m = sum(s1, s2);
      const float m1 = a.rms ? 0.f : m.x * inv, m2 = m.y * inv;
#pragma unroll
      for (int k = 0; k < E; ++k) d[k] += rs2 * (dn[k] - m1 - x[k] * m2);
    }
    // d: the gradient of r
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = a.alpha * d[k];
    ng_store<T, VEC, NTH, E>((T*)a.dx + row * D, l, D, v);
    branch(v);
    get(NG_GT, w);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float dp = s == 0.f ? 0.f : d[k] * s;
      sums[NG_DGATE][k] += dp * v[k];
      d[k] = s == 0.f ? 0.f : dp * w[k];
    }
    if (a.post) {
      float s1 = 0.f, s2 = 0.f;
      get(NG_WP, w);
#pragma unroll
      for (int k = 0; k < E; ++k) {
        sums[NG_DWP][k] += d[k] * y[k];
        sums[NG_DBP][k] += d[k];
        d[k] *= w[k];
        s1 += d[k];
        s2 += d[k] * y[k];
      }
      const float2 m = sum(s1, s2);
      const float m1 = a.rms ? 0.f : m.x * inv, m2 = m.y * inv;
#pragma unroll
      for (int k = 0; k < E; ++k) d[k] = rs1 * (d[k] - m1 - y[k] * m2);
    }
    ng_store<T, VEC, NTH, E>((T*)a.dy + row * D, l, D, d);
  }
  if (!a.part) return;
  float* o = a.part + (long)blockIdx.x * NG_SUMS * D;
  if (W == 1) {
#pragma unroll
    for (int o = G; o < 64; o *= 2)                       // the wave's other rows
#pragma unroll
      for (int q = 0; q < NG_SUMS; ++q)
#pragma unroll
        for (int k = 0; k < E; ++k) sums[q][k] += __shfl_xor(sums[q][k], o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) < G)
#pragma unroll
      for (int q = 0; q < NG_SUMS; ++q) ng_store<float, VEC, NTH, E>(vec + (ft_wave() * NG_SUMS + q) * Dp, l, D, sums[q]);
    __syncthreads();
    const int st = NG_SUMS * Dp;
    for (int c = threadIdx.x; c < NG_SUMS * D; c += 256) {
      const float* f = vec + c / D * Dp + c % D;
      o[c] = (f[0] + f[st]) + (f[2 * st] + f[3 * st]);
    }
  } else {
#pragma unroll
    for (int q = 0; q < NG_SUMS; ++q)
      ng_each<VEC, NTH, E>(l, D, [&](int k, int c) {
        constexpr int STEP = VEC == 8 ? 8 : 1;
#pragma unroll
        for (int i = 0; i < STEP; ++i) o[q * D + c + i] = sums[q][k + i];
      });
  }
}

// out[c] = sum over workgroups of their partial sums: 64 columns by 16 slices of the workgroups.  blockIdx.y: 0 to 3 the four weights, from 4 on gate
// vectors, each workgroup every (gridDim.y - 4)th of them (there may be more than a launch has workgroups in y)
struct NgOut { float* p[NG_SUMS]; };
__global__ void __launch_bounds__(1024) k_ng_sum(const float* part, int D, long blocks, long groups, NgOut out) {
  __shared__ double red[16][64];
  const int q = blockIdx.y < 4 ? blockIdx.y : NG_DGATE, c = blockIdx.x * 64 + (threadIdx.x & 63), sl = threadIdx.x >> 6;
  if (!out.p[q]) return;
  for (long g = blockIdx.y < 4 ? 0 : blockIdx.y - 4; g < (q == NG_DGATE ? groups : 1); g += gridDim.y - 4) {
    const long b0 = g * blocks, b1 = q == NG_DGATE ? b0 + blocks : groups * blocks;
    double v = 0;
    if (c < D)
#pragma unroll 4
      for (long b = b0 + sl; b < b1; b += 16) v += (double)part[(b * NG_SUMS + q) * D + c];
    __syncthreads();                                   // the vector before has been read
    red[sl][threadIdx.x & 63] = v;
    __syncthreads();
    if (sl == 0 && c < D) {
#pragma unroll
      for (int i = 1; i < 16; ++i) v += red[i][threadIdx.x & 63];
      out.p[q][g * D + c] = (float)v;
    }
    if (q != NG_DGATE) return;
  }
}

// ---------------------------------------------------------------- host
// Waves of a row, values of a lane, and lanes of a row that is shorter than a wave (262144 x 64 bf16: 24 and 49 us forward and backward, 112 and 252 with
// a wave a row; 131072 x 256: 49 and 95, 62 and 141).  A wave alone needs no barriers for its sums, so one takes a row as long as 16 values a lane are enough
// (12608 x 768 bf16: 19 and 41 us forward and backward, 30 and 67 by four waves of 8 values; 16384 x 1024: 30 and 50, 39 and 82); above, backward 16 values leave two workgroups a
// CU instead of one of twice the waves (65536 x 4096 bf16: 667 us against 1151), forward 8 are as good.
static void ng_form(long D, bool bwd, int& W, int& E, int& G) {
  G = D <= 64 ? 8 : D <= 128 ? 16 : D <= 256 ? 32 : 64;
  W = D <= 1024 ? 1 : D <= 2048 || (bwd && D <= 4096) ? 4 : 8;
  E = D <= 512 || (D > 1024 && D <= 2048) || (!bwd && D <= 4096 && D > 2048) ? 8 : 16;
}
// workgroups of a gate vector's rows: in all as many as the chip holds at once, each wave with the same number of rows.  deep: waves a SIMD that
// the registers of the form in most use allow.  (By the compiler's report others hold one fewer, so that their last workgroups start when the
// first end: forward, rows no whole eights wide up to 256, from 513 to 1024 and from 4097 on, and fp32 up to 256; backward, bf16 rows no whole eights wide
// from 257 to 512.)
static void ng_split(long T, long gate_rows, long D, bool bwd, int deep, long& per, long& blocks) {
  int W, E, G;
  ng_form(D, bwd, W, E, G);
  const long groups = T / gate_rows, at_once = W == 1 ? 256 / G : 1, waves = 4 * 256 * deep, want = waves / (W == 1 ? 4 : W);
  const long b = (want + groups - 1) / groups;
  per = ft_up((gate_rows + b - 1) / b, at_once);
  blocks = (gate_rows + per - 1) / per;
}
static int ng_deep(long D, bool bwd, int dt) {
  int W, E, G;
  ng_form(D, bwd, W, E, G);
  if (bwd) return E == 16 ? 2 : dt && G == 64 ? 4 : 3;
  return W == 8 ? (E == 16 ? 2 : 4) : E == 16 ? 3 : 5;
}
static bool ng_aligned(const NgArgs& a, int dt) {
  size_t p = (size_t)a.y | (size_t)a.x | (size_t)a.dr | (size_t)a.dh | (size_t)a.r | (size_t)a.h | (size_t)a.dy | (size_t)a.dx | (size_t)a.wp | (size_t)a.bp |
             (size_t)a.gate | (size_t)a.wn | (size_t)a.bn;
  const long m = dt ? 8 : 4;
  return (p & 15) == 0 && a.D % 8 == 0 && a.ldy % m == 0 && a.ldx % m == 0 && a.lddr % m == 0 && a.lddh % m == 0;
}
template <typename T, bool BWD> static int ng_launch(const NgArgs& a, int dt, hipStream_t s) {
  const dim3 g((unsigned)(a.T / a.gate_rows * a.blocks));
  const bool v = ng_aligned(a, dt);
#define NG_RUN(VEC, W, E, G)                                                                                           \
  do {                                                                                                                \
    if constexpr (BWD) {                                                                                              \
      static FtLds allowed;                                                                                           \
      constexpr int rows = W == 1 ? 4 * NG_SUMS : NG_VECS;                                                            \
      FC_TRY(allowed.allow((const void*)k_ng_bwd<T, VEC, W, E, G>, rows * W * 64 * E * 4));                              \
      hipLaunchKernelGGL((k_ng_bwd<T, VEC, W, E, G>), g, dim3(W == 8 ? 512 : 256), rows * ((a.D + 7) & ~7) * 4, s, a);   \
    } else {                                                                                                          \
      hipLaunchKernelGGL((k_ng_fwd<T, VEC, W, E, G>), g, dim3(W == 8 ? 512 : 256), 0, s, a);                             \
    }                                                                                                                 \
  } while (0)
#define NG_PICK(W, E, G) do { if (v) NG_RUN(8, W, E, G); else NG_RUN(1, W, E, G); } while (0)
  int W, E, G;
  ng_form(a.D, BWD, W, E, G);
  if (G == 8) NG_PICK(1, 8, 8);
  else if (G == 16) NG_PICK(1, 8, 16);
  else if (G == 32) NG_PICK(1, 8, 32);
  else if (W == 1 && E == 8) NG_PICK(1, 8, 64);
  else if (W == 1) NG_PICK(1, 16, 64);
  else if (W == 4 && E == 8) NG_PICK(4, 8, 64);
  else if (W == 4) { if constexpr (BWD) NG_PICK(4, 16, 64); }
  else if (E == 8) { if constexpr (!BWD) NG_PICK(8, 8, 64); }
  else NG_PICK(8, 16, 64);
#undef NG_PICK
#undef NG_RUN
  FC_LAUNCH_CHECK();
  return 0;
}
// a launch has fewer than 2^32 threads in a dimension; the backward has no more workgroups than the forward, nor larger ones
static int ng_grid(const char* what, const NgArgs& a, bool bwd) {
  int W, E, G;
  ng_form(a.D, bwd, W, E, G);
  FC_REQUIRE(a.T / a.gate_rows * a.blocks * (W == 8 ? 512 : 256) < (1L << 32), "%s: too many samples (%ld gate vectors)", what, a.T / a.gate_rows);
  return 0;
}
static int ng_check(const char* what, int dt, int kind, const NgArgs& a, const void* out) {
  FC_REQUIRE(dt == FC_PREC_FP32 || dt == FC_PREC_BF16, "%s: dt %d", what, dt);
  FC_REQUIRE(kind == FC_NORM_LAYER || kind == FC_NORM_RMS, "%s: norm %d", what, kind);
  FC_REQUIRE(a.T >= 0 && a.T < (1L << 40) && a.D >= 1 && a.D <= 8192, "%s: bad sizes (%ld rows, width %d: 1 to 8192)", what, a.T, a.D);
  FC_REQUIRE(a.T == 0 || (a.y && a.x && out), "%s: null pointer", what);
  FC_REQUIRE(a.ldy >= a.D && a.ldx >= a.D, "%s: rows %ld and %ld apart", what, a.ldy, a.ldx);
  FC_REQUIRE(a.eps > 0.f, "%s: eps %g", what, (double)a.eps);
  FC_REQUIRE(a.gate_rows >= 1 && a.scale_rows >= 1 && a.T % a.gate_rows == 0 && a.T % a.scale_rows == 0, "%s: %ld rows are no whole number of samples", what, a.T);
  FC_REQUIRE((!a.bp || a.wp) && (!a.bn || a.wn), "%s: a bias without its weight", what);
  FC_REQUIRE(kind == FC_NORM_LAYER || (!a.bp && !a.bn), "%s: RMSNorm has no bias", what);
  return ft_check_device(a.x, what);
}
extern "C" size_t fc_norm_gate_workspace_bytes(int64_t T, int32_t D, int64_t gate_rows) {
  if (T <= 0 || D < 1 || gate_rows < 0) return 256;
  long per, blocks, more;
  const long gr = gate_rows ? gate_rows : T;
  if (T % gr) return 256;
  ng_split(T, gr, D, true, ng_deep(D, true, FC_PREC_BF16), per, blocks);
  ng_split(T, gr, D, true, ng_deep(D, true, FC_PREC_FP32), per, more);
  return (size_t)(T / gr) * (blocks > more ? blocks : more) * NG_SUMS * D * sizeof(float) + 256;
}
extern "C" int fc_norm_gate_fwd(int32_t dt, int32_t kind, const void* y, int64_t ldy, const void* x, int64_t ldx, int64_t T, int32_t D, const float* post_w,
                                const float* post_b, const float* gate, int64_t gate_rows, const float* row_scale, int64_t scale_rows, float alpha,
                                const float* pre_w, const float* pre_b, float eps, void* r, void* h, void* stream) {
  NgArgs a = {};
  a.y = y; a.x = x; a.ldy = ldy; a.ldx = ldx; a.r = r; a.h = h;
  a.wp = post_w; a.bp = post_b; a.gate = gate; a.scale = row_scale; a.wn = pre_w; a.bn = pre_b;
  a.alpha = alpha; a.eps = eps; a.rms = kind == FC_NORM_RMS; a.post = post_w != nullptr; a.pre = pre_w != nullptr; a.D = D; a.T = T;
  a.gate_rows = gate && gate_rows ? gate_rows : T ? T : 1;
  a.scale_rows = row_scale && scale_rows ? scale_rows : T ? T : 1;
  FC_TRY(ng_check("fc_norm_gate_fwd", dt, kind, a, r));
  FC_REQUIRE(!a.pre || h || T == 0, "fc_norm_gate_fwd: no place for the second norm's output");
  if (T == 0) return 0;
  ng_split(T, a.gate_rows, D, false, ng_deep(D, false, dt), a.per, a.blocks);
  FC_TRY(ng_grid("fc_norm_gate_fwd", a, false));
  return dt ? ng_launch<bf16_t, false>(a, dt, (hipStream_t)stream) : ng_launch<float, false>(a, dt, (hipStream_t)stream);
}
extern "C" int fc_norm_gate_bwd(int32_t dt, int32_t kind, const void* dr, int64_t lddr, const void* dh, int64_t lddh, const void* y, int64_t ldy, const void* x,
                                int64_t ldx, int64_t T, int32_t D, const float* post_w, const float* post_b, const float* gate, int64_t gate_rows,
                                const float* row_scale, int64_t scale_rows, float alpha, const float* pre_w, float eps, void* dy, void* dx, float* d_post_w,
                                float* d_post_b, float* d_pre_w, float* d_pre_b, float* d_gate, void* workspace, size_t workspace_bytes, void* stream) {
  NgArgs a = {};
  a.y = y; a.x = x; a.ldy = ldy; a.ldx = ldx; a.dr = dr; a.dh = dh; a.lddr = dr ? lddr : 0; a.lddh = dh ? lddh : 0; a.dy = dy; a.dx = dx;
  a.wp = post_w; a.bp = post_b; a.gate = gate; a.scale = row_scale; a.wn = pre_w;
  a.alpha = alpha; a.eps = eps; a.rms = kind == FC_NORM_RMS; a.post = post_w != nullptr; a.pre = pre_w != nullptr && dh != nullptr; a.D = D; a.T = T;
  a.gate_rows = gate && gate_rows ? gate_rows : T ? T : 1;
  a.scale_rows = row_scale && scale_rows ? scale_rows : T ? T : 1;
  FC_TRY(ng_check("fc_norm_gate_bwd", dt, kind, a, dy));
  FC_REQUIRE((dx || T == 0) && (!dr || lddr >= D) && (!dh || lddh >= D) && (!dh || pre_w), "fc_norm_gate_bwd: null pointer, rows too close, or a gradient without its norm");
  const long groups = T ? T / a.gate_rows : gate_rows ? 0 : 1;      // (no rows: the one vector's gradient is zeros; how many others there are is not known)
  NgOut out = {{d_post_w, d_post_b, d_pre_w, d_pre_b, gate ? d_gate : nullptr}};
  const bool sums = out.p[0] || out.p[1] || out.p[2] || out.p[3] || out.p[4];
  hipStream_t s = (hipStream_t)stream;
  if (T) {
    ng_split(T, a.gate_rows, D, true, ng_deep(D, true, dt), a.per, a.blocks);
    FC_TRY(ng_grid("fc_norm_gate_bwd", a, true));
    if (sums) {
      FC_REQUIRE(workspace && ((size_t)workspace & 255) == 0 && workspace_bytes >= (size_t)groups * a.blocks * NG_SUMS * D * sizeof(float), "fc_norm_gate_bwd: workspace too small or not aligned to 256 bytes");
      a.part = (float*)workspace;
    }
    FC_TRY(dt ? (ng_launch<bf16_t, true>(a, dt, s)) : (ng_launch<float, true>(a, dt, s)));
  }
  if (sums) {
    hipLaunchKernelGGL(k_ng_sum, dim3((D + 63) / 64, (unsigned)(4 + (!out.p[NG_DGATE] ? 0 : groups < 60000 ? groups : 60000))), dim3(1024), 0, s, a.part, D, a.blocks, groups, out);
    FC_LAUNCH_CHECK();
  }
  return 0;
}
