// Gated feed-forward block:  [g | u] = x w_in^T;  h = act(g) u;  y = h w_out^T     (w_in [2 F, D]: gate rows, then up rows; w_out [D, F])
//
// Forward: one product computes both projections -- a tile's columns are gate and up rows of the same hidden units, interleaved by half a
// wave's columns, so that g and u of a unit are in one lane -- and its epilogue applies the activation and the product; h is all that
// reaches memory.  A second product gives y.
// Backward: nothing but the inputs is kept.  dh = dy w_out goes to the workspace in 32 bits; the product of the forward is run again, and its
// epilogue, which has g and u in 32 bits, reads dh and writes
//   h = act(g) u,   dg = dh u act'(g),   du = dh act(g)
// each rounded once; then dx = [dg | du] w_in, dw_in = [dg | du]^T x, dw_out = dy^T h.  That is 16 T D F operations for the 12 of a backward
// pass that reads g and u back.  Kept in 32 bits (in 16 they would be rounded once more than here) these are 8 T F bytes, four times h, for as long as the
// layers above run, and 16 T F of traffic: at the rate of a copy 292 us for 8192 x 4096 x 11000, where the product takes 1100; at widths of about 1050 both
// cost the same.  What is saved here is that memory.  (dh on the same tile as g and
// u, without its 8 bytes a unit through memory, leaves registers for 128 x 256 tiles only: 2300 us for 8192 x 4096 x 11000, 2000 in two kernels;
// 70 against 74 for 12608 x 384 x 1024.)
#include <math.h>

#include "../../include/fedcola_hip.h"
#include "fc_tiles.h"

struct GmArgs {
  FtMat x, w_in, w_out, dy;
  int T, D, F, act;
  bool b32;                     // fp32: w_in and w_out are the fp32 matrices themselves
  long up;                      // rows between a unit's gate and up row in w_in
  bf16_t *h, *dgu;              // planes of [T][ldh], [T][2 ldh]: h; dg | du
  long ldh;                     // whole 128-byte lines: a row that straddles one more costs every tile load an L2 request more
  const float* dh;              // [dh_parts][T][ldd], to be added up
  long ldd;
  int dh_parts;
};

// act(g) and act'(g); FAST, for bf16 operands: through v_exp_f32 and v_rcp_f32 (an ulp each), gelu's erf by a polynomial that is off by up to 1.5e-7: gates
// under about -5, where gelu is smaller than that, keep its size and not its digits
template <bool FAST> __device__ __forceinline__ void gm_act(int act, float g, float& a, float& da) {
  if (act == FC_ACT_SILU) {
    const float s = FAST ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f)) : 1.f / (1.f + expf(-g));
    a = g * s;
    da = s * (1.f + g * (1.f - s));
  } else if (FAST) {
    float cdf, pdf;
    gelu_fast_parts(g, cdf, pdf);
    a = g * cdf;
    da = cdf + g * pdf;
  } else {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752440f));
    a = g * cdf;
    da = cdf + g * expf(-0.5f * g * g) * 0.39894228040143267794f;
  }
}

template <class S, int NPROD>
__device__ __forceinline__ void gm_gate_up(const GmArgs& a, char* smem, ft_f4 (&acc)[S::NI][S::NJ], const FtTile& t, int wave, int lane) {
  constexpr int WC = S::NJ * 16, HC = WC / 2;            // columns of a wave: HC gate rows and the HC up rows of the same units
  const int wm = wave / S::WN, wn = wave % S::WN, m0 = t.m * S::TM, f0 = t.n * (S::TN / 2);
  FtPipe<S, TK, TK> pipe(smem);
  pipe.sa.init(a.x, m0, a.D, wave, lane, [&](int r) { return m0 + r < a.T ? (long)m0 + r : -1L; });
  pipe.sb.init(a.w_in, f0, a.D, wave, lane, [&](int r) {
    const int in = r % WC, f = f0 + (r / WC) * HC + in % HC;
    return f < a.F ? (long)f + (in < HC ? 0 : a.up) : -1L;
  });
  ft_zero(acc);
  pipe.fill(0);
  pipe.run(0, (a.D + 63) / 64, acc);
  pipe.drain();
}

// Planes of h, dg and du: fp32's three; bf16's one, each value rounded once to bf16, which is half of a result's error (2.35e-3 in norm, 1.66e-3 without);
// two (16 bits of mantissa) for up to 32 rows, whose products read the weights once all the same: there the second plane costs no time.
template <class S, int NPROD> constexpr int gm_planes() { return NPROD == 6 ? 3 : S::TM == 32 ? 2 : 1; }
// one row block of values, J columns of 16, into the planes' LDS images
template <class S, int NPROD>
__device__ __forceinline__ void gm_put(char* img, int i, const ft_f4 (&v)[S::NJ / 2], int wm, int wn, int lane) {
  constexpr int J = S::NJ / 2, FC = S::TN / 2, IMG = S::TM * FC * 2;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int r = (wm * S::NI + i) * 16 + (lane & 15), c = wn * J * 16 + 16 * j + 4 * (lane >> 4);
    constexpr int PL = gm_planes<S, NPROD>();
    if (PL == 1) {
      ft_img_put<FC>(img, r, c, v[j][0], v[j][1], v[j][2], v[j][3]);
    } else {
      float h[3][4];
#pragma unroll
      for (int x = 0; x < 4; ++x) ft_split(v[j][x], h[0][x], h[1][x], h[2][x]);
#pragma unroll
      for (int p = 0; p < PL; ++p) ft_img_put<FC>(img + p * IMG, r, c, h[p][0], h[p][1], h[p][2], h[p][3]);
    }
  }
}
// the planes' images to the columns f0.. of rows of `ld` values
template <class S, int NPROD> __device__ __forceinline__ void gm_out(const char* img, bf16_t* out, long plane, long ld, const GmArgs& a, int m0, int f0) {
  constexpr int FC = S::TN / 2, IMG = S::TM * FC * 2;
  const FtRows rows;
#pragma unroll
  for (int p = 0; p < gm_planes<S, NPROD>(); ++p) ft_img_out<S::TM, FC, S::NT>(img + p * IMG, out + p * plane, ld, m0, f0, a.T, (int)a.ldh, rows, true);
}

// GRAD: the backward's pass over the same product.  (The large tile with its 128 accumulators, dh and the activation's values takes all 256 registers and
// spills 144 bytes a lane: 1307 us of the 6600 of 8192 x 4096 x 11000.)
template <class S, int NPROD, bool GRAD>
__global__ void __launch_bounds__(S::NT, S::NT == 512 ? 2 : 1) k_gm_act(GmArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int J = S::NJ / 2, FC = S::TN / 2, SET = gm_planes<S, NPROD>() * S::TM * FC * 2;     // bytes of an output's images
  constexpr bool TURN = 2 * SET <= S::LDS;                                                      // room for two outputs' in turn
  static_assert(SET <= S::LDS, "an output's images fit");
  const int wave = ft_wave(), lane = threadIdx.x & 63, wm = wave / S::WN, wn = wave % S::WN;
  const FtTile t = ft_tile((a.T + S::TM - 1) / S::TM, (a.F + FC - 1) / FC, 1, blockIdx.x);
  if (!t.any) return;
  const int m0 = t.m * S::TM, f0 = t.n * FC;
  ft_f4 acc[S::NI][S::NJ];
  gm_gate_up<S, NPROD>(a, smem, acc, t, wave, lane);
#pragma unroll
  for (int i = 0; i < S::NI; ++i) {
    ft_f4 h[J], d[J];
    if (GRAD) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int m = m0 + (wm * S::NI + i) * 16 + (lane & 15), f = f0 + wn * J * 16 + 16 * j + 4 * (lane >> 4);
        const bool in = m < a.T && f < a.ldd;                   // (ldd is F in whole eights)
        const float* at = a.dh + (in ? (long)m * a.ldd + f : 0);
        ft_f4 v = *(const ft_f4*)at;
        if (S::TM < 256)                                        // (the large tile's registers are full, and its products are long enough unsliced)
          for (int q = 1; q < a.dh_parts; ++q) v += *(const ft_f4*)(at + (long)q * a.T * a.ldd);
#pragma unroll
        for (int x = 0; x < 4; ++x) d[j][x] = in && f + x < a.F ? v[x] : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float v, dv;
        const float u = acc[i][j + J][x];
        gm_act<NPROD == 1>(a.act, acc[i][j][x], v, dv);
        if (GRAD) {
          acc[i][j][x] = d[j][x] * u * dv;
          acc[i][j + J][x] = d[j][x] * v;
        }
        h[j][x] = v * u;
      }
    gm_put<S, NPROD>(smem, i, h, wm, wn, lane);
    if (GRAD && (i & 1)) __builtin_amdgcn_sched_barrier(0);      // two rows' loads at a time: all of them together do not fit the registers
  }
  ft_barrier();
  gm_out<S, NPROD>(smem, a.h, a.T * a.ldh, a.ldh, a, m0, f0);
  if (GRAD) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      char* img = smem + (TURN ? (q ^ 1) * SET : 0);
      if (!TURN) ft_barrier();
#pragma unroll
      for (int i = 0; i < S::NI; ++i) {
        ft_f4 v[J];
#pragma unroll
        for (int j = 0; j < J; ++j) v[j] = acc[i][j + q * J];
        gm_put<S, NPROD>(img, i, v, wm, wn, lane);
      }
      ft_barrier();
      gm_out<S, NPROD>(img, a.dgu + q * a.ldh, a.T * 2 * a.ldh, 2 * a.ldh, a, m0, f0);
    }
  }
}

// The same from partial sums of [g | u] (few tiles and a long reduction, which then runs in slices): eight lanes share eight units of a row,
// each with every eighth slice.  PL: planes of h, dg and du.
struct GmJoin {
  GmArgs a;
  const float* gu;
  long ldp;
  int parts;
};
__device__ __forceinline__ void gm_sum8(const float* p, long step, int parts, int q0, int cols, float (&v)[8]) {
#pragma unroll
  for (int x = 0; x < 8; ++x) v[x] = 0.f;
#pragma unroll 2
  for (int q = q0; q < parts; q += 8)
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < cols) v[x] += p[q * step + x];
#pragma unroll
  for (int o = 1; o < 8; o *= 2)
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] += __shfl_xor(v[x], o, 64);
}
template <int PL> __device__ __forceinline__ void gm_store8(bf16_t* o, long plane, const float (&v)[8]) {
  float h[3][8];
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    if (PL == 1) h[0][x] = v[x]; else ft_split(v[x], h[0][x], h[1][x], h[2][x]);
  }
#pragma unroll
  for (int p = 0; p < PL; ++p) *(uint4*)(o + p * plane) = make_uint4(f2bf2(h[p][0], h[p][1]), f2bf2(h[p][2], h[p][3]), f2bf2(h[p][4], h[p][5]), f2bf2(h[p][6], h[p][7]));
}
template <int PL, bool GRAD> __global__ void __launch_bounds__(256) k_gm_join(GmJoin j) {
  const GmArgs& a = j.a;
  const long e = ((long)blockIdx.x * 256 + threadIdx.x) / 8, cw = a.ldh / 8, m = e / cw;
  const int q0 = threadIdx.x & 7, f = (int)(e - m * cw) * 8, cols = a.F - f;
  if (m >= a.T) return;
  float g[8], u[8], d[8];
  const float* at = j.gu + m * j.ldp + f;
  gm_sum8(at, a.T * j.ldp, j.parts, q0, cols, g);
  gm_sum8(at + a.F, a.T * j.ldp, j.parts, q0, cols, u);
  if (GRAD) gm_sum8(a.dh + m * a.ldd + f, a.T * a.ldd, a.dh_parts, q0, cols, d);
  if (q0) return;
  float h[8];
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    float v, dv;
    gm_act<PL != 3>(a.act, g[x], v, dv);
    h[x] = v * u[x];
    if (GRAD) {
      g[x] = d[x] * u[x] * dv;
      u[x] = d[x] * v;
    }
  }
  gm_store8<PL>(a.h + m * a.ldh + f, a.T * a.ldh, h);
  if (GRAD) {
    bf16_t* o = a.dgu + m * 2 * a.ldh + f;
    gm_store8<PL>(o, a.T * 2 * a.ldh, g);
    gm_store8<PL>(o + a.ldh, a.T * 2 * a.ldh, u);
  }
}

// ---------------------------------------------------------------- host
typedef FtShape<256, 256, 2, 4, 2> GmBig;
typedef FtShape<128, 128, 2, 2, 2> GmMid;
typedef FtShape<32, 64, 2, 2, 6> GmRow;
typedef FtShape<128, 128, 2, 4, 3, 32, 3> GmPlanes;
typedef FtShape<32, 64, 2, 2, 5, 32, 3, true> GmRows32;
typedef FtShape<128, 128, 2, 4, 3, 32, 3, true> GmMid32;

template <class S, int NPROD, bool GRAD> static int gm_act_launch(const GmArgs& a, hipStream_t s) {
  const long tiles = (long)((a.T + S::TM - 1) / S::TM) * ((a.F + S::TN / 2 - 1) / (S::TN / 2));
  FC_REQUIRE(tiles < (1L << 31), "gated_mlp: too many tiles");
  static FtLds lds;
  FC_TRY(lds.allow((const void*)k_gm_act<S, NPROD, GRAD>, S::LDS));
  hipLaunchKernelGGL((k_gm_act<S, NPROD, GRAD>), dim3((unsigned)tiles), dim3(S::NT), S::LDS, s, a);
  FC_LAUNCH_CHECK();
  return 0;
}
// 256 x 256 or 128 x 128 tiles by the model of the time, 32 x 64 (ft_few) for a few rows (forward, 12608 x 384 x 1024, 400
// large tiles: 55 us, 59 with 128 x 128; 2048 x 768 x 2048, 128 tiles: 46 and 42).  Backward: 256 x 256 only where the product is long; the epilogue
// (8 bytes a unit in, 6 out) stands still while it runs, and two 128 x 128 workgroups a CU cover each other's (12608 x 384 x 1024: 52 us against 70;
// 8192 x 4096 x 11000 the other way, 1571 against 1310)
static bool gm_big(int dt, long T, long D, long F, bool grad) { return dt && (!grad || D >= 1024) && ft_large(T, 2 * F, D); }
template <int NPROD, bool GRAD> static int gm_act_run(const GmArgs& a, hipStream_t s) {
  if constexpr (NPROD == 6) {
    return !a.b32 ? gm_act_launch<GmPlanes, NPROD, GRAD>(a, s) : ft_few(6, a.T) ? gm_act_launch<GmRows32, NPROD, GRAD>(a, s) : gm_act_launch<GmMid32, NPROD, GRAD>(a, s);
  } else {
    if (ft_few(1, a.T)) return gm_act_launch<GmRow, NPROD, GRAD>(a, s);
    if (gm_big(1, a.T, a.D, a.F, GRAD)) return gm_act_launch<GmBig, NPROD, GRAD>(a, s);
    return gm_act_launch<GmMid, NPROD, GRAD>(a, s);
  }
}

struct GmSizes { size_t x, w_in, w_out, dy, h, gu, dgu, dh, part; FtPlan plan_gu, plan_dh, plan[3]; bool group; };
// [g | u] in slices, where that is much faster by the model of the products' time (fp32, 45 x 3200 x 448: 41 us forward, 134 by whole tiles;
// bf16, 256 x 4096 x 1024: 39 and 57)
static FtProduct gm_gu_product(int dt, long T, long D, long F, bool b32) {
  FtProduct p;
  p.nprod = dt ? 1 : 6;
  p.b32 = b32;
  p.M = (int)T; p.N = (int)(2 * F); p.K = (int)D;
  return p;
}
template <bool GRAD> static int gm_act_any(const GmArgs& a, int dt, const FtPlan& gu, float* part, hipStream_t s) {
  if (!gu.target) return dt ? gm_act_run<1, GRAD>(a, s) : gm_act_run<6, GRAD>(a, s);
  FtProduct p = gm_gu_product(dt, a.T, a.D, a.F, a.b32);
  p.a = a.x;
  p.b = a.w_in;
  FC_TRY(ft_product(p, gu, part, false, s));
  GmJoin j;
  j.a = a; j.gu = part; j.ldp = ft_part_ld(p.N); j.parts = ft_parts(p, gu);
  const dim3 g((unsigned)((a.T * a.ldh + 255) / 256));
  if (!dt) hipLaunchKernelGGL((k_gm_join<3, GRAD>), g, dim3(256), 0, s, j);
  else if (a.T <= 32) hipLaunchKernelGGL((k_gm_join<2, GRAD>), g, dim3(256), 0, s, j);
  else hipLaunchKernelGGL((k_gm_join<1, GRAD>), g, dim3(256), 0, s, j);
  FC_LAUNCH_CHECK();
  return 0;
}

// bf16, few rows: h, dg and du are two planes, which are rows behind each other, of the result (y, dx) or of the reduction (dw_in, dw_out: one k-step)
static bool gm_two(int dt, long T) { return dt && T <= 32; }
// dx = [dg | du] w_in, dw_in = [dg | du]^T x, dw_out = dy^T h
static void gm_products(int dt, long T, long D, long F, const GmArgs& a, FtProduct (&p)[3]) {
  p[0].b32 = a.b32;
  const long Fp = ft_up(F, 64);
  for (FtProduct& q : p) { q.am = TR; q.bm = TR; q.nprod = dt ? 1 : 6; q.K = (int)T; }
  p[0].am = TK;
  p[0].M = (int)T; p[0].N = (int)D; p[0].K = (int)F;
  p[0].segs = 2; p[0].a2 = Fp; p[0].b2 = F * a.w_in.ld;
  p[0].a.p = p[1].a.p = a.dgu;
  p[0].a.ld = p[1].a.ld = 2 * Fp;
  p[0].a.plane = p[1].a.plane = T * 2 * Fp;
  p[0].b = a.w_in;
  p[1].M = (int)(2 * Fp); p[1].N = (int)D;
  if (Fp != F) { p[1].rows.half = (int)Fp; p[1].rows.to = (int)F; }
  p[1].b = a.x;
  p[2].M = (int)D; p[2].N = (int)F;
  p[2].a = a.dy;
  p[2].b.p = a.h; p[2].b.ld = Fp; p[2].b.plane = T * Fp;
  if (gm_two(dt, T)) {
    p[0].M = (int)(2 * T);
    p[0].fold = (int)T;
    p[1].K = p[2].K = (int)(2 * T);
    p[1].b.wrap = p[2].a.wrap = (int)T;
  }
}
// dh = dy w_out, whose slices' sums the activation's pass adds up
static FtProduct gm_dh_product(int dt, long T, long D, long F, bool b32) {
  FtProduct p;
  p.am = TK; p.bm = TR; p.nprod = dt ? 1 : 6; p.b32 = b32;
  p.M = (int)T; p.N = (int)F; p.K = (int)D;
  return p;
}
static FtProduct gm_y_product(int dt, long T, long D, long F, bool b32) {
  FtProduct p;
  p.nprod = dt ? 1 : 6;
  p.b32 = b32;
  p.M = (int)T; p.N = (int)D; p.K = (int)F;
  if (gm_two(dt, T)) {
    p.M = (int)(2 * T);
    p.fold = (int)T;
  }
  return p;
}
// b32: fp32 weights read where they are; packed: what is not planes anyway is laid out
static GmSizes gm_sizes(int dt, long T, long D, long F, bool b32, bool packed, bool backward) {
  GmSizes z = {};
  const long Dp = ft_up(D, 64), Fp = ft_up(F, 64), e = dt ? 2 : 6, eh = dt && ft_few(1, T) ? 4 : e;
  if (packed || !dt) {
    z.x = ft_up(T * Dp * e, 256);
    z.dy = backward ? z.x : 0;
  }
  if (dt ? packed : !b32) {
    z.w_in = ft_up(2 * F * Dp * e, 256);
    z.w_out = ft_up(D * Fp * e, 256);
  }
  z.h = ft_up(T * Fp * eh, 256);
  z.plan_gu = ft_plan(gm_gu_product(dt, T, D, F, b32), false);
  if (z.plan_gu.gain < 1.3) z.plan_gu.target = 0;
  z.gu = z.plan_gu.target ? ft_up(ft_part_floats(T, 2 * F, z.plan_gu) * 4, 256) : 0;
  if (!backward) {
    z.part = ft_product_part_floats(gm_y_product(dt, T, D, F, b32)) * 4;
    return z;
  }
  z.dgu = ft_up(T * 2 * Fp * eh, 256);
  z.plan_dh = ft_plan(gm_dh_product(dt, T, D, F, b32), false);
  if (gm_big(dt, T, D, F, true) && !z.plan_gu.target) z.plan_dh.target = 0;
  z.dh = ft_up(ft_part_floats(T, F, z.plan_dh) * 4, 256);
  FtProduct p[3];
  GmArgs a = {};
  a.b32 = b32;
  gm_products(dt, T, D, F, a, p);
  z.group = ft_group_plan(p, 3, z.plan);
  for (int i = 0; i < 3; ++i) {
    if (z.group) {
      z.part += z.plan[i].target ? ft_up(ft_part_floats(p[i].M, p[i].N, z.plan[i]) * 4, 256) : 0;
    } else {
      const size_t n = ft_product_part_floats(p[i]) * 4;
      z.part = z.part > n ? z.part : n;
    }
  }
  return z;
}
static size_t gm_total(const GmSizes& z) { return z.x + z.w_in + z.w_out + z.dy + z.h + z.gu + z.dgu + z.dh + z.part; }

// a matrix as the products take it: where it is, or as one of the packs
static void gm_matrix(int dt, bool b32, const void* p, long ld, long R, long C, char*& ws, FtMat& m, FtPacks& l) {
  if (b32) {
    m = ft_mat32(p, ld, R, C);
    return;
  }
  if (ft_direct(dt, p, ld, C)) {
    m.p = (const bf16_t*)p;
    m.ld = ld;
    return;
  }
  FtPack k;
  k.src = p; k.lds = ld; k.dt = dt; k.R = R; k.C = C; k.dst = (bf16_t*)ws; k.ldd = ft_up(C, 64);
  m.p = k.dst; m.ld = k.ldd; m.plane = R * k.ldd;
  ws += ft_up((dt ? 2 : 6) * R * k.ldd, 256);
  l.add(k);
}
struct GmCall { int dt, act; long T, D, F; const void *x, *w_in, *w_out, *dy; long ldx, ld_in, ld_out, lddy; };
static int gm_check(const char* what, const GmCall& c, const void* ws) {
  FC_REQUIRE(c.dt == FC_PREC_FP32 || c.dt == FC_PREC_BF16, "%s: dt %d", what, c.dt);
  FC_REQUIRE(c.act == FC_ACT_SILU || c.act == FC_ACT_GELU, "%s: activation %d", what, c.act);
  FC_REQUIRE(c.T >= 0 && c.T <= (1L << 28) && c.D >= 1 && c.F >= 1 && c.D <= (1L << 18) && c.F <= (1L << 20), "%s: bad sizes (%ld rows, width %ld, hidden %ld)", what,
             c.T, c.D, c.F);
  FC_REQUIRE(c.w_in && c.w_out && ws && (c.x || c.T == 0), "%s: null pointer", what);
  FC_REQUIRE(c.ldx >= c.D && c.ld_in >= c.D && c.ld_out >= c.F && c.ldx < (1L << 21) && c.ld_in < (1L << 21) && c.ld_out < (1L << 21), "%s: row strides %ld, %ld, %ld", what,
             c.ldx, c.ld_in, c.ld_out);
  FC_REQUIRE((c.F + 512) * (c.ld_in > c.D + 64 ? c.ld_in : c.D + 64) < (1L << 30), "%s: the up rows are past a tile load's reach (%ld x %ld)", what, c.F, c.ld_in);
  FC_REQUIRE(((size_t)ws & 255) == 0, "%s: the workspace is aligned to 256 bytes", what);
  return ft_check_device(c.w_in, what);
}
static bool gm_direct(const GmCall& c) {
  return ft_direct(c.dt, c.x, c.ldx, c.D) && ft_direct(c.dt, c.w_in, c.ld_in, c.D) && ft_direct(c.dt, c.w_out, c.ld_out, c.F) &&
         (!c.dy || ft_direct(c.dt, c.dy, c.lddy, c.D));
}
// fp32, few rows: both weights are read where they are, where the up rows are within a tile load's reach
static bool gm_b32(const GmCall& c) {
  return ft_b32(c.dt, c.T, c.w_in, c.ld_in) && ft_b32(c.dt, c.T, c.w_out, c.ld_out) && (c.F + 512) * c.ld_in < (1L << 29);
}
// the operands as the products take them; what of them cannot be taken as it is goes to the workspace
static int gm_operands(const GmCall& c, char*& ws, GmArgs& a, hipStream_t s) {
  a.b32 = gm_b32(c);
  a.T = (int)c.T; a.D = (int)c.D; a.F = (int)c.F; a.act = c.act; a.up = c.F; a.ldh = ft_up(c.F, 64);
  FtPacks l;
  gm_matrix(c.dt, false, c.x, c.ldx, c.T, c.D, ws, a.x, l);
  if (c.dy) gm_matrix(c.dt, false, c.dy, c.lddy, c.T, c.D, ws, a.dy, l);
  gm_matrix(c.dt, a.b32, c.w_out, c.ld_out, c.D, c.F, ws, a.w_out, l);
  gm_matrix(c.dt, a.b32, c.w_in, c.ld_in, 2 * c.F, c.D, ws, a.w_in, l);
  return ft_pack(l, s);
}

extern "C" int32_t fc_gated_mlp_form(int32_t dt, int32_t T, int32_t D, int32_t F, int32_t packed, int32_t backward) {
  if (T < 1 || D < 1 || F < 1) return 0;
  const bool b32 = !dt && !packed && T <= FT_B32;
  const GmSizes z = gm_sizes(dt, T, D, F, b32, packed || F % 8 || D % 8, backward != 0);
  const int group = z.group ? FC_FORM_GROUP : 0;
  if (z.plan_gu.target) return z.plan_gu.TM | FC_FORM_SLICED | group;
  if (dt ? ft_few(1, T) : b32 && ft_few(6, T)) return 32 | group;
  return (gm_big(dt, T, D, F, backward != 0) ? 256 : 128) | group;
}
extern "C" size_t fc_gated_mlp_workspace_bytes(int32_t dt, int32_t T, int32_t D, int32_t F, int32_t packed, int32_t backward) {
  if (T < 0 || D < 1 || F < 1) return 0;
  const bool few = !dt && T <= FT_B32;
  const size_t n = gm_total(gm_sizes(dt, T, D, F, few, packed || F % 8 || D % 8, backward != 0)) + 256;
  if (!few || !packed) return n;
  const size_t planes = gm_total(gm_sizes(dt, T, D, F, false, true, backward != 0)) + 256;      // (weights said to be packed may still be read in place)
  return n > planes ? n : planes;
}
extern "C" int fc_gated_mlp_fwd(int32_t dt, int32_t act, const void* x, int64_t ldx, const void* w_in, int64_t ld_in, const void* w_out, int64_t ld_out,
                                int32_t T, int32_t D, int32_t F, void* y, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
  GmCall c = {dt, act, T, D, F, x, w_in, w_out, nullptr, ldx, ld_in, ld_out, 0};
  FC_TRY(gm_check("fc_gated_mlp_fwd", c, workspace));
  FC_REQUIRE((y || T == 0) && ldy >= D, "fc_gated_mlp_fwd: output missing or its rows %ld apart", (long)ldy);
  const GmSizes z = gm_sizes(dt, T, D, F, gm_b32(c), !gm_direct(c), false);
  FC_REQUIRE(workspace_bytes >= gm_total(z), "fc_gated_mlp_fwd: workspace too small");
  if (T == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  GmArgs a = {};
  FC_TRY(gm_operands(c, ws, a, s));
  a.h = (bf16_t*)ws;
  ws += z.h;
  FC_TRY(gm_act_any<false>(a, dt, z.plan_gu, (float*)ws, s));
  ws += z.gu;
  FtProduct p = gm_y_product(dt, T, D, F, a.b32);
  p.a.p = a.h; p.a.ld = a.ldh; p.a.plane = (long)T * a.ldh;
  p.b = a.w_out;
  p.out = y; p.ldo = ldy;
  return ft_product_out(p, (float*)ws, z.part / 4, s);
}
extern "C" int fc_gated_mlp_bwd(int32_t dt, int32_t act, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w_in, int64_t ld_in,
                                const void* w_out, int64_t ld_out, int32_t T, int32_t D, int32_t F, void* dx, int64_t lddx, void* dw_in,
                                int64_t ldd_in, void* dw_out, int64_t ldd_out, void* workspace, size_t workspace_bytes, void* stream) {
  GmCall c = {dt, act, T, D, F, x, w_in, w_out, dy, ldx, ld_in, ld_out, lddy};
  FC_TRY(gm_check("fc_gated_mlp_bwd", c, workspace));
  FC_REQUIRE((dy || T == 0) && lddy >= D && lddy < (1L << 21) && (!dx || lddx >= D) && (!dw_in || ldd_in >= D) && (!dw_out || ldd_out >= F),
             "fc_gated_mlp_bwd: dy missing, or rows too close");
  const GmSizes z = gm_sizes(dt, T, D, F, gm_b32(c), !gm_direct(c), true);
  FC_REQUIRE(workspace_bytes >= gm_total(z), "fc_gated_mlp_bwd: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  GmArgs a = {};
  FC_TRY(gm_operands(c, ws, a, s));
  a.h = (bf16_t*)ws;
  ws += z.h;
  float* gu = (float*)ws;
  ws += z.gu;
  a.dgu = (bf16_t*)ws;
  ws += z.dgu;
  char* part = ws + z.dh;
  if (T) {
    FtProduct p = gm_dh_product(dt, T, D, F, a.b32);
    p.a = a.dy;
    p.b = a.w_out;
    FC_TRY(ft_product(p, z.plan_dh, (float*)ws, false, s));
    a.dh_parts = ft_parts(p, z.plan_dh);
    a.dh = (const float*)ws;
    a.ldd = ft_part_ld(F);
    FC_TRY(gm_act_any<true>(a, dt, z.plan_gu, gu, s));
  }
  FtProduct p[3], q[3];
  FtPlan plan[3];
  float* at[3];
  FtSums sums;
  int n = 0;
  gm_products(dt, T, D, F, a, p);
  p[0].out = T ? dx : nullptr; p[0].ldo = lddx;
  p[1].out = dw_in; p[1].ldo = ldd_in;
  p[2].out = dw_out; p[2].ldo = ldd_out;
  for (int i = 0; i < 3; ++i) {
    if (!p[i].out) continue;
    if (!z.group) {
      FC_TRY(ft_product_out(p[i], (float*)part, z.part / 4, s));
      continue;
    }
    q[n] = p[i];
    plan[n] = z.plan[i];
    at[n] = z.plan[i].target ? (float*)part : nullptr;
    if (at[n]) {
      sums.add(q[n], plan[n], at[n], nullptr, q[n].fold ? q[n].fold : q[n].M);
      part += ft_up(ft_part_floats(q[n].M, q[n].N, plan[n]) * 4, 256);
    }
    ++n;
  }
  if (!n) return 0;
  FC_TRY(ft_group(q, plan, n, at, s));
  return ft_reduce(sums, s);
}
