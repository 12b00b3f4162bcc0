// Gated feed-forward block:  [g | u] = x w_in^T;  h = act(g) u;  y = h w_out^T     (w_in [2 F, D]: gate rows, then up rows; w_out [D, F])
//
// Forward: one product computes both projections -- a tile's columns are gate and up rows of the same hidden units, interleaved by half a
// wave's columns, so that g and u of a unit are in one lane -- and its epilogue applies the activation and the product; h is all that
// reaches memory.  A second product gives y.
// Backward: nothing but the inputs is kept.  One kernel forms g and u again and, on the same tile, dh = dy w_out, and writes
//   h = act(g) u,   dg = dh u act'(g),   du = dh act(g)
// each rounded once from 32 bits; then dx = [dg | du] w_in, dw_in = [dg | du]^T x, dw_out = dy^T h.  That is 16 T D F operations for the
// 12 of a backward pass that reads g and u back; these would have to be stored in 32 bits (16 bytes a hidden unit to write and read, as
// much time as the 4 D operations at D of about 1000) or rounded once more than here.
#include <math.h>

#include "../../include/fedcola_hip.h"
#include "fc_tiles.h"

struct GmArgs {
  FtMat x, w_in, w_out, dy;
  int T, D, F, act;
  long up;                      // rows between a unit's gate and up row in w_in
  bf16_t *h, *dgu;              // planes of [T][ldh], [T][2 ldh]: h; dg | du
  long ldh;
};

// act(g) and act'(g); FAST: through v_exp_f32 and v_rcp_f32, for bf16 operands
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
  FtStager<TK, S::TM, S::NW> sa;
  FtStager<TK, S::TN, S::NW> sb;
  sa.init(a.x, m0, a.D, wave, lane, [&](int r) { return m0 + r < a.T ? (long)m0 + r : -1L; });
  sb.init(a.w_in, f0, a.D, wave, lane, [&](int r) {
    const int in = r % WC, f = f0 + (r / WC) * HC + in % HC;
    return f < a.F ? (long)f + (in < HC ? 0 : a.up) : -1L;
  });
#pragma unroll
  for (int i = 0; i < S::NI; ++i)
#pragma unroll
    for (int j = 0; j < S::NJ; ++j) acc[i][j] = ft_f4{0.f, 0.f, 0.f, 0.f};
  ft_loop<S, TK, TK, NPROD, S::NJ>(sa, sb, smem, 0, (a.D + 63) / 64, acc, wm, wn, wave, lane);
}

// one plane of v[i][j], the values of S::TM rows and S::TN / 2 units, as an LDS image
template <class S, int NPROD, int J>
__device__ __forceinline__ void gm_image(char* img, const ft_f4 (&v)[S::NI][J], int pl, int wm, int wn, int lane) {
#pragma unroll
  for (int i = 0; i < S::NI; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float o[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (NPROD == 1) { o[x] = v[i][j][x]; continue; }
        float h[3];
        ft_split(v[i][j][x], h[0], h[1], h[2]);
        o[x] = h[pl];
      }
      ft_img_put<S::TN / 2>(img, (wm * S::NI + i) * 16 + (lane & 15), wn * J * 16 + 16 * j + 4 * (lane >> 4), o[0], o[1], o[2], o[3]);
    }
}

template <class S, int NPROD>
__global__ void __launch_bounds__(S::NT, S::NT == 512 ? 2 : 1) k_gm_act(GmArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int wave = ft_wave(), lane = threadIdx.x & 63, wm = wave / S::WN, wn = wave % S::WN;
  const FtTile t = ft_tile((a.T + S::TM - 1) / S::TM, (a.F + S::TN / 2 - 1) / (S::TN / 2), 1);
  if (!t.any) return;
  ft_f4 acc[S::NI][S::NJ], h[S::NI][S::NJ / 2];
  gm_gate_up<S, NPROD>(a, smem, acc, t, wave, lane);
#pragma unroll
  for (int i = 0; i < S::NI; ++i)
#pragma unroll
    for (int j = 0; j < S::NJ / 2; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float v, dv;
        gm_act<NPROD == 1>(a.act, acc[i][j][x], v, dv);
        h[i][j][x] = v * acc[i][j + S::NJ / 2][x];
      }
  const FtRows rows;
#pragma unroll
  for (int pl = 0; pl < (NPROD == 1 ? 1 : 3); ++pl) {
    if (pl) ft_barrier();
    gm_image<S, NPROD, S::NJ / 2>(smem, h, pl, wm, wn, lane);
    ft_barrier();
    ft_img_out<S::TM, S::TN / 2, S::NT>(smem, a.h + pl * a.T * a.ldh, a.ldh, t.m * S::TM, t.n * (S::TN / 2), a.T, (int)a.ldh, rows, true);
  }
}

template <class S, int NPROD>
__global__ void __launch_bounds__(S::NT, S::NT == 512 ? 2 : 1) k_gm_grad(GmArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int J = S::NJ / 2, FC = S::TN / 2;
  const int wave = ft_wave(), lane = threadIdx.x & 63, wm = wave / S::WN, wn = wave % S::WN;
  const FtTile t = ft_tile((a.T + S::TM - 1) / S::TM, (a.F + FC - 1) / FC, 1);
  if (!t.any) return;
  const int m0 = t.m * S::TM, f0 = t.n * FC;
  ft_f4 acc[S::NI][S::NJ], dh[S::NI][J];
  gm_gate_up<S, NPROD>(a, smem, acc, t, wave, lane);
  FtStager<TK, S::TM, S::NW> sa;
  FtStager<TR, FC, S::NW> sb;
  sa.init(a.dy, m0, a.D, wave, lane, [&](int r) { return m0 + r < a.T ? (long)m0 + r : -1L; });
  sb.init(a.w_out, f0, a.D, wave, lane, [&](int r) { return f0 + r < a.F ? (long)f0 + r : -1L; });
#pragma unroll
  for (int i = 0; i < S::NI; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) dh[i][j] = ft_f4{0.f, 0.f, 0.f, 0.f};
  ft_loop<S, TK, TR, NPROD, J>(sa, sb, smem, 0, (a.D + 63) / 64, dh, wm, wn, wave, lane);
#pragma unroll
  for (int i = 0; i < S::NI; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float v, dv;
        const float u = acc[i][j + J][x], d = dh[i][j][x];
        gm_act<NPROD == 1>(a.act, acc[i][j][x], v, dv);
        acc[i][j][x] = d * u * dv;
        acc[i][j + J][x] = d * v;
        dh[i][j][x] = v * u;
      }
  const FtRows rows;
  ft_f4 dv[S::NI][J];
#pragma unroll
  for (int pl = 0; pl < (NPROD == 1 ? 1 : 3); ++pl) {
    if (pl) ft_barrier();
    constexpr int IMG = S::TM * FC * 2;
    static_assert(3 * IMG <= S::LDS, "three images at once");
    gm_image<S, NPROD, J>(smem, dh, pl, wm, wn, lane);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int i = 0; i < S::NI; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j) dv[i][j] = acc[i][j + q * J];
      gm_image<S, NPROD, J>(smem + (1 + q) * IMG, dv, pl, wm, wn, lane);
    }
    ft_barrier();
    ft_img_out<S::TM, FC, S::NT>(smem, a.h + pl * a.T * a.ldh, a.ldh, m0, f0, a.T, (int)a.ldh, rows, true);
#pragma unroll
    for (int q = 0; q < 2; ++q)
      ft_img_out<S::TM, FC, S::NT>(smem + (1 + q) * IMG, a.dgu + pl * a.T * 2 * a.ldh + q * a.ldh, 2 * a.ldh, m0, f0, a.T, (int)a.ldh, rows, true);
  }
}

// ---------------------------------------------------------------- host
typedef FtShape<256, 256, 2, 4, 2> GmBig;
typedef FtShape<128, 128, 2, 2, 2> GmMid;
typedef FtShape<32, 64, 2, 2, 4> GmRow;
typedef FtShape<128, 256, 2, 4, 3> GmGrad;     // 144 KB; 64 + 32 accumulators a lane

template <class S, int NPROD> static int gm_act_launch(const GmArgs& a, hipStream_t s) {
  const long tiles = (long)((a.T + S::TM - 1) / S::TM) * ((a.F + S::TN / 2 - 1) / (S::TN / 2));
  FC_REQUIRE(tiles < (1L << 31), "gated_mlp: too many tiles");
  FC_TRY(ft_allow_lds((const void*)k_gm_act<S, NPROD>, S::LDS));
  hipLaunchKernelGGL((k_gm_act<S, NPROD>), dim3((unsigned)tiles), dim3(S::NT), S::LDS, s, a);
  FC_LAUNCH_CHECK();
  return 0;
}
template <int NPROD> static int gm_act_run(const GmArgs& a, hipStream_t s) {
  if (a.T <= 32) return gm_act_launch<GmRow, NPROD>(a, s);
  if ((long)((a.T + 255) / 256) * ((a.F + 127) / 128) >= 128) return gm_act_launch<GmBig, NPROD>(a, s);
  return gm_act_launch<GmMid, NPROD>(a, s);
}
template <int NPROD> static int gm_grad_run(const GmArgs& a, hipStream_t s) {
  typedef GmGrad S;
  const long tiles = (long)((a.T + S::TM - 1) / S::TM) * ((a.F + S::TN / 2 - 1) / (S::TN / 2));
  FC_REQUIRE(tiles < (1L << 31), "gated_mlp: too many tiles");
  FC_TRY(ft_allow_lds((const void*)k_gm_grad<S, NPROD>, S::LDS));
  hipLaunchKernelGGL((k_gm_grad<S, NPROD>), dim3((unsigned)tiles), dim3(S::NT), S::LDS, s, a);
  FC_LAUNCH_CHECK();
  return 0;
}

struct GmSizes { size_t x, w_in, w_out, dy, h, dgu, part; };
static GmSizes gm_sizes(int dt, long T, long D, long F, bool packed, bool backward) {
  GmSizes z = {};
  const long D8 = ft_up(D, 8), F8 = ft_up(F, 8), e = dt ? 2 : 6;
  const int np = dt ? 1 : 6;
  if (packed) {
    z.x = ft_up(T * D8 * e, 256);
    z.w_in = ft_up(2 * F8 * D8 * e, 256);
    z.w_out = ft_up(D * F8 * e, 256);
    z.dy = backward ? z.x : 0;
  }
  z.h = ft_up(T * F8 * e, 256);
  if (!backward) {
    z.part = ft_product_part_floats(TK, TK, np, T, D, F) * 4;
    return z;
  }
  z.dgu = ft_up(T * 2 * F8 * e, 256);
  const size_t a = ft_product_part_floats(TK, TR, np, T, D, 2 * F8), b = ft_product_part_floats(TR, TR, np, 2 * F8, D, T),
               c = ft_product_part_floats(TR, TR, np, D, F, T);
  z.part = 4 * (a > b ? a > c ? a : c : b > c ? b : c);
  return z;
}
static size_t gm_total(const GmSizes& z) { return z.x + z.w_in + z.w_out + z.dy + z.h + z.dgu + z.part; }

static int gm_matrix(int dt, const void* p, long ld, long R, long C, bool use_direct, char*& ws, FtMat& m, hipStream_t s) {
  if (use_direct) {
    m.p = (const bf16_t*)p;
    m.ld = ld;
    return 0;
  }
  FtPack k;
  k.src = p; k.lds = ld; k.dt = dt; k.R = R; k.C = C; k.dst = (bf16_t*)ws; k.ldd = ft_up(C, 8); k.Rd = R;
  m.p = k.dst; m.ld = k.ldd; m.plane = R * k.ldd;
  ws += ft_up((dt ? 1 : 3) * R * k.ldd * 2, 256);
  return ft_pack(k, s);
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
  FC_REQUIRE((c.F + 512) * (c.ld_in > c.D + 8 ? c.ld_in : c.D + 8) < (1L << 30), "%s: the up rows are past a tile load's reach (%ld x %ld)", what, c.F, c.ld_in);
  FC_REQUIRE(((size_t)ws & 255) == 0, "%s: the workspace is aligned to 256 bytes", what);
  return ft_check_device(c.w_in, what);
}
static bool gm_direct(const GmCall& c) {
  return ft_direct(c.dt, c.x, c.ldx, c.D) && ft_direct(c.dt, c.w_in, c.ld_in, c.D) && ft_direct(c.dt, c.w_out, c.ld_out, c.F) &&
         (!c.dy || ft_direct(c.dt, c.dy, c.lddy, c.D));
}
// the operands as the products take them; what of them cannot be taken as it is goes to the workspace
static int gm_operands(const GmCall& c, char*& ws, GmArgs& a, hipStream_t s) {
  const long F8 = ft_up(c.F, 8);
  a.T = (int)c.T; a.D = (int)c.D; a.F = (int)c.F; a.act = c.act;
  FC_TRY(gm_matrix(c.dt, c.x, c.ldx, c.T, c.D, ft_direct(c.dt, c.x, c.ldx, c.D), ws, a.x, s));
  if (c.dy) FC_TRY(gm_matrix(c.dt, c.dy, c.lddy, c.T, c.D, ft_direct(c.dt, c.dy, c.lddy, c.D), ws, a.dy, s));
  FC_TRY(gm_matrix(c.dt, c.w_out, c.ld_out, c.D, c.F, ft_direct(c.dt, c.w_out, c.ld_out, c.F), ws, a.w_out, s));
  if (ft_direct(c.dt, c.w_in, c.ld_in, c.D) && F8 == c.F) {
    a.w_in.p = (const bf16_t*)c.w_in;
    a.w_in.ld = c.ld_in;
    a.up = c.F;
  } else {     // halves of F8 rows, so that [dg | du] has 16-byte columns and meets w_in row by row
    FtPack k;
    k.src = c.w_in; k.lds = c.ld_in; k.dt = c.dt; k.R = 2 * c.F; k.C = c.D; k.dst = (bf16_t*)ws; k.ldd = ft_up(c.D, 8); k.Rd = 2 * F8; k.half = F8; k.to = c.F;
    a.w_in.p = k.dst; a.w_in.ld = k.ldd; a.w_in.plane = k.Rd * k.ldd;
    a.up = F8;
    ws += ft_up((c.dt ? 1 : 3) * k.Rd * k.ldd * 2, 256);
    FC_TRY(ft_pack(k, s));
  }
  a.ldh = F8;
  return 0;
}

extern "C" size_t fc_gated_mlp_workspace_bytes(int32_t dt, int32_t T, int32_t D, int32_t F, int32_t packed, int32_t backward) {
  if (T < 0 || D < 1 || F < 1) return 0;
  return gm_total(gm_sizes(dt, T, D, F, !dt || packed || F % 8 || D % 8, backward != 0)) + 256;
}
extern "C" int fc_gated_mlp_fwd(int32_t dt, int32_t act, const void* x, int64_t ldx, const void* w_in, int64_t ld_in, const void* w_out, int64_t ld_out,
                                int32_t T, int32_t D, int32_t F, void* y, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
  GmCall c = {dt, act, T, D, F, x, w_in, w_out, nullptr, ldx, ld_in, ld_out, 0};
  FC_TRY(gm_check("fc_gated_mlp_fwd", c, workspace));
  FC_REQUIRE((y || T == 0) && ldy >= D, "fc_gated_mlp_fwd: output missing or its rows %ld apart", (long)ldy);
  const GmSizes z = gm_sizes(dt, T, D, F, !gm_direct(c), false);
  FC_REQUIRE(workspace_bytes >= gm_total(z), "fc_gated_mlp_fwd: workspace too small");
  if (T == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  GmArgs a = {};
  FC_TRY(gm_operands(c, ws, a, s));
  a.h = (bf16_t*)ws;
  ws += z.h;
  FC_TRY(dt ? gm_act_run<1>(a, s) : gm_act_run<6>(a, s));
  FtProduct p;
  p.nprod = dt ? 1 : 6;
  p.a.p = a.h; p.a.ld = a.ldh; p.a.plane = (long)T * a.ldh;
  p.b = a.w_out;
  p.M = T; p.N = D; p.K = F; p.out = y; p.ldo = ldy;
  return ft_product_out(p, (float*)ws, z.part / 4, s);
}
extern "C" int fc_gated_mlp_bwd(int32_t dt, int32_t act, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w_in, int64_t ld_in,
                                const void* w_out, int64_t ld_out, int32_t T, int32_t D, int32_t F, void* dx, int64_t lddx, void* dw_in,
                                int64_t ldd_in, void* dw_out, int64_t ldd_out, void* workspace, size_t workspace_bytes, void* stream) {
  GmCall c = {dt, act, T, D, F, x, w_in, w_out, dy, ldx, ld_in, ld_out, lddy};
  FC_TRY(gm_check("fc_gated_mlp_bwd", c, workspace));
  FC_REQUIRE((dy || T == 0) && lddy >= D && lddy < (1L << 21) && (!dx || lddx >= D) && (!dw_in || ldd_in >= D) && (!dw_out || ldd_out >= F),
             "fc_gated_mlp_bwd: dy missing, or rows too close");
  const GmSizes z = gm_sizes(dt, T, D, F, !gm_direct(c), true);
  FC_REQUIRE(workspace_bytes >= gm_total(z), "fc_gated_mlp_bwd: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  GmArgs a = {};
  FC_TRY(gm_operands(c, ws, a, s));
  a.h = (bf16_t*)ws;
  ws += z.h;
  a.dgu = (bf16_t*)ws;
  ws += z.dgu;
  if (T) FC_TRY(dt ? gm_grad_run<1>(a, s) : gm_grad_run<6>(a, s));
  FtProduct p;
  p.nprod = dt ? 1 : 6;
  p.a.p = a.dgu; p.a.ld = 2 * a.ldh; p.a.plane = (long)T * 2 * a.ldh;
  if (dx && T) {
    p.am = TK; p.bm = TR;
    p.b = a.w_in;
    p.M = T; p.N = D; p.K = (int)(2 * a.ldh); p.out = dx; p.ldo = lddx;
    FC_TRY(ft_product_out(p, (float*)ws, z.part / 4, s));
  }
  p.am = TR; p.bm = TR;
  p.K = T;
  if (dw_in) {
    p.b = a.x;
    p.M = (int)(2 * a.ldh); p.N = D; p.out = dw_in; p.ldo = ldd_in;
    if (a.ldh != F) { p.rows.half = (int)a.ldh; p.rows.to = F; }
    FC_TRY(ft_product_out(p, (float*)ws, z.part / 4, s));
    p.rows = FtRows();
  }
  if (dw_out) {
    p.a = a.dy;
    p.b.p = a.h; p.b.ld = a.ldh; p.b.plane = (long)T * a.ldh;
    p.M = D; p.N = F; p.out = dw_out; p.ldo = ldd_out;
    FC_TRY(ft_product_out(p, (float*)ws, z.part / 4, s));
  }
  return 0;
}
