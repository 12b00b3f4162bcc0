// Softmax cross entropy of a linear layer over a large vocabulary, the logits not kept (but for a few rows, whose logits are little).
//
//   L[t, v] = x[t] . w[v];   lse[t] = log sum_v exp L[t, v];   row[t] = lse[t] - L[t, y[t]]      (0 where y[t] is the ignored index)
//   dL[t, v] = (exp(L[t, v] - lse[t]) - [v = y[t]]) g[t];      dx = dL w;   dw = dL^T x
//
// Forward: rows that count are gathered once (aligned; three bf16 planes for fp32), so ignored rows cost no products and what they hold
// touches nothing.  One tiled product; each tile leaves its columns' maximum and sum of exponentials per row, and the target's logit,
// behind (8 bytes for TN logits); a second pass joins them.  Backward: the logits are formed again in pieces of the vocabulary, dL of a
// piece goes to the workspace in the operands' precision, and two products read it.  That is 8 T V D operations for 6 T V D; keeping the
// exponentials instead costs another rounding (their sum is not known yet when they are stored) or 8 bytes a logit of traffic, more than
// the 2 D operations they save up to D of about 1500.  A piece's dL (<= 192 MB) is written once and read twice.
// Everything is added in a fixed order; nothing is zero-filled by a memset.
#include <math.h>

#include "../../include/fedcola_hip.h"
#include "fc_tiles.h"

#define CE_LOG2E 1.4426950408889634f

// ---- what the forward leaves for the backward, at the caller's address
struct CeSaved {
  int* n;          // rows that count
  int *pos, *idx, *y;   // row -> place among them or -1; place -> row; place -> target, -1 for one outside of the vocabulary
  float* lse;      // [place]
  FtMat x;         // gathered rows
  float* logits;   // [place][ldg] where they are kept, else null
  long ldg;
  size_t bytes;
};
// columns of the vocabulary in a piece: what dL of T rows takes stays under 192 MB, in whole 256-column tiles
static long ce_piece(int dt, long T, long V) {
  const long most = (192L << 20) / ((T ? T : 1) * (dt ? 2 : 6)) / 256 * 256, all = ft_up(V, 256);
  return most < 256 ? 256 : most < all ? most : all;
}
// The logits of a few rows are little beside the weight, which forming them again would read once more (1 x 3648 x 59042 fp32 with gradients: 625 us,
// 1017 without this and the outer product of fc_tiles.hip): up to 32 rows, and up to 128 while they are an eighth of it.
static bool ce_keep(int dt, long T, long V, long D) {
  return T > 0 && (T <= 32 || (T <= 128 && T * 32 <= D * (dt ? 2 : 4))) && T * ft_up(V, 8) <= (1L << 25) && ce_piece(dt, T, V) >= V;
}
static CeSaved ce_saved(void* base, int dt, long T, long V, long D) {
  CeSaved s;
  char* p = (char*)base;
  const long ld = ft_up(D, 64), t4 = ft_up(T * 4, 256);
  s.n = (int*)p;
  s.pos = (int*)(p + 256);
  s.idx = (int*)(p + 256 + t4);
  s.y = (int*)(p + 256 + 2 * t4);
  s.lse = (float*)(p + 256 + 3 * t4);
  s.x.p = (bf16_t*)(p + 256 + 4 * t4);
  s.x.ld = ld;
  s.x.plane = T * ld;
  s.bytes = 256 + 4 * t4 + ft_up((dt ? 1 : 3) * T * ld * 2, 256);
  const bool keep = ce_keep(dt, T, V, D);
  s.ldg = ft_up(V, 8);
  s.logits = keep ? (float*)(p + s.bytes) : nullptr;
  s.bytes += keep ? T * s.ldg * 4 : 0;
  return s;
}

// ---- which rows count, and their copies.  Workgroup b takes rows [b R, (b + 1) R) after counting the targets before them.
template <typename T, int PL>
__global__ void __launch_bounds__(256) k_ce_rows(const T* x, long ldx, const int64_t* y, long T_, int R, int V, int64_t ignore, int D, bool vec, CeSaved s) {
  __shared__ int red[4], src[64];
  const int tid = threadIdx.x, lane = tid & 63;
  const long r0 = (long)blockIdx.x * R, r1 = r0 + R < T_ ? r0 + R : T_;
  int c = 0;
  for (long i = tid; i < r0; i += 256) c += y[i] != ignore;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
  if (lane == 0) red[tid >> 6] = c;
  __syncthreads();
  int at = red[0] + red[1] + red[2] + red[3];
  const int cw = (int)(s.x.ld / 8);
  for (long b = r0; b < r1; b += 64) {
    const long r = b + lane;
    const int64_t t = r < r1 ? y[r] : ignore;
    const bool on = r < r1 && t != ignore;
    const unsigned long long m = __ballot(on);
    const int k = __popcll(m & ((1ull << lane) - 1)), n = __popcll(m);
    if (tid < 64) {
      if (r < r1) s.pos[r] = on ? at + k : -1;
      if (on) {
        s.idx[at + k] = (int)r;
        s.y[at + k] = t >= 0 && t < V ? (int)t : -1;
        src[k] = (int)(r - b);
      }
    }
    __syncthreads();
    for (int e = tid; e < n * cw; e += 256) {
      const int i = e / cw, c0 = (e - i * cw) * 8;
      const T* p = x + (b + src[i]) * ldx + c0;
      bf16_t* d = (bf16_t*)s.x.p + (long)(at + i) * s.x.ld + c0;
      if (PL == 1 && vec) {                                    // (D in whole chunks; the row's padding is zeros, and nothing behind its D values is read)
        *(uint4*)d = c0 < D ? *(const uint4*)p : make_uint4(0, 0, 0, 0);
        continue;
      }
      float v[8], h[3][8];
      ft_row8(p, D - c0, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (PL == 1) h[0][j] = v[j]; else ft_split(v[j], h[0][j], h[1][j], h[2][j]);
      }
#pragma unroll
      for (int q = 0; q < PL; ++q)
        *(uint4*)(d + q * s.x.plane) = make_uint4(f2bf2(h[q][0], h[q][1]), f2bf2(h[q][2], h[q][3]), f2bf2(h[q][4], h[q][5]), f2bf2(h[q][6], h[q][7]));
    }
    at += n;
    __syncthreads();
  }
  if (r1 == T_ && tid == 0) *s.n = at;
}

// exp(v - m): through v_exp_f32 for bf16 operands, whose logits carry 2^-9 each; expf for fp32
template <int NPROD> __device__ __forceinline__ float ce_exp(float v, float m) {
  return NPROD == 1 ? __builtin_amdgcn_exp2f((v - m) * CE_LOG2E) : expf(v - m);
}
struct CePart { float m, s; };   // maximum, and sum of exp(. - maximum)
template <int NPROD> __device__ __forceinline__ CePart ce_join(CePart a, CePart b) {
  CePart r;
  r.m = fmaxf(a.m, b.m);
  // a side without a finite or infinite maximum holds nothing, unless it holds NaN in its sum
  const float x = a.m == r.m ? 1.f : ce_exp<NPROD>(a.m, r.m), y = b.m == r.m ? 1.f : ce_exp<NPROD>(b.m, r.m);
  r.s = a.s * x + b.s * y;
  return r;
}

struct CeArgs {
  FtMat x, w;
  bool b32;                   // fp32: w is the fp32 matrix itself
  int T, V, D, v0, nv;        // this launch's columns [v0, v0 + nv) of the vocabulary
  const int *n, *y, *idx;
  CePart* part;               // [tiles of columns][T]
  float* tlogit;              // [T]
  float* logits;              // [T][ldg], where they are kept
  long ldg;
  const float *lse, *g;
  int reduction;
  bf16_t* dl;                 // planes of [T][ldl]
  long ldl, plane;
};

// the tiles of a workgroup: the product's in turn, epilogue(tile, acc, pipe) after each
template <class S, class F> __device__ __forceinline__ void ce_tiles(const CeArgs& a, char* smem, int M, F epilogue) {
  const int tm = (M + S::TM - 1) / S::TM, tn = (a.nv + S::TN - 1) / S::TN, nk = (a.D + 63) / 64;
  int b = blockIdx.x;
  FtTile t = ft_tile(tm, tn, 1, b);
  if (!t.any) return;
  FtPipe<S, TK, TK> pipe(smem);
  auto go = [&](const FtTile& u) {
    const int m0 = u.m * S::TM, n0 = a.v0 + u.n * S::TN, lane = ft_fresh(pipe.lane);
    pipe.sa.init(a.x, m0, a.D, pipe.wave, lane, [&](int r) { return m0 + r < M ? (long)m0 + r : -1L; });
    pipe.sb.init(a.w, n0, a.D, pipe.wave, lane, [&](int r) { return n0 + r < a.V ? (long)n0 + r : -1L; });
  };
  go(t);
  pipe.fill(0);
  for (;;) {
    ft_f4 acc[S::NI][S::NJ];
    ft_zero(acc);
    const FtTile u = ft_tile(tm, tn, 1, b += gridDim.x);
    pipe.run(0, nk, acc, [&] {
      if (u.any) { go(u); pipe.seek(0); }
    });
    epilogue(t, acc, pipe);
    if (!u.any) break;
    t = u;
  }
  pipe.drain();
}

template <class S> constexpr int ce_red_bytes() { return S::WN * S::TM * (int)sizeof(CePart); }
template <class S, int NPROD>
__global__ void __launch_bounds__(S::NT, S::NT == 512 ? 2 : 1) k_ce_stats(CeArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int M = min(a.T, *a.n);
  CePart* red = (CePart*)(smem + S::LDS);                // [WN][TM]
  ce_tiles<S>(a, smem, M, [&](const FtTile& t, ft_f4 (&acc)[S::NI][S::NJ], auto& pipe) {
    const int lane = ft_fresh(pipe.lane), wm = pipe.wm, wn = pipe.wn, g = lane >> 4, m0 = t.m * S::TM, n0 = t.n * S::TN + wn * S::NJ * 16;
    const bool edge = n0 + S::NJ * 16 > a.V;
#pragma unroll
    for (int i = 0; i < S::NI; ++i) {
      const int r = (wm * S::NI + i) * 16 + (lane & 15), m = m0 + r;
      if (edge)
#pragma unroll
        for (int j = 0; j < S::NJ; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (n0 + 16 * j + 4 * g + x >= a.V) acc[i][j][x] = -__builtin_inff();
      if constexpr (S::TM < 256)                                                // (the few rows whose logits are kept never take the large tiles)
        if (a.logits && m < M)
#pragma unroll
          for (int j = 0; j < S::NJ; ++j)
            if (n0 + 16 * j + 4 * g < a.ldg) *(ft_f4*)(a.logits + m * a.ldg + n0 + 16 * j + 4 * g) = acc[i][j];
      CePart p;
      p.m = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < S::NJ; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) p.m = fmaxf(p.m, acc[i][j][x]);
      p.m = fmaxf(p.m, __shfl_xor(p.m, 16, 64));
      p.m = fmaxf(p.m, __shfl_xor(p.m, 32, 64));
      p.s = 0.f;
      // a maximum of -inf: columns past the vocabulary alone, logits of -inf, or NaN, which fmaxf leaves out and the sum must not
      const float base = p.m == -__builtin_inff() ? 0.f : p.m;
#pragma unroll
      for (int j = 0; j < S::NJ; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) p.s += ce_exp<NPROD>(acc[i][j][x], base);
      p.s += __shfl_xor(p.s, 16, 64);
      p.s += __shfl_xor(p.s, 32, 64);
      if (g == 0) red[wn * S::TM + r] = p;
      const int rel = (m < M ? a.y[m] : -1) - n0;          // the target's logit, where this wave holds it
      if (rel >= 0 && rel < S::NJ * 16 && ((rel >> 2) & 3) == g) {
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < S::NJ; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (16 * j + x == (rel & ~12)) v = acc[i][j][x];
        a.tlogit[m] = v;
      }
    }
    ft_barrier();
    pipe.settle();
    for (int r = pipe.wave * 64 + lane; r < S::TM; r += S::NT)
      if (m0 + r < M) {
        CePart p = red[r];
#pragma unroll
        for (int q = 1; q < S::WN; ++q) p = ce_join<NPROD>(p, red[q * S::TM + r]);
        a.part[(long)t.n * a.T + m0 + r] = p;
      }
  });
}

// joins the tiles' partial sums: ROWS rows a workgroup, 256 / ROWS lanes a row (16: whole lines of neighbouring rows; 1: a scoring call's few rows)
template <int NPROD, int ROWS>
__global__ void __launch_bounds__(256) k_ce_join(const CePart* part, int tiles, const float* tlogit, CeSaved s, float* rows, long T) {
  constexpr int LANES = 256 / ROWS;
  __shared__ CePart red[LANES][ROWS];
  const int r = threadIdx.x % ROWS, q = threadIdx.x / ROWS;
  const long t = (long)blockIdx.x * ROWS + r;
  const int at = t < T ? s.pos[t] : -1;
  CePart p = {-__builtin_inff(), 0.f};
  if (at >= 0)
#pragma unroll 4
    for (int i = q; i < tiles; i += LANES) p = ce_join<NPROD>(p, part[(long)i * T + at]);
  red[q][r] = p;
  __syncthreads();
  if (q < 16 && LANES > 16) {
#pragma unroll
    for (int i = 1; i < LANES / 16; ++i) p = ce_join<NPROD>(p, red[q + 16 * i][r]);
    red[q][r] = p;
  }
  if (LANES > 16) __syncthreads();
  if (q == 0 && t < T) {
#pragma unroll
    for (int i = 1; i < 16; ++i) p = ce_join<NPROD>(p, red[i][r]);
    float l = 0.f;
    if (at >= 0) {
      const bool in = s.y[at] >= 0;
      const float lse = in ? p.m + logf(p.s) : __builtin_nanf("");   // a target outside of the vocabulary: NaN, in the loss and in the gradients
      s.lse[at] = lse;
      l = in ? lse - tlogit[at] : lse;
    }
    rows[t] = l;
  }
}
// sum or mean of the rows, in fp64 and in one order
__global__ void __launch_bounds__(1024) k_ce_loss(const float* rows, long T, const int* n, int reduction, float* loss) {
  __shared__ double red[16];
  double v = 0;
  for (long i = threadIdx.x; i < T; i += 1024) v += (double)rows[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) v += red[i];
    *loss = (float)(reduction == FC_REDUCE_MEAN ? v / (double)*n : v);    // no row counts: 0 / 0, NaN, as torch's mean
  }
}

// dL of the tile's logits, rounded once to the operands' precision.  A factor that all rows share (g, g / count) is applied to the products'
// results instead: multiplied in here, it gives the targets' entries, which are all close to -1, all the same rounding error.
template <class S> constexpr int ce_img_bytes() { return 16 * S::NJ * 16 * 2; }         // of a wave: 16 rows
template <class S, int NPROD>
__global__ void __launch_bounds__(S::NT, S::NT == 512 ? 2 : 1) k_ce_grad(CeArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int W = S::NJ * 16;
  const int M = min(a.T, *a.n);
  ce_tiles<S>(a, smem, M, [&](const FtTile& t, ft_f4 (&acc)[S::NI][S::NJ], auto& pipe) {
    const int lane = ft_fresh(pipe.lane), g = lane >> 4, m0 = t.m * S::TM + pipe.wm * S::NI * 16, c0 = t.n * S::TN + pipe.wn * W, n0 = a.v0 + c0;
    char* img = smem + S::LDS + pipe.wave * ce_img_bytes<S>();
#pragma unroll
    for (int i = 0; i < S::NI; ++i) {
      const int m = m0 + i * 16 + (lane & 15);
      const bool live = m < M;
      const float lse = live ? a.lse[m] : 0.f;
      const int rel = (live ? a.y[m] : -1) - n0 - 4 * g;
      const float sc = live && a.reduction == FC_REDUCE_NONE ? a.g[a.idx[m]] : 1.f;
#pragma unroll
      for (int j = 0; j < S::NJ; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float p = ce_exp<NPROD>(acc[i][j][x], lse);
          if (rel == 16 * j + x) p -= 1.f;
          acc[i][j][x] = live && n0 + 16 * j + 4 * g + x < a.V ? p * sc : 0.f;
        }
      if (i == 0) pipe.settle();
#pragma unroll
      for (int pl = 0; pl < (NPROD == 1 ? 1 : 3); ++pl) {
#pragma unroll
        for (int j = 0; j < S::NJ; ++j) {
          float v[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if (NPROD == 1) { v[x] = acc[i][j][x]; continue; }
            float h[3];
            ft_split(acc[i][j][x], h[0], h[1], h[2]);
            v[x] = h[pl];
          }
          ft_wimg_put<W>(img, lane & 15, 16 * j + 4 * g, v[0], v[1], v[2], v[3]);
        }
        ft_wimg_out<W>(img, a.dl + pl * a.plane, a.ldl, m0 + i * 16, c0, M, (int)a.ldl, lane);
      }
    }
  });
}

// ---- few tiles and a long reduction: the logits come as fp32 partial sums of slices of it, for the rows really there
struct CeSlices {
  const float* part;            // [slices][M][ldp]
  long ldp, K;
  int target, TM, TN, nprod;
  __device__ __forceinline__ int count(int M, int V) const { return ft_slices((long)((M + TM - 1) / TM) * ((V + TN - 1) / TN), K, target, nprod); }
  __device__ __forceinline__ ft_f4 at(long row, int col, int M, int slices) const {
    const float* p = part + row * ldp + col;
    ft_f4 v = *(const ft_f4*)p;
#pragma unroll 4
    for (int q = 1; q < slices; ++q) v += *(const ft_f4*)(p + (long)q * M * ldp);
    return v;
  }
};
// a workgroup a row: log-sum-exp and loss
template <int NPROD>
__global__ void __launch_bounds__(256) k_ce_row(CeSlices l, int V, CeSaved s, float* rows) {
  __shared__ CePart red[4];
  __shared__ float target;
  const long t = blockIdx.x;
  const int at = s.pos[t], tid = threadIdx.x, M = *s.n;
  if (at < 0) {
    if (tid == 0) rows[t] = 0.f;
    return;
  }
  const int y = s.y[at], slices = l.count(M, V);
  if (tid == 0) target = __builtin_nanf("");             // a target outside of the vocabulary: NaN, in the loss and in the gradients
  __syncthreads();
  CePart p = {-__builtin_inff(), 0.f};
  for (int c = tid * 4; c < V; c += 1024) {
    const ft_f4 v = l.at(at, c, M, slices);
    if (s.logits) *(ft_f4*)(s.logits + at * s.ldg + c) = v;
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (c + x < V) {
        p = ce_join<NPROD>(p, CePart{v[x], 1.f});
        if (c + x == y) target = v[x];
      }
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) p = ce_join<NPROD>(p, CePart{__shfl_xor(p.m, o, 64), __shfl_xor(p.s, o, 64)});
  if ((tid & 63) == 0) red[tid >> 6] = p;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int i = 1; i < 4; ++i) p = ce_join<NPROD>(p, red[i]);
    const float lse = y >= 0 ? p.m + logf(p.s) : target;
    s.lse[at] = lse;
    rows[t] = lse - target;
  }
}
// dL, eight columns a lane
template <int NPROD> __global__ void __launch_bounds__(256) k_ce_dl(CeSlices l, CeArgs a) {
  const int M = min(a.T, *a.n), cw = (a.V + 7) / 8;
  const long e = (long)blockIdx.x * 256 + threadIdx.x, m = e / cw;
  const int c0 = (int)(e - m * cw) * 8;
  if (m >= M) return;
  const int slices = l.count(M, a.V);
  const ft_f4 v[2] = {l.at(m, c0, M, slices), l.at(m, c0 + 4, M, slices)};
  const float lse = a.lse[m], sc = a.reduction == FC_REDUCE_NONE ? a.g[a.idx[m]] : 1.f;
  const int y = a.y[m];
  float h[3][8];
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    float p = ce_exp<NPROD>(v[x >> 2][x & 3], lse);
    if (c0 + x == y) p -= 1.f;
    p = c0 + x < a.V ? p * sc : 0.f;
    if (NPROD == 1) h[0][x] = p; else ft_split(p, h[0][x], h[1][x], h[2][x]);
  }
#pragma unroll
  for (int q = 0; q < (NPROD == 1 ? 1 : 3); ++q)
    *(uint4*)(a.dl + q * a.plane + m * a.ldl + c0) = make_uint4(f2bf2(h[q][0], h[q][1]), f2bf2(h[q][2], h[q][3]), f2bf2(h[q][4], h[q][5]), f2bf2(h[q][6], h[q][7]));
}

// ---------------------------------------------------------------- host
typedef FtShape<256, 256, 2, 4, 2> CeBig;
typedef FtShape<128, 128, 2, 2, 2> CeMid;
typedef FtShape<32, 64, 2, 2, 6> CeRow;
typedef FtShape<128, 128, 2, 4, 3, 32, 3> CePlanes;
typedef FtShape<32, 64, 2, 2, 5, 32, 3, true> CeRows32;
typedef FtShape<128, 128, 2, 4, 3, 32, 3, true> CeMid32;
// 256 x 256 or 128 x 128 tiles by the model of the time (forward, 768 wide: 512 x 32768 36 us, 42 with 128 x 128; 256 x 32768 32 and 27.5; of 13 sizes
// around the border it takes the faster every time), 128 x 128 for fp32, 32 x 64 (ft_few) for the few rows of a scoring call.  Kept logits are
// written by tiles of up to 128 rows alone, whatever the model says of the large ones.
static int ce_shape(int dt, long T, long V, long D, bool b32) {
  if ((dt || b32) && ft_few(dt ? 1 : 6, T)) return 2;
  return dt && !ce_keep(dt, T, V, D) && ft_large(T, V, D) ? 0 : 1;
}
static int ce_tn(int shape) { return shape == 0 ? 256 : shape == 1 ? 128 : 64; }

template <class S, int NPROD, bool GRAD> static int ce_launch(const CeArgs& a, hipStream_t s) {
  const long tiles = (long)((a.T + S::TM - 1) / S::TM) * ((a.nv + S::TN - 1) / S::TN);
  FC_REQUIRE(tiles < (1L << 31), "linear_ce: too many tiles");
  const dim3 g((unsigned)ft_walkers<S>(tiles, a.D));
  if (GRAD) {
    constexpr int bytes = S::LDS + S::NW * ce_img_bytes<S>();
    static FtLds lds;
    FC_TRY(lds.allow((const void*)k_ce_grad<S, NPROD>, bytes));
    hipLaunchKernelGGL((k_ce_grad<S, NPROD>), g, dim3(S::NT), bytes, s, a);
  } else {
    constexpr int bytes = S::LDS + ce_red_bytes<S>();
    static FtLds lds;
    FC_TRY(lds.allow((const void*)k_ce_stats<S, NPROD>, bytes));
    hipLaunchKernelGGL((k_ce_stats<S, NPROD>), g, dim3(S::NT), bytes, s, a);
  }
  FC_LAUNCH_CHECK();
  return 0;
}
template <bool GRAD> static int ce_run(int dt, int shape, const CeArgs& a, hipStream_t s) {
  if (a.T == 0 || a.nv == 0) return 0;
  if (dt) return shape == 0 ? ce_launch<CeBig, 1, GRAD>(a, s) : shape == 1 ? ce_launch<CeMid, 1, GRAD>(a, s) : ce_launch<CeRow, 1, GRAD>(a, s);
  return shape != 1 ? ce_launch<CeRows32, 6, GRAD>(a, s) : a.b32 ? ce_launch<CeMid32, 6, GRAD>(a, s) : ce_launch<CePlanes, 6, GRAD>(a, s);
}

static FtProduct ce_logits(int dt, long T, long V, long D, bool b32, const int* n) {
  FtProduct p;
  p.nprod = dt ? 1 : 6;
  p.b32 = b32;
  p.M = (int)T; p.N = (int)V; p.K = (int)D; p.Mdyn = n;
  return p;
}
static CeSlices ce_slices(const FtProduct& p, const FtPlan& plan, const float* part) {
  CeSlices l;
  l.part = part; l.ldp = ft_part_ld(p.N); l.K = p.K; l.target = plan.target; l.TM = plan.TM; l.TN = plan.TN; l.nprod = p.nprod;
  return l;
}
struct CeSizes { size_t w, part, rows, dl, dxp, dwp; long piece; FtPlan logits, dx, dw; bool group; };
// dx = dL w and dw = dL^T x of nv columns; n: device, the rows that count
static void ce_products(int dt, long T, long D, long nv, bool b32, const int* n, FtProduct& x, FtProduct& w) {
  x.am = TK; x.bm = TR; x.nprod = dt ? 1 : 6; x.b32 = b32; x.M = (int)T; x.N = (int)D; x.K = (int)nv; x.Mdyn = n;
  w.am = TR; w.bm = TR; w.nprod = x.nprod; w.M = (int)nv; w.N = (int)D; w.K = (int)T; w.Kdyn = n;
}
static CeSizes ce_sizes(int dt, long T, long V, long D, bool direct_w, bool grad) {
  CeSizes z = {};
  const bool b32 = !dt && direct_w;
  z.w = direct_w ? 0 : (size_t)ft_up((dt ? 2 : 6) * V * ft_up(D, 64), 256);
  // slices pay where the model of the products' time says so by much (122 x 2263 x 326 fp32: 38 us forward, 115 by whole tiles; 64 x 4096 x 1000
  // bf16: 23 and 31), and where the logits are one piece
  z.piece = ce_piece(dt, T, V);
  z.logits = ft_plan(ce_logits(dt, T, V, D, b32, nullptr), false);
  if (z.logits.gain < 1.3 || z.piece < V || (grad && ce_keep(dt, T, V, D))) z.logits.target = 0;
  if (z.logits.target) z.part = (size_t)ft_up(ft_part_floats(T, V, z.logits) * 4, 256);
  if (!grad) {
    const int tn = ce_tn(ce_shape(dt, T, V, D, b32));
    if (!z.logits.target) z.part = (size_t)ft_up((V + tn - 1) / tn * T * (long)sizeof(CePart), 256);
    z.rows = (size_t)ft_up(T * 4, 256) * 2;
    return z;
  }
  z.dl = (size_t)ft_up((dt ? 1 : 3) * T * z.piece * 2, 256);
  if (z.piece >= V) {                     // one piece: its two products may run together
    FtProduct p[2];
    FtPlan plan[2];
    ce_products(dt, T, D, V, b32, nullptr, p[0], p[1]);
    if (ft_group_plan(p, 2, plan)) {
      z.group = true;
      z.dx = plan[0];
      z.dw = plan[1];
      z.dxp = (size_t)ft_up(ft_part_floats(T, D, z.dx) * 4, 256);
      z.dwp = z.dw.target ? (size_t)ft_up(ft_part_floats(V, D, z.dw) * 4, 256) : 0;
      return z;
    }
  }
  FtProduct px, pw;
  ce_products(dt, T, D, z.piece, b32, nullptr, px, pw);
  z.dx = ft_plan(px, true);
  z.dxp = (size_t)ft_up(ft_part_floats(T, D, z.dx) * 4, 256);
  for (long nv : {z.piece < V ? z.piece : V, V % z.piece}) {
    pw.M = (int)nv;
    const size_t n = nv ? (size_t)ft_up(ft_product_part_floats(pw) * 4, 256) : 0;
    z.dwp = z.dwp > n ? z.dwp : n;
  }
  return z;
}
static int ce_args(const char* what, int dt, long T, long V, long D, long ldw, const void* w) {
  FC_REQUIRE(dt == FC_PREC_FP32 || dt == FC_PREC_BF16, "%s: dt %d", what, dt);
  FC_REQUIRE(T >= 0 && T <= (1L << 28) && V >= 1 && V <= (1L << 30) && D >= 1 && D <= (1L << 20), "%s: bad sizes (%ld rows, %ld classes, width %ld)", what, T, V, D);
  FC_REQUIRE(w && ldw >= D && ldw < (1L << 21), "%s: weight missing or its rows %ld apart", what, ldw);
  return ft_check_device(w, what);
}
// the weight as the products take it: where it is, or laid out in the workspace
static bool ce_direct(int dt, const void* w, long ldw, long T, long D) { return dt ? ft_direct(dt, w, ldw, D) : ft_b32(dt, T, w, ldw); }
static int ce_weight(int dt, const void* w, long ldw, bool direct, long V, long D, char*& ws, FtMat& m, hipStream_t s) {
  if (direct) {
    if (dt) { m.p = (const bf16_t*)w; m.ld = ldw; } else { m = ft_mat32(w, ldw, V, D); }
    return 0;
  }
  FtPack k;
  k.src = w; k.lds = ldw; k.dt = dt; k.R = V; k.C = D; k.dst = (bf16_t*)ws; k.ldd = ft_up(D, 64);
  m.p = k.dst; m.ld = k.ldd; m.plane = V * k.ldd;
  ws += (size_t)ft_up((dt ? 2 : 6) * V * k.ldd, 256);
  FtPacks l;
  l.add(k);
  return ft_pack(l, s);
}

template <class S> static bool ce_walks(long T, long nv, long D) {
  const long tiles = ((T + S::TM - 1) / S::TM) * ((nv + S::TN - 1) / S::TN);
  return ft_walkers<S>(tiles, D) < tiles;
}
extern "C" int32_t fc_linear_ce_form(int32_t dt, int32_t T, int32_t V, int32_t D, int32_t packed, int32_t backward) {
  if (T < 1 || V < 1 || D < 1) return 0;
  if (backward && ce_keep(dt, T, V, D)) return FC_FORM_KEPT;
  const bool direct = !packed && (dt || T <= FT_B32), b32 = !dt && direct;
  const CeSizes z = ce_sizes(dt, T, V, D, direct, backward != 0);
  if (z.logits.target) return z.logits.TM | FC_FORM_SLICED;
  const long nv = backward && z.piece < V ? z.piece : V;
  const int shape = ce_shape(dt, T, nv, D, b32);
  const bool walk = shape == 0 ? ce_walks<CeBig>(T, nv, D) : shape == 2 ? false : dt ? ce_walks<CeMid>(T, nv, D) : b32 ? ce_walks<CeMid32>(T, nv, D) : ce_walks<CePlanes>(T, nv, D);
  return (shape == 0 ? 256 : shape == 1 ? 128 : 32) | (walk ? FC_FORM_WALK : 0) | (nv < V ? FC_FORM_PIECES : 0);
}
extern "C" size_t fc_linear_ce_saved_bytes(int32_t dt, int32_t T, int32_t V, int32_t D) {
  return T < 0 || V < 1 || D < 1 ? 0 : ce_saved(nullptr, dt, T, V, D).bytes;
}
extern "C" size_t fc_linear_ce_workspace_bytes(int32_t dt, int32_t T, int32_t V, int32_t D, int32_t packed, int32_t backward) {
  if (T < 0 || V < 1 || D < 1) return 0;
  size_t most = 0;
  for (bool direct : {false, true}) {                 // (a weight said to be packed may still be read in place)
    if (!packed && !direct && (dt || T <= FT_B32)) continue;
    if (direct && !dt && T > FT_B32) continue;
    const CeSizes z = ce_sizes(dt, T, V, D, direct, backward != 0);
    const size_t n = z.w + z.part + z.rows + z.dl + z.dxp + z.dwp + 256;
    most = most > n ? most : n;
  }
  return most;
}
extern "C" int fc_linear_ce_fwd(int32_t dt, const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* y, int32_t T, int32_t V, int32_t D,
                                int64_t ignore_index, int32_t reduction, float* loss, void* saved, size_t saved_bytes, void* workspace,
                                size_t workspace_bytes, void* stream) {
  FC_TRY(ce_args("fc_linear_ce_fwd", dt, T, V, D, ldw, w));
  FC_REQUIRE(reduction >= FC_REDUCE_NONE && reduction <= FC_REDUCE_SUM, "fc_linear_ce_fwd: reduction %d", reduction);
  FC_REQUIRE((loss || (T == 0 && reduction == FC_REDUCE_NONE)) && saved && workspace && ((x && y && ldx >= D) || T == 0), "fc_linear_ce_fwd: null pointer, or rows %ld apart", (long)ldx);
  FC_REQUIRE((((size_t)saved | (size_t)workspace) & 255) == 0, "fc_linear_ce_fwd: saved and workspace are aligned to 256 bytes");
  const CeSaved sv = ce_saved(saved, dt, T, V, D);
  const bool direct = ce_direct(dt, w, ldw, T, D);
  const CeSizes z = ce_sizes(dt, T, V, D, direct, false);
  FC_REQUIRE(saved_bytes >= sv.bytes && workspace_bytes >= z.w + z.part + z.rows, "fc_linear_ce_fwd: saved or workspace too small");
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  CeArgs a = {};
  FC_TRY(ce_weight(dt, w, ldw, direct, V, D, ws, a.w, s));
  a.x = sv.x;
  a.b32 = !dt && direct;
  a.T = T; a.V = V; a.D = D; a.v0 = 0; a.nv = V;
  a.n = sv.n; a.y = sv.y; a.idx = sv.idx;
  a.logits = sv.logits; a.ldg = sv.ldg;
  a.part = (CePart*)ws;
  a.tlogit = (float*)(ws + z.part);
  float* rows = reduction == FC_REDUCE_NONE ? loss : (float*)(ws + z.part + z.rows / 2);
  // 16 rows a workgroup, more where its count of the targets before it would cost more than the copy
  const int R = (int)ft_up(T > 16384 ? (T + 1023) / 1024 : 16, 16), blocks = T ? (T + R - 1) / R : 1;
  if (dt) {
    const bool vec = ft_direct(1, x, ldx, D);
    hipLaunchKernelGGL((k_ce_rows<bf16_t, 1>), dim3(blocks), dim3(256), 0, s, (const bf16_t*)x, (long)ldx, y, (long)T, R, V, ignore_index, D, vec, sv);
  } else {
    hipLaunchKernelGGL((k_ce_rows<float, 3>), dim3(blocks), dim3(256), 0, s, (const float*)x, (long)ldx, y, (long)T, R, V, ignore_index, D, false, sv);
  }
  FC_LAUNCH_CHECK();
  if (z.logits.target) {
    FtProduct p = ce_logits(dt, T, V, D, a.b32, sv.n);
    p.a = a.x;
    p.b = a.w;
    FC_TRY(ft_product(p, z.logits, (float*)ws, false, s));
    const CeSlices l = ce_slices(p, z.logits, (const float*)ws);
    if (dt) hipLaunchKernelGGL(k_ce_row<1>, dim3(T), dim3(256), 0, s, l, V, sv, rows);
    else hipLaunchKernelGGL(k_ce_row<6>, dim3(T), dim3(256), 0, s, l, V, sv, rows);
    FC_LAUNCH_CHECK();
  } else {
    const int shape = ce_shape(dt, T, V, D, a.b32), tn = ce_tn(shape), tiles = (V + tn - 1) / tn;
    FC_TRY(ce_run<false>(dt, shape, a, s));
    if (T) {
      const dim3 gj((unsigned)(T <= 64 ? T : (T + 15) / 16));
      if (dt && T <= 64) hipLaunchKernelGGL((k_ce_join<1, 1>), gj, dim3(256), 0, s, a.part, tiles, a.tlogit, sv, rows, (long)T);
      else if (dt) hipLaunchKernelGGL((k_ce_join<1, 16>), gj, dim3(256), 0, s, a.part, tiles, a.tlogit, sv, rows, (long)T);
      else if (T <= 64) hipLaunchKernelGGL((k_ce_join<6, 1>), gj, dim3(256), 0, s, a.part, tiles, a.tlogit, sv, rows, (long)T);
      else hipLaunchKernelGGL((k_ce_join<6, 16>), gj, dim3(256), 0, s, a.part, tiles, a.tlogit, sv, rows, (long)T);
      FC_LAUNCH_CHECK();
    }
  }
  if (reduction != FC_REDUCE_NONE) {
    hipLaunchKernelGGL(k_ce_loss, dim3(1), dim3(1024), 0, s, rows, (long)T, sv.n, reduction, loss);
    FC_LAUNCH_CHECK();
  }
  return 0;
}
extern "C" int fc_linear_ce_bwd(int32_t dt, const void* w, int64_t ldw, int32_t T, int32_t V, int32_t D, int32_t reduction, const float* gloss,
                                const void* saved, size_t saved_bytes, void* dx, int64_t lddx, void* dw, int64_t lddw, void* workspace,
                                size_t workspace_bytes, void* stream) {
  FC_TRY(ce_args("fc_linear_ce_bwd", dt, T, V, D, ldw, w));
  FC_REQUIRE((gloss || T == 0) && saved && workspace && (!dx || lddx >= D) && (!dw || lddw >= D), "fc_linear_ce_bwd: null pointer, or an output's rows too close");
  FC_REQUIRE(reduction >= FC_REDUCE_NONE && reduction <= FC_REDUCE_SUM, "fc_linear_ce_bwd: reduction %d", reduction);
  FC_REQUIRE((((size_t)saved | (size_t)workspace) & 255) == 0, "fc_linear_ce_bwd: saved and workspace are aligned to 256 bytes");
  const CeSaved sv = ce_saved((void*)saved, dt, T, V, D);
  const bool direct = ce_direct(dt, w, ldw, T, D);
  const CeSizes z = ce_sizes(dt, T, V, D, direct, true);
  FC_REQUIRE(saved_bytes >= sv.bytes && workspace_bytes >= z.w + z.part + z.dl + z.dxp + z.dwp, "fc_linear_ce_bwd: saved or workspace too small");
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  CeArgs a = {};
  FC_TRY(ce_weight(dt, w, ldw, direct, V, D, ws, a.w, s));
  a.x = sv.x;
  a.b32 = !dt && direct;
  a.T = T; a.V = V; a.D = D;
  a.n = sv.n; a.y = sv.y; a.idx = sv.idx;
  a.lse = sv.lse; a.g = gloss; a.reduction = reduction;
  float* part = (float*)ws;
  ws += z.part;
  a.dl = (bf16_t*)ws;
  a.ldl = z.piece;
  a.plane = (long)T * z.piece;
  float* dxp = (float*)(ws + z.dl);
  float* dwp = (float*)(ws + z.dl + z.dxp);
  const int es = dt ? 2 : 4;
  FtProduct px, pw;
  ce_products(dt, T, D, z.piece, a.b32, sv.n, px, pw);
  px.out = dx; px.ldo = lddx;
  px.a.p = a.dl; px.a.ld = a.ldl; px.a.plane = a.plane;
  pw.a = px.a;
  pw.b = sv.x;
  pw.ldo = lddw;
  if (reduction != FC_REDUCE_NONE) {
    px.alpha = pw.alpha = gloss;
    if (reduction == FC_REDUCE_MEAN) px.alpha_over = pw.alpha_over = sv.n;
  }
  for (long v0 = 0; v0 < V; v0 += z.piece) {
    a.v0 = (int)v0;
    a.nv = (int)(V - v0 < z.piece ? V - v0 : z.piece);
    if (z.logits.target || sv.logits) {
      FtProduct p = ce_logits(dt, T, V, D, a.b32, sv.n);
      p.a = a.x;
      p.b = a.w;
      if (!sv.logits) FC_TRY(ft_product(p, z.logits, part, false, s));
      const CeSlices l = ce_slices(p, z.logits, sv.logits ? sv.logits : part);
      const dim3 g((unsigned)(((long)T * ((V + 7) / 8) + 255) / 256));
      if (dt) hipLaunchKernelGGL(k_ce_dl<1>, g, dim3(256), 0, s, l, a);
      else hipLaunchKernelGGL(k_ce_dl<6>, g, dim3(256), 0, s, l, a);
      FC_LAUNCH_CHECK();
    } else {
      FC_TRY(ce_run<true>(dt, ce_shape(dt, T, a.nv, D, a.b32), a, s));
    }
    if (z.group) {
      px.K = pw.M = a.nv;
      px.b = a.w;
      pw.out = dw;
      FtProduct p[2];
      FtPlan plan[2];
      float* part[2];
      FtSums l;
      int n = 0;
      if (dx && T) {
        p[n] = px; plan[n] = z.dx; part[n++] = dxp;
        l.add(px, z.dx, dxp, sv.pos, T);
      }
      if (dw) {
        p[n] = pw; plan[n] = z.dw; part[n++] = z.dw.target ? dwp : nullptr;
        if (z.dw.target) l.add(pw, z.dw, dwp, nullptr, V);
      }
      if (!n) return 0;
      FC_TRY(ft_group(p, plan, n, part, s));
      return ft_reduce(l, s);
    }
    px.Ks = (int)z.piece;
    if (dw) {
      pw.M = a.nv;
      pw.out = (char*)dw + v0 * lddw * es;
      FC_TRY(ft_product_out(pw, dwp, z.dwp / 4, s));
    }
    if (dx && T) {
      px.K = a.nv;
      px.b = a.w;
      px.b.p = a.w.p + v0 * a.w.ld;
      FC_TRY(ft_product(px, z.dx, dxp, v0 > 0, s));
    }
  }
  if (dx && T) FC_TRY(ft_reduce(px, z.dx, dxp, sv.pos, T, s));
  return 0;
}
