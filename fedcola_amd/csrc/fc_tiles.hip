// The plain tiled product of fc_tiles.h with its choice of tile and of slices of the reduction, the sum of the slices, and the packing
// of operands that the tile loads cannot take as they are.
#include "fc_tiles.h"

int ft_check_device(const void* p, const char* what) {
  hipPointerAttribute_t at;
  int cur = 0;
  if (!p) return 0;
  if (hipPointerGetAttributes(&at, p) != hipSuccess) { (void)hipGetLastError(); fc_set_error("%s: not a device pointer", what); return -1; }
  FC_CHECK_HIP(hipGetDevice(&cur));
  FC_REQUIRE(at.type == hipMemoryTypeDevice || at.type == hipMemoryTypeManaged, "%s: not a device pointer", what);
  FC_REQUIRE(at.device == cur, "%s: the buffers are on device %d, the current device is %d", what, at.device, cur);
  return 0;
}

// ---------------------------------------------------------------- packing
template <typename T, int PL>
__global__ void __launch_bounds__(256) k_ft_pack(FtPacks l) {
  const long e = (long)blockIdx.x * 256 + threadIdx.x;
  if (e >= l.first[l.n]) return;
  int w = 0;
#pragma unroll
  for (int i = 1; i < 4; ++i)
    if (i < l.n && e >= l.first[i]) w = i;
  FtPack a = l.p[0];
  long e0 = 0;
#pragma unroll
  for (int i = 1; i < 4; ++i)
    if (w == i) { a = l.p[i]; e0 = l.first[i]; }
  const long cw = a.ldd / 8, r = (e - e0) / cw;
  const int c0 = (int)(e - e0 - r * cw) * 8;
  float v[8];
  ft_row8((const T*)a.src + r * a.lds + c0, (int)(a.C - c0), v);
  float h[3][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (PL == 1) h[0][j] = v[j]; else ft_split(v[j], h[0][j], h[1][j], h[2][j]);
  }
#pragma unroll
  for (int p = 0; p < PL; ++p)
    *(uint4*)(a.dst + (size_t)p * a.R * a.ldd + r * a.ldd + c0) =
        make_uint4(f2bf2(h[p][0], h[p][1]), f2bf2(h[p][2], h[p][3]), f2bf2(h[p][4], h[p][5]), f2bf2(h[p][6], h[p][7]));
}
int ft_pack(const FtPacks& p, hipStream_t s) {
  const long n = p.first[p.n];
  if (n == 0) return 0;
  const dim3 g((unsigned)((n + 255) / 256));
  if (p.p[0].dt) hipLaunchKernelGGL((k_ft_pack<bf16_t, 1>), g, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((k_ft_pack<float, 3>), g, dim3(256), 0, s, p);
  FC_LAUNCH_CHECK();
  return 0;
}

typedef FtShape<256, 256, 2, 4, 2> FtBig;      // 128 KB of LDS, one workgroup a CU
typedef FtShape<128, 128, 2, 2, 2> FtMid;      // 64 KB, two
typedef FtShape<32, 64, 2, 2, 6> FtRow;        // 72 KB, two: few rows, the reading of B is what counts (TK x TK alone)
typedef FtShape<128, 128, 2, 4, 3, 32, 3> FtPlanes;          // fp32, all in planes: 144 KB, one workgroup of eight waves a CU
typedef FtShape<128, 128, 2, 4, 3, 32, 3, true> FtMid32;     // fp32, B in 32 bits: 120 KB
typedef FtShape<32, 64, 2, 2, 5, 32, 3, true> FtRows32;      // the same of few rows: 70 KB, two

// ---------------------------------------------------------------- the product
// workgroup b of a product: into p.out, or (part) as partial sums
template <class S, int AM, int BMO, int NPROD>
__device__ __forceinline__ void ft_product_tile(const FtProduct& p, float* part, int target, int add, int b, char* smem) {
  const int M = p.Mdyn ? min(p.M, *p.Mdyn) : p.M, K = p.Kdyn ? min(p.K, *p.Kdyn) : p.K, N = p.N;
  const int tm = (M + S::TM - 1) / S::TM, tn = (N + S::TN - 1) / S::TN, Ks = (p.Ks ? p.Ks : K) * p.segs, splits = ft_slices((long)tm * tn, Ks, target, NPROD);
  const FtTile t = ft_tile(tm, tn, splits, b);
  if (!t.any) return;
  FtPipe<S, AM, BMO> pipe(smem);
  const int wave = pipe.wave, lane = pipe.lane, wm = pipe.wm, wn = pipe.wn, m0 = t.m * S::TM, n0 = t.n * S::TN;
  pipe.sa.init(p.a, m0, K, wave, lane, [&](int r) { return m0 + r < M ? (long)m0 + r : -1L; });
  pipe.sb.init(p.b, n0, K, wave, lane, [&](int r) { return n0 + r < N ? (long)n0 + r : -1L; });
  ft_f4 acc[S::NI][S::NJ];
  ft_zero(acc);
  const int nk = (K + 63) / 64, all = nk * p.segs, per = (p.segs == 1 ? (Ks + 63) / 64 + splits - 1 : all + splits - 1) / splits, kt0 = min(all, t.split * per),
            kt1 = min(all, kt0 + per);
  auto part_of = [&](int k0, int k1) {
    pipe.fill(k0);
    pipe.run(k0, k1, acc);
    pipe.drain();
  };
  part_of(kt0 < nk ? kt0 : nk, kt1 < nk ? kt1 : nk);
  if (kt1 > nk) {
    pipe.sa.p += p.a2;
    pipe.sb.p += p.b2;
    part_of(kt0 > nk ? kt0 - nk : 0, kt1 - nk);
  }
  const int mr = wm * S::NI * 16 + (lane & 15), nc = wn * S::NJ * 16 + 4 * (lane >> 4);
  if (part) {
    const long ldp = ft_part_ld(N);
    float* o = part + (long)t.split * M * ldp;
#pragma unroll
    for (int i = 0; i < S::NI; ++i) {
      const int m = m0 + mr + 16 * i;
      if (m >= M) continue;
#pragma unroll
      for (int j = 0; j < S::NJ; ++j) {
        const int n = n0 + nc + 16 * j;
        if (n >= ldp) continue;
        ft_f4* q = (ft_f4*)(o + (long)m * ldp + n);
        *q = add ? *q + acc[i][j] : acc[i][j];
      }
    }
    return;
  }
  const float al = p.factor();
#pragma unroll
  for (int i = 0; i < S::NI; ++i)
#pragma unroll
    for (int j = 0; j < S::NJ; ++j) acc[i][j] *= al;
  if constexpr (NPROD == 1 && S::TM == 32) {
    if (p.fold) {                                         // both terms of every row are in this tile
      constexpr int LD = S::TN + 4;
      float* sum = (float*)smem;
#pragma unroll
      for (int i = 0; i < S::NI; ++i)
#pragma unroll
        for (int j = 0; j < S::NJ; ++j) *(ft_f4*)(sum + (mr + 16 * i) * LD + nc + 16 * j) = acc[i][j];
      ft_barrier();
      for (int e = threadIdx.x; e < p.fold * S::TN; e += S::NT) {
        const int r = e / S::TN, c = e % S::TN;
        if (n0 + c < N) ((bf16_t*)p.out)[r * p.ldo + n0 + c] = f2bf(sum[r * LD + c] + sum[(r + p.fold) * LD + c]);
      }
      return;
    }
  }
  if (NPROD == 1) {
#pragma unroll
    for (int i = 0; i < S::NI; ++i)
#pragma unroll
      for (int j = 0; j < S::NJ; ++j) ft_img_put<S::TN>(smem, mr + 16 * i, nc + 16 * j, acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
    ft_barrier();
    const bool vec = p.ldo % 8 == 0 && ((size_t)p.out & 15) == 0;
    ft_img_out<S::TM, S::TN, S::NT>(smem, (bf16_t*)p.out, p.ldo, m0, n0, M, N, p.rows, vec);
  } else {
    const bool vec = p.ldo % 4 == 0 && ((size_t)p.out & 15) == 0;
#pragma unroll
    for (int i = 0; i < S::NI; ++i) {
      const int m = m0 + mr + 16 * i;
      const long row = m < M ? p.rows.at(m) : -1;
      if (row < 0) continue;
#pragma unroll
      for (int j = 0; j < S::NJ; ++j) {
        const int n = n0 + nc + 16 * j;
        float* q = (float*)p.out + row * p.ldo + n;
        if (vec && n + 4 <= N) {
          *(ft_f4*)q = acc[i][j];
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (n + x < N) q[x] = acc[i][j][x];
        }
      }
    }
  }
}

template <class S, int AM, int BMO, int NPROD>
__global__ void __launch_bounds__(S::NT, S::NT == 512 ? 2 : 1) k_ft_product(FtProduct p, float* part, int target, int add) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  ft_product_tile<S, AM, BMO, NPROD>(p, part, target, add, blockIdx.x, smem);
}
// several products in one launch: B is TR in all of them
template <class S, int NPROD>
__global__ void __launch_bounds__(S::NT, S::NT == 512 ? 2 : 1) k_ft_group(FtGroup g) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int b = blockIdx.x, i = b < g.first[1] ? 0 : b < g.first[2] ? 1 : 2;
  const FtProduct& p = g.p[i];
  if constexpr (NPROD == 6) {
    if (p.b32) return ft_product_tile<FtMid32, TK, TR, NPROD>(p, g.part[i], g.target[i], g.add[i], b - g.first[i], smem);
  }
  if (p.am == TK) ft_product_tile<S, TK, TR, NPROD>(p, g.part[i], g.target[i], g.add[i], b - g.first[i], smem);
  else ft_product_tile<S, TR, TR, NPROD>(p, g.part[i], g.target[i], g.add[i], b - g.first[i], smem);
}

struct FtCost { double step, fixed; int slots; };   // us a k-step with the chip full, us a tile besides, tiles at once
static const FtCost kCost[6] = {{1.6, 7.0, 256}, {1.15, 5.0, 512}, {0.45, 4.0, 512}, {2.6, 6.0, 256}, {1.0, 5.0, 512}, {2.8, 6.0, 256}};
static const int kTM[6] = {256, 128, 32, 128, 32, 128}, kTN[6] = {256, 128, 64, 128, 64, 128};

static long tiles_of(const FtPlan& pl, long M, long N) { return ((M + kTM[pl.shape] - 1) / kTM[pl.shape]) * ((N + kTN[pl.shape] - 1) / kTN[pl.shape]); }
// The cheaper of the shapes and slice counts by a model of the time: rounds of tiles over the chip times (k-steps of a slice x time of a
// step + time of a tile's start and end), plus the partial sums' way to memory and back.  The constants are measured: 256 x 256 tiles run
// a k-step in 1.6 us on all CUs (1.3 PFLOP/s), 128 x 128 ones in 1.15 us, two a CU (0.93), and where they leave half of the chip idle, 0.8; 32 x 64 ones in 0.45.
// fp32, in 64 k: 2.6 us from planes, 2.8 with B split on the way, 1.0 for 32 rows.
static double rounds_of(long wg, int slots) { return wg <= 4 * slots ? (double)((wg + slots - 1) / slots) : (double)wg / slots + 0.5; }
bool ft_large(long M, long N, long K) {
  double t[2];
  for (int sh = 0; sh < 2; ++sh) {
    const long tiles = tiles_of(FtPlan{sh, 0}, M, N);
    t[sh] = rounds_of(tiles, kCost[sh].slots) * ((double)((K + 63) / 64) * kCost[sh].step * (sh && 2 * tiles <= kCost[sh].slots ? 0.7 : 1.0) + kCost[sh].fixed);
  }
  return t[0] < t[1];
}
FtPlan ft_plan(const FtProduct& p, bool dynamic_rows) {
  const long M = p.M, N = p.N, K = (long)p.K * p.segs;
  const int nprod = p.nprod;
  FtPlan best;
  double least = 1e30, whole = 1e30;
  for (int sh = 0; sh < 6; ++sh) {
    if (nprod == 6 ? sh != (!p.b32 ? 3 : ft_few(6, M) ? 4 : 5) : sh > 2 || (sh == 2 && (p.am != TK || p.bm != TK || !ft_few(1, M)))) continue;
    const long tiles = ((M + kTM[sh] - 1) / kTM[sh]) * ((N + kTN[sh] - 1) / kTN[sh]), nk = (K + 63) / 64;
    for (int want = 1; want <= 32; ++want) {
      const int sp = ft_slices(tiles, K, (int)(tiles * want > (1 << 20) ? 0 : tiles * want), nprod);
      const long per = (nk + sp - 1) / sp, wg = tiles * sp, slots = kCost[sh].slots;
      double t = rounds_of(wg, slots) * ((double)per * kCost[sh].step * (2 * wg <= slots && sh ? 0.7 : 1.0) + kCost[sh].fixed);
      if (sp > 1) t += 4.0 + (double)sp * M * N * 8.0 / 4e6;
      else if (t < whole) whole = t;
      if (t < least) {
        least = t;
        best.shape = sh;
        best.target = sp > 1 ? (int)(tiles * sp) : 0;
        if (dynamic_rows && best.target < slots) best.target = (int)slots;
      }
      if (sp < want) break;
    }
  }
  if (p.fold && !best.target && !(best.shape == 2 && M <= kTM[2])) best.target = (int)tiles_of(best, M, N);
  best.TM = kTM[best.shape];
  best.TN = kTN[best.shape];
  best.gain = whole / least;
  return best;
}
// slices x tiles stays under max(target, tiles), and rows x columns under tiles x a tile
size_t ft_part_floats(long M, long N, const FtPlan& pl) {
  const long tiles = tiles_of(pl, M, N), wg = tiles > pl.target ? tiles : pl.target;
  return (size_t)wg * kTM[pl.shape] * kTN[pl.shape];
}

int ft_parts(const FtProduct& p, const FtPlan& pl) { return ft_slices(tiles_of(pl, p.M, p.N), (long)(p.Ks ? p.Ks : p.K) * p.segs, pl.target, p.nprod); }
// workgroups of a product: rows really there may be fewer, and the slices then more, but never more of both than this
static long workgroups(const FtProduct& p, const FtPlan& pl, bool part) {
  const long tiles = tiles_of(pl, p.M, p.N);
  if (!part) return tiles;
  if (p.Mdyn) return tiles > pl.target ? tiles : pl.target;
  return tiles * ft_parts(p, pl);
}
template <class S, int AM, int BMO, int NPROD>
static int launch(const FtProduct& p, const FtPlan& pl, float* part, bool add, hipStream_t s) {
  const long n = workgroups(p, pl, part != nullptr);
  FC_REQUIRE(n < (1L << 31), "product of %d x %d: too many tiles", p.M, p.N);
  if (n == 0) return 0;
  static FtLds lds;
  FC_TRY(lds.allow((const void*)k_ft_product<S, AM, BMO, NPROD>, S::LDS));
  hipLaunchKernelGGL((k_ft_product<S, AM, BMO, NPROD>), dim3((unsigned)n), dim3(S::NT), S::LDS, s, p, part, part ? pl.target : 0, add ? 1 : 0);
  FC_LAUNCH_CHECK();
  return 0;
}
template <class S, int NPROD> static int by_mode(const FtProduct& p, const FtPlan& pl, float* part, bool add, hipStream_t s) {
  if (p.am == TK && p.bm == TK) return launch<S, TK, TK, NPROD>(p, pl, part, add, s);
  if constexpr (S::F32) {
    if (p.am == TK) return launch<S, TK, TR, NPROD>(p, pl, part, add, s);
  }
  if constexpr (S::TN >= 128 && !S::F32) {
    if (p.am == TK) return launch<S, TK, TR, NPROD>(p, pl, part, add, s);
    if (p.bm == TR) return launch<S, TR, TR, NPROD>(p, pl, part, add, s);
  }
  fc_set_error("no such product");
  return -1;
}
int ft_product(const FtProduct& p, const FtPlan& plan, float* part, bool add, hipStream_t s) {
  // 32-bit offsets inside a tile: 256 rows of a TK operand, 64 of a TR one, and a whole row of columns
  FC_REQUIRE(p.a.ld < (1L << 21) && p.b.ld < (1L << 21), "an operand's rows are too far apart (%ld, %ld elements)", p.a.ld, p.b.ld);
  switch (plan.shape) {
    case 0: return by_mode<FtBig, 1>(p, plan, part, add, s);
    case 1: return by_mode<FtMid, 1>(p, plan, part, add, s);
    case 2: return by_mode<FtRow, 1>(p, plan, part, add, s);
    case 3: return by_mode<FtPlanes, 6>(p, plan, part, add, s);
    case 4: return by_mode<FtRows32, 6>(p, plan, part, add, s);
    default: return by_mode<FtMid32, 6>(p, plan, part, add, s);
  }
}

// ---------------------------------------------------------------- sums of the slices
// L lanes share a group of eight columns, each with every L-th slice: one where there are many groups, eight where few rows leave the chip
// waiting for one lane's loads (512 groups, 32 slices of two terms: 15 us with one, 5 with eight; 122880 groups of 4 slices: 8 and 15), and for
// rows of two terms
template <typename T, int L>
__global__ void __launch_bounds__(256) k_ft_reduce(FtSums l) {
  const long e0 = ((long)blockIdx.x * 256 + threadIdx.x) / L;
  const int q0 = threadIdx.x % L;
  if (e0 >= l.first[l.n]) return;
  const int w = e0 < l.first[1] ? 0 : e0 < l.first[2] ? 1 : 2;
  const long e = e0 - l.first[w];
  const FtProduct& p = l.p[w];
  const int M = p.Mdyn ? min(p.M, *p.Mdyn) : p.M, K = p.Kdyn ? min(p.K, *p.Kdyn) : p.K, N = p.N, TM = l.TM[w], TN = l.TN[w];
  const long ldp = ft_part_ld(N), cw = ldp / 8;
  const int splits = ft_slices((long)((M + TM - 1) / TM) * ((N + TN - 1) / TN), (long)(p.Ks ? p.Ks : K) * p.segs, l.target[w], p.nprod);
  const int* pos = l.pos[w];
  const int two = L > 1 && p.fold ? 1 : 0;
  const long m = e / cw;
  const int n = (int)(e - m * cw) * 8;
  const long src = pos ? pos[m] : m, row = pos ? m : p.rows.at((int)m);
  if (row < 0) return;
  ft_f4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  if (src >= 0 && src < M)
#pragma unroll 4
    for (int q = q0; q < splits << two; q += L) {
      const ft_f4* a = (const ft_f4*)(l.part[w] + ((long)(q >> two) * M + src + (q & two) * p.fold) * ldp + n);
      v[0] += a[0];
      v[1] += a[1];
    }
  if (L > 1) {
#pragma unroll
    for (int o = 1; o < L; o *= 2)
#pragma unroll
      for (int x = 0; x < 8; ++x) v[x >> 2][x & 3] += __shfl_xor(v[x >> 2][x & 3], o, 64);
    if (q0) return;
  }
  const float al = p.factor();
  v[0] *= al;
  v[1] *= al;
  T* o = (T*)p.out + row * p.ldo + n;
  if (sizeof(T) == 2 && n + 8 <= N && p.ldo % 8 == 0 && ((size_t)p.out & 15) == 0) {
    *(uint4*)o = make_uint4(f2bf2(v[0][0], v[0][1]), f2bf2(v[0][2], v[0][3]), f2bf2(v[1][0], v[1][1]), f2bf2(v[1][2], v[1][3]));
    return;
  }
#pragma unroll
  for (int x = 0; x < 8; ++x)
    if (n + x < N) Io<T>::st(o, x, v[x >> 2][x & 3]);
}
void FtSums::add(const FtProduct& q, const FtPlan& plan, const float* partial, const int* places, long rows) {
  p[n] = q; part[n] = partial; pos[n] = places; target[n] = plan.target; TM[n] = kTM[plan.shape]; TN[n] = kTN[plan.shape];
  first[n + 1] = first[n] + rows * (ft_part_ld(q.N) / 8);
  for (int i = ++n; i < 3; ++i) first[i + 1] = first[i];
}
int ft_reduce(const FtSums& l, hipStream_t s) {
  const long n = l.first[l.n];
  if (n == 0) return 0;
  const int L = n <= 16384 || l.p[0].fold || l.p[1].fold || l.p[2].fold ? 8 : 1;
  const dim3 g((unsigned)((n * L + 255) / 256));
  if (l.p[0].nprod == 1 && L == 1) hipLaunchKernelGGL((k_ft_reduce<bf16_t, 1>), g, dim3(256), 0, s, l);
  else if (l.p[0].nprod == 1) hipLaunchKernelGGL((k_ft_reduce<bf16_t, 8>), g, dim3(256), 0, s, l);
  else if (L == 1) hipLaunchKernelGGL((k_ft_reduce<float, 1>), g, dim3(256), 0, s, l);
  else hipLaunchKernelGGL((k_ft_reduce<float, 8>), g, dim3(256), 0, s, l);
  FC_LAUNCH_CHECK();
  return 0;
}
int ft_reduce(const FtProduct& p, const FtPlan& plan, const float* part, const int* pos, long R, hipStream_t s) {
  FtSums l;
  l.add(p, plan, part, pos, R);
  return ft_reduce(l, s);
}

// ---------------------------------------------------------------- products that wait for nothing of each other
// One launch of 128 x 128 tiles while the chip would run less than about 160 k-steps of them: launches of 100 to 500 workgroups one after
// the other leave part of it idle each (12608 x 384 x 1024, three products and their sums: 109 us apart, 80 together).  Above, tiles of 256 x 256
// in launches of their own are faster.  Slices: of about half of a slot's share of the work, so that what is long and what is short packs well.
bool ft_group_plan(const FtProduct* p, int n, FtPlan* plan) {
  const int sh = p[0].nprod == 1 ? 1 : 3, slots = kCost[sh].slots;
  double work = 0;
  for (int i = 0; i < n; ++i)
    if (p[i].b32 && ft_few(6, p[i].M)) return false;
  for (int i = 0; i < n; ++i) work += (double)tiles_of(FtPlan{sh, 0}, p[i].M, p[i].N) * (double)((p[i].K + 63) / 64 * p[i].segs);
  if (work > 160.0 * slots) return false;
  const double share = work / slots / 2 > 4 ? work / slots / 2 : 4;
  for (int i = 0; i < n; ++i) {
    const long tiles = tiles_of(FtPlan{sh, 0}, p[i].M, p[i].N), nk = (long)(p[i].K + 63) / 64 * p[i].segs;
    const long want = nk <= 2 * share ? 1 : (long)((double)nk / share + 0.5);
    plan[i].shape = sh;
    plan[i].target = want > 1 ? (int)(tiles * want < (1 << 20) ? tiles * want : 0) : 0;
    if (p[i].Mdyn && plan[i].target < slots) plan[i].target = slots;
    if (p[i].fold && !plan[i].target) plan[i].target = (int)tiles;
  }
  return true;
}
int ft_group(const FtProduct* p, const FtPlan* plan, int n, float* const* part, hipStream_t s) {
  FtGroup g;
  for (int i = 0; i < n; ++i) {
    FC_REQUIRE(p[i].bm == TR && p[i].a.ld < (1L << 21) && p[i].b.ld < (1L << 21), "an operand's rows are too far apart");
    g.p[i] = p[i];
    g.part[i] = part[i];
    g.target[i] = part[i] ? plan[i].target : 0;
    g.add[i] = 0;
    g.first[i + 1] = g.first[i] + (int)ft_up(workgroups(p[i], plan[i], part[i] != nullptr), 8);      // whole rounds over the XCDs
  }
  for (int i = n; i < 3; ++i) g.first[i + 1] = g.first[i];
  if (g.first[n] == 0) return 0;
  if (plan[0].shape == 1) {
    static FtLds lds;
    FC_TRY(lds.allow((const void*)k_ft_group<FtMid, 1>, FtMid::LDS));
    hipLaunchKernelGGL((k_ft_group<FtMid, 1>), dim3(g.first[n]), dim3(FtMid::NT), FtMid::LDS, s, g);
  } else {
    static FtLds lds;
    FC_TRY(lds.allow((const void*)k_ft_group<FtPlanes, 6>, FtPlanes::LDS));
    hipLaunchKernelGGL((k_ft_group<FtPlanes, 6>), dim3(g.first[n]), dim3(FtPlanes::NT), FtPlanes::LDS, s, g);
  }
  FC_LAUNCH_CHECK();
  return 0;
}

// ---------------------------------------------------------------- fp32, a reduction over few rows: C[m, n] = sum_k A[k, m] B[k, n], k < 32
// All that costs time is the writing of C, of which the tiles, one workgroup of eight waves a CU, reach half the rate (38227 x 2816, 11 rows: 178 us;
// here 72, 6 TB/s).  A wave's lanes hold four columns each of all rows of B; the values of A, of `per` rows of C, come from LDS.
// Where C is small and the rows are not the fewest, the tiles' start is the shorter one (gated block with gradients, 768 x 2048, 32 rows: 99 us with
// tiles, 120 here; 4096 x 11008: 731 and 700; 4 rows: 98 and 95, 701 and 585).
template <int KM>
__global__ void __launch_bounds__(256) k_ft_outer(FtProduct p, int per, int cols) {      // cols: waves of a workgroup side by side
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* sa = (float*)smem;                                                            // [per][KM]
  const int K = p.Kdyn ? min(p.K, *p.Kdyn) : p.K, wave = ft_wave(), lane = threadIdx.x & 63;
  const long m0 = (long)blockIdx.x * per;
  const int rows = (int)min((long)per, p.M - m0), n = (blockIdx.y * cols + wave % cols) * 256 + lane * 4;
  auto whole = [](const FtMat& a, long at) {          // four values (the rows of planes are whole groups of 64, zeros behind the last value)
    ft_f4 v[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      const uint2 u = *(const uint2*)(a.p + q * a.plane + at);
      v[q] = ft_f4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
    }
    return v[0] + (v[1] + v[2]);
  };
  for (int e = threadIdx.x; e < KM * (per / 4); e += 256) {
    const int k = e / (per / 4), r = (e - k * (per / 4)) * 4;
    const ft_f4 v = k < K && r < rows ? whole(p.a, k * p.a.ld + m0 + r) : ft_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 4; ++x) sa[(r + x) * KM + k] = v[x];
  }
  ft_f4 b[KM];
#pragma unroll
  for (int k = 0; k < KM; ++k) b[k] = k < K && n < p.N ? whole(p.b, k * p.b.ld + n) : ft_f4{0.f, 0.f, 0.f, 0.f};
  __syncthreads();
  if (n >= p.N) return;
  const float al = p.factor();
  const bool vec = p.ldo % 4 == 0 && ((size_t)p.out & 15) == 0 && n + 4 <= p.N;
  for (int r = wave / cols; r < rows; r += 4 / cols) {
    ft_f4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KM; k += 4) {
      const ft_f4 v = *(const ft_f4*)(sa + r * KM + k);
#pragma unroll
      for (int x = 0; x < 4; ++x) c += v[x] * b[k + x];
    }
    const long row = p.rows.at((int)(m0 + r));
    if (row < 0) continue;
    c *= al;
    float* o = (float*)p.out + row * p.ldo + n;
    if (vec) {
      *(ft_f4*)o = c;
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (n + x < p.N) o[x] = c[x];
    }
  }
}
static bool ft_is_outer(const FtProduct& p) { return p.nprod == 6 && p.am == TR && p.bm == TR && p.segs == 1 && p.K <= 32 && (p.K <= 8 || (long)p.M * p.N >= (1L << 24)); }
static int ft_outer(const FtProduct& p, hipStream_t s) {
  if (p.M == 0 || p.N == 0) return 0;
  const int waves = (p.N + 255) / 256, cols = waves >= 3 ? 4 : waves, by = (waves + cols - 1) / cols;
  int per = 128;
  while (per > 16 && (long)by * ((p.M + per - 1) / per) < 1024) per /= 2;
  const dim3 g((unsigned)((p.M + per - 1) / per), (unsigned)by);
  if (p.K <= 8) hipLaunchKernelGGL(k_ft_outer<8>, g, dim3(256), per * 8 * 4, s, p, per, cols);
  else if (p.K <= 16) hipLaunchKernelGGL(k_ft_outer<16>, g, dim3(256), per * 16 * 4, s, p, per, cols);
  else hipLaunchKernelGGL(k_ft_outer<32>, g, dim3(256), per * 32 * 4, s, p, per, cols);
  FC_LAUNCH_CHECK();
  return 0;
}

size_t ft_product_part_floats(const FtProduct& p) {
  if (ft_is_outer(p)) return 0;
  const FtPlan plan = ft_plan(p, false);
  return plan.target ? ft_part_floats(p.M, p.N, plan) : 0;
}
int ft_product_out(const FtProduct& p, float* part, size_t part_floats, hipStream_t s) {
  if (ft_is_outer(p)) return ft_outer(p, s);
  const FtPlan plan = ft_plan(p, false);
  if (!plan.target) return ft_product(p, plan, nullptr, false, s);
  FC_REQUIRE(part && part_floats >= ft_part_floats(p.M, p.N, plan), "workspace too small for the partial sums");
  FC_TRY(ft_product(p, plan, part, false, s));
  return ft_reduce(p, plan, part, nullptr, p.fold ? p.fold : p.M, s);
}
