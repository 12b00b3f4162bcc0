// Tiled products for the fused vocabulary cross entropy (fc_linear_ce.hip) and the gated feed-forward block (fc_gated_mlp.hip):
//
//     C[m, n] = sum_k A(m, k) B(n, k)
//
// with each operand stored either with k contiguous ("TK": rows are m or n) or with k as its row index ("TR"), bf16, on
// v_mfma_f32_16x16x32_bf16.  fp32 operands are taken as three bf16 planes hi + mid + lo (24 bits of mantissa) and the
// products of the six plane pairs that are above 2^-24 of the whole (NPROD = 6), so that the result is that of an fp32 product.  The planes are
// laid out in memory first, but for a B that few rows meet: that one is split when its fragments are formed (FtB32).
//
// One k-step is 64 deep (fp32: two stages of 32).  Operand tiles go global -> LDS by buffer_load ... lds (16 B a lane), NS stages deep, one
// barrier a step.  The loads are issued by inline asm: with the builtin the compiler waits for every load in flight in front of the LDS reads
// it cannot tell apart from the load's destination.  They have no register results; ft_dma_wait() in front of each barrier waits for them.
// Rows, columns and k past the end read as zero: by the descriptor's size or by an offset outside of it.
// LDS images (both conflict-free): TK [rows][64 k], 128-B rows, 16-B chunk c of row r at chunk c ^ ((r >> 1) & 7), read by ds_read_b128;
// TR [64 k][W cols], 32-B unit u of row k at unit u ^ (((k >> 3) & 1) << 2 | (k & 3)), read by ds_read_b64_tr_b16.
// The MFMA's operands are swapped, so a lane's accumulator acc[i][j] is row 16 i + (lane & 15), columns 16 j + 4 (lane >> 4) .. + 3.
#pragma once
#include <atomic>
#include <type_traits>

#include "fc_common.h"

typedef __attribute__((ext_vector_type(8))) short ft_b8;
typedef __attribute__((ext_vector_type(4))) short ft_b4;
typedef __attribute__((ext_vector_type(4))) float ft_f4;
typedef __attribute__((ext_vector_type(4))) int ft_i4;
typedef __attribute__((address_space(3))) ft_b4 ft_lds_b4;

enum { TK = 0, TR = 1 };
#define FT_OOB 0x80000000u       // outside of every descriptor below (their sizes stay under 2^31)
#define FT_MAX_BYTES 0x7fffff00L

// one operand: element (row, k) of plane q at p[q * plane + row * ld + k] (TK), (k, col) at p[q * plane + k * ld + col] (TR)
struct FtMat {
  const bf16_t* p = nullptr;
  long ld = 0, plane = 0;
  int wrap = 0;                    // TR, > 0: rows k from there on are rows k - wrap again (up to 2 wrap, at most 64: one k-step)
  const bf16_t* end = nullptr;     // an fp32 matrix read where it is (FtB32): one past its last element
};

__device__ __forceinline__ int ft_wave() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }
__device__ __forceinline__ unsigned ft_lds_addr(const char* p) {
  return (unsigned)__builtin_amdgcn_readfirstlane((int)(size_t)(__attribute__((address_space(3))) const char*)p);
}
template <int N> __device__ __forceinline__ void ft_dma_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ft_barrier() {   // LDS hand-off: this wave's LDS traffic is done, its global stores need not be
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// m0 (a reserved register, no operand of anything else in these kernels) takes the LDS address of the wave's piece
__device__ __forceinline__ void ft_dma16(ft_i4 rsrc, unsigned lds, unsigned voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory");
}
__device__ __forceinline__ ft_i4 ft_rsrc(const void* p, long bytes) {
  const unsigned long long a = (unsigned long long)p;
  const long b = bytes < 0 ? 0 : bytes > FT_MAX_BYTES ? FT_MAX_BYTES : bytes;
  ft_i4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32) & 0xffff);
  r[2] = __builtin_amdgcn_readfirstlane((int)b);
  r[3] = 0x00020000;
  return r;
}

// the same value, of which nothing is computed ahead of time and kept in registers over a loop that needs them all
__device__ __forceinline__ int ft_fresh(int v) { asm volatile("" : "+v"(v)); return v; }

// the XOR of a TK row's 16-B chunks: rows that would meet in a bank differ in it
template <int KS> __device__ __forceinline__ int ft_tk_swz(int row) { return KS == 64 ? (row >> 1) & 7 : (row >> 2) & 3; }

// Stages one operand's tile of W rows (TK) or columns (TR), KS k deep, by NW waves, in pieces of 1 KB.
template <int MODE, int W, int KS, int NW> struct FtStager {
  static constexpr int NP = W * KS / 512 / NW, RP = 512 / KS, CR = KS / 8;      // pieces of a wave; TK: rows of a piece, chunks of a row
  static_assert(NP >= 1 && NP * NW * 512 == W * KS, "a wave moves whole pieces");
  static_assert(MODE == TK || W >= 128, "a TR row holds at least the swizzle's eight units");
  const bf16_t* p;
  long ld, plane;
  int K, kc[2];                     // TK: first k, inside the stage, of the lane's chunk in an even and an odd piece
  unsigned voff[NP];
  // of the stage that is being loaded: descriptor, start, bytes and k left; and where the next one starts
  ft_i4 r;
  const bf16_t *cur, *at;
  long cur_bytes, bytes;
  int left, left_next;

  // map(r): row (TK) / column (TR) of the matrix that tile position r takes, < 0 for none.  TR positions come in eights: map(r + i) = map(r) + i.
  // TK: offsets are taken from row `base`, the least row of the tile.
  template <class F> __device__ __forceinline__ void init(const FtMat& m, long base, int K_, int wave, int lane, F map) {
    ld = m.ld; plane = m.plane; K = K_;
    p = m.p + (MODE == TK ? base * ld : 0);
#pragma unroll
    for (int i = 0; i < 2; ++i) kc[i] = (lane % CR ^ ft_tk_swz<KS>(i * RP + lane / CR)) * 8;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int piece = wave * NP + i;
      if (MODE == TK) {
        const int t = piece * RP + lane / CR;
        const long row = map(t);
        voff[i] = row >= 0 ? (unsigned)(((row - base) * ld + (lane % CR ^ ft_tk_swz<KS>(t)) * 8) * 2) : FT_OOB;
      } else {
        const int k = piece * (512 / W) + lane * 8 / W, pc = lane % (W / 8), kr = m.wrap && k >= m.wrap ? k - m.wrap : k;
        const int s = (((k >> 3) & 1) << 2) | (k & 3);
        const int c = (((pc >> 1) ^ s) << 1) | (pc & 1);
        const long col = map(c * 8);
        voff[i] = col >= 0 && (!m.wrap || kr < m.wrap) ? (unsigned)(((long)kr * ld + col) * 2) : FT_OOB;
      }
    }
  }
  __device__ __forceinline__ void seek(long k0) {              // the next stage is the one at k0, of the first plane
    at = p + (MODE == TK ? k0 : k0 * ld);
    left_next = K - k0 < -KS ? -KS : (int)(K - k0);
    bytes = (K - k0) * ld * 2;
  }
  __device__ __forceinline__ void step() {                     // past the end: no k left, no bytes, and so zeros
    cur = at;
    cur_bytes = bytes;
    r = ft_rsrc(cur, MODE == TK ? FT_MAX_BYTES : cur_bytes);
    left = left_next;
    left_next -= KS;
    at += MODE == TK ? KS : KS * ld;
    bytes -= 2 * KS * ld;
  }
  __device__ __forceinline__ unsigned offset(int i, int wave) const {
    const int k = NP % 2 == 0 ? kc[i & 1] : (wave * NP + i) & 1 ? kc[1] : kc[0];
    return MODE == TK ? (k < left ? voff[i] : FT_OOB) : voff[i];
  }
  __device__ __forceinline__ void piece(int i, unsigned lds, int wave) const { ft_dma16(r, lds + (wave * NP + i) * 1024, offset(i, wave)); }
  __device__ __forceinline__ void piece_of(int pl, int i, unsigned lds, int wave) const {      // the same k of plane pl
    ft_dma16(ft_rsrc(cur + pl * plane, MODE == TK ? FT_MAX_BYTES : cur_bytes), lds + (wave * NP + i) * 1024, offset(i, wave));
  }
};

// one wave's fragment of 16 rows / columns starting at rb (a multiple of 16) for 32 k, the ks-th of a stage
template <int MODE, int W, int KS> __device__ __forceinline__ ft_b8 ft_frag(const char* tile, int rb, int ks, int lane) {
  const int g = lane >> 4;
  if (MODE == TK) {
    const int c = (ks * 4 + g) ^ ft_tk_swz<KS>(lane & 15);
    return *(const ft_b8*)(tile + (rb + (lane & 15)) * (KS * 2) + (c << 4));
  }
  const int q = (lane >> 2) & 3, s = ((g & 1) << 2) | q;
  const char* a = tile + (ks * 32 + 8 * g + q) * (W * 2) + ((((rb >> 4) ^ s)) << 5) + (lane & 3) * 8;
  const ft_b4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ft_lds_b4*)a);
  const ft_b4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ft_lds_b4*)(a + 4 * W * 2));
  return ft_b8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// the three planes of an fp32 value, exact for every finite one: above bf16's largest (3.3895e38) the first plane is that, not infinity.  An infinity
// or no number gives planes with no number among them, and so does every product with it.
__device__ __forceinline__ void ft_split(float x, float& hi, float& mid, float& lo) {
  constexpr float top = 3.38953138925153547590470800371487867e38f;       // 0x7f7f0000
  hi = __builtin_amdgcn_fmed3f(bf2f(f2bf(x)), -top, top);
  const float r = x - hi;
  mid = bf2f(f2bf(r));
  lo = r - mid;
}

// fp32 tiles of 32 rows (a scoring call's): 32 rows of A's three planes, 32 k deep, are six pieces by four waves, the last two of them moved
// twice so that every wave moves as many
struct FtRowsA {
  static constexpr int NP = 2;
  const bf16_t* p;
  long ld, plane, at;
  int K, kc[2];
  unsigned voff[2];
  template <class F> __device__ __forceinline__ void init(const FtMat& m, long base, int K_, int wave, int lane, F map) {
    ld = m.ld; plane = m.plane; K = K_;
    p = m.p + base * ld;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = (id(i, wave) & 1) * 16 + (lane >> 2), c = (lane & 3) ^ ft_tk_swz<32>(t);
      const long row = map(t);
      kc[i] = c * 8;
      voff[i] = row >= 0 ? (unsigned)(((row - base) * ld + c * 8) * 2) : FT_OOB;
    }
  }
  static __device__ __forceinline__ int id(int i, int wave) { return i ? 4 + (wave & 1) : wave; }
  __device__ __forceinline__ void load(int i, long k0, unsigned lds, int wave) const {
    const int q = id(i, wave);
    ft_dma16(ft_rsrc(p + (q >> 1) * plane + k0, FT_MAX_BYTES), lds + q * 1024, kc[i] < (K - k0 < 32 ? (int)(K - k0) : 32) ? voff[i] : FT_OOB);
  }
};
// An fp32 B that is read where it is, in 32 bits, and split when its fragments are formed: its tile is a bf16 stager's with two columns to a
// value, [rows][64] (TK) or [32][2 columns] (TR).  Any alignment of a float does: buffer loads of 16 bytes start at any dword and are clipped at the
// descriptor's size dword by dword.  What a row's last 16 bytes take of the next row is masked (TK) or belongs to columns that are not there (TR).
template <int MODE, int W, int NW> struct FtB32 : FtStager<MODE, MODE == TK ? W : 2 * W, MODE == TK ? 64 : 32, NW> {
  typedef FtStager<MODE, MODE == TK ? W : 2 * W, MODE == TK ? 64 : 32, NW> Base;
  const bf16_t* end;
  // the matrix' ld counts bf16 units, two to a value
  template <class F> __device__ __forceinline__ void init(const FtMat& m, long base, int K_, int wave, int lane, F map) {
    end = m.end;
    if (MODE == TK) Base::init(m, base, 2 * K_, wave, lane, map);
    else Base::init(m, base, K_, wave, lane, [&](int r) { const long c = map(r >> 1); return c < 0 ? -1L : 2 * c; });
  }
  __device__ __forceinline__ void seek(long k0) { Base::seek(MODE == TK ? 2 * k0 : k0); }
  __device__ __forceinline__ int left_at(long k0) const { return (int)((MODE == TK ? this->K / 2 : this->K) - k0); }
  __device__ __forceinline__ void step() {
    Base::step();
    const long rest = (end - this->cur) * 2;
    this->r = ft_rsrc(this->cur, MODE == TK || rest < this->cur_bytes ? rest : this->cur_bytes);
  }
  // a stage with `left` k to come
  static __device__ __forceinline__ void mask(int left, int g, float (&v)[8]) {
    if (MODE == TK && left < 32)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 8 * g + i < left ? v[i] : 0.f;
  }
  // eight k of column r (the lane's)
  static __device__ __forceinline__ void read(const char* t, int r, int g, float (&v)[8]) {
    if (MODE == TK) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const ft_f4 u = *(const ft_f4*)(t + r * 128 + (((2 * g + h) ^ ft_tk_swz<64>(r)) << 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * h + i] = u[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = *(const float*)(t + (8 * g + i) * (W * 4) + (((r >> 3) ^ (((g & 1) << 2) | (i & 3))) << 5) + (r & 7) * 4);
    }
  }
};
// eight fp32 values of a B fragment as the fragments of their three planes
__device__ __forceinline__ void ft_split8(const float (&v)[8], ft_b8& f0, ft_b8& f1, ft_b8& f2) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float h[2], m[2], l[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) ft_split(v[i + j], h[j], m[j], l[j]);
    ((unsigned*)&f0)[i / 2] = f2bf2(h[0], h[1]);
    ((unsigned*)&f1)[i / 2] = f2bf2(m[0], m[1]);
    ((unsigned*)&f2)[i / 2] = f2bf2(l[0], l[1]);
  }
}

// tile shape: TM x TN by WM x WN waves, NS LDS stages of KS k and PL planes (F32: of A alone, B as it is)
template <int TM_, int TN_, int WM_, int WN_, int NS_, int KS_ = 64, int PL_ = 1, bool F32_ = false> struct FtShape {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, NS = NS_, KS = KS_, PL = PL_, NW = WM * WN, NT = NW * 64;
  static constexpr bool F32 = F32_;
  static constexpr int NI = TM / WM / 16, NJ = TN / WN / 16, STAGE = F32 ? TM * KS * 2 * PL + TN * KS * 4 : (TM + TN) * KS * 2 * PL, LDS = NS * STAGE;
};
template <class S, int MODE, bool F32> struct FtStagers {
  typedef FtStager<MODE, S::TM, S::KS, S::NW> A;
  typedef FtStager<MODE, S::TN, S::KS, S::NW> B;
};
template <class S, int MODE> struct FtStagers<S, MODE, true> {
  typedef typename std::conditional<S::TM == 32, FtRowsA, FtStager<TK, S::TM < 128 ? 128 : S::TM, S::KS, S::NW>>::type A;
  typedef FtB32<MODE, S::TN, S::NW> B;
};
template <class S, int MODE> using FtStageA = typename FtStagers<S, MODE, S::F32>::A;
template <class S, int MODE> using FtStageB = typename FtStagers<S, MODE, S::F32>::B;

// The loops over k: acc += the k-steps [kt0, kt1).
//
// For the large tiles (NS < 4) the loads run on from one tile of a workgroup to its next (k_ce_stats, k_ce_grad; 2560 x 768 x 30522 with gradients
// 483 us, 495 without): fill() loads the first tile's first NS stages, run() takes a tile's steps and, when the last of its loads is issued, calls
// advance(), which sets the stagers to the next tile; what a tile's last NS steps load is the next one's beginning, which arrives while the
// epilogue runs.  Steps past the end of the matrices load zeros.  settle() in front of the epilogue's first store keeps the next run from waiting
// for these stores; drain() in front of LDS reuse and the kernel's end leaves no load in flight.
//
// bf16: a step's two halves of 32 k are held in registers in turn: while the MFMAs of one run, the fragments of the next are read, one read to
// every few MFMAs, so that neither the LDS nor the matrix pipe waits for the other.  The one barrier stands between the halves: there a wave has
// the step's second half in registers, so its stage is free for the loads of the step NS on, and the next stage, loaded for NS - 1 steps by then,
// is read from there on.
// fp32: all three planes of both operands (F32: of A, and B in 32 bits) in a stage of 32 k, six products from one read of each fragment.  (A plane
// pair a step would load every plane twice and meet six barriers for one here.)  The fragments of the next stage are read under the MFMAs of this
// one, whose barrier stands under the first of them; B's of F32 are split a few groups of MFMAs later.
template <class S, int AM, int BMO> struct FtPipe {
  static constexpr bool ROWS = S::NS >= 4, PLANES = S::PL == 3;
  static constexpr int NI = S::NI, NJ = S::NJ, PA1 = FtStageA<S, AM>::NP, PB1 = FtStageB<S, BMO>::NP;
  static constexpr int PA = PA1 * (PLANES && !ROWS ? 3 : 1), PB = PB1 * (PLANES && !S::F32 ? 3 : 1), P = PA + PB;      // loads of a wave a stage
  static constexpr int TA = S::TM * S::KS * 2, TB = S::TN * S::KS * 2;                                                // bytes of a plane's tile
  typedef ft_f4 Acc[S::NI][S::NJ];
  FtStageA<S, AM> sa;
  FtStageB<S, BMO> sb;
  char* smem;
  unsigned lds0;
  int wave, lane, wm, wn, at = 0;
  bool landed = false;

  __device__ __forceinline__ FtPipe(char* smem_) : smem(smem_), lds0(ft_lds_addr(smem_)), wave(ft_wave()), lane(threadIdx.x & 63) {
    wm = wave / S::WN;
    wn = wave % S::WN;
  }
  __device__ __forceinline__ void seek(int kt) {
    if constexpr (!(ROWS && PLANES)) sa.seek((long)kt * 64);
    sb.seek((long)kt * 64);
  }
  __device__ __forceinline__ void next() { sa.step(); sb.step(); }
  __device__ __forceinline__ void piece(int i, int slot) const {
    const unsigned l = lds0 + slot * S::STAGE;
    if constexpr (!PLANES) {
      if (i < PA) sa.piece(i, l, wave); else sb.piece(i - PA, l + TA, wave);
    } else {
      if (i < PA) sa.piece_of(i / PA1, i % PA1, l + i / PA1 * TA, wave);
      else if (S::F32) sb.piece(i - PA, l + 3 * TA, wave);
      else sb.piece_of((i - PA) / PB1, (i - PA) % PB1, l + 3 * TA + (i - PA) / PB1 * TB, wave);
    }
  }
  __device__ __forceinline__ void fill(int kt0) {
    if constexpr (!ROWS) {
      seek(kt0);
#pragma unroll
      for (int st = 0; st < S::NS; ++st) {
        next();
#pragma unroll
        for (int i = 0; i < P; ++i) piece(i, st);
      }
      ft_dma_wait<(S::NS - 1) * P>();
      ft_barrier();
      at = 0;
      landed = false;
    }
  }
  __device__ __forceinline__ void settle() {
    if constexpr (!ROWS) { ft_dma_wait<0>(); landed = true; }
  }
  __device__ __forceinline__ void drain() {
    if constexpr (!ROWS) { ft_dma_wait<0>(); ft_barrier(); }
  }
  // (every stage but the one that the next step reads may be on its way; a settled pipe's are all there)
  __device__ __forceinline__ void await(bool first) const {
    if (!(first && landed)) ft_dma_wait<(S::NS - 2) * P>();
    ft_barrier();
  }
  __device__ __forceinline__ static int following(int slot) { return slot + 1 == S::NS ? 0 : slot + 1; }

  template <class F> __device__ __forceinline__ void run(int kt0, int kt1, Acc& acc, F advance) {
    if constexpr (ROWS && S::F32) rows32(kt0, kt1, acc);
    else if constexpr (ROWS) rows(kt0, kt1, acc);
    else if constexpr (PLANES) planes(kt0, kt1, acc, advance);
    else halves(kt0, kt1, acc, advance);
    landed = false;
  }
  __device__ __forceinline__ void run(int kt0, int kt1, Acc& acc) { run(kt0, kt1, acc, [] {}); }

  template <class F> __device__ __forceinline__ void halves(int kt0, int kt1, Acc& acc, F advance) {
    constexpr int NF = NI + NJ, NM = NI * NJ;
    const int steps = kt1 - kt0;
    ft_b8 f[2][NF];                           // [half][B fragments, then A fragments]
    auto read = [&](int i, int ks, int slot) {
      const char* t = smem + slot * S::STAGE;
      f[ks][i] = i < NJ ? ft_frag<BMO, S::TN, 64>(t + TA, (wn * NJ + i) * 16, ks, lane) : ft_frag<AM, S::TM, 64>(t, (wm * NI + i - NJ) * 16, ks, lane);
    };
    auto mfma = [&](int m, int ks) {
      const int i = m / NJ, j = m % NJ;
      acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[ks][j], f[ks][NJ + i], acc[i][j], 0, 0, 0);
    };
#pragma unroll
    for (int i = 0; i < NF; ++i) read(i, 0, at);
    // a half: reads spread over the first three quarters of its MFMAs, so that the last ones cover the last read's way
    constexpr int RM = NM * 3 / 4 / NF > 0 ? NM * 3 / 4 / NF : 1;
    auto half = [&](int ks, int slot, auto before) {
#pragma unroll
      for (int g = 0; g < NF; ++g) {
        before(g);
        read(g, ks ^ 1, slot);
#pragma unroll
        for (int m = g * RM; m < (g + 1 < NF ? (g + 1) * RM : NM); ++m) mfma(m, ks);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    for (int s = 0; s < steps; ++s) {
      if (s == steps - S::NS) advance();
      half(0, at, [&](int g) { if (g == 0) next(); });
      await(s == 0);
      const int to = following(at);
      half(1, to, [&](int g) {
#pragma unroll
        for (int i = g * P / NF; i < (g + 1) * P / NF; ++i) piece(i, at);
      });
      at = to;
    }
  }

  template <class F> __device__ __forceinline__ void planes(int kt0, int kt1, Acc& acc, F advance) {
    static_assert(S::KS == 32, "a stage is one fragment deep");
    constexpr int NM = 6 * NI * NJ, NF = 3 * NI + (S::F32 ? NJ : 3 * NJ);
    const int steps = (kt1 - kt0) * 2;
    ft_b8 fa[2][3][NI], fb[2][3][NJ];
    float raw[NJ][8];
    int left = 0;                                       // k from the stage that is read on (F32)
    auto split = [&](int j, int h) {
      if constexpr (S::F32) FtStageB<S, BMO>::mask(left, lane >> 4, raw[j]);
      ft_split8(raw[j], fb[h][0][j], fb[h][1][j], fb[h][2][j]);
    };
    auto read = [&](int i, int h, int slot) {             // in the order of use: both first planes, then the others
      const char* t = smem + slot * S::STAGE;
      if constexpr (S::F32) {
        if (i < NJ) FtStageB<S, BMO>::read(t + 3 * TA, (wn * NJ + i) * 16 + (lane & 15), lane >> 4, raw[i]);
        else fa[h][(i - NJ) / NI][(i - NJ) % NI] = ft_frag<AM, S::TM, 32>(t + (i - NJ) / NI * TA, (wm * NI + (i - NJ) % NI) * 16, 0, lane);
      } else {
        const int pl = i / (NI + NJ), k = i % (NI + NJ);
        if (k < NJ) fb[h][pl][k] = ft_frag<BMO, S::TN, 32>(t + 3 * TA + pl * TB, (wn * NJ + k) * 16, 0, lane);
        else fa[h][pl][k - NJ] = ft_frag<AM, S::TM, 32>(t + pl * TA, (wm * NI + k - NJ) * 16, 0, lane);
      }
    };
    auto mfma = [&](int m, int h) {
      constexpr int qa[6] = {0, 0, 1, 1, 0, 2}, qb[6] = {0, 1, 0, 1, 2, 0};
      const int q = m / (NI * NJ), i = m % (NI * NJ) / NJ, j = m % NJ;
      acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[h][qb[q]][j], fa[h][qa[q]][i], acc[i][j], 0, 0, 0);
    };
#pragma unroll
    for (int i = 0; i < NF; ++i) read(i, 0, at);
    if constexpr (S::F32) {
      left = sb.left_at((long)kt0 * 64);
#pragma unroll
      for (int j = 0; j < NJ; ++j) split(j, 0);
    }
    constexpr int M0 = NM / 8, RM = (NM - M0) / NF, LATE = 4;
    static_assert(RM >= 1 && (!S::F32 || LATE + 2 * NJ <= NF), "an MFMA to every read, and the splits' places");
    auto stage = [&](int h, bool first) {
      const int to = following(at);
      next();
      if (S::F32) left -= 32;
#pragma unroll
      for (int m = 0; m < M0; ++m) mfma(m, h);
      __builtin_amdgcn_sched_barrier(0);
      await(first);                                     // slot `to` is there, and slot `at` read by everybody
#pragma unroll
      for (int g = 0; g < NF; ++g) {
#pragma unroll
        for (int i = g * P / NF; i < (g + 1) * P / NF; ++i) piece(i, at);
        read(g, h ^ 1, to);
        if constexpr (S::F32)
          if (g >= LATE && (g - LATE) % 2 == 0 && (g - LATE) / 2 < NJ) split((g - LATE) / 2, h ^ 1);
#pragma unroll
        for (int m = M0 + g * RM; m < (g + 1 < NF ? M0 + (g + 1) * RM : NM); ++m) mfma(m, h);
        __builtin_amdgcn_sched_barrier(0);
      }
      at = to;
    };
    static_assert(S::NS % 2 == 1, "the last load of a tile is issued in an odd stage");
    for (int s = 0; s < steps; s += 2) {
      stage(0, s == 0);
      if (s + 1 == steps - S::NS) advance();
      stage(1, false);
    }
  }

  // few rows: a step is short, and its loads' way from memory long.  Nothing is in flight before and after.
  __device__ __forceinline__ void rows(int kt0, int kt1, Acc& acc) {
    const int steps = kt1 - kt0;
    int slot = 0, free_slot = S::NS - 1;
    seek(kt0);
    auto put = [&](int to) {
      next();
#pragma unroll
      for (int i = 0; i < P; ++i) piece(i, to);
    };
#pragma unroll
    for (int s = 0; s < S::NS - 1; ++s) put(s);
    for (int s = 0; s < steps; ++s) {
      await(false);
      put(free_slot);
      const char* ta = smem + slot * S::STAGE;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        ft_b8 af[NI], bf[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) bf[j] = ft_frag<BMO, S::TN, 64>(ta + TA, (wn * NJ + j) * 16, ks, lane);
#pragma unroll
        for (int i = 0; i < NI; ++i) af[i] = ft_frag<AM, S::TM, 64>(ta, (wm * NI + i) * 16, ks, lane);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[j], af[i], acc[i][j], 0, 0, 0);
      }
      free_slot = slot;
      slot = following(slot);
    }
    ft_dma_wait<0>();
    ft_barrier();
  }
  __device__ __forceinline__ void rows32(int kt0, int kt1, Acc& acc) {
    static_assert(S::TM == 32 && S::NW == 4 && S::KS == 32 && S::PL == 3 && S::NI == 1, "two waves by two");
    const int steps = (kt1 - kt0) * 2, g = lane >> 4;
    int slot = 0, free_slot = S::NS - 1, left = sb.left_at((long)kt0 * 64);
    long k0 = (long)kt0 * 64;
    sb.seek(k0);
    auto put = [&](int to) {
      const unsigned l = lds0 + to * S::STAGE;
      sb.step();
#pragma unroll
      for (int i = 0; i < PA; ++i) sa.load(i, k0, l, wave);
#pragma unroll
      for (int i = 0; i < PB; ++i) sb.piece(i, l + 3 * TA, wave);
      k0 += 32;
    };
#pragma unroll
    for (int s = 0; s < S::NS - 1; ++s) put(s);
    for (int s = 0; s < steps; ++s) {
      await(false);
      put(free_slot);
      const char* ta = smem + slot * S::STAGE;
      const char* tb = ta + 3 * TA;
      ft_b8 fa[3], fb[NJ][3];
#pragma unroll
      for (int p = 0; p < 3; ++p) fa[p] = ft_frag<TK, 32, 32>(ta + p * TA, wm * 16, 0, lane);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        float v[8];
        sb.read(tb, (wn * NJ + j) * 16 + (lane & 15), g, v);
        sb.mask(left, g, v);
        ft_split8(v, fb[j][0], fb[j][1], fb[j][2]);
      }
#pragma unroll
      for (int q = 0; q < 6; ++q)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          constexpr int qa[6] = {0, 0, 1, 1, 0, 2}, qb[6] = {0, 1, 0, 1, 2, 0};
          acc[0][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j][qb[q]], fa[qa[q]], acc[0][j], 0, 0, 0);
        }
      left -= 32;
      free_slot = slot;
      slot = following(slot);
    }
    ft_dma_wait<0>();
    ft_barrier();
  }
};
template <int NI, int NJ> __device__ __forceinline__ void ft_zero(ft_f4 (&acc)[NI][NJ]) {
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = ft_f4{0.f, 0.f, 0.f, 0.f};
}

// ---- which tile a workgroup takes.  Consecutive ids share an XCD's L2 (workgroups are dealt to the 8 XCDs in turn), and ids walk the
// tiles in groups of 8 tile rows, column by column, so that the tiles in flight on an XCD share few operand panels.
struct FtTile { int m, n, split; bool any; };
__device__ __forceinline__ FtTile ft_tile(int tm, int tn, int splits, int b) {
  FtTile t;
  const int total = tm * tn * splits;
  t.any = b < total;
  if (!t.any) { t.m = t.n = t.split = 0; return t; }
  const int q = total >> 3, r = total & 7, xcd = b & 7;
  int id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (b >> 3);
  t.split = id / (tm * tn);
  id -= t.split * tm * tn;
  const int per = 8 * tn, gi = id / per, first = gi * 8, gs = tm - first < 8 ? tm - first : 8, in = id - gi * per;
  t.m = first + in % gs;
  t.n = in / gs;
  return t;
}

// ---- rows of an output: position i of `half` rows each goes to row (i / half) * to + i % half, none where i % half >= to (0: as it is)
struct FtRows {
  int half = 0, to = 0;
  __device__ __forceinline__ long at(int i) const {
    if (!half) return i;
    const int h = i >= half ? 1 : 0, f = i - h * half;
    return f < to ? (long)h * to + f : -1;
  }
};

// a bf16 image of the tile in LDS, rows of IW columns: 16-B chunk c of row r at chunk c ^ (r & 15)
template <int IW> __device__ __forceinline__ int ft_img(int row, int chunk) { return row * (IW * 2) + ((chunk ^ (row & 15 & (IW / 8 - 1))) << 4); }
template <int IW> __device__ __forceinline__ void ft_img_put(char* img, int row, int col, float a, float b, float c, float d) {
  *(uint2*)(img + ft_img<IW>(row, col >> 3) + (col & 4) * 2) = make_uint2(f2bf2(a, b), f2bf2(c, d));
}
// image -> global: rows m0 + r < M, columns n0 + c < N of a row-major bf16 matrix
template <int IR, int IW, int NT>
__device__ __forceinline__ void ft_img_out(const char* img, bf16_t* out, long ld, int m0, int n0, int M, int N, const FtRows& rows, bool vec) {
  if (!vec) {                             // rows at any element: a wave's lanes write neighbouring ones
#pragma unroll 4
    for (int e = threadIdx.x; e < IR * IW; e += NT) {
      const int r = e / IW, c = e % IW, m = m0 + r, n = n0 + c;
      if (m >= M || n >= N) continue;
      const long row = rows.at(m);
      if (row >= 0) out[row * ld + n] = *(const bf16_t*)(img + ft_img<IW>(r, c >> 3) + (c & 7) * 2);
    }
    return;
  }
#pragma unroll 4
  for (int e = threadIdx.x; e < IR * (IW / 8); e += NT) {
    const int r = e / (IW / 8), c = e % (IW / 8), m = m0 + r, n = n0 + c * 8;
    if (m >= M || n >= N) continue;
    const long row = rows.at(m);
    if (row < 0) continue;
    const uint4 v = *(const uint4*)(img + ft_img<IW>(r, c));
    bf16_t* o = out + row * ld + n;
    if (n + 8 <= N) {
      *(uint4*)o = v;
    } else {
      const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < N) o[i] = (bf16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// the same for one wave's 16 rows of W columns, in 16 * W * 2 bytes of its own: no barrier
template <int W> __device__ __forceinline__ int ft_wimg(int row, int chunk) { return row * (W * 2) + ((chunk ^ (W == 64 ? row & 7 : (row >> 1) & 3 & (W / 8 - 1))) << 4); }
template <int W> __device__ __forceinline__ void ft_wimg_put(char* img, int row, int col, float a, float b, float c, float d) {
  *(uint2*)(img + ft_wimg<W>(row, col >> 3) + (col & 4) * 2) = make_uint2(f2bf2(a, b), f2bf2(c, d));
}
template <int W> __device__ __forceinline__ void ft_wimg_out(const char* img, bf16_t* out, long ld, int m0, int n0, int M, int N, int lane) {
#pragma unroll
  for (int q = 0; q < W / 32; ++q) {
    const int e = q * 64 + lane, r = e / (W / 8), c = e % (W / 8);
    const uint4 v = *(const uint4*)(img + ft_wimg<W>(r, c));
    if (m0 + r < M && n0 + c * 8 < N) *(uint4*)(out + (long)(m0 + r) * ld + n0 + c * 8) = v;
  }
}

// eight values of a row, fewer where it ends, 0 behind its end.  bf16 rows may start at any element: whole dwords are read, from the one that
// holds the first value to the one that holds the last, and shifted.
template <typename T> __device__ __forceinline__ void ft_row8(const T* p, int cols, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    if (cols >= 8) {
      const bool odd = ((size_t)p & 2) != 0;
      const unsigned* q = (const unsigned*)((size_t)p & ~(size_t)3);
      unsigned w[5];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = q[j];
      w[4] = odd ? q[4] : 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned u = odd ? w[j] >> 16 | w[j + 1] << 16 : w[j];
        v[2 * j] = __uint_as_float(u << 16);
        v[2 * j + 1] = __uint_as_float(u & 0xffff0000u);
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < cols ? Io<T>::ld(p, j) : 0.f;
}

// ---------------------------------------------------------------- host side (fc_tiles.hip)
// C = A B^T written to `out` (bf16 for nprod 1, fp32 for 6), or as fp32 partial sums for ft_reduce().
struct FtProduct {
  int am = TK, bm = TK, nprod = 1;
  bool b32 = false;               // fp32: B is the fp32 matrix itself (its ld in bf16 units), not its planes
  FtMat a, b;
  int M = 0, N = 0, K = 0;
  int Ks = 0;                     // > 0: the length that the slices are cut from, >= K (products added onto each other's partial sums)
  const int* Mdyn = nullptr;      // device: the rows (M) / reduction length (K) really there, at most M / K
  const int* Kdyn = nullptr;
  int fold = 0;                   // > 0: A's rows are two terms of each of `fold` rows, first terms first, and the result is their sum
  int segs = 1;                   // 2: the reduction is two pieces of length K, the second a2 / b2 elements on in A / B
  long a2 = 0, b2 = 0;
  const float* alpha = nullptr;   // device: factor of the result (null: 1), over *alpha_over where that is given
  const int* alpha_over = nullptr;
  void* out = nullptr;
  long ldo = 0;
  FtRows rows;
  __device__ __forceinline__ float factor() const {
    if (!alpha) return 1.f;
    return alpha_over ? (*alpha_over > 0 ? *alpha / (float)*alpha_over : 0.f) : *alpha;
  }
};
// shape: index of the tile shape (TM x TN); target: workgroups wanted, by which the reduction is sliced (0: it is not)
struct FtPlan {
  int shape = 0, target = 0, TM = 0, TN = 0;
  double gain = 1;      // time of the best unsliced form over this one's, by the model
};
FtPlan ft_plan(const FtProduct& p, bool dynamic_rows);
// whether a bf16 product that cannot be sliced is faster in tiles of 256 x 256 than of 128 x 128, by the same model
bool ft_large(long M, long N, long K);
__host__ __device__ static inline long ft_part_ld(long N) { return (N + 7) / 8 * 8; }
// slices of a reduction of length K for `tiles` output tiles: as many as the target asks for, none under four k-steps (one of fp32's six products)
__host__ __device__ static inline int ft_slices(long tiles, long K, int target, int nprod) {
  if (target <= 0 || tiles <= 0) return 1;
  long s = target / tiles;
  const long most = nprod == 1 ? (K + 63) / 64 / 4 : (K + 63) / 64;
  s = s < most ? s : most;
  return s < 1 ? 1 : s > 32 ? 32 : (int)s;
}
size_t ft_part_floats(long M, long N, const FtPlan& plan);     // for any number of rows up to M
int ft_parts(const FtProduct& p, const FtPlan& plan);          // slices of a product whose rows are all there
// partial sums [slices][rows there][ft_part_ld(N)] into `part` (or, part null, the product into p.out); add: onto what is there
int ft_product(const FtProduct& p, const FtPlan& plan, float* part, bool add, hipStream_t s);
// up to three products in one launch, and the sums of their slices in one
struct FtGroup {
  FtProduct p[3];
  float* part[3] = {nullptr, nullptr, nullptr};
  int target[3] = {0, 0, 0}, add[3] = {0, 0, 0}, first[4] = {0, 0, 0, 0};      // first workgroup of each
};
struct FtSums {
  FtProduct p[3];
  const float* part[3] = {nullptr, nullptr, nullptr};
  const int* pos[3] = {nullptr, nullptr, nullptr};
  int target[3] = {0, 0, 0}, TM[3] = {0, 0, 0}, TN[3] = {0, 0, 0}, n = 0;
  long first[4] = {0, 0, 0, 0};                                                // first group of eight columns of each
  void add(const FtProduct& q, const FtPlan& plan, const float* partial, const int* places, long rows);
};
int ft_reduce(const FtSums& l, hipStream_t s);
// whether they are better run as a group, and how; part[i] null: straight into out
bool ft_group_plan(const FtProduct* p, int n, FtPlan* plan);
int ft_group(const FtProduct* p, const FtPlan* plan, int n, float* const* part, hipStream_t s);
// out = the sum over the slices, in one order, of ft_product's partial sums; with `pos`: out[r] = row pos[r] of the sums, 0 where pos[r] < 0, for R rows
int ft_reduce(const FtProduct& p, const FtPlan& plan, const float* part, const int* pos, long R, hipStream_t s);
// the product into p.out, by way of partial sums in `part` where the plan slices the reduction
int ft_product_out(const FtProduct& p, float* part, size_t part_floats, hipStream_t s);
size_t ft_product_part_floats(const FtProduct& p);

// an operand as the products take it: rows of whole 128-byte lines, and in planes for fp32
struct FtPack {
  const void* src = nullptr;
  long lds = 0;                   // elements between source rows
  int dt = 1;
  long R = 0, C = 0;
  bf16_t* dst = nullptr;
  long ldd = 0;                   // multiple of 64, >= C: the columns in between are written as zeros
};
struct FtPacks {                  // up to four of one type in one launch
  FtPack p[4];
  int n = 0;
  long first[5] = {0, 0, 0, 0, 0};   // 16-byte chunks before each
  void add(const FtPack& q) { p[n] = q; first[n + 1] = first[n] + q.R * (q.ldd / 8); ++n; }
};
int ft_pack(const FtPacks& p, hipStream_t s);
// rows up to which tiles are 32 rows high: their reading of B is what counts (bf16, 64 rows of 4096 x 11008: 77 us forward, 88 with 128 x 128 tiles;
// fp32, where every 32 rows split B's fragments once more, 64 rows: 271 us, 222 with 128 x 128)
static inline bool ft_few(int nprod, long T) { return T <= (nprod == 1 ? 64 : 32); }
// fp32: up to how many rows a weight is not worth laying out in planes (gated block forward, 4096 x 11008: 96 rows 229 us, 564 with planes; 512 rows 767
// and 997; with gradients, 384 x 1024, 1000 rows: 147 and 136), and whether it can be read where it is
#define FT_B32 512
static inline bool ft_b32(int dt, long T, const void* p, long ld) { return !dt && T <= FT_B32 && ((size_t)p & 3) == 0 && ld < (1L << 20); }
static inline FtMat ft_mat32(const void* p, long ld, long R, long C) {
  FtMat m;
  m.p = (const bf16_t*)p;
  m.ld = 2 * ld;
  m.end = m.p + 2 * ((R - 1) * ld + C);
  return m;
}
static inline bool ft_direct(int dt, const void* p, long ld, long cols) { return dt == 1 && ((size_t)p & 15) == 0 && ld % 8 == 0 && cols % 8 == 0; }
// workgroups of a kernel whose workgroups walk the tiles: as many as run at once, where the loads of two tiles can follow each other (FtPipe)
template <class S> static inline long ft_walkers(long tiles, long K) {
  return S::NT == 512 && (K + 63) / 64 * (S::KS == 32 ? 2 : 1) >= S::NS && tiles > 256 ? 256 : tiles;
}
static inline long ft_up(long v, long m) { return (v + m - 1) / m * m; }
// > 64 KB of LDS for a kernel: asked for once on each device (a static of the launch that needs it)
struct FtLds {
  std::atomic<unsigned long long> done{0};      // a bit for each of the first 64 devices
  int allow(const void* kernel, int bytes) {
    int dev = 0;
    FC_CHECK_HIP(hipGetDevice(&dev));
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return 0;
    FC_CHECK_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
    return 0;
  }
};
// the device that holds p has to be the current one
int ft_check_device(const void* p, const char* what);
