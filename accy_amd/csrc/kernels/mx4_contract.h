// Products of microscaled 4-bit floats on gfx950: C[m, n] = sum_k A[m, k] B[n, k], both operands' rows blocked along k, on
// v_mfma_scale_f32_32x32x64_f8f6f4, which takes codes and scales as they are: a lane's 16 bytes are one block, its scale a
// byte beside it. Included after gemm.h and mx4.h.
//
// C supplies M, N, K (K a multiple of 32); the epilogue receives (0, m, n, f32 sum) for every output.
#pragma once

namespace accy {
namespace mx4 {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Bytes SA of sa and SB of sb are the scales of the lane's blocks.
template <int SA = 0, int SB = 0>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c, u32_t sa, u32_t sb) {
  const i32x8 aw = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, bw = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(aw, bw, c, 4, 4, SA, (int)sa, SB, (int)sb);
}

// Matrix instructions read every lane's operands whatever the execution mask: this keeps the compiler from moving one, with what
// computes its operands, behind the branch around a store that only some lanes take.
__device__ __forceinline__ void settle(f32x16& acc) { asm volatile("" : "+a"(acc)); }

// Small tiles, BM x BN outputs (multiples of 16) of a workgroup whose WK waves share K, each keeping sums of the whole tile, which
// meet in LDS at the end: for few rows, where every weight is read once, and for products too small to fill the chip with
// larger tiles. Bound by the operands' bytes, of which a CU takes about 52 KB a us (tile (16, 32): 16 x 8192 x 8192 6.7
// us, 2.4 of them a launch; 16 x 28672 x 8192, from HBM, 22.5).
//
// A wave takes 256 values of every row at a time (every WK-th 256), up to four stages ahead, on its own: its codes go straight to
// its own part of LDS, an instruction 128 bytes of eight rows, and its scales through registers, eight bytes a row. (Operands
// straight to registers in the matrix instruction's order, whose neighbouring lanes are rows apart, take a cache access
// per lane: 10.3 and 29.5 us for the above.) v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds row l % 16 and, of the eight
// blocks, 2 g and 2 g + 1, g = l / 16, with their scales as bytes 0 and 1 of one word. Rows past the end read the last
// row and are not stored. A block past K reads the last one with the scales 2^-127 on both sides, whose products vanish in f32
// (below 36 x 2^-254).
//
// C supplies M, N, K, BM, BN and WK.
template <int S>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c, u32_t sa, u32_t sb) {
  const i32x8 aw = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, bw = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(aw, bw, c, 4, 4, S, (int)sa, S, (int)sb);
}

// The scales of blocks b .. b + 7 of a row (b a multiple of eight), 0 for those past K.
template <long K>
__device__ __forceinline__ u32x2 scale_eight(const u8_t* __restrict__ row, long b) {
  typedef u32x2 __attribute__((aligned(1))) any;
  constexpr long BLOCKS = K / 32, REST = BLOCKS % 8;
  if (REST == 0 || b + 8 <= BLOCKS) return *(const any*)(row + b);
  u32x2 w = {0, 0};
#pragma unroll
  for (int e = 0; e < (int)REST; ++e) w[e >> 2] |= (u32_t)row[BLOCKS - REST + e] << (8 * (e & 3));
  return w;
}

template <class C, class Epi>
__device__ __forceinline__ void contract_direct(const u8_t* __restrict__ A, const u8_t* __restrict__ AS, const u8_t* __restrict__ B,
                                                const u8_t* __restrict__ BS, const Epi& epi) {
  constexpr int TM = C::BM / 16, TN = C::BN / 16, WK = C::WK, ROWS = C::BM + C::BN, D = ROWS / 8, E = (ROWS + 63) / 64;
  constexpr long TILES_N = (C::N + C::BN - 1) / C::BN, BLOCKS = C::K / 32, ITERS = (BLOCKS + 7) / 8;
  constexpr int S = ITERS >= 4 * WK ? 4 : (int)((ITERS + WK - 1) / WK);  // no more stages than a wave has steps
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  const long m0 = (long)blockIdx.x / TILES_N * C::BM, n0 = (long)blockIdx.x % TILES_N * C::BN;
  __shared__ __attribute__((aligned(1024))) u8_t c0[WK][ROWS * 128], c1[S > 1 ? WK : 1][S > 1 ? ROWS * 128 : 16],
      c2[S > 2 ? WK : 1][S > 2 ? ROWS * 128 : 16], c3[S > 3 ? WK : 1][S > 3 ? ROWS * 128 : 16];
  __shared__ __attribute__((aligned(16))) u8_t words[WK][ROWS * 8];
  u8_t* const stage[4] = {c0[wave], c1[S > 1 ? wave : 0], c2[S > 2 ? wave : 0], c3[S > 3 ? wave : 0]};
  // codes: an instruction moves 128 bytes of eight rows, lane l the chunk l % 8 ^ (row / 2 mod 8) of row l / 8
  const u8_t* src[D];
  int chunk[D];
#pragma unroll
  for (int i = 0; i < D; ++i) {
    const int r = 8 * i + (lane >> 3);
    const long m = m0 + r < C::M ? m0 + r : C::M - 1, n = n0 + r - C::BM < C::N ? n0 + r - C::BM : C::N - 1;
    src[i] = 8 * i < C::BM ? A + m * (C::K / 2) : B + n * (C::K / 2);
    chunk[i] = (lane & 7) ^ ((r >> 1) & 7);
  }
  // scales: lane l those of rows l, 64 + l ..
  const u8_t* ssrc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int r = 64 * i + lane < ROWS ? 64 * i + lane : ROWS - 1;
    const long m = m0 + r < C::M ? m0 + r : C::M - 1, n = n0 + r - C::BM < C::N ? n0 + r - C::BM : C::N - 1;
    ssrc[i] = r < C::BM ? AS + m * BLOCKS : BS + n * BLOCKS;
  }
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  u32x2 sc[S][E];
  auto load = [&](int s, long it) {
#pragma unroll
    for (int i = 0; i < D; ++i) {
      long at = 8 * it + chunk[i];
      if constexpr (BLOCKS % 8 != 0) at = at < BLOCKS ? at : BLOCKS - 1;
      gemm::dma16(src[i] + 16 * at, (ACCY_LDS void*)(stage[s] + 1024 * i));
    }
#pragma unroll
    for (int i = 0; i < E; ++i) sc[s][i] = scale_eight<C::K>(ssrc[i], 8 * it);
  };
  auto frag = [&](int s, int row0, int e) {
    const int r = row0 + (lane & 15);
    return *(const u32x4*)(stage[s] + r * 128 + 16 * ((2 * g + e) ^ ((r >> 1) & 7)));
  };
  long it = wave;
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (it + s * WK < ITERS) load(s, it + s * WK);
  for (; it < ITERS; it += S * WK) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const long now = it + s * WK, ahead = now + (S - 1) * WK;
      if (now >= ITERS) break;
      // The stage's codes have landed when no more is outstanding than the three stages after it (their scales not counted);
      // where no stage follows, when nothing is.
      if (ahead < ITERS) {
        load((s + S - 1) % S, ahead);
        gemm::wait_vmcnt<(S - 1) * D>();
      } else {
        gemm::wait_vmcnt<0>();
      }
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (ROWS % 64 == 0 || 64 * i + lane < ROWS) *(u32x2*)(words[wave] + 8 * (64 * i + lane)) = sc[s][i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      u32x4 a[TM][2], b[TN][2];
      u32_t sa[TM], sb[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        a[i][0] = frag(s, 16 * i, 0), a[i][1] = frag(s, 16 * i, 1);
        sa[i] = *(const u16_t*)(words[wave] + 8 * (16 * i + (lane & 15)) + 2 * g);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        b[j][0] = frag(s, C::BM + 16 * j, 0), b[j][1] = frag(s, C::BM + 16 * j, 1);
        sb[j] = *(const u16_t*)(words[wave] + 8 * (C::BM + 16 * j + (lane & 15)) + 2 * g);
      }
      __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8));  // lgkmcnt(0): the stage may be overwritten
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          acc[i][j] = mfma16<0>(a[i][0], b[j][0], acc[i][j], sa[i], sb[j]);
          acc[i][j] = mfma16<1>(a[i][1], b[j][1], acc[i][j], sa[i], sb[j]);
        }
    }
  }
  // Element e of lane l of tile (i, j) is output (16 i + 4 (l / 16) + e, 16 j + l % 16).
  // A wave's sums take the place of its first stage, which every load has reached and every read has left.
  constexpr int ALL = C::BM * C::BN;
  static_assert(ALL * 4 <= ROWS * 128, "a wave's sums fit its stage");
  float* const mine = (float*)c0[wave];
#pragma unroll
  for (int t = 0; t < TM * TN; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) mine[(t * 4 + e) * 64 + lane] = acc[t / TN][t % TN][e];
  __syncthreads();
  for (int x = tid; x < ALL; x += 64 * WK) {
    const int m = x / C::BN, n = x % C::BN, at = (((m >> 4) * TN + (n >> 4)) * 4 + (m & 3)) * 64 + ((m >> 2) & 3) * 16 + (n & 15);
    float v = ((const float*)c0[0])[at];
#pragma unroll
    for (int w = 1; w < WK; ++w) v += ((const float*)c0[w])[at];
    if ((C::M % C::BM == 0 || m0 + m < C::M) && (C::N % C::BN == 0 || n0 + n < C::N)) epi(0, m0 + m, n0 + n, v);
  }
}

// Tiles of BM x BN outputs by four waves (2 x 2), operands' codes straight to LDS: the direct-to-LDS pipeline of gemm.h with
// the codes as its 16-bit elements (K / 4 of them to a row; a K step of 128 values is 64 bytes of a row, four stages of
// them), a fragment's 16 bytes one block of the row. A step's 2 x TM x TN matrix instructions take 32 clocks each against
// (BM + BN) x 64 bytes of LDS written and twice that read, at 128 bytes a clock: with 256 x 256 tiles three quarters of the
// LDS's rate. At that size registers alone reach 6.2-6.6 PFLOP/s of random codes and 8.3-8.8 of
// zeros, this kernel 4.0 and 5.2: the board's power takes a quarter of either, the structure over a third.
//
// A row's scales are four bytes to a step. Fetched 16 bytes a row and four steps, straight to registers, they take a line of
// the row each time (8192^3: 297 us; without any scales 255), so 64 bytes of each row go to LDS at once, for 16 steps, in
// the 32 KB that the stages of 256 x 256 tiles leave: 273 us. (Laid out by groups of rows before: 267, and a launch more.) Every
// wave has read the last of them into registers when the barrier of the step after is passed, and the next 64 bytes
// land during the three steps that follow. Rows are 4 x STEPS bytes apart: the operand's own rows where K is a multiple of
// 128, else a copy with zeros (2^-127 on both sides: nothing, see contract_direct) for the blocks past K (pad_scales).
//
// C supplies M, N, K, BM, BN, GROUP_M and SPLITS; split blockIdx.z takes an equal share of the groups of four steps.
template <class C> struct Codes {
  static __device__ __forceinline__ long row(long i) { return i * (C::K / 4); }
  static __device__ __forceinline__ long k(long i) { return i; }
};

template <class C>
struct Tile {
  static constexpr int BM = C::BM, BN = C::BN, TM = BM / 64, TN = BN / 64, NF = TM + TN, NM = TM * TN, S = 4;
  static constexpr int DA = BM / 64, DB = BN / 64, PER = DA + DB;  // direct-to-LDS instructions of a wave and step
  static constexpr long STEPS = (C::K + 127) / 128;

  struct Frags {
    u32x4 a[TM], b[TN];
    __device__ __forceinline__ void load_one(int q, const u16_t* as, const u16_t* bs, int s, int lane, int wm, int wn) {
      if (q < TM) a[q] = gemm::frag<BM, true>(as, wm * (BM / 2) + q * 32, s, lane);
      else b[q - TM] = gemm::frag<BN, true>(bs, wn * (BN / 2) + (q - TM) * 32, s, lane);
    }
  };
  struct Scales {
    u32x4 a[TM], b[TN];
  };

  // One step on stage I, whose f0 holds the first sub-step's fragments: the matrix instructions of f0 with the loads of step kt
  // + 3 and the reads of the second sub-step between them, the wait for step kt + 1, and the second sub-step's
  // instructions with the reads of step kt + 1's first between them (see gemm.h).
  template <int I, class Acc>
  static __device__ __forceinline__ void step(const u16_t* __restrict__ A, const u16_t* __restrict__ B, long m0, long n0, long kt,
                                              u16_t* const (&as)[4], u16_t* const (&bs)[4], Frags& f0, const Scales& sc, Acc& acc,
                                              int wave, int lane, int wm, int wn) {
    constexpr int NEXT = (I + 3) % 4;
    const long ahead = (kt + 3 < STEPS ? kt + 3 : STEPS - 1) * 32;
    Frags f1;
#pragma unroll
    for (int t = 0; t < NM; ++t) {
      acc[t / TN][t % TN] = mfma32<0, 0>(f0.a[t / TN], f0.b[t % TN], acc[t / TN][t % TN], sc.a[t / TN][I], sc.b[t % TN][I]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = t * (NF + PER) / NM; k < (t + 1) * (NF + PER) / NM; ++k) {
        if (k < NF) f1.load_one(k, as[I], bs[I], 1, lane, wm, wn);
        else if (k - NF < DA) gemm::dma_part<BM, true, Codes<C>, C::M, C::K / 4>(A, m0, ahead, as[NEXT], wave, lane, k - NF);
        else gemm::dma_part<BN, true, Codes<C>, C::N, C::K / 4>(B, n0, ahead, bs[NEXT], wave, lane, k - NF - DA);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    gemm::wait_vmcnt<2 * PER>();
    gemm::lds_reads_done_barrier();
#pragma unroll
    for (int t = 0; t < NM; ++t) {
      acc[t / TN][t % TN] = mfma32<2, 2>(f1.a[t / TN], f1.b[t % TN], acc[t / TN][t % TN], sc.a[t / TN][I], sc.b[t % TN][I]);
      __builtin_amdgcn_sched_barrier(0);
      static_assert(NF <= NM, "fragment reads fit one per matrix instruction");
      if (t < NF) f0.load_one(t, as[(I + 1) % 4], bs[(I + 1) % 4], 0, lane, wm, wn);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// Both operands' scale rows, 4 x STEPS bytes apart.
template <class C>
__device__ __forceinline__ void pad_scales(const u8_t* __restrict__ AS, const u8_t* __restrict__ BS, u32_t* __restrict__ a, u32_t* __restrict__ b) {
  constexpr long BLOCKS = C::K / 32, STEPS = (C::K + 127) / 128;
  const bool first = blockIdx.y == 0;
  const long all = (first ? C::M : C::N) * STEPS;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long)gridDim.x * 256) {
    const u8_t* const row = (first ? AS : BS) + i / STEPS * BLOCKS;
    u32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i % STEPS * 4 + e < BLOCKS) w |= (u32_t)row[i % STEPS * 4 + e] << (8 * e);
    (first ? a : b)[i] = w;
  }
}

template <class C, class Epi>
__device__ __forceinline__ void contract_tile(const u8_t* __restrict__ A8, const u8_t* __restrict__ AS, const u8_t* __restrict__ B8,
                                              const u8_t* __restrict__ BS, const Epi& epi) {
  typedef Tile<C> T;
  constexpr int BM = C::BM, BN = C::BN, TM = T::TM, TN = T::TN;
  constexpr long TILES_M = (C::M + BM - 1) / BM, TILES_N = (C::N + BN - 1) / BN, PITCH = 4 * T::STEPS;
  constexpr long GROUPS = (T::STEPS + 3) / 4, SHARE = (GROUPS + C::SPLITS - 1) / C::SPLITS;
  const u16_t *__restrict__ A = (const u16_t*)A8, *__restrict__ B = (const u16_t*)B8;
  // distinct arrays per stage (see gemm.h)
  constexpr int A_ST = BM * 32, B_ST = BN * 32;
  __shared__ __attribute__((aligned(1024))) u16_t a0[A_ST], a1[A_ST], a2[A_ST], a3[A_ST];
  __shared__ __attribute__((aligned(1024))) u16_t b0[B_ST], b1[B_ST], b2[B_ST], b3[B_ST];
  u16_t* const as[4] = {a0, a1, a2, a3};
  u16_t* const bs[4] = {b0, b1, b2, b3};
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1, half = lane >> 5;
  long tm, tn;
  gemm::tile_of<TILES_M, TILES_N, C::GROUP_M>(blockIdx.x, tm, tn);
  const long m0 = tm * BM, n0 = tn * BN;
  long group = C::SPLITS > 1 ? (long)blockIdx.z * SHARE : 0;
  const long last = C::SPLITS > 1 && (group + SHARE) * 4 < T::STEPS ? (group + SHARE) * 4 : T::STEPS;
  long kt = group * 4;

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};

  // Scales: of the fragments' rows, the four words of a group.
  typename T::Scales now;
  __shared__ __attribute__((aligned(1024))) u8_t ss[(BM + BN) * 64];
  // Groups g .. g + 3 (g a multiple of four) of every row to LDS, A's rows and then B's. The 16-byte chunk at position p of a
  // row is its chunk p ^ (row / 4 mod 4), so that 16 rows read at one chunk cover 256 distinct bytes. An instruction
  // moves 16 rows, 16 bytes a lane, where rows are whole chunks, else four rows, a step's four bytes a lane. What lies past
  // the row's end reads its last bytes, which no step uses.
  // The offsets are computed each time (the lane's number is opaque here): kept, they would push accumulators out of the registers.
  constexpr int UNIT = PITCH % 16 == 0 ? 16 : 4, LPR = 64 / UNIT, RPI = 64 / LPR;  // lanes per row, rows per instruction
  const u8_t *const ab = AS + m0 * PITCH, *const bb = BS + n0 * PITCH;
  const int rows_a = C::M - m0 < BM ? (int)(C::M - m0) : BM, rows_b = C::N - n0 < BN ? (int)(C::N - n0) : BN;
  auto fetch = [&](long g) {
    u32_t l = (u32_t)lane;
    asm volatile("" : "+v"(l));
    const u32_t row = l / LPR, at = l % LPR * UNIT;
#pragma unroll
    for (int i = 0; i < (BM + BN) / 4 / RPI; ++i) {
      const int gi = wave * ((BM + BN) / 4 / RPI) + i, r0 = RPI * gi;
      const bool a = r0 < BM;
      const u32_t end = (u32_t)(a ? rows_a - 1 : rows_b - 1);
      u32_t r = (u32_t)(a ? r0 : r0 - BM) + row, c = 16 * ((u32_t)g + ((at >> 4) ^ (((u32_t)r0 + row) >> 2 & 3))) + (at & 15);
      r = r < end ? r : end;
      c = c < (u32_t)(PITCH - UNIT) ? c : (u32_t)(PITCH - UNIT);
      const u8_t* const p = (a ? ab : bb) + (r * (u32_t)PITCH + c);
      ACCY_LDS void* const to = (ACCY_LDS void*)(ss + gi * 64 * UNIT);
      if constexpr (UNIT == 16) __builtin_amdgcn_global_load_lds(p, to, 16, 0, 0);
      else __builtin_amdgcn_global_load_lds(p, to, 4, 0, 0);
    }
  };
  auto read = [&](int row0, int q) {
    const int r = row0 + (lane & 31);
    return *(const u32x4*)(ss + r * 64 + 16 * (q ^ ((r >> 2) & 3)));
  };
  // A wave's halves hold the even and the odd blocks: bytes 2 s of the words are then those of the lane's block in sub-step s.
  auto take = [&](int q) {
#pragma unroll
    for (int i = 0; i < TM; ++i) now.a[i] = read(wm * (BM / 2) + 32 * i, q) >> 8 * half;
#pragma unroll
    for (int j = 0; j < TN; ++j) now.b[j] = read(BM + wn * (BN / 2) + 32 * j, q) >> 8 * half;
  };

  if (kt < last) {
    fetch(group & ~3L);
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      const long at = (kt + s < T::STEPS ? kt + s : T::STEPS - 1) * 32;
      gemm::dma_tile<BM, true, Codes<C>, C::M, C::K / 4>(A, m0, at, as[s], wave, lane);
      gemm::dma_tile<BN, true, Codes<C>, C::N, C::K / 4>(B, n0, at, bs[s], wave, lane);
    }
    typename T::Frags f0;
    gemm::wait_vmcnt<2 * T::PER>();
    gemm::lds_reads_done_barrier();
#pragma unroll
    for (int q = 0; q < T::NF; ++q) f0.load_one(q, as[0], bs[0], 0, lane, wm, wn);
    // Whole groups of four steps, then what the last split has left.
    for (; kt + 4 <= last; kt += 4) {
      take((int)(group & 3));
      ++group;
      T::template step<0>(A, B, m0, n0, kt, as, bs, f0, now, acc, wave, lane, wm, wn);
      if ((group & 3) == 0) fetch(group);
      T::template step<1>(A, B, m0, n0, kt + 1, as, bs, f0, now, acc, wave, lane, wm, wn);
      T::template step<2>(A, B, m0, n0, kt + 2, as, bs, f0, now, acc, wave, lane, wm, wn);
      T::template step<3>(A, B, m0, n0, kt + 3, as, bs, f0, now, acc, wave, lane, wm, wn);
    }
    constexpr int REST = (int)(T::STEPS % 4);
    if constexpr (REST > 0) {
      if (C::SPLITS == 1 || kt < last) {
        take((int)(group & 3));
        T::template step<0>(A, B, m0, n0, kt, as, bs, f0, now, acc, wave, lane, wm, wn);
        if constexpr (REST > 1) T::template step<1>(A, B, m0, n0, kt + 1, as, bs, f0, now, acc, wave, lane, wm, wn);
        if constexpr (REST > 2) T::template step<2>(A, B, m0, n0, kt + 2, as, bs, f0, now, acc, wave, lane, wm, wn);
      }
    }
    gemm::wait_vmcnt<0>();  // loads past the last step, which nobody reads
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) settle(acc[i][j]);
  const long col = n0 + wn * (BN / 2) + (lane & 31), row = m0 + wm * (BM / 2) + half * 4;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const long m = row + i * 32 + (e >> 2) * 8 + (e & 3), n = col + j * 32;
        if ((C::M % BM == 0 || m < C::M) && (C::N % BN == 0 || n < C::N)) epi(0, m, n, acc[i][j][e]);
      }
}

}  // namespace mx4
}  // namespace accy
