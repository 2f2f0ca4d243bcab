// Microscaled 4-bit floats on gfx950: quantisation, and a paged cache with the attention that reads it (products:
// mx4_contract.h).
//
// The format: blocks of 32 values along one axis; a value is e2m1 (sign, two exponent bits, one mantissa bit: 0, 0.5, 1,
// 1.5, 2, 3, 4, 6) times its block's scale, a power of two held as its biased exponent in one byte (e8m0; 255 is NaN).
// Two codes share a byte, the first in its low half. A block of largest magnitude A takes the scale 2^(floor(log2 A) - 2),
// at least 2^-127: the largest value lands in [4, 8), where 6 is the last code; codes are rounded to nearest, ties
// to the even code. A block with a NaN or an infinity takes scale 255 and reads as NaN throughout.
//
// v_cvt_scalef32_pk_fp4_f32 divides by the scale and rounds two values exactly so (ties, saturation and the scales 2^-127 and
// 2^127 included), v_cvt_scalef32_pk_{f32,bf16}_fp4 is the way back, exact in both types.
#pragma once

namespace accy {
namespace mx4 {

typedef u32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Element types: 0 bf16, 1 f16, 2 f32. Results round to nearest even in all of them (the operators' own rounding; the
// elementwise operations of a program truncate bf16, see common.h).
template <int DT> struct Elem { typedef u16_t type; };
template <> struct Elem<2> { typedef float type; };

template <int DT> __device__ __forceinline__ typename Elem<DT>::type to_elem(float v) {
  if constexpr (DT == 0) return __builtin_bit_cast(u16_t, (__bf16)v);
  else if constexpr (DT == 1) return f32_to_f16(v);
  else return v;
}
template <int DT> __device__ __forceinline__ float from_elem(typename Elem<DT>::type v) {
  if constexpr (DT == 0) return bf16_to_f32(v);
  else if constexpr (DT == 1) return f16_to_f32(v);
  else return v;
}
// The value of a result of type DT.
template <int DT> __device__ __forceinline__ float rounded(float v) { return from_elem<DT>(to_elem<DT>(v)); }

// A scale byte as the f32 whose exponent the conversions take.
__device__ __forceinline__ float scale_of(u32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Eight consecutive values at a time, as one lane of the four that share a block; 16-byte accesses where the type has them.
template <int DT> __device__ __forceinline__ void load8(const typename Elem<DT>::type* __restrict__ p, float (&x)[8]) {
  if constexpr (DT == 2) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    const u32x4 w = *(const u32x4*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = from_elem<DT>((u16_t)(w[i >> 1] >> (16 * (i & 1))));
  }
}
template <int DT> __device__ __forceinline__ void store8(typename Elem<DT>::type* __restrict__ p, const float (&x)[8]) {
  if constexpr (DT == 2) {
    *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
    *(f32x4*)(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (u32_t)to_elem<DT>(x[2 * i]) | ((u32_t)to_elem<DT>(x[2 * i + 1]) << 16);
    *(u32x4*)p = w;
  }
}

// The scale byte of the block that four adjacent lanes hold eight values each of (all four call it), and the codes of
// this lane's eight. The exponent of the largest magnitude comes from its bits: the unsigned order of the bits without
// the sign is the order of the magnitudes, with infinity and NaN above all of them. The scale's exponent is 2 less, and
// 2^-127 (byte 0) for everything below 2^-125, subnormals and zero among it.
__device__ __forceinline__ u32_t block_scale(const float (&x)[8]) {
  u32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const u32_t b = __builtin_bit_cast(u32_t, x[i]) & 0x7fffffffu;
    top = top > b ? top : b;
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const u32_t b = (u32_t)__shfl_xor((int)top, o, 64);
    top = top > b ? top : b;
  }
  const u32_t e = top >> 23;
  return e == 255 ? 255 : e < 2 ? 0 : e - 2;
}
__device__ __forceinline__ u32_t encode8(const float (&x)[8], u32_t byte) {
  const float s = scale_of(byte);
  u32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  return w;
}
__device__ __forceinline__ void decode8(u32_t w, u32_t byte, float (&x)[8]) {
  const float s = scale_of(byte);
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
  x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1], x[4] = c[0], x[5] = c[1], x[6] = d[0], x[7] = d[1];
}

// The values of codes and scales, eight per thread: N values, a multiple of 32.
template <int DT, class I, I N>
__device__ __forceinline__ void values(const u8_t* __restrict__ codes, const u8_t* __restrict__ scales,
                                       typename Elem<DT>::type* __restrict__ out) {
  for (I i = ((I)blockIdx.x * 256 + threadIdx.x) * 8; i < N; i += (I)gridDim.x * 2048) {
    float x[8];
    decode8(*(const u32_t*)(codes + i / 2), scales[i / 32], x);
    store8<DT>(out + i, x);
  }
}

// ---------------------------------------------------------------------------------------------
// The paged cache: u8 [page, kv_head, PB]. A page of T tokens holds per head, in this order, T rows of HD / 2 key codes, T
// rows of HD / 2 value codes, T rows of HD / 32 key scales and T rows of HD / 32 value scales: PB = T (HD + HD / 16). A token's
// place is its slot, page * T + row.
//
// C supplies DT, HD, H (key-value heads), T (a multiple of 32), P (pages).
// ---------------------------------------------------------------------------------------------

template <class C> struct Page {
  static constexpr long BYTES = (long)C::T * (C::HD + C::HD / 16), CODES = (long)C::T * C::HD / 2, SCALES = (long)C::T * C::HD / 32;
  static __device__ __forceinline__ const u8_t* head(const u8_t* cache, long page, long h) { return cache + (page * C::H + h) * BYTES; }
  static __device__ __forceinline__ long codes(bool value, long row) { return (value ? CODES : 0) + row * (C::HD / 2); }
  static __device__ __forceinline__ long scales(bool value, long row) { return 2 * CODES + (value ? SCALES : 0) + row * (C::HD / 32); }
};

// The rows of TOKENS tokens, keys and values [token, head, dim], quantised into their slots: TW tokens per workgroup, eight
// values of both per thread and step. A slot outside the cache writes nothing, and of two tokens of one slot the later
// one is kept, so that codes and scales are always one token's. With few tokens every workgroup looks through the slots
// after its own for them; with OWNERS, `owner` holds the last token of each slot (claim, before).
template <class C> struct Write {
  static constexpr int ROW = C::H * C::HD / 8, TW = ROW >= 512 ? 1 : 512 / ROW;
};
template <class C, bool OWNERS>
__device__ __forceinline__ void cache_write(u8_t* __restrict__ cache, const typename Elem<C::DT>::type* __restrict__ keys,
                                            const typename Elem<C::DT>::type* __restrict__ values, const int* __restrict__ slots,
                                            const int* __restrict__ owner) {
  constexpr int ROW = Write<C>::ROW, TW = Write<C>::TW;
  __shared__ int place[TW];
  const int tid = threadIdx.x;
  const long t0 = (long)blockIdx.x * TW;
  if (tid < TW) {
    int s = t0 + tid < C::TOKENS ? slots[t0 + tid] : -1;
    if (s < 0 || s >= C::P * C::T) s = -1;
    if constexpr (OWNERS) {
      if (s >= 0 && owner[s] != (int)(t0 + tid)) s = -1;
    }
    place[tid] = s;
  }
  __syncthreads();
  if constexpr (!OWNERS) {
    for (long j = t0 + 1 + tid; j < C::TOKENS; j += 256) {
      const int s = slots[j];
      for (int w = 0; w < TW && t0 + w < j; ++w)
        if (place[w] == s) place[w] = -1;
    }
    __syncthreads();
  }
  for (int i = tid; i < TW * ROW; i += 256) {
    const int w = i / ROW, h = i % ROW / (C::HD / 8), c = i % (C::HD / 8) * 8, s = place[w];
    if (s < 0) continue;
    const long at = (t0 + w) * C::H * C::HD + h * C::HD + c;
    float k[8], v[8];
    load8<C::DT>(keys + at, k);
    load8<C::DT>(values + at, v);
    u8_t* const page = cache + ((long)(s / C::T) * C::H + h) * Page<C>::BYTES;
    const u32_t ks = block_scale(k), vs = block_scale(v);
    *(u32_t*)(page + Page<C>::codes(false, s % C::T) + c / 2) = encode8(k, ks);
    *(u32_t*)(page + Page<C>::codes(true, s % C::T) + c / 2) = encode8(v, vs);
    if (c % 32 == 0) {
      page[Page<C>::scales(false, s % C::T) + c / 32] = (u8_t)ks;
      page[Page<C>::scales(true, s % C::T) + c / 32] = (u8_t)vs;
    }
  }
}

// The last token of each slot that a token has: FIRST puts -1 there, then the largest token number is taken.
template <class C, bool FIRST>
__device__ __forceinline__ void claim(const int* __restrict__ slots, int* __restrict__ owner) {
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  if (t >= C::TOKENS) return;
  const int s = slots[t];
  if (s < 0 || s >= C::P * C::T) return;
  if constexpr (FIRST) owner[s] = -1;
  else atomicMax(&owner[s], (int)t);
}

// The keys or values of N slots; zeros for a slot outside the cache.
template <class C, bool VALUE>
__device__ __forceinline__ void cache_read(const u8_t* __restrict__ cache, const int* __restrict__ slots,
                                           typename Elem<C::DT>::type* __restrict__ out) {
  constexpr long N = (long)C::TOKENS * C::H * C::HD;
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8; i < N; i += (long)gridDim.x * 2048) {
    const long row = i / C::HD, h = row % C::H, c = i % C::HD;
    const int slot = slots[row / C::H];
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (slot >= 0 && slot < C::P * C::T) {
      const u8_t* const page = Page<C>::head(cache, slot / C::T, h);
      decode8(*(const u32_t*)(page + Page<C>::codes(VALUE, slot % C::T) + c / 2), page[Page<C>::scales(VALUE, slot % C::T) + c / 32], x);
    }
    store8<C::DT>(out + i, x);
  }
}

// ---------------------------------------------------------------------------------------------
// Attention over the cache: O[b, i, h] = softmax(q[b, i, h] . k_j / sqrt(HD)) v over the keys j < len[b] - (Q - 1 - i) of
// key-value head h / G; key j is row j % T of page pages[b, j / T]. Pages outside the cache hold no keys, and a row that sees no
// key is 0. Scores, softmax and sums are f32.
//
// The Q x G rows that share a key-value head are the columns of 16-wide matrix instructions, NR sixteens of them per wave, so
// the cache is read once for all of them. Per 32 keys (a step) a wave computes S^T = K Q^T (two v_mfma_f32_16x16x32_bf16 tiles of
// 16 keys per 32 dims): lane l holds row l % 16 and, g = l / 16, keys 4 g + i and 16 + 4 g + i, which is how the B operand of
// O^T = V^T P^T wants them when its k index 8 g + j means key 4 g + j (j < 4) or 12 + 4 g + j, so P never leaves the lane. Of
// K's dims, of which any order will do, lane l takes the HD / 4 from g HD / 4 on of key l % 16: they are contiguous. V's rows are
// keys while its A operand wants eight keys of one dim: ds_read_b64_tr_b8 hands a lane one byte (two dims) of eight rows.
//
// fp4 with its scale is exact in bf16. Queries are split into PARTS bf16 parts (bf16 1, f16 2, f32 3: exact, or 24 bits), and the
// probabilities likewise (PP), one matrix instruction each: the sums keep f32's accuracy whatever the type. A row's running
// maximum follows the scores only where one exceeds it by 2^8: till then probabilities are at most 2^8 and sums need no
// rescaling, nor the maximum its way through the lanes.
//
// A step's codes (32 HD bytes) and scales go straight to LDS, three stages of them per wave, each wave on its own: loads that
// are in order, and 8 KB in flight per wave without a register. Rows of a power of two of 16-byte chunks are
// swizzled so that the reads above meet every bank once.
//
// Each wave takes every fourth step of the workgroup's range; the waves join through LDS, the SPLITS workgroups of a
// sequence and head through memory (m, l, O per row) and a second kernel. A range is a share of the sequence's own length.
//
// C supplies, besides the cache's, Q, G, MAXP (pages per sequence), SEQS, NR, SPLITS and SL = log2(e) / sqrt(HD).
// ---------------------------------------------------------------------------------------------

#define ACCY_MX4_LDS __attribute__((address_space(3)))

template <int DT> constexpr int query_parts() { return DT + 1; }

// x as bf16 numbers whose sum is x (to 8 bits a part): the next part; x becomes what is left.
__device__ __forceinline__ __bf16 take_part(float& x) {
  const __bf16 h = (__bf16)x;
  x -= (float)h;
  return h;
}

// Nothing is subtracted while a row has seen no key.
__device__ __forceinline__ float base_of(float m) { return m == -__builtin_inff() ? 0.0f : m; }

template <class C> struct Rows {
  static constexpr int R = C::Q * C::G, TILES = (R + 15) / 16, GROUPS = (TILES + C::NR - 1) / C::NR;
};

// Where 16-byte chunk c of key's row lies within the row's chunks in LDS: 16 rows that are read at one chunk (keys; 32 lanes of
// values read 16 rows, four of each eight) fall into different banks.
template <int CH> __device__ __forceinline__ int key_chunk(int key, int c) {
  if constexpr (CH == 2 || CH == 4 || CH == 8) return c ^ (key / (16 / CH) & (CH - 1));
  else return c;
}
template <int CH> __device__ __forceinline__ int value_chunk(int key, int c) {
  if constexpr (CH == 2) return c ^ (key >> 4 & 1);
  else if constexpr (CH == 4) return c ^ ((key >> 2 & 1) | (key >> 3 & 2));
  else if constexpr (CH == 8) return c ^ ((key >> 1 & 3) | (key >> 2 & 4));
  else return c;
}

// Four bf16 pairs as the eight elements of a matrix operand.
__device__ __forceinline__ bf16x8 eight(bf16x2 a, bf16x2 b, bf16x2 c, bf16x2 d) { return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]}; }

template <int I> __device__ __forceinline__ bf16x2 pair_of_byte(u32_t w, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, I);
}

template <int N> struct Number { static constexpr int value = N; };

template <class C>
__device__ __forceinline__ void attend(const typename Elem<C::DT>::type* __restrict__ Q, const u8_t* __restrict__ cache,
                                       const int* __restrict__ pages, const int* __restrict__ lengths,
                                       typename Elem<C::DT>::type* __restrict__ out, float* __restrict__ part) {
  typedef Page<C> P;
  typedef Rows<C> RS;
  constexpr int HD = C::HD, NB = HD / 32, PARTS = query_parts<C::DT>(), PP = C::DT == 2 ? 3 : 2, NR = C::NR;
  constexpr int CODES = 16 * HD, SCALES = 32 * NB;  // bytes of a step's keys, or values, in LDS
  constexpr int DC = 2 * HD / 64, DS = (16 * NB + 63) / 64, PER = DC + DS;  // load instructions of a step
  constexpr int STAGE = 2 * CODES + 256 * DS;
  // One array per stage: the compiler can then tell a stage's reads from the loads still on their way into the others.
  __shared__ __attribute__((aligned(1024))) u8_t l0[4 * STAGE], l1[4 * STAGE], l2[4 * STAGE];
  // the waves' meeting place, once the steps are done (every load has landed by then): two waves' rows
  constexpr int JOIN = 16 * (HD + 4) * 4;
  static_assert(JOIN <= 4 * STAGE, "a stage of the four waves holds a wave's rows");
  auto joined = [&](int w) { return (float*)(w ? l1 : l0); };
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, r = lane & 15;
  auto stage = [&](auto s) -> u8_t* {
    if constexpr (decltype(s)::value == 0) return l0;
    else if constexpr (decltype(s)::value == 1) return l1;
    else return l2;
  };
  const long bh = blockIdx.x / RS::GROUPS, b = bh / C::H, h = bh % C::H;
  const int row0 = (int)(blockIdx.x % RS::GROUPS) * NR * 16;
  int len = C::P > 0 ? lengths[b] : 0;
  len = len < 0 ? 0 : len > C::MAXP * C::T ? C::MAXP * C::T : len;
  len = __builtin_amdgcn_readfirstlane(len);
  const int steps = (len + 31) / 32, per = (steps + C::SPLITS - 1) / C::SPLITS;
  const int first = (int)blockIdx.y * per, end = first + per < steps ? first + per : steps;
  const int sure = len - (C::Q - 1);  // keys below it are seen by every row

  // queries: the B operand of S^T, row r of each tile, dims g HD / 4 + 8 s + j at step s
  bf16x8 q[NR][NB][PARTS];
  int limit[NR];
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    const int row = row0 + 16 * t + r, i = row / C::G;
    limit[t] = row < RS::R ? len - (C::Q - 1 - i) : 0;
    const long at = ((b * C::Q + i) * C::H * C::G + h * C::G + row % C::G) * HD + g * (HD / 4);
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (row < RS::R) load8<C::DT>(Q + at + 8 * s, x);
#pragma unroll
      for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j) q[t][s][p][j] = take_part(x[j]);
    }
  }
  f32x4 o[NR][NB][2];
  float m[NR], l[NR];
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    m[t] = -__builtin_inff();
    l[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < NB; ++d) o[t][d][0] = o[t][d][1] = f32x4{0, 0, 0, 0};
  }

  // Loads: chunk x = 64 i + lane of a step's LDS, keys and then values; then the scales, a word a lane.
  u32_t from[DC], sfrom[DS];
#pragma unroll
  for (int i = 0; i < DC; ++i) {
    const int x = 64 * i + lane, value = x >= HD, y = value ? x - HD : x, row = y / NB, c = y % NB;
    from[i] = value ? (u32_t)P::CODES + row * (HD / 2) + 16 * value_chunk<NB>(row, c) : row * (HD / 2) + 16 * key_chunk<NB>(row, c);
  }
#pragma unroll
  for (int i = 0; i < DS; ++i) {
    const int x = 64 * i + lane < 16 * NB ? 64 * i + lane : 16 * NB - 1, value = x >= 8 * NB;
    sfrom[i] = (u32_t)(2 * P::CODES) + (value ? (u32_t)P::SCALES + 4 * (x - 8 * NB) : 4 * x);
  }
  auto page_of = [&](int step) { return step < end ? __builtin_amdgcn_readfirstlane(pages[b * C::MAXP + step * 32 / C::T]) : 0; };
  auto load = [&](auto s, int step, int page) {
    const int in = step * 32 % C::T;
    const u8_t* const head = P::head(cache, page >= 0 && page < C::P ? page : 0, h);
    const u8_t *const codes = head + in * (HD / 2), *const scales = head + in * NB;
#pragma unroll
    for (int i = 0; i < DC; ++i) __builtin_amdgcn_global_load_lds(codes + from[i], (ACCY_MX4_LDS void*)(stage(s) + wave * STAGE + 1024 * i), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < DS; ++i)
      __builtin_amdgcn_global_load_lds(scales + sfrom[i], (ACCY_MX4_LDS void*)(stage(s) + wave * STAGE + 2 * CODES + 256 * i), 4, 0, 0);
  };
  auto wait = [&](auto left) {
    constexpr int N = decltype(left)::value;
    static_assert(N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));  // vmcnt(N)
    asm volatile("" ::: "memory");
  };

  // Where in a stage the lane reads: its share of key r's codes (of key 16 + r 8 HD bytes on) and key r's scales; a block's bytes of
  // its value row, which lanes 2 t and 2 t + 1 of sixteen have for their t-th key; the scales of values 4 g .. (16 on: those of 16 + 4 g).
  constexpr int KC = NB % 4 == 0 ? NB / 4 : 1;
  u32_t kat[KC], vat[NB];
#pragma unroll
  for (int c = 0; c < KC; ++c)
    kat[c] = wave * STAGE + r * (HD / 2) +
             (NB % 4 == 0 ? 16 * key_chunk<NB>(r, g * KC + c) : NB == 2 ? 16 * key_chunk<NB>(r, g >> 1) + 8 * (g & 1) : g * (HD / 8));
  const u32_t ksat = wave * STAGE + 2 * CODES + r * NB, vsat = wave * STAGE + 2 * CODES + SCALES + 4 * g * NB;
#pragma unroll
  for (int d = 0; d < NB; ++d) {
    const int tk = r >> 1, key = 4 * g + (tk & 3) + (tk >> 2) * 16;
    vat[d] = wave * STAGE + CODES + key * (HD / 2) + 16 * value_chunk<NB>(key, d) + 8 * (r & 1);
  }

  auto compute = [&](auto s, int step, int page, auto tail_) {
    constexpr bool TAIL = decltype(tail_)::value != 0;
    const int k0 = step * 32;
    const u8_t* const lds = stage(s);
    f32x4 sc[NR][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      u32_t kw[NB];
      if constexpr (NB % 4 == 0) {
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const u32x4 w = *(const u32x4*)(lds + kat[c] + u * 8 * HD);
#pragma unroll
          for (int e = 0; e < 4; ++e) kw[4 * c + e] = w[e];
        }
      } else if constexpr (NB == 2) {
        const u32x2 w = *(const u32x2*)(lds + kat[0] + u * 8 * HD);
        kw[0] = w[0], kw[1] = w[1];
      } else {
#pragma unroll
        for (int e = 0; e < NB; ++e) kw[e] = *(const u32_t*)(lds + kat[0] + u * 8 * HD + 4 * e);
      }
#pragma unroll
      for (int t = 0; t < NR; ++t) sc[t][u] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < NB; ++e) {
        const float x = scale_of(lds[ksat + u * 16 * NB + (g * (HD / 4) + 8 * e) / 32]);
        const bf16x8 a = eight(pair_of_byte<0>(kw[e], x), pair_of_byte<1>(kw[e], x), pair_of_byte<2>(kw[e], x), pair_of_byte<3>(kw[e], x));
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
          for (int p = 0; p < PARTS; ++p) sc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[t][e][p], sc[t][u], 0, 0, 0);
      }
    }
    // The scores' maximum over the lane's keys k0 + 16 u + 4 g + i, those that the row does not see left out.
    float top[NR];
    bool above = false;
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      top[t] = -__builtin_inff();
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (TAIL) sc[t][u][i] = k0 + 16 * u + 4 * g + i < limit[t] && page >= 0 && page < C::P ? sc[t][u][i] : -__builtin_inff();
          top[t] = fmaxf(top[t], sc[t][u][i]);
        }
      top[t] *= C::SL;
      above |= top[t] > m[t] + 8.0f;  // also where m is -inf and a key is seen
    }
    if (__builtin_amdgcn_ballot_w64(above) != 0) {
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        top[t] = fmaxf(top[t], __shfl_xor(top[t], 16, 64));
        top[t] = fmaxf(top[t], __shfl_xor(top[t], 32, 64));
        top[t] = fmaxf(top[t], m[t]);
        const float alpha = __builtin_amdgcn_exp2f(m[t] - base_of(top[t]));
        m[t] = top[t];
        l[t] *= alpha;
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][d][e][i] *= alpha;
      }
    }
    bf16x8 pr[NR][PP];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const float base = base_of(m[t]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][j >> 2][j & 3], C::SL, -base));
        l[t] += p;
#pragma unroll
        for (int e = 0; e < PP; ++e) pr[t][e][j] = take_part(p);
      }
    }
    // scale bytes of the lane's eight keys: four rows of NB bytes, twice
    u32_t vw[2][NB];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < NB; ++e) vw[u][e] = *(const u32_t*)(lds + vsat + 16 * u * NB + 4 * e);
    auto vbyte = [&](int j, int d) { const int at = (j & 3) * NB + d; return vw[j >> 2][at >> 2] >> (8 * (at & 3)) & 255; };
    // The conversions take the scale's exponent bits alone, so its other bits may be the neighbouring bytes'.
    auto vscale = [&](int j, int d) {
      const int at = (j & 3) * NB + d, by = 23 - 8 * (at & 3);
      return by >= 0 ? vw[j >> 2][at >> 2] << by : vw[j >> 2][at >> 2] >> -by;
    };
    // A key that only some rows see must not reach the others where it is NaN (0 x NaN): then one query at a time, with
    // what that query does not see left out. Keys past the end are left out always.
    bool apart = false;
    if constexpr (TAIL && C::Q > 1) {
      bool nan = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = k0 + 4 * g + (j & 3) + (j >> 2) * 16;
#pragma unroll
        for (int d = 0; d < NB; ++d) nan |= key >= sure && key < len && vbyte(j, d) == 255;
      }
      apart = __builtin_amdgcn_ballot_w64(nan) != 0;
    }
    auto weigh = [&](int only) {
      const int seen = page >= 0 && page < C::P ? len - (C::Q - 1 - only) : 0;
#pragma unroll
      for (int d = 0; d < NB; ++d) {
        const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((ACCY_MX4_LDS i32x2*)(lds + vat[d]));
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u32_t scale = vscale(j, d);
          if constexpr (TAIL) scale = k0 + 4 * g + (j & 3) + (j >> 2) * 16 < seen ? scale : 0;
          x[j] = __builtin_bit_cast(float, scale);
        }
        const bf16x2 y[8] = {pair_of_byte<0>((u32_t)w[0], x[0]), pair_of_byte<1>((u32_t)w[0], x[1]), pair_of_byte<2>((u32_t)w[0], x[2]),
                             pair_of_byte<3>((u32_t)w[0], x[3]), pair_of_byte<0>((u32_t)w[1], x[4]), pair_of_byte<1>((u32_t)w[1], x[5]),
                             pair_of_byte<2>((u32_t)w[1], x[6]), pair_of_byte<3>((u32_t)w[1], x[7])};
        bf16x8 even, odd;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          even[j] = y[j][0];
          odd[j] = y[j][1];
        }
#pragma unroll
        for (int t = 0; t < NR; ++t) {
          const f32x4 before[2] = {o[t][d][0], o[t][d][1]};
#pragma unroll
          for (int p = 0; p < PP; ++p) {
            o[t][d][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, pr[t][p], o[t][d][0], 0, 0, 0);
            o[t][d][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, pr[t][p], o[t][d][1], 0, 0, 0);
          }
          if constexpr (TAIL && C::Q > 1) {
            const bool mine = !apart || (row0 + 16 * t + r) / C::G == only;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[t][d][e][i] = mine ? o[t][d][e][i] : before[e][i];
          }
        }
      }
    };
    if constexpr (TAIL && C::Q > 1) {
#pragma unroll 1
      for (int only = apart ? 0 : C::Q - 1; only < C::Q; ++only) weigh(only);
    } else {
      weigh(C::Q - 1);
    }
  };

  {
    int step = first + wave, p0 = page_of(step), p1 = page_of(step + 4), p2 = page_of(step + 8);
    // Stage S holds step `now` of page `mine`; the step two stages on goes to stage S + 2, its page into `mine`.
    auto turn = [&](auto s, auto two, int now, int& mine, int next) {
      // This stage has landed when no more than the next one's and the one's after are outstanding; where no more follow, when
      // nothing is.
      const int page = mine;
      if (now + 8 < end) {
        load(two, now + 8, next);
        mine = page_of(now + 12);
        wait(Number<2 * PER>());
      } else {
        wait(Number<0>());
      }
      if (now * 32 + 32 <= sure && page >= 0 && page < C::P) compute(s, now, page, Number<0>());
      else compute(s, now, page, Number<1>());
      __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8));  // lgkmcnt(0): the stage may be overwritten
      asm volatile("" ::: "memory");
    };
    if (step < end) load(Number<0>(), step, p0);
    if (step + 4 < end) load(Number<1>(), step + 4, p1);
    for (; step < end; step += 12) {
      turn(Number<0>(), Number<2>(), step, p0, p2);
      if (step + 4 >= end) break;
      turn(Number<1>(), Number<0>(), step + 4, p1, p0);
      if (step + 8 >= end) break;
      turn(Number<2>(), Number<1>(), step + 8, p2, p1);
    }
  }

  // The waves: 2 and 3 hand theirs to 0 and 1, then 1 to 0. Lane (r, g) holds dims 32 d + 8 g .. + 7 of row r: even ones in
  // [0], odd ones in [1]. A row in LDS: HD outputs, m, then l per lane group.
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    l[t] += __shfl_xor(l[t], 16, 64);
    l[t] += __shfl_xor(l[t], 32, 64);
#pragma unroll
    for (int from = 2; from > 0; from >>= 1) {
      __syncthreads();
      if (wave >= from && wave < 2 * from) {
        float* const p = joined(wave - from) + r * (HD + 4);
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[32 * d + 8 * g + 2 * i] = o[t][d][0][i];
            p[32 * d + 8 * g + 2 * i + 1] = o[t][d][1][i];
          }
        if (g == 0) {
          p[HD] = m[t];
          p[HD + 1] = l[t];
        }
      }
      __syncthreads();
      if (wave < from) {
        const float* const p = joined(wave) + r * (HD + 4);
        const float top = fmaxf(m[t], p[HD]), base = base_of(top);
        const float mine = __builtin_amdgcn_exp2f(m[t] - base), theirs = __builtin_amdgcn_exp2f(p[HD] - base);
        m[t] = top;
        l[t] = l[t] * mine + p[HD + 1] * theirs;
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[t][d][0][i] = o[t][d][0][i] * mine + p[32 * d + 8 * g + 2 * i] * theirs;
            o[t][d][1][i] = o[t][d][1][i] * mine + p[32 * d + 8 * g + 2 * i + 1] * theirs;
          }
      }
    }
  }
  if (wave != 0) return;
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    const int row = row0 + 16 * t + r;
    if (row >= RS::R) continue;
    if constexpr (C::SPLITS == 1) {
      const long at = ((b * C::Q + row / C::G) * C::H * C::G + h * C::G + row % C::G) * HD;
      const float by = l[t] == 0.0f ? 0.0f : 1.0f / l[t];
#pragma unroll
      for (int d = 0; d < NB; ++d) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = o[t][d][i & 1][i >> 1] * by;
        store8<C::DT>(out + at + 32 * d + 8 * g, x);
      }
    } else {
      float* const p = part + ((bh * RS::R + row) * C::SPLITS + blockIdx.y) * (HD + 4);
#pragma unroll
      for (int d = 0; d < NB; ++d) {
        *(f32x4*)(p + 32 * d + 8 * g) = f32x4{o[t][d][0][0], o[t][d][1][0], o[t][d][0][1], o[t][d][1][1]};
        *(f32x4*)(p + 32 * d + 8 * g + 4) = f32x4{o[t][d][0][2], o[t][d][1][2], o[t][d][0][3], o[t][d][1][3]};
      }
      if (g == 0) {
        p[HD] = m[t];
        p[HD + 1] = l[t];
      }
    }
  }
}

// The rows' outputs from their splits' parts, in split order; one thread per output.
template <class C>
__device__ __forceinline__ void attend_join(const float* __restrict__ part, typename Elem<C::DT>::type* __restrict__ out) {
  constexpr long R = Rows<C>::R, N = (long)C::SEQS * C::H * R * C::HD;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= N) return;
  const long bhr = i / C::HD, d = i % C::HD, row = bhr % R, bh = bhr / R;
  const float* const p = part + bhr * C::SPLITS * (C::HD + 4);
  float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
#pragma unroll 8
  for (int s = 0; s < C::SPLITS; ++s) m = fmaxf(m, p[s * (C::HD + 4) + C::HD]);
  const float base = base_of(m);
#pragma unroll 8
  for (int s = 0; s < C::SPLITS; ++s) {
    const float* const x = p + s * (C::HD + 4);
    const float scale = __builtin_amdgcn_exp2f(x[C::HD] - base);
    l += x[C::HD + 1] * scale;
    o += x[d] * scale;
  }
  const long at = ((bh / C::H * C::Q + row / C::G) * C::H * C::G + bh % C::H * C::G + row % C::G) * C::HD;
  out[at + d] = to_elem<C::DT>(l == 0.0f ? 0.0f : o / l);
}

}  // namespace mx4
}  // namespace accy
