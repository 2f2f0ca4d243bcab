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

// The scale byte of the block that 32 / V adjacent lanes hold V values each of (all of them call it), and the codes of
// this lane's. The exponent of the largest magnitude comes from its bits: the unsigned order of the bits without
// the sign is the order of the magnitudes, with infinity and NaN above all of them. The scale's exponent is 2 less, and
// 2^-127 (byte 0) for everything below 2^-125, subnormals and zero among it.
template <int V> __device__ __forceinline__ u32_t block_scale(const float (&x)[V]) {
  u32_t top = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const u32_t b = __builtin_bit_cast(u32_t, x[i]) & 0x7fffffffu;
    top = top > b ? top : b;
  }
#pragma unroll
  for (int o = 1; o < 32 / V; o <<= 1) {
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
// The same of four values, codes in the low half.
__device__ __forceinline__ u32_t encode4(const float (&x)[4], u32_t byte) {
  const float s = scale_of(byte);
  const u32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], s, 0);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
}
__device__ __forceinline__ void decode4(u32_t w, u32_t byte, float (&x)[4]) {
  const float s = scale_of(byte);
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
  x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
}
template <int DT> __device__ __forceinline__ void store4(typename Elem<DT>::type* __restrict__ p, const float (&x)[4]) {
  if constexpr (DT == 2) {
    *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
  } else {
    *(u32x2*)p = u32x2{(u32_t)to_elem<DT>(x[0]) | ((u32_t)to_elem<DT>(x[1]) << 16), (u32_t)to_elem<DT>(x[2]) | ((u32_t)to_elem<DT>(x[3]) << 16)};
  }
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

// place[w], the slot of token w of TW or -1, becomes -1 where a later one of `left` tokens has the same: the part of thread tid of 256.
template <int TW>
__device__ __forceinline__ void leave_to_later(int* place, const int* __restrict__ slots, int left, int tid) {
  constexpr int W = TW < 4 ? TW : 4;
  for (int j0 = 1 + tid; j0 < left; j0 += 2048) {
    int s[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) s[u] = j0 + 256 * u < left ? slots[j0 + 256 * u] : -1;
    for (int w0 = 0; w0 < TW; w0 += W) {
      int mine[W];
#pragma unroll
      for (int w = 0; w < W; ++w) mine[w] = w0 + w < TW ? place[w0 + w] : -1;
      u32_t lost = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int w = 0; w < W; ++w) lost |= s[u] == mine[w] && j0 + 256 * u > w0 + w ? 1u << w : 0;
      if (lost != 0) {
        // (a token without a slot has nothing to lose, and past TW there is none)
#pragma unroll
        for (int w = 0; w < W; ++w)
          if ((lost >> w & 1) && mine[w] >= 0) place[w0 + w] = -1;
      }
    }
  }
}

// The rows of TOKENS tokens, keys and values [token, head, dim], quantised into their slots: TW tokens per workgroup, eight
// values of both per thread and step. A slot outside the cache writes nothing, and of two tokens of one slot the later
// one is kept, so that codes and scales are always one token's. With few tokens every workgroup looks through the slots
// after its own for them, eight loads at a time and its first rows already on their way; with OWNERS, `owner` holds the last
// token of each slot (claim, before).
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
  float k[2][8], v[2][8];
  auto fetch = [&](int u, int i) {
    const long at = t0 * C::H * C::HD + (long)i * 8;
    if (i < TW * ROW && t0 + i / ROW < C::TOKENS) {
      load8<C::DT>(keys + at, k[u]);
      load8<C::DT>(values + at, v[u]);
    }
  };
  fetch(0, tid);
  fetch(1, 256 + tid);
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
    leave_to_later<TW>(place, slots + t0, (int)(C::TOKENS - t0), tid);
    __syncthreads();
  }
  for (int i0 = 0; i0 < TW * ROW; i0 += 512) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = i0 + 256 * u + tid;
      if (i0 > 0) fetch(u, i);
      if (i >= TW * ROW) continue;
      const int w = i / ROW, h = i % ROW / (C::HD / 8), c = i % (C::HD / 8) * 8, s = place[w];
      if (s < 0) continue;
      u8_t* const page = cache + ((long)(s / C::T) * C::H + h) * Page<C>::BYTES;
      const u32_t ks = block_scale(k[u]), vs = block_scale(v[u]);
      *(u32_t*)(page + Page<C>::codes(false, s % C::T) + c / 2) = encode8(k[u], ks);
      *(u32_t*)(page + Page<C>::codes(true, s % C::T) + c / 2) = encode8(v[u], vs);
      if (c % 32 == 0) {
        page[Page<C>::scales(false, s % C::T) + c / 32] = (u8_t)ks;
        page[Page<C>::scales(true, s % C::T) + c / 32] = (u8_t)vs;
      }
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

// The keys, the values or both of N slots (none: nullptr); zeros for a slot outside the cache.
template <class C>
__device__ __forceinline__ void cache_read(const u8_t* __restrict__ cache, const int* __restrict__ slots,
                                           typename Elem<C::DT>::type* __restrict__ keys, typename Elem<C::DT>::type* __restrict__ values) {
  constexpr long N = (long)C::TOKENS * C::H * C::HD;
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8; i < N; i += (long)gridDim.x * 2048) {
    const long row = i / C::HD, h = row % C::H, c = i % C::HD;
    const int slot = slots[row / C::H];
#pragma unroll
    for (int value = 0; value < 2; ++value) {
      typename Elem<C::DT>::type* const out = value ? values : keys;
      if (!out) continue;
      float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (slot >= 0 && slot < C::P * C::T) {
        const u8_t* const page = Page<C>::head(cache, slot / C::T, h);
        decode8(*(const u32_t*)(page + Page<C>::codes(value != 0, slot % C::T) + c / 2),
                page[Page<C>::scales(value != 0, slot % C::T) + c / 32], x);
      }
      store8<C::DT>(out + i, x);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Attention over the cache: O[b, i, h] = softmax(q[b, i, h] . k_j / sqrt(HD)) v over the keys j < len[b] - (Q - 1 - i) of
// key-value head h / G; key j is row j % T of page pages[b, j / T]. Pages outside the cache hold no keys, and a row that sees no
// key is 0. Scores, softmax and sums are f32.
//
// The Q x G rows that share a key-value head are the columns of 16-wide matrix instructions, 16 rows to a workgroup (two sixteens to
// a wave, so that the cache is read once for 32 rows, run out of registers: with keys unwidened and probabilities in 17 bits 24 x 8 heads x
// 8000 keys of 128, 32 rows, bf16, took 94 us so, and 65 in twice the workgroups). Per 32 keys (a step) a wave computes S^T = K Q^T, two tiles of 16 keys, on
// v_mfma_f32_16x16x32_bf16, with K widened to bf16, in which fp4 with its scale is exact, and the queries as QP bf16 numbers whose
// sum they are, all bits of them (bf16 1, f16 2, f32 3). Lane group g of four holds dims g HD / 4 .. of a key and of a
// row, so that a lane's codes are adjacent, and of an instruction's eight dims one block's. (The scaled 4-bit instruction takes
// keys as they lie and saves 32 VALU instructions a step of 128 dims, but queries as three e4m3 numbers on their block's scale
// lose what lies 2^-20 below its largest, and it is no faster: 48 x 8 x 8 heads x 16000 keys 116 us either way, 8 x 16 x 4096 18.3 against
// 16.7.)
// Lane l then holds row l % 16 and, g = l / 16, keys 4 g + i and 16 + 4 g + i, which is how the B operand of O^T = V^T P^T
// (the same instruction) wants them when its k index 8 g + j means key 4 g + j (j < 4) or 12 + 4 g + j, so P never leaves
// the lane. V's blocks lie along its dims and not along the keys that are summed, so V is widened to bf16, in which fp4 with its
// scale is exact; its rows are keys while the A operand wants eight keys of one dim: ds_read_b64_tr_b8 hands a lane one byte (two
// dims) of eight rows. The probabilities are split into three bf16 numbers, one matrix instruction each, which is all bits of
// them (with two, 17 bits, 48 x 8 x 8 heads x 16000 keys of 128 bf16 take 117 us instead of 122, and one of 400 results is the neighbour
// of f32's rounded). A row's running maximum follows the scores only where one exceeds it by 2^8: till then
// probabilities are at most 2^8 and sums need no rescaling, nor the maximum its way through the lanes.
//
// A step's codes (32 HD bytes) and scales go straight to LDS, three stages of them per wave, each wave on its own: loads that
// are in order, and 8 KB in flight per wave without a register. Rows of a power of two of 16-byte chunks are
// swizzled so that the reads above meet every bank once.
//
// Each wave takes every fourth step of the workgroup's range; the waves join through LDS, the SPLITS workgroups of a
// sequence and head through memory (m, l, O per row) and a second kernel. A range is a share of the sequence's own length.
//
// C supplies, besides the cache's, Q, G, MAXP (pages per sequence), SEQS, SPLITS and SL = log2(e) / sqrt(HD).
// ---------------------------------------------------------------------------------------------

#define ACCY_MX4_LDS __attribute__((address_space(3)))

// The upper eight bits of a number's significand, as a bf16 number; x becomes what is left, exactly.
__device__ __forceinline__ u32_t take_top(float& x) {
  const u32_t w = __builtin_bit_cast(u32_t, x) & 0xffff0000u;
  x -= __builtin_bit_cast(float, w);
  return w >> 16;
}

// Two values as bf16 numbers whose sums they are (to 8 bits a part): the next part of both; x becomes what is left.
__device__ __forceinline__ u32_t take_parts(f32x2& x) {
  const u32_t w = __builtin_bit_cast(u32_t, __builtin_convertvector(x, bf16x2));
  x[0] -= __builtin_bit_cast(float, w << 16);
  x[1] -= __builtin_bit_cast(float, w & 0xffff0000u);
  return w;
}

// Nothing is subtracted while a row has seen no key.
__device__ __forceinline__ float base_of(float m) { return m == -__builtin_inff() ? 0.0f : m; }

template <class C> struct Rows {
  static constexpr int R = C::Q * C::G, GROUPS = (R + 15) / 16;
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

template <int I> __device__ __forceinline__ bf16x2 pair_of_byte(u32_t w, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, I);
}

template <int N> struct Number { static constexpr int value = N; };

// Shared keys: C::PREFIXES, PSPLITS (workgroups along a prefix), PREFIX_MAXP (pages of one); without them 0. The rows of a prefix are those of
// its sequences, one sequence after the other, sixteen to a workgroup: at most so many groups.
template <class C, class = void> struct Shared {
  static constexpr int N = 0, SPLITS = 0, MAXP = 0;
};
template <class C> struct Shared<C, decltype((void)C::PREFIXES)> {
  static constexpr int N = C::PREFIXES, SPLITS = C::PSPLITS, MAXP = C::PREFIX_MAXP;
};
template <class C> constexpr int PREFIXES = Shared<C>::N;
template <class C> constexpr int PSPLITS = Shared<C>::SPLITS;
template <class C> constexpr int PREFIX_PAGES = Shared<C>::MAXP;
template <class C> constexpr int PREFIX_GROUPS = (int)(C::SEQS * Rows<C>::R / 16) + Shared<C>::N;

// The prefix that group `group` of the prefixes' rows belongs to (-1: there is no such group), the group's first row of the prefix's, and how
// many those are. The sequences of the group's rows go to `list`, in order. All threads; `list` has room for 16 and the counts.
struct Members {
  int prefix, row0, rows;
};
template <class C> __device__ __forceinline__ Members members_of(const int* __restrict__ of, int group, int* list) {
  constexpr int R = Rows<C>::R, N = PREFIXES<C>;
  int* const count = list + 16;
  int* const waves = count + N;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < N; i += 256) count[i] = 0;
  __syncthreads();
  for (long s = tid; s < C::SEQS; s += 256) {
    const int p = of[s];
    if (p >= 0 && p < N) atomicAdd(&count[p], 1);
  }
  __syncthreads();
  Members m = {-1, 0, 0};
  for (int p = 0; p < N; ++p) {
    const int groups = (count[p] * R + 15) / 16;
    if (group < groups) {
      m = {p, group * 16, count[p] * R};
      break;
    }
    group -= groups;
  }
  if (m.prefix < 0) return m;
  // its sequences number first .. last in order
  const int first = m.row0 / R, last = (m.row0 + 15) / R;
  int before = 0;
  for (long s0 = 0; s0 < C::SEQS && before <= last; s0 += 256) {
    const bool mine = s0 + tid < C::SEQS && of[s0 + tid] == m.prefix;
    const u64_t ballot = __builtin_amdgcn_ballot_w64(mine);
    if (lane == 0) waves[wave] = __builtin_popcountll(ballot);
    __syncthreads();
    int k = before + __builtin_popcountll(ballot & ((1ull << lane) - 1));
    for (int w = 0; w < 4; ++w) {
      if (w < wave) k += waves[w];
      before += waves[w];
    }
    if (mine && k >= first && k <= last) list[k - first] = (int)(s0 + tid);
    __syncthreads();
  }
  return m;
}

// What a workgroup's keys are: all of its sequence's, or with shared keys its sequence's own or those of a prefix.
enum Keys { ALL, OWN, PREFIX };

// What the stages of a workgroup's loads take, and the numbers that follow from C.
template <class C> struct Stages {
  static constexpr int NB = C::HD / 32, CODES = 16 * C::HD, SCALES = 32 * NB;  // bytes of a step's keys, or values, in LDS
  static constexpr int DC = 2 * C::HD / 64, DS = (16 * NB + 63) / 64, PER = DC + DS;  // load instructions of a step
  static constexpr int STAGE = 2 * CODES + 256 * DS;
};

template <class C, Keys KEYS>
__device__ __forceinline__ void attend_keys(const typename Elem<C::DT>::type* __restrict__ Q, const u8_t* __restrict__ cache,
                                            const int* __restrict__ pages, const int* __restrict__ lengths, const int* __restrict__ of,
                                            typename Elem<C::DT>::type* __restrict__ out, float* __restrict__ part, const int block, const int split,
                                            u8_t (&l0)[4 * Stages<C>::STAGE], u8_t (&l1)[4 * Stages<C>::STAGE], u8_t (&l2)[4 * Stages<C>::STAGE]) {
  typedef Page<C> P;
  typedef Rows<C> RS;
  typedef Stages<C> ST;
  constexpr int HD = C::HD, NB = ST::NB, QP = C::DT + 1, PP = 3;
  constexpr int W = NB % 4 == 0 ? 4 : NB % 2 == 0 ? 2 : 1;  // eights of a key's dims to a read, all of one block
  constexpr int CODES = ST::CODES, SCALES = ST::SCALES, DC = ST::DC, DS = ST::DS, PER = ST::PER, STAGE = ST::STAGE;
  // A cache that one workgroup alone reads streams by with the non-temporal hint (48 x 8 x 8 heads x 16000 keys of 128 bf16 122 us,
  // 138 without).
  constexpr int ONCE = KEYS != PREFIX && RS::GROUPS == 1 ? 2 : 0;
  // where the waves meet, once the steps are done (every load has landed by then): two waves' rows to a stage
  constexpr int JOIN = 16 * (HD + 4);
  static_assert(2 * JOIN * 4 <= 4 * STAGE, "a stage of the four waves holds two waves' rows");
  auto joined = [&](int k) { return (float*)(k < 2 ? l0 : l1) + (k & 1) * JOIN; };
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, r = lane & 15;
  auto stage = [&](auto s) -> u8_t* {
    if constexpr (decltype(s)::value == 0) return l0;
    else if constexpr (decltype(s)::value == 1) return l1;
    else return l2;
  };
  // A head's groups of rows lie eight workgroups apart, on one XCD: its cache comes through that one's L2 (24 x 8 heads x 8000 keys
  // of 128, 32 rows bf16: 70 us side by side, 68 so).
  constexpr int SETS = KEYS == PREFIX ? C::H * PSPLITS<C> : (int)(C::SEQS * C::H), GROUPS = KEYS == PREFIX ? PREFIX_GROUPS<C> : RS::GROUPS;
  const int set = block / (8 * GROUPS), in = block % (8 * GROUPS);
  const int wide = SETS - 8 * set < 8 ? SETS - 8 * set : 8;
  // b: the sequence or the prefix; row0: the first of the workgroup's rows among those of its head and sequence or prefix, `rows` in all.
  long bh = 8 * set + in % wide, b = bh / C::H, h = bh % C::H;
  int row0 = in / wide * 16, rows = RS::R, share = split;
  int member = 0;
  if constexpr (KEYS == PREFIX) {
    h = bh % C::H;
    share = (int)(bh / C::H);
    const Members m = members_of<C>(of, in / wide, (int*)l0);
    if (m.prefix < 0) return;  // (there are fewer groups than there could be)
    b = m.prefix;
    row0 = m.row0;
    rows = m.rows;
    member = row0 + (lane & 15) < rows ? ((const int*)l0)[(row0 + (lane & 15)) / RS::R - row0 / RS::R] : 0;
    __syncthreads();  // the list's place is a stage's
  }
  constexpr int MAXP = KEYS == PREFIX ? PREFIX_PAGES<C> : C::MAXP, SHARES = KEYS == PREFIX ? PSPLITS<C> : C::SPLITS;
  int len = C::P > 0 ? lengths[b] : 0;
  len = len < 0 ? 0 : len > MAXP * C::T ? MAXP * C::T : len;
  len = __builtin_amdgcn_readfirstlane(len);
  const int steps = (len + 31) / 32, per = (steps + SHARES - 1) / SHARES;
  const int first = share * per, end = first + per < steps ? first + per : steps;
  const int sure = KEYS == PREFIX ? len : len - (C::Q - 1);  // keys below it are seen by every row

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
  auto page_of = [&](int step) { return step < end ? __builtin_amdgcn_readfirstlane(pages[b * MAXP + step * 32 / C::T]) : 0; };
  auto load = [&](auto s, int step, int page) {
    const int in = step * 32 % C::T;
    const u8_t* const head = P::head(cache, page >= 0 && page < C::P ? page : 0, h);
    const u8_t *const codes = head + in * (HD / 2), *const scales = head + in * NB;
#pragma unroll
    for (int i = 0; i < DC; ++i) __builtin_amdgcn_global_load_lds(codes + from[i], (ACCY_MX4_LDS void*)(stage(s) + wave * STAGE + 1024 * i), 16, 0, ONCE);
#pragma unroll
    for (int i = 0; i < DS; ++i)
      __builtin_amdgcn_global_load_lds(scales + sfrom[i], (ACCY_MX4_LDS void*)(stage(s) + wave * STAGE + 2 * CODES + 256 * i), 4, 0, ONCE);
  };
  int step = first + wave, p0 = page_of(step), p1 = page_of(step + 4), p2 = page_of(step + 8);
  // The queries are asked for before the steps' loads, which would have to land first otherwise, and worked on after.
  float x[NB][8];
  // (a row of a prefix is one of its sequences' rows, one sequence after the other)
  const int row = row0 + r, inner = KEYS == PREFIX ? row % RS::R : row;
  const long seq = KEYS == PREFIX ? (long)member : b;
  const long at = ((seq * C::Q + inner / C::G) * C::H * C::G + h * C::G + inner % C::G) * HD;
#pragma unroll
  for (int t = 0; t < NB; ++t) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[t][j] = 0;
    if (row < rows) load8<C::DT>(Q + at + 8 * (g * NB + t), x[t]);
  }
  __builtin_amdgcn_sched_barrier(0);
  if (step < end) load(Number<0>(), step, p0);
  if (step + 4 < end) load(Number<1>(), step + 4, p1);

  // Queries: the B operand of S^T, row r, eight dims to an instruction. Infinities become NaN, as their scores do.
  u32x4 q[NB][QP];
  const int limit = row < rows ? len - (KEYS == PREFIX ? 0 : C::Q - 1 - row / C::G) : 0;
#pragma unroll
  for (int t = 0; t < NB; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float y[2] = {x[t][2 * j] + (x[t][2 * j] - x[t][2 * j]), x[t][2 * j + 1] + (x[t][2 * j + 1] - x[t][2 * j + 1])};
#pragma unroll
      for (int p = 0; p < QP; ++p) {
        const u32_t first = take_top(y[0]);
        q[t][p][j] = first | take_top(y[1]) << 16;
      }
    }
  f32x4 o[NB][2];
  float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
  for (int d = 0; d < NB; ++d) o[d][0] = o[d][1] = f32x4{0, 0, 0, 0};

  auto wait = [&](auto left) {
    constexpr int N = decltype(left)::value;
    static_assert(N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));  // vmcnt(N)
    asm volatile("" ::: "memory");
  };

  // Where in a stage the lane reads: W eights of key r (of key 16 + r 8 HD bytes on) and their block's scale; a block's bytes
  // of its value row, which lanes 2 t and 2 t + 1 of sixteen have for their t-th key; the scales of values 4 g .. (16 on: those
  // of 16 + 4 g).
  u32_t kat[NB / W], ksat[NB / W], vat[NB];
#pragma unroll
  for (int c = 0; c < NB / W; ++c) {
    const int eight = g * NB + c * W;
    kat[c] = wave * STAGE + r * (HD / 2) + 16 * key_chunk<NB>(r, eight / 4) + eight % 4 * 4;
    ksat[c] = wave * STAGE + 2 * CODES + r * NB + eight / 4;
  }
  const u32_t vsat = wave * STAGE + 2 * CODES + SCALES + 4 * g * NB;
#pragma unroll
  for (int d = 0; d < NB; ++d) {
    const int tk = r >> 1, key = 4 * g + (tk & 3) + (tk >> 2) * 16;
    vat[d] = wave * STAGE + CODES + key * (HD / 2) + 16 * value_chunk<NB>(key, d) + 8 * (r & 1);
  }

  // sc[u][i]: key 16 u + 4 g + i of the stage against row r.
  auto scores = [&](auto s, f32x4 (&sc)[2]) {
    const u8_t* const lds = stage(s);
    sc[0] = sc[1] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < NB / W; ++c) {
      typedef u32_t codes_t __attribute__((ext_vector_type(W)));
      codes_t w[2];
      float scale[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        w[u] = *(const codes_t*)(lds + kat[c] + u * 8 * HD);
        scale[u] = scale_of(lds[ksat[c] + u * 16 * NB]);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const bf16x2 y[4] = {pair_of_byte<0>(w[u][e], scale[u]), pair_of_byte<1>(w[u][e], scale[u]), pair_of_byte<2>(w[u][e], scale[u]),
                               pair_of_byte<3>(w[u][e], scale[u])};
          bf16x8 k;
#pragma unroll
          for (int j = 0; j < 8; ++j) k[j] = y[j >> 1][j & 1];
#pragma unroll
          for (int p = 0; p < QP; ++p)
            sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, __builtin_bit_cast(bf16x8, q[c * W + e][p]), sc[u], 0, 0, 0);
        }
        // a block's widened codes at a time: the registers of more would cost a CU its third workgroup
        if ((c + 1) * W % 4 == 0) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  auto compute = [&](auto s, f32x4 (&sc)[2], int step, int page, auto tail_) {
    constexpr bool TAIL = decltype(tail_)::value != 0;
    const int k0 = step * 32;
    const u8_t* const lds = stage(s);
    // The scores' maximum over the lane's keys k0 + 16 u + 4 g + i, those that the row does not see left out.
    float top = -__builtin_inff();
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (TAIL) sc[u][i] = k0 + 16 * u + 4 * g + i < limit && page >= 0 && page < C::P ? sc[u][i] : -__builtin_inff();
        top = fmaxf(top, sc[u][i]);
      }
    top *= C::SL;
    if (__builtin_amdgcn_ballot_w64(top > m + 8.0f) != 0) {  // also where m is -inf and a key is seen
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      top = fmaxf(top, m);
      const float alpha = __builtin_amdgcn_exp2f(m - base_of(top));
      m = top;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][e][i] *= alpha;
    }
    u32x4 pr[PP];
    const float base = base_of(m);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      f32x2 p = {__builtin_amdgcn_exp2f(__builtin_fmaf(sc[j >> 2][j & 3], C::SL, -base)),
                 __builtin_amdgcn_exp2f(__builtin_fmaf(sc[(j + 1) >> 2][(j + 1) & 3], C::SL, -base))};
      l += p[0];
      l += p[1];
#pragma unroll
      for (int e = 0; e < PP; ++e) pr[e][j >> 1] = take_parts(p);
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
    // A key that only some rows see must not reach the others where its value is NaN or, with the two scales whose larger codes are
    // beyond f32, infinite (0 x NaN): then one query of the workgroup's rows at
    // a time, with what that query does not see left out. Keys past the end are left out always.
    bool apart = false;
    if constexpr (TAIL && C::Q > 1 && KEYS != PREFIX) {
      bool nan = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = k0 + 4 * g + (j & 3) + (j >> 2) * 16;
#pragma unroll
        for (int d = 0; d < NB; ++d) nan |= key >= sure && key < len && vbyte(j, d) >= 253;
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
        const f32x4 before[2] = {o[d][0], o[d][1]};
#pragma unroll
        for (int p = 0; p < PP; ++p) {
          o[d][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, __builtin_bit_cast(bf16x8, pr[p]), o[d][0], 0, 0, 0);
          o[d][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, __builtin_bit_cast(bf16x8, pr[p]), o[d][1], 0, 0, 0);
        }
        if constexpr (TAIL && C::Q > 1 && KEYS != PREFIX) {
          const bool mine = !apart || (row0 + r) / C::G == only;
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][e][i] = mine ? o[d][e][i] : before[e][i];
        }
      }
    };
    if constexpr (TAIL && C::Q > 1 && KEYS != PREFIX) {
      const int most = (row0 + 15) / C::G < C::Q ? (row0 + 15) / C::G : C::Q - 1;  // the last query of the workgroup's rows
#pragma unroll 1
      for (int only = apart ? row0 / C::G : C::Q - 1; only <= (apart ? most : C::Q - 1); ++only) weigh(only);
    } else {
      weigh(C::Q - 1);
    }
  };

  {
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
      f32x4 sc[2];
      scores(s, sc);
      if (now * 32 + 32 <= sure && page >= 0 && page < C::P) compute(s, sc, now, page, Number<0>());
      else compute(s, sc, now, page, Number<1>());
      __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8));  // lgkmcnt(0): the stage may be overwritten
      asm volatile("" ::: "memory");
    };
    for (; step < end; step += 12) {
      turn(Number<0>(), Number<2>(), step, p0, p2);
      if (step + 4 >= end) break;
      turn(Number<1>(), Number<0>(), step + 4, p1, p0);
      if (step + 8 >= end) break;
      turn(Number<2>(), Number<1>(), step + 8, p2, p1);
    }
  }

  // The waves meet: lane (r, g) holds dims 32 d + 8 g .. + 7 of row r, even ones in [0], odd ones in [1]. A row in LDS is HD
  // outputs, m and l; then every thread joins the four waves' four dims of a row.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  __syncthreads();
  float* const p = joined(wave) + r * (HD + 4);
#pragma unroll
  for (int d = 0; d < NB; ++d) {
    *(f32x4*)(p + 32 * d + 8 * g) = f32x4{o[d][0][0], o[d][1][0], o[d][0][1], o[d][1][1]};
    *(f32x4*)(p + 32 * d + 8 * g + 4) = f32x4{o[d][0][2], o[d][1][2], o[d][0][3], o[d][1][3]};
  }
  if (g == 0) {
    p[HD] = m;
    p[HD + 1] = l;
    if (KEYS == PREFIX && wave == 0) p[HD + 2] = __builtin_bit_cast(float, member);
  }
  __syncthreads();
  for (int at = tid; at < 16 * HD / 4; at += 256) {
    const int rr = at / (HD / 4), d = at % (HD / 4) * 4, row = row0 + rr;
    if (row >= rows) continue;
    const int from = rr * (HD + 4);
    float top = joined(0)[from + HD], sum = 0.0f;
#pragma unroll
    for (int k = 1; k < 4; ++k) top = fmaxf(top, joined(k)[from + HD]);
    const float base = base_of(top);
    f32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float* const w = joined(k) + from;
      const float scale = __builtin_amdgcn_exp2f(w[HD] - base);
      const f32x4 y = *(const f32x4*)(w + d);
      sum += w[HD + 1] * scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += y[i] * scale;
    }
    if constexpr (KEYS == ALL && C::SPLITS == 1) {
      const long to = ((b * C::Q + row / C::G) * C::H * C::G + h * C::G + row % C::G) * HD + d;
      const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[to + i] = to_elem<C::DT>(v[i] * by);
    } else {
      // a row's parts: those of its prefix, then those of its own keys
      constexpr int PARTS = KEYS == ALL ? C::SPLITS : C::SPLITS + PSPLITS<C>;
      const long whose = KEYS == PREFIX ? ((long)__builtin_bit_cast(int, joined(0)[from + HD + 2]) * C::H + h) * RS::R + row % RS::R : bh * RS::R + row;
      float* const to = part + (whose * PARTS + (KEYS == OWN ? PSPLITS<C> : 0) + share) * (HD + 4);
      *(f32x4*)(to + d) = v;
      if (d == 0) {
        to[HD] = top;
        to[HD + 1] = sum;
      }
    }
  }
}

template <class C>
__device__ __forceinline__ void attend(const typename Elem<C::DT>::type* __restrict__ Q, const u8_t* __restrict__ cache,
                                       const int* __restrict__ pages, const int* __restrict__ lengths,
                                       typename Elem<C::DT>::type* __restrict__ out, float* __restrict__ part) {
  // One array per stage: the compiler can then tell a stage's reads from the loads still on their way into the others.
  __shared__ __attribute__((aligned(1024))) u8_t l0[4 * Stages<C>::STAGE], l1[4 * Stages<C>::STAGE], l2[4 * Stages<C>::STAGE];
  attend_keys<C, ALL>(Q, cache, pages, lengths, nullptr, out, part, (int)blockIdx.x, (int)blockIdx.y, l0, l1, l2);
}

// With keys that sequences share: a wave's step of 32 keys costs about 1840 cycles for its sixteen rows, 210 VALU and 32 matrix instructions one
// after the other for the most part, whoever's rows they are; what is saved is the steps of rows that would be alone (64 sequences of 4 rows to
// each of 4 heads of 128 over 8192 shared keys and up to 1024 of their own: a call 25 us, 62 with all of the keys each one's own). (32 rows to a
// wave, keys and values widened once for both sixteens: 256 registers, two workgroups to a CU, 33 us against 28.) The first workgroups take the
// prefixes, the rows of all of a prefix's sequences together, the others each sequence's own keys. Every row's parts are joined by the next kernel.
template <class C>
__device__ __forceinline__ void attend_shared(const typename Elem<C::DT>::type* __restrict__ Q, const u8_t* __restrict__ cache,
                                              const int* __restrict__ pages, const int* __restrict__ lengths, const int* __restrict__ prefix_pages,
                                              const int* __restrict__ prefix_lengths, const int* __restrict__ of, float* __restrict__ part) {
  __shared__ __attribute__((aligned(1024))) u8_t l0[4 * Stages<C>::STAGE], l1[4 * Stages<C>::STAGE], l2[4 * Stages<C>::STAGE];
  constexpr int FIRST = PREFIX_GROUPS<C> * C::H * PSPLITS<C>, EACH = (int)(C::SEQS * C::H * Rows<C>::GROUPS);
  const int block = (int)blockIdx.x - FIRST;
  if (block < 0) attend_keys<C, PREFIX>(Q, cache, prefix_pages, prefix_lengths, of, nullptr, part, (int)blockIdx.x, 0, l0, l1, l2);
  else attend_keys<C, OWN>(Q, cache, pages, lengths, of, nullptr, part, block % EACH, block / EACH, l0, l1, l2);
}

// The rows' outputs from their splits' parts, in split order; one thread per output. `of`: with shared keys, whose parts come first and
// are not there for a sequence without a prefix.
template <class C>
__device__ __forceinline__ void attend_join(const float* __restrict__ part, typename Elem<C::DT>::type* __restrict__ out, const int* __restrict__ of = nullptr) {
  constexpr long R = Rows<C>::R, N = (long)C::SEQS * C::H * R * C::HD;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= N) return;
  const long bhr = i / C::HD, d = i % C::HD, row = bhr % R, bh = bhr / R;
  constexpr int PARTS = C::SPLITS + PSPLITS<C>;
  const float* const p = part + bhr * PARTS * (C::HD + 4);
  float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
  int from = 0;
  if constexpr (PSPLITS<C> > 0) {
    const int x = of[bh / C::H];
    if (x < 0 || x >= PREFIXES<C>) from = PSPLITS<C>;
  }
#pragma unroll 8
  for (int s = from; s < PARTS; ++s) m = fmaxf(m, p[s * (C::HD + 4) + C::HD]);
  const float base = base_of(m);
#pragma unroll 8
  for (int s = from; s < PARTS; ++s) {
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
