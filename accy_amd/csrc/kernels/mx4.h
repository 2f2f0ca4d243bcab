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
// the cache is read once for all of them. Per 32 keys a wave computes S^T = K Q^T (two v_mfma_f32_16x16x32_bf16 tiles of 16
// keys per 32 dims): lane l holds row l % 16 and, g = l / 16, keys 4 g + i and 16 + 4 g + i, which is how the B operand of
// O^T = V^T P^T wants them when its k index 8 g + j means key 4 g + j (j < 4) or 12 + 4 g + j, so P never leaves the lane. K's
// codes go from memory to the A operand's lanes as they lie: lane l's HD / 4 dims of key l % 16 (g HD / 4 on) are
// contiguous, and step s takes eight of them. V's rows are keys while its A operand wants eight keys of one dim: its codes
// pass through LDS, where ds_read_b64_tr_b8 hands a lane one byte (two dims) of eight rows.
//
// fp4 with its scale is exact in bf16. Queries are split into PARTS bf16 parts (bf16 1, f16 2, f32 3: exact, or 24 bits), and the
// probabilities likewise (PPARTS), one matrix instruction each: the sums keep f32's accuracy whatever the type.
//
// Each wave takes every fourth 32 keys of the workgroup's range; the waves join through LDS, the SPLITS workgroups of a
// sequence and head through memory (m, l, O per row) and a second kernel. A range is a share of the sequence's own length.
//
// C supplies, besides the cache's, Q, G, MAXP (pages per sequence), SEQS, NR, SPLITS and SL = log2(e) / sqrt(HD).
// ---------------------------------------------------------------------------------------------

#define ACCY_MX4_LDS __attribute__((address_space(3)))

template <int DT> constexpr int query_parts() { return DT + 1; }

// x as `PARTS` bf16 numbers whose sum is x (to 8 bits a part): the part, and what is left.
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

template <class C>
__device__ __forceinline__ void attend(const typename Elem<C::DT>::type* __restrict__ Q, const u8_t* __restrict__ cache,
                                       const int* __restrict__ pages, const int* __restrict__ lengths,
                                       typename Elem<C::DT>::type* __restrict__ out, float* __restrict__ part) {
  typedef Page<C> P;
  typedef Rows<C> RS;
  constexpr int HD = C::HD, NB = HD / 32, PARTS = query_parts<C::DT>(), PP = C::DT == 2 ? 3 : 2, NR = C::NR;
  constexpr int KB = HD / 8;             // bytes of a lane's share of a key
  constexpr int VPITCH = HD / 2 + 8;     // LDS pitch of a value row
  constexpr int VCH = (32 * HD / 2 + 1023) / 1024;  // 16-byte chunks per lane of 32 value rows
  __shared__ __attribute__((aligned(16))) u8_t vs[4][32 * VPITCH];
  __shared__ float joined[2][16 * (HD + 4)];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, r = lane & 15;
  const long bh = blockIdx.x / RS::GROUPS, b = bh / C::H, h = bh % C::H;
  const int row0 = (int)(blockIdx.x % RS::GROUPS) * NR * 16;
  int len = lengths[b];
  len = len < 0 ? 0 : len > C::MAXP * C::T ? C::MAXP * C::T : len;
  const int steps = (len + 31) / 32, per = (steps + C::SPLITS - 1) / C::SPLITS;
  const int first = (int)blockIdx.y * per, end = first + per < steps ? first + per : steps;

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
  const int sure = len - (C::Q - 1);  // keys below it are seen by every row

  f32x4 o[NR][NB][2];
  float m[NR], l[NR];
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    m[t] = -__builtin_inff();
    l[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < NB; ++d) o[t][d][0] = o[t][d][1] = f32x4{0, 0, 0, 0};
  }

  for (int step = first + wave; step < end; step += 4) {
    const int k0 = step * 32, page = pages[b * C::MAXP + k0 / C::T];
    if (page < 0 || page >= C::P) continue;
    const u8_t* const head = P::head(cache, page, h);
    const int in = k0 % C::T;
    // values into LDS
#pragma unroll
    for (int c = 0; c < VCH; ++c) {
      const int chunk = c * 64 + lane;
      if (32 * HD / 2 % 1024 == 0 || chunk < 32 * HD / 32) {
        const u32x4 w = *(const u32x4*)(head + P::codes(true, in) + 16 * chunk);
        u8_t* const p = &vs[wave][chunk / (HD / 32) * VPITCH + chunk % (HD / 32) * 16];
        *(u32x2*)p = u32x2{w[0], w[1]};
        *(u32x2*)(p + 8) = u32x2{w[2], w[3]};
      }
    }
    // other lanes' rows are read below: no access may move across
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // scores
    f32x4 sc[NR][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = in + 16 * u + r;
      u32_t kw[NB];
      const u8_t* const kp = head + P::codes(false, key) + g * KB;
#pragma unroll
      for (int s = 0; s < NB; ++s) kw[s] = *(const u32_t*)(kp + 4 * s);
#pragma unroll
      for (int t = 0; t < NR; ++t) sc[t][u] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < NB; ++s) {
        const float scale = scale_of(head[P::scales(false, key) + (g * (HD / 4) + 8 * s) / 32]);
        bf16x8 a;
        const bf16x2 a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(kw[s], scale, 0), a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(kw[s], scale, 1);
        const bf16x2 a2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(kw[s], scale, 2), a3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(kw[s], scale, 3);
        a[0] = a0[0], a[1] = a0[1], a[2] = a1[0], a[3] = a1[1], a[4] = a2[0], a[5] = a2[1], a[6] = a3[0], a[7] = a3[1];
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
          for (int p = 0; p < PARTS; ++p) sc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[t][s][p], sc[t][u], 0, 0, 0);
      }
    }
    // softmax: lane's keys are k0 + 16 u + 4 g + i
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      float top = m[t];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float s = sc[t][u][i] * C::SL;
          sc[t][u][i] = k0 + 16 * u + 4 * g + i < limit[t] ? s : -__builtin_inff();
          top = fmaxf(top, sc[t][u][i]);
        }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float base = base_of(top), alpha = __builtin_amdgcn_exp2f(m[t] - base);
      m[t] = top;
      l[t] *= alpha;
#pragma unroll
      for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][d][e][i] *= alpha;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[t][u][i] = __builtin_amdgcn_exp2f(sc[t][u][i] - base);
          l[t] += sc[t][u][i];
        }
    }
    // scale bytes of the lane's eight keys
    u8_t vb[8][NB];
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int key = 4 * g + (j & 3) + (j >> 2) * 16;
#pragma unroll
      for (int d = 0; d < NB; ++d) {
        vb[j][d] = head[P::scales(true, in + key) + d];
        nan |= k0 + key >= sure && k0 + key < len && vb[j][d] == 255;
      }
    }
    // A key that only some rows see must not reach the others where it is NaN (0 x NaN): then one query at a time, with
    // what that query does not see left out. Keys past the end are left out always.
    const bool apart = C::Q > 1 && __builtin_amdgcn_ballot_w64(nan) != 0;
#pragma unroll 1
    for (int only = apart ? 0 : C::Q - 1; only < C::Q; ++only) {
      const int seen = len - (C::Q - 1 - only);
#pragma unroll
      for (int d = 0; d < NB; ++d) {
        // lanes 2 t and 2 t + 1 of sixteen address the block's bytes of their t-th key
        const int t = r >> 1, key = 4 * g + (t & 3) + (t >> 2) * 16;
        const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((ACCY_MX4_LDS i32x2*)&vs[wave][key * VPITCH + 16 * d + 8 * (r & 1)]);
        bf16x8 even, odd;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = 4 * g + (j & 3) + (j >> 2) * 16;
          const float scale = scale_of(k0 + key < seen ? vb[j][d] : 0);
          const u32_t word = (u32_t)w[j >> 2];
          bf16x2 x;
          if ((j & 3) == 0) x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0);
          else if ((j & 3) == 1) x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1);
          else if ((j & 3) == 2) x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2);
          else x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3);
          even[j] = x[0];
          odd[j] = x[1];
        }
#pragma unroll
        for (int t = 0; t < NR; ++t) {
          const bool mine = !apart || (row0 + 16 * t + r) / C::G == only;
          const f32x4 before[2] = {o[t][d][0], o[t][d][1]};
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = sc[t][j >> 2][j & 3];
#pragma unroll
          for (int p = 0; p < PP; ++p) {
            bf16x8 pr;
#pragma unroll
            for (int j = 0; j < 8; ++j) pr[j] = take_part(x[j]);
            o[t][d][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, pr, o[t][d][0], 0, 0, 0);
            o[t][d][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, pr, o[t][d][1], 0, 0, 0);
          }
          if constexpr (C::Q > 1) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[t][d][e][i] = mine ? o[t][d][e][i] : before[e][i];
          }
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
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
        float* const p = &joined[wave - from][r * (HD + 4)];
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
        const float* const p = &joined[wave][r * (HD + 4)];
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
