// Log probabilities of given tokens, entropies and the top alternatives of rows of logits, and the gradient.
//
// With m a row's maximum, y = (x - m) log2 e, l = sum 2^y and s = sum 2^y y: log p = (y - log2 l) ln 2, and the entropy is (log2 l - s /
// l) ln 2. One pass over the row gives l, s and the alternatives: each thread keeps a maximum of its own elements, lets it follow only where
// a batch of them has a larger one, and the threads' (m, l, s) are joined at the end. That is a conversion, a maximum, a multiply-add, an
// exponential and two more operations an element, about what HBM delivers one in; so the alternatives have to come almost free.
//
// Alternatives: an element is compared with a bound below the row's K-th largest only where its batch's maximum reaches the bound. After the first
// batch each wave takes the largest bound that a quarter (its share of K) of its lanes' maxima reach, and the least of the waves' bounds stands
// for the row. What reaches the bound goes to a list in LDS as a 64-bit key, the value's order above and the index's below, so that all
// keys differ and ties go to the lowest index. A list that is full raises the bound to its own K-th key and the batch is taken
// again (equal or ascending logits do that, a few times); at the end the keys of the list are ranked against each other.
//
// Rows start anywhere: chunks of 16 bytes are read on their own grid, and what lies before or after the row is masked.
//
// C supplies DT (0 bf16, 1 f16, 2 f32), ROWS, V (elements of a row), K (alternatives, 0: none), SPLITS (workgroups of a row), NT (threads), U
// (chunks that a thread has on their way at once).
#pragma once

namespace accy {
namespace logits {

typedef u32_t u32x4 __attribute__((ext_vector_type(4)));

template <int DT> struct Elem { typedef u16_t type; };
template <> struct Elem<2> { typedef float type; };

constexpr float LN2 = 0x1.62e43p-1f, L2E = 0x1.715476p+0f;
// An element is left out of products with its y below this (2^y is 0 there, and y may be -inf).
constexpr float LEAST = -200.0f;

template <class C> struct Chunks {
  static constexpr int SIZE = C::DT == 2 ? 4 : 2, PER = 16 / SIZE;  // elements of a chunk
  static constexpr long TOTAL = C::ROWS * C::V;
};

// The elements of a chunk as f32; those of another row are -inf, which weighs nothing.
template <class C> __device__ __forceinline__ void widen(const u32x4& w, float (&x)[Chunks<C>::PER]) {
  if constexpr (C::DT == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32_t bits = w[i];  // (a vector's element is no object to cast the bits of)
      x[i] = __builtin_bit_cast(float, bits);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = C::DT == 0 ? bf16_of(w[i >> 1], i) : f16_of(w[i >> 1], i);
  }
}

// Chunk c (of the whole buffer), of which the row has elements lo .. hi - 1; a chunk that the buffer ends in is read element by element.
template <class C>
__device__ __forceinline__ u32x4 read(const typename Elem<C::DT>::type* __restrict__ x, long c) {
  typedef Chunks<C> K;
  if (K::TOTAL % K::PER == 0 || (c + 1) * K::PER <= K::TOTAL) return *(const u32x4*)(x + c * K::PER);
  u32x4 w = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < K::PER; ++i) {
    if (c * K::PER + i >= K::TOTAL) continue;
    if constexpr (C::DT == 2) w[i] = __builtin_bit_cast(u32_t, x[c * K::PER + i]);
    else w[i >> 1] |= (u32_t)x[c * K::PER + i] << (16 * (i & 1));
  }
  return w;
}

// The part of a row that belongs to split z: elements first .. end - 1 of the buffer, chunks c0 .. c1 - 1.
struct Range {
  long first, end, c0, c1;
};
template <class C> __device__ __forceinline__ Range range_of(long row, int z) {
  typedef Chunks<C> K;
  const long begin = row * C::V, finish = begin + C::V, a = begin / K::PER, b = (finish + K::PER - 1) / K::PER;
  const long per = ((b - a) + C::SPLITS - 1) / C::SPLITS;
  Range r;
  r.c0 = a + z * per < b ? a + z * per : b;
  r.c1 = r.c0 + per < b ? r.c0 + per : b;
  r.first = r.c0 * K::PER > begin ? r.c0 * K::PER : begin;
  r.end = r.c1 * K::PER < finish ? r.c1 * K::PER : finish;
  return r;
}
template <class C> __device__ __forceinline__ void mask(const Range& r, long c, float (&x)[Chunks<C>::PER]) {
  constexpr int PER = Chunks<C>::PER;
  if (c * PER >= r.first && (c + 1) * PER <= r.end) return;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (c * PER + i < r.first || c * PER + i >= r.end) x[i] = -__builtin_inff();
}

__device__ __forceinline__ float base_of(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// A thread's, or a range's: its maximum, and sums of 2^y and of 2^y y with y measured from that maximum.
struct Sums {
  float m = -__builtin_inff(), l = 0.0f, s = 0.0f;
  // The same measured from a maximum that is no smaller.
  __device__ __forceinline__ void rebase(float to) {
    const float shift = fmaxf((base_of(m) - base_of(to)) * L2E, LEAST), scale = __builtin_amdgcn_exp2f(l == 0.0f ? LEAST : shift);
    s = (s + l * shift) * scale;
    l *= scale;
    m = to;
  }
  // An element; base: base_of(m).
  __device__ __forceinline__ void add(float x, float base) {
    const float y = (x - base) * L2E, e = __builtin_amdgcn_exp2f(y);
    l += e;
    s = __builtin_fmaf(e, fmaxf(y, LEAST), s);
  }
  __device__ __forceinline__ void join(Sums o) {
    const float top = fmaxf(m, o.m);
    rebase(top);
    o.rebase(top);
    l += o.l;
    s += o.s;
  }
};

// The order of values, in the order of unsigned numbers: +0 and -0 are one, NaN is below all.
__device__ __forceinline__ u32_t order(float x) {
  const u32_t b = __builtin_bit_cast(u32_t, x + 0.0f);
  return x != x ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(u32_t o) { return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ u64_t key_of(float x, u32_t index) { return (u64_t)order(x) << 32 | (u32_t)~index; }

// The list of a workgroup: up to CAP keys, in no order. Below the bound nothing is of interest.
template <class C> struct List {
  static constexpr int CAP = C::K > 0 ? 1024 : 1, BEST = C::K > 0 ? C::K : 1;
  u64_t key[CAP], best[BEST], bound;
  u32_t share[C::NT / 64];
  int count;

  // The K largest of the first n keys to `best`, in order; what is missing is 0. All threads.
  __device__ void rank(int n) {
    for (int i = threadIdx.x; i < BEST; i += C::NT) best[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += C::NT) {
      const u64_t mine = key[i];
      int above = 0;
      for (int j = 0; j < n; ++j) above += key[j] > mine;
      if (above < BEST) best[above] = mine;
    }
    __syncthreads();
  }
};

// One range: sums of all of its elements, and its K largest keys in list.best.
template <class C>
__device__ __forceinline__ Sums scan(const typename Elem<C::DT>::type* __restrict__ x, const Range r, long begin, List<C>& list) {
  typedef Chunks<C> CH;
  constexpr int PER = CH::PER, WAVES = C::NT / 64;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  Sums a;
  if constexpr (C::K > 0) {
    if (tid == 0) {
      list.bound = 1ull << 32;  // everything but NaN
      list.count = 0;
    }
    __syncthreads();
  }
  bool first = true;
  for (long c0 = r.c0; c0 < r.c1; c0 += C::NT * C::U) {
    u32x4 w[C::U];
    float top = -__builtin_inff();
#pragma unroll
    for (int u = 0; u < C::U; ++u) {
      const long c = c0 + u * C::NT + tid;
      if (c < r.c1) w[u] = read<C>(x, c);
    }
#pragma unroll
    for (int u = 0; u < C::U; ++u) {
      const long c = c0 + u * C::NT + tid;
      if (c >= r.c1) continue;
      float v[PER];
      widen<C>(w[u], v);
      mask<C>(r, c, v);
#pragma unroll
      for (int i = 0; i < PER; ++i) top = fmaxf(top, v[i]);
    }
    if (top > a.m) a.rebase(top);
    const float base = base_of(a.m);
#pragma unroll
    for (int u = 0; u < C::U; ++u) {
      const long c = c0 + u * C::NT + tid;
      if (c >= r.c1) continue;
      float v[PER];
      widen<C>(w[u], v);
      mask<C>(r, c, v);
#pragma unroll
      for (int i = 0; i < PER; ++i) a.add(v[i], base);
    }
    if constexpr (C::K > 0) {
      if (first) {
        first = false;
        // The largest 16 bits that a share of this wave's lanes reach.
        constexpr int SHARE = (C::K + WAVES - 1) / WAVES;
        const u32_t mine = order(top) >> 16;
        u32_t least = 0;
        for (u32_t bit = 1u << 15; bit; bit >>= 1)
          if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(mine >= (least | bit))) >= SHARE) least |= bit;
        if (lane == 0) list.share[wave] = least;
        __syncthreads();
        if (tid == 0) {
          u32_t b = list.share[0];
          for (int i = 1; i < WAVES; ++i) b = b < list.share[i] ? b : list.share[i];
          if (b > 0) list.bound = (u64_t)b << 48;
        }
        __syncthreads();
      }
      int before = list.count;
      __syncthreads();
      for (;;) {
        const u64_t bound = list.bound;
        if (order(top) >= (u32_t)(bound >> 32)) {
#pragma unroll
          for (int u = 0; u < C::U; ++u) {
            const long c = c0 + u * C::NT + tid;
            if (c >= r.c1) continue;
            float v[PER];
            widen<C>(w[u], v);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const long at = c * PER + i;
              const u64_t key = key_of(v[i], (u32_t)(at - begin));
              if (key >= bound && at >= r.first && at < r.end) {
                const int place = atomicAdd(&list.count, 1);
                if (place < List<C>::CAP) list.key[place] = key;
              }
            }
          }
        }
        __syncthreads();
        const int found = list.count;
        if (found <= List<C>::CAP) break;
        // Full: its K-th key bounds the range's. Of what was there before the batch the keys that reach it stay, K at most, and the
        // batch is taken again. (CAP different keys reach the old bound and K of them the new one, so that it rises by CAP - K keys every time.)
        list.rank(List<C>::CAP);
        const u64_t higher = list.best[C::K - 1];
        u64_t kept[List<C>::CAP / C::NT];
#pragma unroll
        for (int i = 0; i < List<C>::CAP / C::NT; ++i) kept[i] = i * C::NT + tid < before ? list.key[i * C::NT + tid] : 0;
        __syncthreads();
        if (tid == 0) {
          list.bound = higher;
          list.count = 0;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < List<C>::CAP / C::NT; ++i)
          if (kept[i] >= higher) list.key[atomicAdd(&list.count, 1)] = kept[i];
        __syncthreads();
        before = list.count;
        __syncthreads();
      }
    }
  }
  if constexpr (C::K > 0) {
    __syncthreads();
    list.rank(list.count);
  }
  // the threads' sums
  __shared__ float lds[WAVES][3];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    Sums b;
    b.m = __shfl_xor(a.m, o, 64);
    b.l = __shfl_xor(a.l, o, 64);
    b.s = __shfl_xor(a.s, o, 64);
    a.join(b);
  }
  if (lane == 0) {
    lds[wave][0] = a.m;
    lds[wave][1] = a.l;
    lds[wave][2] = a.s;
  }
  __syncthreads();
  a = Sums();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    Sums b;
    b.m = lds[i][0];
    b.l = lds[i][1];
    b.s = lds[i][2];
    a.join(b);
  }
  return a;
}

// What a row's outputs are made of.
__device__ __forceinline__ float log_prob(const Sums& a, float x) {
  if (a.l == 0.0f) return -__builtin_inff();
  return (x - base_of(a.m)) - __builtin_amdgcn_logf(a.l) * LN2;
}
__device__ __forceinline__ float entropy(const Sums& a) { return a.l == 0.0f ? 0.0f : (__builtin_amdgcn_logf(a.l) - a.s / a.l) * LN2; }

template <class C>
__device__ __forceinline__ void write(const typename Elem<C::DT>::type* __restrict__ x, const int* __restrict__ tokens, long row, const Sums& a,
                                      const u64_t* best, float* __restrict__ token, float* __restrict__ entropies, float* __restrict__ top,
                                      int* __restrict__ top_tokens) {
  const int tid = threadIdx.x;
  if (tid == 0 && token) {
    const int t = tokens[row];
    float v = 0.0f;
    if (t >= 0 && t < C::V) {
      const typename Elem<C::DT>::type e = x[row * C::V + t];
      if constexpr (C::DT == 2) v = log_prob(a, e);
      else v = log_prob(a, C::DT == 0 ? bf16_to_f32(e) : f16_to_f32(e));
    }
    token[row] = v;
  }
  if (tid == 0 && entropies) entropies[row] = entropy(a);
  if (tid < C::K) {
    const u64_t key = best[tid];
    if (top) top[row * C::K + tid] = key ? log_prob(a, value_of((u32_t)(key >> 32))) : __builtin_nanf("");
    if (top_tokens) top_tokens[row * C::K + tid] = key ? (int)~(u32_t)key : -1;
  }
}

// One workgroup for each row (SPLITS 1), or for each part of one, which goes to `part` [row][split]: Sums, then K keys.
template <class C> struct Part {
  u64_t key[C::K > 0 ? C::K : 1];
  Sums a;
};
template <class C>
__device__ __forceinline__ void log_probs(const typename Elem<C::DT>::type* __restrict__ x, const int* __restrict__ tokens, float* __restrict__ token,
                                          float* __restrict__ entropies, float* __restrict__ top, int* __restrict__ top_tokens, float* __restrict__ part) {
  __shared__ List<C> list;
  const long row = blockIdx.x;
  const Sums a = scan<C>(x, range_of<C>(row, (int)blockIdx.y), row * C::V, list);
  if constexpr (C::SPLITS == 1) {
    write<C>(x, tokens, row, a, list.best, token, entropies, top, top_tokens);
  } else {
    Part<C>* const to = (Part<C>*)part + row * C::SPLITS + blockIdx.y;
    if (threadIdx.x < C::K) to->key[threadIdx.x] = list.best[threadIdx.x];
    if (threadIdx.x == 0) to->a = a;
  }
}

// A row's parts joined, in split order.
template <class C> __device__ __forceinline__ Sums join_sums(const float* __restrict__ part, long row) {
  const Part<C>* const from = (const Part<C>*)part + row * C::SPLITS;
  Sums a;
#pragma unroll 4
  for (int z = 0; z < C::SPLITS; ++z) a.join(from[z].a);
  return a;
}
template <class C>
__device__ __forceinline__ void log_probs_join(const typename Elem<C::DT>::type* __restrict__ x, const int* __restrict__ tokens,
                                               const float* __restrict__ part, float* __restrict__ token, float* __restrict__ entropies,
                                               float* __restrict__ top, int* __restrict__ top_tokens) {
  __shared__ List<C> list;
  const long row = blockIdx.x;
  const Part<C>* const from = (const Part<C>*)part + row * C::SPLITS;
  if constexpr (C::K > 0) {
    static_assert(C::SPLITS * C::K <= List<C>::CAP, "the splits' keys fit a list");
    if (threadIdx.x == 0) list.count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < C::SPLITS * C::K; i += C::NT) {
      const u64_t key = from[i / C::K].key[i % C::K];
      if (key) list.key[atomicAdd(&list.count, 1)] = key;
    }
    __syncthreads();
    list.rank(list.count);
  }
  write<C>(x, tokens, row, join_sums<C>(part, row), list.best, token, entropies, top, top_tokens);
}

// ---- the gradient ----
//
// d x = g (1 at the token) - p (g + h (log p + H)), g and h the gradients of the token's log probability and of the entropy H: with z = log2 p,
// p (A + B z) with A = g + h H and B = h ln 2.
template <class C> struct Slope {
  float base, log_l, a, b, g;  // z = (x - base) log2 e - log2 l
  long at;                     // the token's element, or -1
};
template <class C>
__device__ __forceinline__ Slope<C> slope_of(const Sums& s, long row, const int* __restrict__ tokens, const float* __restrict__ d_token,
                                             const float* __restrict__ d_entropy) {
  Slope<C> k;
  const int t = tokens[row];
  const bool inside = t >= 0 && t < C::V;
  const float h = d_entropy[row];
  k.g = inside ? d_token[row] : 0.0f;
  k.at = inside && s.l != 0.0f ? row * C::V + t : -1;
  k.base = base_of(s.m);
  k.log_l = s.l == 0.0f ? 0.0f : __builtin_amdgcn_logf(s.l);
  k.a = k.g + h * entropy(s);
  k.b = h * LN2;
  return k;
}
template <class C> __device__ __forceinline__ float slope_at(const Slope<C>& k, float x, long at) {
  const float z = __builtin_fmaf(x - k.base, L2E, -k.log_l);
  const float d = __builtin_amdgcn_exp2f(z) * __builtin_fmaf(k.b, fmaxf(z, LEAST), k.a);
  return at == k.at ? k.g - d : -d;
}
template <int DT> __device__ __forceinline__ typename Elem<DT>::type to_elem(float v) {
  if constexpr (DT == 0) return __builtin_bit_cast(u16_t, (__bf16)v);
  else if constexpr (DT == 1) return f32_to_f16(v);
  else return v;
}
// The gradient of a chunk's elements.
template <class C>
__device__ __forceinline__ void put(typename Elem<C::DT>::type* __restrict__ dx, const Range& r, const Slope<C>& k, long c, const u32x4& w) {
  constexpr int PER = Chunks<C>::PER;
  float v[PER];
  widen<C>(w, v);
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = slope_at(k, v[i], c * PER + i);
  if (c * PER >= r.first && (c + 1) * PER <= r.end) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (C::DT == 2) o[i] = __builtin_bit_cast(u32_t, v[i]);
      else o[i] = (u32_t)to_elem<C::DT>(v[2 * i]) | (u32_t)to_elem<C::DT>(v[2 * i + 1]) << 16;
    }
    *(u32x4*)(dx + c * PER) = o;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (c * PER + i >= r.first && c * PER + i < r.end) dx[c * PER + i] = to_elem<C::DT>(v[i]);
  }
}

// A row whose chunks fit the workgroup's registers, U of them a thread: read once, written once.
template <class C>
__device__ __forceinline__ void grad_row(const typename Elem<C::DT>::type* __restrict__ x, const int* __restrict__ tokens, const float* __restrict__ d_token,
                                         const float* __restrict__ d_entropy, typename Elem<C::DT>::type* __restrict__ dx) {
  constexpr int PER = Chunks<C>::PER, WAVES = C::NT / 64;
  __shared__ float tops[WAVES], ls[WAVES], ss[WAVES];
  const long row = blockIdx.x;
  const Range r = range_of<C>(row, 0);
  const int tid = threadIdx.x;
  u32x4 w[C::U];
#pragma unroll
  for (int u = 0; u < C::U; ++u)
    if (r.c0 + u * C::NT + tid < r.c1) w[u] = read<C>(x, r.c0 + u * C::NT + tid);
  Sums a;
  auto each = [&](auto f) {
#pragma unroll
    for (int u = 0; u < C::U; ++u) {
      const long c = r.c0 + u * C::NT + tid;
      if (c >= r.c1) continue;
      float v[PER];
      widen<C>(w[u], v);
      mask<C>(r, c, v);
#pragma unroll
      for (int i = 0; i < PER; ++i) f(v[i]);
    }
  };
  each([&](float v) { a.m = fmaxf(a.m, v); });
  a.m = block_reduce<C::NT>(a.m, MaxOp(), tops);
  const float base = base_of(a.m);
  each([&](float v) { a.add(v, base); });
  a.l = block_reduce<C::NT>(a.l, SumOp(), ls);
  a.s = block_reduce<C::NT>(a.s, SumOp(), ss);
  const Slope<C> k = slope_of<C>(a, row, tokens, d_token, d_entropy);
#pragma unroll
  for (int u = 0; u < C::U; ++u) {
    const long c = r.c0 + u * C::NT + tid;
    if (c < r.c1) put<C>(dx, r, k, c, w[u]);
  }
}

// Rows that several workgroups share: the sums come from `part` (log_probs with K = 0), each workgroup writes a part of the row.
template <class C>
__device__ __forceinline__ void grad_split(const typename Elem<C::DT>::type* __restrict__ x, const int* __restrict__ tokens, const float* __restrict__ d_token,
                                           const float* __restrict__ d_entropy, const float* __restrict__ part, typename Elem<C::DT>::type* __restrict__ dx) {
  const long row = blockIdx.x;
  const Range r = range_of<C>(row, (int)blockIdx.y);
  const Slope<C> k = slope_of<C>(join_sums<C>(part, row), row, tokens, d_token, d_entropy);
  for (long c = r.c0 + threadIdx.x; c < r.c1; c += C::NT) put<C>(dx, r, k, c, read<C>(x, c));
}

}  // namespace logits
}  // namespace accy
