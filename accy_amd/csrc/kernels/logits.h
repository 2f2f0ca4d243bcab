// Log probabilities of given tokens, entropies and the top alternatives of rows of logits, and the gradient.
//
// With m near a row's maximum, y = (x - m) log2 e, l = sum 2^y and s = sum 2^y y: log p = (y - log2 l) ln 2, and the entropy is (log2 l - s /
// l) ln 2. One pass over the row gives l, s and the alternatives: each thread measures from an m of its own, the maximum of its first chunk,
// and the threads' (m, l, s) are joined at the end, measured from the row's maximum. That is a conversion, half a maximum, a multiply-add, an
// exponential and two more operations an element, more than HBM delivers one in; so the alternatives have to come almost free
// (2048 x 50257 bf16 55-58 us, 3.7 TB/s, with 20 alternatives, 49 with one; 8 x 32000 f32 in 31 parts a row 5.2 us of kernel and 6.4 of the parts' join). The
// gradient reads a row once and writes it: 1001 x 50257 f16 47 us, 4.3 TB/s.
//
// Alternatives: an element is compared with a bound below the row's K-th largest only where its batch's maximum reaches the bound. After the first
// batch each wave takes the largest bound that a quarter (its share of K) of its lanes' maxima reach, and the least of the waves' bounds stands
// for the row. What reaches the bound goes to a list in LDS as a 64-bit key, the value's order above and the index's below, so that all
// keys differ and ties go to the lowest index. A list that is full raises the bound to its own K-th key and the batch is taken
// again (equal or ascending logits do that, a few times); at the end the keys of the list are ranked against each other.
//
// Rows start anywhere: whole chunks of 16 bytes are read on their own grid, and the few elements before the first and after the last one
// are a lane's each.
//
// C supplies DT (0 bf16, 1 f16, 2 f32), ROWS, V (elements of a row), K (alternatives, 0: none), SPLITS (workgroups of a row), NT (threads), U
// (chunks that a thread holds at once), ONCE (with the non-temporal hint).
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
};

// The elements of a chunk as f32.
template <class C> __device__ __forceinline__ void widen(const u32x4& w, float (&x)[Chunks<C>::PER]) {
#pragma unroll
  for (int i = 0; i < Chunks<C>::PER; ++i) {
    const u32_t bits = w[C::DT == 2 ? i : i >> 1];  // (a vector's element is no object to cast the bits of)
    x[i] = C::DT == 2 ? __builtin_bit_cast(float, bits) : C::DT == 0 ? bf16_of(bits, i) : f16_of(bits, i);
  }
}

template <int DT> __device__ __forceinline__ float value(typename Elem<DT>::type e) {
  if constexpr (DT == 2) return e;
  else return DT == 0 ? bf16_to_f32(e) : f16_to_f32(e);
}

// The part of a row that belongs to split z: chunks from .. to - 1, counted from element `at` of the buffer, which `base` points to, and the
// elements besides, `head` before the row's first whole chunk and `tail` after its last one, counted the same way. The row begins at element `lead`.
template <class C> struct Range {
  const typename Elem<C::DT>::type* base;
  long at;
  int from, to, lead, head, tail, after;
  // The element of this thread of those besides, or -1.
  __device__ __forceinline__ int besides() const {
    const int i = (int)threadIdx.x;
    return i < head ? lead + i : i < head + tail ? after + i - head : -1;
  }
};
template <class C> __device__ __forceinline__ Range<C> range_of(const typename Elem<C::DT>::type* x, long row, int z) {
  constexpr int PER = Chunks<C>::PER;
  const long begin = row * C::V;
  Range<C> r;
  r.at = begin / PER * PER;
  r.base = x + r.at;
  r.lead = (int)(begin - r.at);
  const int end = r.lead + (int)C::V, first = (r.lead + PER - 1) / PER, last = end / PER > first ? end / PER : first;
  const int per = (last - first + C::SPLITS - 1) / C::SPLITS;
  r.from = first + z * per < last ? first + z * per : last;
  r.to = r.from + per < last ? r.from + per : last;
  r.after = last * PER;
  r.head = z == 0 ? (first * PER < end ? first * PER : end) - r.lead : 0;
  r.tail = z == C::SPLITS - 1 && end > r.after ? end - r.after : 0;
  return r;
}
// f(0), .., f(N - 1) with numbers that are constants from the start: an array that they index is registers, whatever stands between.
template <int I> struct Index { static constexpr int value = I; };
template <int N, class F> __device__ __forceinline__ void each(F f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(Index<N - 1>());
  }
}
// Keeps the compiler from carrying widened elements from one pass over to the next in twice the registers.
__device__ __forceinline__ void opaque(u32x4& w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u32_t x = w[i];
    asm("" : "+v"(x));
    w[i] = x;
  }
}

// What a chunk makes of these is there before the next chunk begins: the compiler would begin with all of a row's chunks, and put some aside in memory.
__device__ __forceinline__ void in_order(float& a, float& b, float& c, float& d) { asm("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d)); }

// y = (x - base) log2 e as one multiply-add an element, x L2E - base L2E, takes base L2E rounded, and is off by that rounding, the same for all
// elements of a thread: rest_of(base), which is itself a number. A thread's sums are of such y's, and the rest leaves them where the threads' are
// joined. From FAR on it is beyond 1: there it is none, and y is formed from x - base.
constexpr float FAR = 0x1p+24f;
__device__ __forceinline__ float base_of(float m) { return m == -__builtin_inff() ? 0.0f : m; }
__device__ __forceinline__ bool is_far(float base) { return !(__builtin_fabsf(base) < FAR); }
__device__ __forceinline__ float rest_of(float base) { return is_far(base) ? 0.0f : __builtin_fmaf(base, L2E, -(base * L2E)); }
// With care: the same from x - base, whose rounding is that of a difference.
__device__ __forceinline__ float careful(float x, float base, float rest) { return __builtin_fmaf(x - base, L2E, rest); }

// A thread's, or a range's: sums of 2^y and of 2^y y with y measured from m, a maximum or near one.
struct Sums {
  float m = -__builtin_inff(), l = 0.0f, s = 0.0f;
  // The same measured from another m, with y's that are larger by `more`.
  __device__ __forceinline__ void rebase(float to, float more = 0.0f) {
    // (a sum of nothing is measured from nothing: its shift may be beyond f32)
    const float shift = l == 0.0f ? 0.0f : fmaxf(careful(base_of(m), base_of(to), more), LEAST), scale = __builtin_amdgcn_exp2f(shift);
    s = (s + l * shift) * scale;  // (no multiply-add: the rest of an element that is alone in its row leaves 0 behind)
    l *= scale;
    m = to;
  }
};

// Of a thread's U chunks, `first` its first one, those before `to`.
template <class C> __device__ __forceinline__ int present(int first, int to) {
  const int n = (to - first + C::NT - 1) / C::NT;
  return first >= to ? 0 : n < C::U ? n : C::U;
}
// Chunk c from `base`, a whole workgroup's: a row's bytes are counted in 32 bits.
template <class C> __device__ __forceinline__ const u32x4& chunk(const typename Elem<C::DT>::type* base, int c) { return *(const u32x4*)((const u8_t*)base + (u32_t)c * 16u); }
template <class C> __device__ __forceinline__ void fetch(const Range<C>& r, int first, int n, u32x4 (&w)[C::U]) {
  each<C::U>([&](auto u) {
    if (u.value < n) {
      if constexpr (C::ONCE) w[u.value] = __builtin_nontemporal_load(&chunk<C>(r.base, first + u.value * C::NT));
      else w[u.value] = chunk<C>(r.base, first + u.value * C::NT);
    }
  });
}
template <class C> __device__ __forceinline__ float largest(const u32x4& w) {
  float top = -__builtin_inff(), v[Chunks<C>::PER];
  widen<C>(w, v);
#pragma unroll
  for (int i = 0; i < Chunks<C>::PER; ++i) top = fmaxf(top, v[i]);
  return top;
}
// One element, with care: the sums of it alone.
__device__ __forceinline__ Sums sums_of(float x) {
  Sums a;
  a.m = fmaxf(x, a.m);
  const float y = careful(x, base_of(a.m), rest_of(base_of(a.m)));
  a.l = __builtin_amdgcn_exp2f(y);
  a.s = a.l * fmaxf(y, LEAST);
  return a;
}
// The first n of U chunks added to the sums; `top` becomes their maximum. They are widened once: y is measured from the m that there is, that of the
// first chunk to begin with. Where an element lies 32 above it (or it is that of nothing but masked elements), or m is far from 0, they are added
// again with care. (Masked elements cost one
// maximum each; when they made the batch one to be added again, 2048 x 50257 bf16, a third of every seventh row masked, took 66 us instead of 61.)
template <class C> __device__ __forceinline__ void add(Sums& a, const u32x4 (&w)[C::U], int n, float& top) {
  top = -__builtin_inff();
  if (n <= 0) return;
  if (a.l == 0.0f) a.m = largest<C>(w[0]);
  const float base = base_of(a.m);
  float v[Chunks<C>::PER], dl = 0.0f, ds = 0.0f, from = base * L2E;
  each<C::U>([&](auto u) {
    if (u.value >= n) return;
    if constexpr (C::U > 4) in_order(from, dl, ds, top);
    widen<C>(w[u.value], v);
#pragma unroll
    for (int i = 0; i < Chunks<C>::PER; ++i) top = fmaxf(top, v[i]);
#pragma unroll
    for (int i = 0; i < Chunks<C>::PER; ++i) {
      const float y = __builtin_fmaf(v[i], L2E, -from), e = __builtin_amdgcn_exp2f(y);
      dl += e;
      ds = __builtin_fmaf(e, fmaxf(y, LEAST), ds);
    }
  });
  if (is_far(base) || top - a.m > 32.0f) {
    asm volatile("");  // (a branch: computed either way it would cost as much again)
    if (top > a.m) a.rebase(top, rest_of(top) - rest_of(base_of(a.m)));
    float base = base_of(a.m), rest = rest_of(base);
    dl = ds = 0.0f;
    each<C::U>([&](auto u) {
      if (u.value >= n) return;
      u32x4 again = w[u.value];
      if constexpr (C::U > 4) in_order(base, dl, ds, rest);
      if constexpr (C::DT != 2) opaque(again);
      widen<C>(again, v);
#pragma unroll
      for (int i = 0; i < Chunks<C>::PER; ++i) {
        const float y = careful(v[i], base, rest), e = __builtin_amdgcn_exp2f(y);
        dl += e;
        ds = __builtin_fmaf(e, fmaxf(y, LEAST), ds);
      }
    });
  }
  a.l += dl;
  a.s += ds;
}

// The order of values, in the order of unsigned numbers: +0 and -0 are one, NaN is below all.
__device__ __forceinline__ u32_t order(float x) {
  const u32_t b = __builtin_bit_cast(u32_t, x + 0.0f);
  return x != x ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(u32_t o) { return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ u64_t key_of(float x, u32_t index) { return (u64_t)order(x) << 32 | (u32_t)~index; }

// The list of a workgroup: up to CAP keys, in no order.
template <class C> struct List {
  static constexpr int CAP = C::K > 0 ? 1024 : 1, BEST = C::K > 0 ? C::K : 1;
  u64_t key[CAP], best[BEST];
  // What up to LAID lanes of each wave lay out for the others: their chunks, which lane it is and how many chunks it has.
  static constexpr int LAID = C::K > 0 ? 16 : 1;
  u32x4 chunk[C::NT / 64][LAID][C::U];
  int who[C::NT / 64][LAID];
  u32_t share[2][C::NT / 64];
  int count[3];

  // The K largest of the first n keys to `best`, in order; what is missing is 0. All threads.
  __device__ void rank(int n) {
    for (int i = threadIdx.x; i < BEST; i += C::NT) best[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += C::NT) {
      const u64_t mine = key[i];
      int above = 0;
#pragma unroll 4  // (eight: 84 registers in place of 72, a workgroup to a CU less, 2048 x 50257 bf16 62 us in place of 58)
      for (int j = 0; j < n; ++j) above += key[j] > mine;
      if (above < BEST) best[above] = mine;
    }
    __syncthreads();
  }
};

// The threads' sums: the same in all of them. peak: a thread's maximum.
template <int WAVES> __device__ __forceinline__ Sums join_threads(Sums a, float peak, float (&lds)[WAVES][3]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  a.rebase(wave_reduce(peak, MaxOp()), -rest_of(base_of(a.m)));
  a.l = wave_reduce(a.l, SumOp());
  a.s = wave_reduce(a.s, SumOp());
  if (lane == 0) {
    lds[wave][0] = a.m;
    lds[wave][1] = a.l;
    lds[wave][2] = a.s;
  }
  __syncthreads();
  // A wave's lanes take a wave's sums each.
  const int from = lane % WAVES;
  a.m = lds[from][0];
  a.l = lds[from][1];
  a.s = lds[from][2];
  float top = a.m;
#pragma unroll
  for (int o = 1; o < WAVES; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  a.rebase(top);
#pragma unroll
  for (int o = 1; o < WAVES; o <<= 1) {
    a.l += __shfl_xor(a.l, o, 64);
    a.s += __shfl_xor(a.s, o, 64);
  }
  // The maximum's own 2^y is 1: a sum below it is so by its roundings alone, and would make a log probability one above 0.
  if (a.l > 0.0f && a.l < 1.0f) a.l = 1.0f;
  return a;
}

// The largest 16 bits that the wave's share of K lanes reach with their maxima.
template <class C> __device__ __forceinline__ u32_t share_of(float top) {
  constexpr int SHARE = (C::K + C::NT / 64 - 1) / (C::NT / 64);
  const u32_t mine = order(top) >> 16;
  u32_t least = 0;
#pragma unroll
  for (u32_t bit = 1u << 15; bit; bit >>= 1)
    if (__builtin_popcountll(__builtin_amdgcn_uicmp(mine, least | bit, 35)) >= SHARE) least |= bit;  // lanes of mine >= ..
  return least;
}
// The bound that all waves' shares reach together.
template <class C> __device__ __forceinline__ u64_t bound_of(const u32_t (&share)[C::NT / 64]) {
  u32_t b = share[0];
#pragma unroll
  for (int i = 1; i < C::NT / 64; ++i) b = b < share[i] ? b : share[i];
  return b > 0 ? (u64_t)b << 48 : 1ull << 32;  // (anything but NaN)
}

// One range: sums of all of its elements, and its K largest keys in list.best. The next batch is on its way while one is worked on.
template <class C>
__device__ __forceinline__ Sums scan(const Range<C> r, List<C>& list) {
  constexpr int PER = Chunks<C>::PER, WAVES = C::NT / 64;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  auto keep = [&](float v, int at, u64_t bound, int had, int turn) {
    const u64_t key = key_of(v, (u32_t)(at - r.lead));
    if (key < bound) return;
    const int place = had + atomicAdd(&list.count[turn], 1);
    if (place < List<C>::CAP) list.key[place] = key;
  };
  u32x4 next[C::U];
  fetch<C>(r, r.from + tid, present<C>(r.from + tid, r.to), next);
  const int besides = r.besides();
  float x = 0.0f, peak = -__builtin_inff();
  Sums a;
  if (besides >= 0) {
    x = value<C::DT>(r.base[besides]);
    a = sums_of(x);
    peak = fmaxf(peak, x);
  }
  if constexpr (C::K > 0) {
    if (tid < 3) list.count[tid] = 0;
    __syncthreads();
  }
  // Of the list: what is in it after the last batch, and the bound that keys have to reach; batch: counted from 0 and, in turns of three,
  // whose counter is in use. (The counter after that is cleared before the batch's barrier, all having read it before the last one.)
  int had = 0, batch = 0, turn = 0, rise = 0;
  u64_t bound = 0;
  for (int c0 = r.from; batch == 0 || c0 < r.to; c0 += C::NT * C::U, ++batch) {
    u32x4 w[C::U];
    each<C::U>([&](auto u) { w[u.value] = next[u.value]; });
    const int n = present<C>(c0 + tid, r.to), following_chunk = c0 + C::NT * C::U + tid;
    fetch<C>(r, following_chunk, present<C>(following_chunk, r.to), next);
    float top;
    add<C>(a, w, n, top);
    peak = fmaxf(peak, top);
    if constexpr (C::K > 0) {
      // Bounds come from the threads' maxima so far: the first batch's from itself, the others' from the batches before. They rise by less and
      // less: new ones are taken after 1, 2, 4, .. batches.
      const bool rises = (batch & (batch + 1)) == 0;
      if (rises) {
        const u32_t share = share_of<C>(peak);
        if (lane == 0) list.share[rise][wave] = share;
      }
      if (batch == 0) {
        __syncthreads();
        bound = bound_of<C>(list.share[0]);
      }
      const int following = turn == 2 ? 0 : turn + 1;
      if (tid == 0) list.count[following] = 0;
      for (;;) {
        if (batch == 0 && besides >= 0) keep(x, besides, bound, had, turn);
        // Lanes that reach the bound lay out their chunks, sixteen lanes at a time, and the whole wave looks through them. (A lane after the
        // other, each waits for LDS four times over: 2048 x 50257 bf16, 20 alternatives, 81 us.)
        u64_t lanes = __builtin_amdgcn_uicmp(order(top), (u32_t)(bound >> 32), 35);  // those where it is as large
        while (lanes) {
          constexpr int LAID = List<C>::LAID;
          const int rank = __builtin_popcountll(lanes & ((1ull << lane) - 1)), count = __builtin_popcountll(lanes);
          const bool mine = (lanes >> lane & 1) && rank < LAID;
          if (mine) {
            each<C::U>([&](auto u) { list.chunk[wave][rank][u.value] = w[u.value]; });
            list.who[wave][rank] = lane | n << 8;
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll 1
          for (int i = lane; i < (count < LAID ? count : LAID) * C::U * PER; i += 64) {
            const int from = i / (C::U * PER), j = i % (C::U * PER), who = list.who[wave][from];
            if (j >= (who >> 8) * PER) continue;
            keep(value<C::DT>(((const typename Elem<C::DT>::type*)list.chunk[wave][from])[j]), (c0 + j / PER * C::NT + wave * 64 + (who & 255)) * PER + j % PER, bound, had, turn);
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          lanes &= ~__builtin_amdgcn_ballot_w64(mine);
        }
        __syncthreads();
        const int found = had + list.count[turn];
        if (found <= List<C>::CAP) {
          had = found;
          break;
        }
        // Full: its K-th key bounds the range's. Of what was there before the batch the keys that reach it stay, K at most, and the
        // batch is taken again. (CAP different keys reach the old bound and K of them the new one, so that it rises by CAP - K keys every time.)
        list.rank(List<C>::CAP);
        bound = list.best[C::K - 1];
        u64_t kept[List<C>::CAP / C::NT];
#pragma unroll
        for (int i = 0; i < List<C>::CAP / C::NT; ++i) kept[i] = i * C::NT + tid < had ? list.key[i * C::NT + tid] : 0;
        if (tid == 0) list.count[turn] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < List<C>::CAP / C::NT; ++i)
          if (kept[i] >= bound) list.key[atomicAdd(&list.count[turn], 1)] = kept[i];
        __syncthreads();
        had = list.count[turn];
        __syncthreads();
        if (tid == 0) list.count[turn] = 0;
        __syncthreads();
      }
      if (rises) {
        const u64_t higher = bound_of<C>(list.share[rise]);
        bound = higher > bound ? higher : bound;
        rise ^= 1;
      }
      turn = following;
    }
  }
  if constexpr (C::K > 0) {
    __syncthreads();
    list.rank(had);
  }
  __shared__ float lds[WAVES][3];
  return join_threads<WAVES>(a, peak, lds);
}

// What a row's outputs are made of.
__device__ __forceinline__ float log_prob(const Sums& a, float x) {
  if (a.l == 0.0f) return -__builtin_inff();
  return (x - base_of(a.m)) - __builtin_amdgcn_logf(a.l) * LN2;
}
// A difference of numbers up to 46 (where a thread's m lies 32 below its maximum): off by some 2^-24 of that, and below 0 for nothing but that.
__device__ __forceinline__ float entropy(const Sums& a) {
  const float h = a.l == 0.0f ? 0.0f : (__builtin_amdgcn_logf(a.l) - a.s / a.l) * LN2;
  return h < 0.0f ? 0.0f : h;
}

template <class C>
__device__ __forceinline__ void write(const typename Elem<C::DT>::type* __restrict__ x, const int* __restrict__ tokens, long row, const Sums& a,
                                      const u64_t* best, float* __restrict__ token, float* __restrict__ entropies, float* __restrict__ top,
                                      int* __restrict__ top_tokens) {
  const int tid = threadIdx.x;
  if (tid == 0 && token) {
    const int t = tokens[row];
    float v = 0.0f;
    if (t >= 0 && t < C::V) {
      v = log_prob(a, value<C::DT>(x[row * C::V + t]));
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
  const Sums a = scan<C>(range_of<C>(x, row, (int)blockIdx.y), list);
  if constexpr (C::SPLITS == 1) {
    write<C>(x, tokens, row, a, list.best, token, entropies, top, top_tokens);
  } else {
    Part<C>* const to = (Part<C>*)part + row * C::SPLITS + blockIdx.y;
    if (threadIdx.x < C::K) to->key[threadIdx.x] = list.best[threadIdx.x];
    if (threadIdx.x == 0) to->a = a;
  }
}

// A row's parts joined, a lane's each (there are 64 at most): the same in all threads.
template <class C> __device__ __forceinline__ Sums join_sums(const float* __restrict__ part, long row) {
  static_assert(C::SPLITS <= 64, "a wave holds a row's parts");
  const Part<C>* const from = (const Part<C>*)part + row * C::SPLITS;
  const int lane = threadIdx.x & 63;
  Sums a;
  if (lane < C::SPLITS) a = from[lane].a;
  a.rebase(wave_reduce(a.m, MaxOp()));
  a.l = wave_reduce(a.l, SumOp());
  a.s = wave_reduce(a.s, SumOp());
  return a;
}
template <class C>
__device__ __forceinline__ void log_probs_join(const typename Elem<C::DT>::type* __restrict__ x, const int* __restrict__ tokens,
                                               const float* __restrict__ part, float* __restrict__ token, float* __restrict__ entropies,
                                               float* __restrict__ top, int* __restrict__ top_tokens) {
  __shared__ List<C> list;
  const long row = blockIdx.x;
  const Part<C>* const from = (const Part<C>*)part + row * C::SPLITS;
  const Sums a = join_sums<C>(part, row);
  if constexpr (C::K > 0) {
    static_assert(C::SPLITS * C::K <= List<C>::CAP, "the splits' keys fit a list");
    // Keys below what K of the threads' largest reach are left out before the others are ranked (512 keys 5 us otherwise).
    constexpr int KEYS = C::SPLITS * C::K;
    const int tid = threadIdx.x;
    float most = -__builtin_inff();
    for (int i = tid; i < KEYS; i += C::NT) {
      const u64_t key = from[i / C::K].key[i % C::K];
      if (key) most = fmaxf(most, value_of((u32_t)(key >> 32)));
    }
    const u32_t share = share_of<C>(most);
    if ((tid & 63) == 0) list.share[0][tid >> 6] = share;
    if (tid == 0) list.count[0] = 0;
    __syncthreads();
    const u64_t bound = bound_of<C>(list.share[0]);
    for (int i = tid; i < KEYS; i += C::NT) {
      const u64_t key = from[i / C::K].key[i % C::K];
      if (key >= bound) list.key[atomicAdd(&list.count[0], 1)] = key;
    }
    __syncthreads();
    list.rank(list.count[0]);
  }
  write<C>(x, tokens, row, a, list.best, token, entropies, top, top_tokens);
}

// ---- the gradient ----
//
// d x = g (1 at the token) - p (g + h (log p + H)), g and h the gradients of the token's log probability and of the entropy H: p is 2^y / l and log p +
// H is (y - s / l) ln 2, so that this is 2^y (A + B y) with A = (h ln 2 s / l - g) / l and B = -h ln 2 / l.
template <class C> struct Slope {
  float base, a, b, g;
  int at;                      // the token's element counted as a Range's, or -1
};
template <class C>
__device__ __forceinline__ Slope<C> slope_of(const Sums& s, long row, int lead, const int* __restrict__ tokens, const float* __restrict__ d_token,
                                             const float* __restrict__ d_entropy) {
  Slope<C> k;
  const int t = tokens[row];
  const bool inside = t >= 0 && t < C::V;
  const float h = d_entropy[row], by = s.l == 0.0f ? 0.0f : 1.0f / s.l;
  k.g = inside ? d_token[row] : 0.0f;
  k.at = inside && s.l != 0.0f ? lead + t : -1;
  k.base = base_of(s.m);
  k.a = (h * LN2 * (s.s * by) - k.g) * by;
  k.b = -h * LN2 * by;
  return k;
}
template <int DT> __device__ __forceinline__ typename Elem<DT>::type to_elem(float v) {
  if constexpr (DT == 0) return __builtin_bit_cast(u16_t, (__bf16)v);
  else if constexpr (DT == 1) return f32_to_f16(v);
  else return v;
}
// The gradient at an element.
template <class C> __device__ __forceinline__ float slope(const Slope<C>& k, float x) {
  const float y = (x - k.base) * L2E;
  return __builtin_amdgcn_exp2f(y) * __builtin_fmaf(k.b, fmaxf(y, LEAST), k.a);
}
// The gradient of chunk c's elements.
template <class C>
__device__ __forceinline__ void put(typename Elem<C::DT>::type* __restrict__ to, const Slope<C>& k, int c, const u32x4& w) {
  constexpr int PER = Chunks<C>::PER;
  float v[PER];
  widen<C>(w, v);
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = slope<C>(k, v[i]);
  if (k.at >= 0 && k.at / PER == c) {
    asm volatile("");
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] += i == k.at % PER ? k.g : 0.0f;
  }
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (C::DT == 2) o[i] = __builtin_bit_cast(u32_t, v[i]);
    else o[i] = (u32_t)to_elem<C::DT>(v[2 * i]) | (u32_t)to_elem<C::DT>(v[2 * i + 1]) << 16;
  }
  u32x4* const at = (u32x4*)((u8_t*)to + (u32_t)c * 16u);
  if constexpr (C::ONCE) __builtin_nontemporal_store(o, at);
  else *at = o;
}
template <class C> __device__ __forceinline__ void put_besides(typename Elem<C::DT>::type* __restrict__ to, const Slope<C>& k, int besides, float x) {
  if (besides >= 0) to[besides] = to_elem<C::DT>(slope<C>(k, x) + (besides == k.at ? k.g : 0.0f));
}

// A row whose chunks fit the workgroup's registers, U of them a thread: read once, written once.
template <class C>
__device__ __forceinline__ void grad_row(const typename Elem<C::DT>::type* __restrict__ x, const int* __restrict__ tokens, const float* __restrict__ d_token,
                                         const float* __restrict__ d_entropy, typename Elem<C::DT>::type* __restrict__ dx) {
  constexpr int WAVES = C::NT / 64;
  __shared__ float lds[WAVES][3];
  const long row = blockIdx.x;
  const Range<C> r = range_of<C>(x, row, 0);
  const int first = r.from + (int)threadIdx.x, n = present<C>(first, r.to), besides = r.besides();
  u32x4 w[C::U];
  fetch<C>(r, first, n, w);
  float edge = 0.0f, peak;
  Sums a;
  if (besides >= 0) {
    edge = value<C::DT>(r.base[besides]);
    a = sums_of(edge);
  }
  add<C>(a, w, n, peak);
  if (besides >= 0) peak = fmaxf(peak, edge);
  each<C::U>([&](auto u) { opaque(w[u.value]); });
  a = join_threads<WAVES>(a, peak, lds);
  const Slope<C> k = slope_of<C>(a, row, r.lead, tokens, d_token, d_entropy);
  typename Elem<C::DT>::type* const to = dx + r.at;
  put_besides<C>(to, k, besides, edge);
  each<C::U>([&](auto u) {
    if (u.value < n) put<C>(to, k, first + u.value * C::NT, w[u.value]);
  });
}

// Rows that several workgroups share: the sums come from `part` (log_probs with K = 0), each workgroup writes a part of the row.
template <class C>
__device__ __forceinline__ void grad_split(const typename Elem<C::DT>::type* __restrict__ x, const int* __restrict__ tokens, const float* __restrict__ d_token,
                                           const float* __restrict__ d_entropy, const float* __restrict__ part, typename Elem<C::DT>::type* __restrict__ dx) {
  const long row = blockIdx.x;
  const Range<C> r = range_of<C>(x, row, (int)blockIdx.y);
  const int besides = r.besides();
  const Slope<C> k = slope_of<C>(join_sums<C>(part, row), row, r.lead, tokens, d_token, d_entropy);
  typename Elem<C::DT>::type* const to = dx + r.at;
  put_besides<C>(to, k, besides, besides >= 0 ? value<C::DT>(r.base[besides]) : 0.0f);
  for (int c = r.from + (int)threadIdx.x; c < r.to; c += C::NT) put<C>(to, k, c, chunk<C>(r.base, c));
}

}  // namespace logits
}  // namespace accy
