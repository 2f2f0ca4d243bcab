// Page tables of a cache, and copies of its pages.
//
// fork and compact are counting: which pages are in use is a bitmap (a bit a page), the k-th free page the k-th bit that is clear, found by
// the words' running counts. One workgroup of 1024 threads does either in a few passes over the tables, the bitmaps in LDS (beyond
// LDS_PAGES pages in memory), so that a call is one launch; what bounds it is the way to memory and back of each pass and what one
// CU reads and writes, the tables (us of kernel: 8 rows of 64 slots 7.0, 256 of 512 among 16384 pages 14.6 and 4.0 for the rows' tables by themselves, compaction
// of 64 x 256 slots 8.6 and 4.7). No order of atomics shows: bits are set, and ties go to the lowest row or page.
//
// copies are bound by HBM (about 3000 pages of 34 KB 40 us, 5.2 TB/s). Source and target pages of fork and compact differ from each other
// and are all different, so that their copies need no check (C::CHECK false); of other lists the last copy to a page counts, and in place a page
// that is the source of one copy and the target of another is kept aside first.
#pragma once

namespace accy {
namespace pages {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr long LDS_PAGES = 1 << 17;

// ---- bitmaps: in LDS, or in memory, where other threads' bits come from the coherent level ----
template <bool LDS> __device__ __forceinline__ u32_t word(const u32_t* map, long w) {
  if constexpr (LDS) return map[w];
  else return __hip_atomic_load(map + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <bool LDS> __device__ __forceinline__ void put_word(u32_t* map, long w, u32_t v) {
  if constexpr (LDS) map[w] = v;
  else __hip_atomic_store(map + w, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <bool LDS> __device__ __forceinline__ bool bit(const u32_t* map, long p) { return word<LDS>(map, p >> 5) >> (p & 31) & 1; }
// A barrier after which the other threads' stores and bits are seen, in LDS or in memory.
template <bool LDS> __device__ __forceinline__ void meet() {
  if constexpr (!LDS) __threadfence();
  __syncthreads();
}
__device__ __forceinline__ void set_bit(u32_t* map, long p) { atomicOr(map + (p >> 5), 1u << (p & 31)); }

// The running sum of the threads' values before this one's; total: of all. `lds` holds WAVES + 1 elements.
__device__ __forceinline__ int before_me(int v, int* lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int below = __shfl_up(sum, o, 64);
    if (lane >= o) sum += below;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = sum;
  __syncthreads();
  int start = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const int n = lds[w];
    if (w < wave) start += n;
    total += n;
  }
  return start + sum - v;
}

// The words of a bitmap as each thread's share of them, in order.
__device__ __forceinline__ void my_words(long words, long& from, long& to) {
  const long per = (words + THREADS - 1) / THREADS;
  from = (long)threadIdx.x * per < words ? threadIdx.x * per : words;
  to = from + per < words ? from + per : words;
}

// The position of the k-th bit that is set in w (it has more than k).
__device__ __forceinline__ int nth_bit(u32_t w, int k) {
  int at = 0;
#pragma unroll
  for (int half = 16; half > 0; half >>= 1) {
    const int below = __builtin_popcount(w & ((1u << half) - 1));
    if (k >= below) {
      k -= below;
      w >>= half;
      at += half;
    }
  }
  return at;
}

// Pages held as the first word of a bitmap: bytes of `held` that are not 0. Bits past the last page are set: no page either.
template <long P> __device__ __forceinline__ u32_t held_word(const u8_t* __restrict__ held, long w) {
  u32_t bits = 0;
  if (w * 32 + 32 <= P) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const u32_t four = *(const u32_t*)(held + w * 32 + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) bits |= (four >> (8 * j) & 255u) ? 1u << (4 * i + j) : 0u;
    }
  } else {
    for (int i = 0; i < 32; ++i) bits |= w * 32 + i >= P || held[w * 32 + i] ? 1u << i : 0u;
  }
  return bits;
}

// ---------------------------------------------------------------------------------------------
// fork: C supplies SEQS, ROWS, SLOTS, P (pages), T (tokens of a page), NEW (tokens of a row whose slots are asked for), WIDE (the tables are written by fork_rows).
// ---------------------------------------------------------------------------------------------

// What row r becomes: its parent (-1: empty), the parent's length, the slots that its tokens take and those that it is to have.
struct Fork {
  int parent, length, kept, want;
  bool partial;
};
template <class C>
__device__ __forceinline__ Fork fork_of(const int* __restrict__ lengths, const int* __restrict__ parents, const int* __restrict__ room, long r) {
  Fork f = {-1, 0, 0, 0, false};
  constexpr long MOST = C::SLOTS * C::T;
  const int p = parents[r];
  if (p < 0 || p >= C::SEQS) return f;
  f.parent = p;
  const int n = lengths[p], more = room[r];
  const long length = n < 0 ? 0 : n > MOST ? MOST : n, all = length + (more < 0 ? 0 : more);
  f.length = (int)length;
  f.kept = (int)((length + C::T - 1) / C::T);
  f.want = (int)(((all > MOST ? MOST : all) + C::T - 1) / C::T);
  f.partial = length % C::T != 0;
  return f;
}
// The page in a slot, -1 for none.
template <class C> __device__ __forceinline__ int page_at(const int* __restrict__ table, int parent, int slot) {
  const int p = table[(long)parent * C::SLOTS + slot];
  return p >= 0 && p < C::P ? p : -1;
}

// What fork_rows needs of a row: the first `kept` slots are its parent's, `asked` pages from number `first` of the fresh ones follow.
struct Row {
  int parent, kept, first, asked;
};

// `map` and `counts`: (P + 31) / 32 words each; `firsts` [P]: work space where there are more than THREADS rows; `rows` [ROWS] and
// `fresh` [ROWS x SLOTS]: where the tables are written by another kernel (C::WIDE).
template <class C, bool LDS>
__device__ __forceinline__ void fork_with(u32_t* map, int* counts, const int* __restrict__ table, const int* __restrict__ lengths,
                                          const int* __restrict__ parents, const int* __restrict__ room, const u8_t* __restrict__ held,
                                          int* __restrict__ out_table, int* __restrict__ out_lengths, int* __restrict__ source,
                                          int* __restrict__ target, int* __restrict__ left, int* __restrict__ slots, int* __restrict__ firsts,
                                          Row* __restrict__ rows, int* __restrict__ fresh_pages) {
  constexpr long WORDS = (C::P + 31) / 32;
  constexpr int SLOTS = C::SLOTS > 0 ? (int)C::SLOTS : 1;
  // With a thread for every row its numbers stay in registers; else they are formed again where they are needed.
  constexpr bool ONE = C::ROWS <= THREADS;
  __shared__ int parent[THREADS], kept[THREADS], place[THREADS], sums[WAVES + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto row_of = [&](long r) {
    const Fork none = {-1, 0, 0, 0, false};
    return r < C::ROWS ? fork_of<C>(lengths, parents, room, r) : none;
  };
  auto partly = [&](const Fork& f) { return f.partial ? page_at<C>(table, f.parent, f.kept - 1) : -1; };
  Fork mine = row_of(tid);
  int last = partly(mine);
  for (long w = tid; w < WORDS; w += THREADS) put_word<LDS>(map, w, held_word<C::P>(held, w));
  meet<LDS>();
  // Pages that a row has filled: a wave takes eight rows at once, 64 slots of each.
  for (long r0 = 0; r0 < C::ROWS; r0 += THREADS) {
    if constexpr (!ONE) mine = row_of(r0 + tid);
    parent[tid] = mine.parent;
    kept[tid] = mine.kept - (mine.partial ? 1 : 0);
    __syncthreads();
    const int n = (int)(C::ROWS - r0 < THREADS ? C::ROWS - r0 : THREADS);
    for (int r = wave; r < n; r += 8 * WAVES) {
      int most = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = r + i * WAVES < n && kept[r + i * WAVES] > most ? kept[r + i * WAVES] : most;
      for (int j = lane; j < most; j += 64) {
        int p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = r + i * WAVES;
          p[i] = row < n && j < kept[row] ? page_at<C>(table, parent[row], j) : -1;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (p[i] >= 0) set_bit(map, p[i]);
      }
    }
    meet<LDS>();
  }
  // Pages that a row has filled in part: whose they are. `source` says which rows copy theirs.
  bool copied = false;
  if constexpr (ONE) {
    place[tid] = last;
    __syncthreads();
    if (last >= 0) {
      copied = bit<LDS>(map, last);
#pragma unroll 8
      for (int r = 0; r < tid; ++r) copied |= place[r] == last;
    }
    __syncthreads();
    if (last >= 0) set_bit(map, last);
  } else {
    for (long r = tid; r < C::ROWS; r += THREADS) {
      last = partly(row_of(r));
      if (last >= 0) __hip_atomic_store(firsts + last, (int)C::ROWS, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    meet<false>();
    for (long r = tid; r < C::ROWS; r += THREADS) {
      last = partly(row_of(r));
      if (last >= 0) atomicMin(firsts + last, (int)r);
    }
    meet<false>();
    for (long r = tid; r < C::ROWS; r += THREADS) {
      last = partly(row_of(r));
      source[r] = last >= 0 && (bit<LDS>(map, last) || __hip_atomic_load(firsts + last, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != (int)r) ? last : -1;
    }
    __syncthreads();
    for (long r = tid; r < C::ROWS; r += THREADS) {
      last = partly(row_of(r));
      if (last >= 0) set_bit(map, last);
    }
  }
  meet<LDS>();
  // Free pages before each word.
  long from, to;
  my_words(WORDS, from, to);
  int free = 0, all;
  for (long w = from; w < to; ++w) free += __builtin_popcount(~word<LDS>(map, w));
  const int so_far = before_me(free, sums, all);
  int at = so_far;
  for (long w = from; w < to; ++w) {
    put_word<LDS>((u32_t*)counts, w, (u32_t)at);
    at += __builtin_popcount(~word<LDS>(map, w));
  }
  meet<LDS>();
  auto fresh = [&](long k) {
    if (k >= all) return -1;
    long lo = 0, hi = WORDS;  // the last word with at most k free pages before it
    while (hi - lo > 1) {
      const long mid = (lo + hi) / 2;
      if ((int)word<LDS>((const u32_t*)counts, mid) <= k) lo = mid;
      else hi = mid;
    }
    return (int)(lo * 32) + nth_bit(~word<LDS>(map, lo), (int)(k - (int)word<LDS>((const u32_t*)counts, lo)));
  };
  // The rows: their copies, and then what they are to have.
  long asked = 0;
  for (long r0 = 0; r0 < C::ROWS; r0 += THREADS) {
    const long r = r0 + tid;
    int old = copied ? last : -1;
    if constexpr (!ONE) {
      __syncthreads();
      mine = row_of(r);
      old = r < C::ROWS ? source[r] : -1;
    }
    const int wanted = (old >= 0) + (mine.want - mine.kept);
    int total;
    const long first = asked + before_me(wanted, sums, total);
    // (the last kept slot of a row that copies is one of those to be filled)
    const int stays = mine.kept - (old >= 0);
    if (r < C::ROWS) {
      out_lengths[r] = mine.length;
      const int page = old >= 0 ? fresh(first) : -1;
      source[r] = page >= 0 ? old : -1;
      target[r] = page;
      if constexpr (C::WIDE) rows[r] = Row{mine.parent, stays, (int)first, wanted};
      // the slots of the row's next tokens, those that it has room for
      const int more = C::NEW > 0 ? room[r] : 0;
      for (int i = 0; i < C::NEW; ++i) {
        const long token = (long)mine.length + i;
        int p = -1;
        if (mine.parent >= 0 && i < more && token < C::SLOTS * C::T) {
          const int k = (int)(token / C::T) - stays;
          p = k < 0 ? page_at<C>(table, mine.parent, (int)(token / C::T)) : fresh(first + k);
        }
        slots[r * C::NEW + i] = p < 0 ? -1 : (int)(p * C::T + token % C::T);
      }
    }
    if constexpr (!C::WIDE) {
      parent[tid] = mine.parent;
      kept[tid] = stays;
      place[tid] = (int)(first - asked);
      __syncthreads();
      const int n = (int)((C::ROWS - r0 < THREADS ? C::ROWS - r0 : THREADS) * C::SLOTS);
#pragma unroll 4
      for (int i = tid; i < n; i += THREADS) {
        const int row = i / SLOTS, j = i % SLOTS, k = j - kept[row];
        const int have = (row + 1 < THREADS && r0 + row + 1 < C::ROWS ? place[row + 1] : total) - place[row];
        int p = -1;
        if (k < 0) p = page_at<C>(table, parent[row], j);
        else if (k < have) p = fresh(asked + place[row] + k);
        out_table[r0 * C::SLOTS + i] = p;
      }
    }
    asked += total;
  }
  if constexpr (C::WIDE) {
    // the pages in the order in which they are given out
    int k = so_far;
    for (long w = from; w < to && k < asked; ++w)
      for (u32_t m = ~word<LDS>(map, w); m && k < asked; m &= m - 1, ++k) fresh_pages[k] = (int)(w * 32) + __builtin_ctz(m);
    for (long k = all + (long)tid; k < asked; k += THREADS) fresh_pages[k] = -1;
  }
  if (tid == 0) left[0] = (int)(all - asked);
}
// `work`: of the bitmap and its counts beyond LDS_PAGES pages, of the rows and fresh pages if C::WIDE, of `firsts`; in this order.
template <class C> struct ForkWork {
  static constexpr bool LDS = C::P <= LDS_PAGES;
  static constexpr long WORDS = (C::P + 31) / 32, ROWS = LDS ? 0 : (2 * WORDS + 3) / 4 * 4, FRESH = ROWS + (C::WIDE ? 4 * C::ROWS : 0),
                        FIRSTS = FRESH + (C::WIDE ? C::ROWS * C::SLOTS : 0);
};
template <class C>
__device__ __forceinline__ void fork(const int* __restrict__ table, const int* __restrict__ lengths, const int* __restrict__ parents,
                                     const int* __restrict__ room, const u8_t* __restrict__ held, int* __restrict__ out_table,
                                     int* __restrict__ out_lengths, int* __restrict__ source, int* __restrict__ target, int* __restrict__ left,
                                     int* __restrict__ slots, int* work) {
  typedef ForkWork<C> W;
  __shared__ u32_t map[W::LDS ? W::WORDS + 1 : 1];
  __shared__ int counts[W::LDS ? W::WORDS + 1 : 1];
  fork_with<C, W::LDS>(W::LDS ? map : (u32_t*)work, W::LDS ? counts : work + W::WORDS, table, lengths, parents, room, held, out_table, out_lengths, source,
                       target, left, slots, work + W::FIRSTS, (Row*)(work + W::ROWS), work + W::FRESH);
}
// Large tables: 1024 slots of a row to a workgroup.
template <class C>
__device__ __forceinline__ void fork_rows(const int* __restrict__ table, const int* __restrict__ work, int* __restrict__ out_table) {
  typedef ForkWork<C> W;
  const long r = blockIdx.x;
  const Row row = ((const Row*)(work + W::ROWS))[r];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = (int)blockIdx.y * 1024 + i * 256 + (int)threadIdx.x, k = j - row.kept;
    if (j >= C::SLOTS) break;
    int p = -1;
    if (k < 0) p = page_at<C>(table, row.parent, j);
    else if (k < row.asked) p = work[W::FRESH + row.first + k];
    out_table[r * C::SLOTS + j] = p;
  }
}

// ---------------------------------------------------------------------------------------------
// compact: C supplies ENTRIES (of the tables), P, MOVES, WIDE (the tables are written by compact_rows).
// ---------------------------------------------------------------------------------------------

// The entries of the tables from `first` on, `stride` apart, with the pages that move under their new numbers: a page that moves is the k-th
// that does by the counts. Four entries at once, since the new numbers are in memory.
template <class C, bool LDS>
__device__ __forceinline__ void renumber(const u32_t* used, const int* counts, int moves, const int* __restrict__ table, const int* target,
                                         int* __restrict__ out_table, long first, long stride) {
  for (long i = first; i < C::ENTRIES; i += 4 * stride) {
    int p[4], k[4], to[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) p[u] = i + u * stride < C::ENTRIES ? table[i + u * stride] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      p[u] = p[u] >= 0 && p[u] < C::P ? p[u] : -1;
      k[u] = -1;
      if (p[u] < 0) continue;
      const u32_t m = word<LDS>(used, p[u] >> 5);
      if (m >> (p[u] & 31) & 1) k[u] = (int)word<LDS>((const u32_t*)counts, p[u] >> 5) + __builtin_popcount(m & ((1u << (p[u] & 31)) - 1));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) to[u] = k[u] >= 0 && k[u] < moves ? __hip_atomic_load(target + k[u], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : p[u];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * stride < C::ENTRIES) out_table[i + u * stride] = to[u];
  }
}

template <class C, bool LDS>
__device__ __forceinline__ void compact_with(u32_t* used, u32_t* busy, int* counts, const int* __restrict__ table, const u8_t* __restrict__ held,
                                             int* __restrict__ out_table, int* __restrict__ source, int* __restrict__ target, int* work) {
  constexpr long WORDS = (C::P + 31) / 32;
  __shared__ int sums[WAVES + 1];
  const int tid = threadIdx.x;
  for (long w = tid; w < WORDS; w += THREADS) put_word<LDS>(used, w, 0);
  meet<LDS>();
#pragma unroll 8
  for (long i = tid; i < C::ENTRIES; i += THREADS) {
    const int p = table[i];
    if (p >= 0 && p < C::P) set_bit(used, p);
  }
  meet<LDS>();
  // Pages in use, `used` or held, are n; what is in use and not held from n on moves into what is free below. `used` becomes those that move.
  long from, to;
  my_words(WORDS, from, to);
  int mine = 0, n;
  for (long w = from; w < to; ++w) {
    const u32_t h = held_word<C::P>(held, w), u = word<LDS>(used, w);
    put_word<LDS>(busy, w, h | u);
    put_word<LDS>(used, w, u & ~h);
    mine += __builtin_popcount(h | u);
  }
  before_me(mine, sums, n);
  n -= (int)(WORDS * 32 - C::P);  // (what lies past the last page counts as held)
  auto below = [&](long w) { return n <= w * 32 ? 0u : n >= w * 32 + 32 ? ~0u : (1u << (n - w * 32)) - 1; };
  int movers = 0, holes = 0, all;
  for (long w = from; w < to; ++w) {
    const u32_t m = word<LDS>(used, w) & ~below(w);
    put_word<LDS>(used, w, m);
    movers += __builtin_popcount(m);
    holes += __builtin_popcount(~word<LDS>(busy, w) & below(w));
  }
  int hole = before_me(holes, sums, all), mover = before_me(movers, sums, all);
  const int moves = all < C::MOVES ? all : (int)C::MOVES;
  for (long w = from; w < to; ++w) {
    put_word<LDS>((u32_t*)counts, w, (u32_t)mover);
    for (u32_t m = word<LDS>(used, w); m; m &= m - 1, ++mover)
      if (mover < moves) source[mover] = (int)(w * 32) + __builtin_ctz(m);
    for (u32_t h = ~word<LDS>(busy, w) & below(w); h; h &= h - 1, ++hole)
      if (hole < moves) target[hole] = (int)(w * 32) + __builtin_ctz(h);
  }
  for (long i = moves + tid; i < C::MOVES; i += THREADS) source[i] = target[i] = -1;
  if (C::WIDE && tid == 0) work[0] = moves;
  if constexpr (C::WIDE && LDS) {
    meet<LDS>();  // (past 32 pages a thread, words are others' than those that wrote them)
    for (long w = tid; w < WORDS; w += THREADS) {
      work[4 + w] = (int)used[w];
      work[4 + WORDS + w] = counts[w];
    }
  }
  if constexpr (!C::WIDE) {
    meet<false>();
    renumber<C, LDS>(used, counts, moves, table, target, out_table, tid, THREADS);
  }
}
// `work`: the moves, and from the fourth word on the bitmaps and counts where they are not in LDS or others read them (C::WIDE).
template <class C>
__device__ __forceinline__ void compact(const int* __restrict__ table, const u8_t* __restrict__ held, int* __restrict__ out_table,
                                        int* __restrict__ source, int* __restrict__ target, int* work) {
  constexpr long WORDS = (C::P + 31) / 32;
  constexpr bool LDS = C::P <= LDS_PAGES;
  __shared__ u32_t used[LDS ? WORDS + 1 : 1], busy[LDS ? WORDS + 1 : 1];
  __shared__ int counts[LDS ? WORDS + 1 : 1];
  compact_with<C, LDS>(LDS ? used : (u32_t*)work + 4, LDS ? busy : (u32_t*)work + 4 + 2 * WORDS, LDS ? counts : work + 4 + WORDS, table, held, out_table,
                       source, target, work);
}
// Large tables: 1024 entries to a workgroup.
template <class C>
__device__ __forceinline__ void compact_rows(const int* __restrict__ table, const int* __restrict__ target, int* work, int* __restrict__ out_table) {
  constexpr long WORDS = (C::P + 31) / 32;
  renumber<C, false>((u32_t*)work + 4, work + 4 + WORDS, work[0], table, target, out_table, (long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256);
}

// ---------------------------------------------------------------------------------------------
// copies: C supplies N (copies), P, BYTES (of a page), PER (bytes of a workgroup), W (bytes of an access), ONCE (with the
// non-temporal hint), CHECK, OWNERS (the last copy to each page is in a table).
// ---------------------------------------------------------------------------------------------

// An access of W bytes.
typedef u32_t u32x4 __attribute__((ext_vector_type(4)));
template <int W> struct Piece { typedef u8_t type; };
template <> struct Piece<2> { typedef u16_t type; };
template <> struct Piece<4> { typedef u32_t type; };
template <> struct Piece<8> { typedef u64_t type; };
template <> struct Piece<16> { typedef u32x4 type; };

template <class C> __device__ __forceinline__ bool pair_of(const int* __restrict__ source, const int* __restrict__ target, long i, int& s, int& t) {
  s = source[i];
  t = target[i];
  return s >= 0 && s < C::P && t >= 0 && t < C::P;
}

// The last copy to each page that copies name: FIRST puts -1 there, then the largest copy's number is taken.
template <class C, bool FIRST>
__device__ __forceinline__ void claim(const int* __restrict__ source, const int* __restrict__ target, int* __restrict__ owner) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  int s, t;
  if (i >= C::N || !pair_of<C>(source, target, i, s, t)) return;
  if constexpr (FIRST) owner[s] = owner[t] = -1;
  else atomicMax(&owner[t], (int)i);
}

// Whether some copy from number `from` on goes to page p. All threads of the workgroup.
template <class C> __device__ __forceinline__ bool goes_to(const int* __restrict__ source, const int* __restrict__ target, long from, int p) {
  int found = 0;
  for (long j = from + threadIdx.x; j < C::N; j += 256) {
    int s, t;
    if (pair_of<C>(source, target, j, s, t)) found |= t == p;
  }
  return __syncthreads_or(found) != 0;
}

// The part blockIdx.y of a page.
template <class C> __device__ __forceinline__ void move(const u8_t* from, u8_t* to) {
  typedef typename Piece<C::W>::type V;
  const long begin = (long)blockIdx.y * C::PER, end = begin + C::PER < C::BYTES ? begin + C::PER : C::BYTES;
#pragma unroll 4
  for (long b = begin + threadIdx.x * C::W; b < end; b += 256 * C::W) {
    const V* const x = (const V*)(from + b);
    if constexpr (C::ONCE) __builtin_nontemporal_store(__builtin_nontemporal_load(x), (V*)(to + b));
    else *(V*)(to + b) = *x;
  }
}

// In place: sources that are a target too, aside. aside [N][BYTES], flags [N]: whether a copy's source is there.
template <class C>
__device__ __forceinline__ void put_aside(const u8_t* from, const u8_t* to, const int* __restrict__ source, const int* __restrict__ target,
                                          const int* __restrict__ owner, u8_t* __restrict__ aside, int* __restrict__ flags) {
  if (from != to) return;
  const long i = blockIdx.x;
  int s, t;
  if (!pair_of<C>(source, target, i, s, t)) return;
  bool hit;
  if constexpr (C::OWNERS) hit = owner[s] >= 0;
  else hit = goes_to<C>(source, target, 0, s);
  if (blockIdx.y == 0 && threadIdx.x == 0) flags[i] = hit;
  if (hit) move<C>(from + (long)s * C::BYTES, aside + i * C::BYTES);
}

template <class C>
__device__ __forceinline__ void copy(const u8_t* from, u8_t* to, const int* __restrict__ source, const int* __restrict__ target,
                                     const int* __restrict__ owner, const u8_t* __restrict__ aside, const int* __restrict__ flags) {
  const long i = blockIdx.x;
  int s, t;
  if (!pair_of<C>(source, target, i, s, t)) return;
  const u8_t* page = from + (long)s * C::BYTES;
  if constexpr (C::CHECK) {
    bool last;
    if constexpr (C::OWNERS) last = owner[t] == (int)i;
    else last = !goes_to<C>(source, target, i + 1, t);
    if (!last) return;
    if (from == to && flags[i]) page = aside + i * C::BYTES;
  }
  move<C>(page, to + (long)t * C::BYTES);
}

}  // namespace pages
}  // namespace accy
