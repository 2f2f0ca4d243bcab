// Heads of queries and keys as attention takes them: each normalised, y = x / sqrt(mean(x^2) + eps) * gain, and turned by its token's
// position: of pair i of the first 2 F dims, (a, b) becomes (a cos - b sin, b cos + a sin) of position * frequency[i]. And the gradient.
//
// Two numbers are read and two written for about eight operations, so a prompt's heads are bound by HBM (8192 tokens of 32 heads of 128 bf16 27 us, 5.0
// TB/s; the gradient of 8192 x 20 x 128 31 us, 4.0 TB/s) and a step's by the launch (one token 3.4 us of kernel in a call of 8). The non-temporal hint gains bf16
// rows 4 % and costs f32 rows of 80 dims half as much again.
// A row (one head of one token) belongs to LANES adjacent lanes, so that its sum is a few shuffles, and each lane holds whole
// pairs: W dims of a pair's first members and the W of its second (16 bytes each where the sizes allow it), which turn without
// leaving the lane. The cosines of a token are the same for all of its heads: a workgroup forms them once for its TT tokens, a pair per
// thread, while its first rows are on their way. Angles: the turns position * frequency / 2 pi in two 64-bit numbers, whose fraction
// is off by 2^-50 at most up to 2^50 turns, which positions of 32 bits do not reach below frequencies of millions, then f32 polynomials on an eighth
// of a turn. (One 64-bit number is off by 2^-52 of the turns: 2^-23 at the largest positions and a frequency of 1.)
//
// C supplies DT (elements: 0 bf16, 1 f16, 2 f32), GT (gains), D, F, HQ, HK (heads of queries and keys), TOKENS, AXES (positions per
// token, 0: one without axes), NEIGHBOURS (pairs 2 i, 2 i + 1, else i, F + i), NORM, EPS, W, LANES, TT.
#pragma once

namespace accy {
namespace heads {

// The same types as the other operators' (0 bf16, 1 f16, 2 f32), results rounded to nearest even in all of them.
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
// W numbers as they lie in memory: one access (two of 32 bytes).
template <int BYTES> struct Bits;
template <> struct Bits<2> { typedef u16_t type; };
template <> struct Bits<4> { typedef u32_t type; };
template <> struct Bits<8> { typedef u32_t type __attribute__((ext_vector_type(2))); };
template <> struct Bits<16> { typedef u32_t type __attribute__((ext_vector_type(4))); };
template <> struct Bits<32> { typedef u32_t type __attribute__((ext_vector_type(8), aligned(16))); };  // gains of f32 beside 16-bit heads
template <int DT, int W> struct Raw { typedef typename Bits<W * (DT == 2 ? 4 : 2)>::type type; };
template <class T, int W> struct alignas(W * sizeof(T) < 16 ? W * sizeof(T) : 16) Chunk { T v[W]; };
template <int DT, int W> __device__ __forceinline__ void widen(const typename Raw<DT, W>::type& raw, float* x) {
  const Chunk<typename Elem<DT>::type, W> c = __builtin_bit_cast(Chunk<typename Elem<DT>::type, W>, raw);
#pragma unroll
  for (int i = 0; i < W; ++i) x[i] = from_elem<DT>(c.v[i]);
}
template <int DT, int W> __device__ __forceinline__ typename Raw<DT, W>::type narrow(const float* x) {
  Chunk<typename Elem<DT>::type, W> c;
#pragma unroll
  for (int i = 0; i < W; ++i) c.v[i] = to_elem<DT>(x[i]);
  return __builtin_bit_cast(typename Raw<DT, W>::type, c);
}

template <class C> struct Row {
  // Units of a row: W pairs each, then what does not turn in 2 W dims each (the last one W where it is odd).
  static constexpr int TURNING = C::F / C::W, UNITS = TURNING + (C::D - 2 * C::F + 2 * C::W - 1) / (2 * C::W), PER = (UNITS + C::LANES - 1) / C::LANES;
  static __device__ __forceinline__ int first(int u) { return u >= TURNING ? 2 * C::F + 2 * C::W * (u - TURNING) : C::NEIGHBOURS ? 2 * C::W * u : C::W * u; }
  static __device__ __forceinline__ int second(int u) { return u >= TURNING || C::NEIGHBOURS ? first(u) + C::W : C::F + C::W * u; }
  // Whether unit u is there, and its second half.
  static __device__ __forceinline__ bool has(int u) { return UNITS % C::LANES == 0 || u < UNITS; }
  static __device__ __forceinline__ bool both(int u) { return (C::D - 2 * C::F) % (2 * C::W) == 0 || u + 1 < UNITS; }
};

__device__ __forceinline__ void turn(int position, float frequency, float& c, float& s) {
  // Twice a product and what its rounding left out, 1 / 2 pi in two numbers.
  constexpr double HI = 0x1.45f306dc9c883p-3, LO = -0x1.6b01ec5417056p-57;
  const double f = frequency, p = position, rate = f * HI, rate_lo = __builtin_fma(f, HI, -rate) + f * LO;
  double t = p * rate;
  const double t_lo = __builtin_fma(p, rate, -t) + p * rate_lo;
  t = (t - __builtin_rint(t)) + t_lo;
  const double k = __builtin_rint(t * 4.0);
  const float r = (float)((t - k * 0.25) * 6.283185307179586);
  const u32_t q = (u32_t)(int)k;
  s = sincos_core(r, q);
  c = sincos_core(r, q + 1);
}

// cos and sin of the pairs of tokens t0 .. t0 + TT - 1.
template <class C>
__device__ __forceinline__ void turns(const int* __restrict__ positions, const float* __restrict__ frequencies, const int* __restrict__ axes,
                                      long t0, float (*c)[C::F], float (*s)[C::F]) {
  for (int i = threadIdx.x; i < C::TT * C::F; i += 256) {
    const int t = i / C::F, f = i % C::F;
    if (t0 + t >= C::TOKENS) break;
    int p = 0;
    if constexpr (C::AXES == 0) {
      p = positions[t0 + t];
    } else {
      const int a = axes[f];
      if (a >= 0 && a < C::AXES) p = positions[(t0 + t) * C::AXES + a];
    }
    turn(p, frequencies[f], c[t][f], s[t][f]);
  }
}

// The units of a row that are this lane's, as they lie in memory; zeros where there is nothing.
template <class C, int DT> struct Units {
  typedef typename Raw<DT, C::W>::type V;
  V v[Row<C>::PER][2];
  __device__ __forceinline__ void load(const typename Elem<DT>::type* __restrict__ row, bool here) {
    typedef Row<C> R;
#pragma unroll
    for (int i = 0; i < R::PER; ++i) {
      const int u = (int)(threadIdx.x % C::LANES) + i * C::LANES;
      v[i][0] = v[i][1] = V{};
      if (!here || !R::has(u)) continue;
      v[i][0] = *(const V*)(row + R::first(u));
      if (R::both(u)) v[i][1] = *(const V*)(row + R::second(u));
    }
  }
  __device__ __forceinline__ void widen_to(float (&x)[Row<C>::PER][2 * C::W]) const {
#pragma unroll
    for (int i = 0; i < Row<C>::PER; ++i) {
      widen<DT, C::W>(v[i][0], x[i]);
      widen<DT, C::W>(v[i][1], x[i] + C::W);
    }
  }
};
template <class C> __device__ __forceinline__ void store_row(typename Elem<C::DT>::type* __restrict__ row, const float (&x)[Row<C>::PER][2 * C::W]) {
  typedef Row<C> R;
  typedef typename Raw<C::DT, C::W>::type V;
#pragma unroll
  for (int i = 0; i < R::PER; ++i) {
    const int u = (int)(threadIdx.x % C::LANES) + i * C::LANES;
    if (!R::has(u)) continue;
    *(V*)(row + R::first(u)) = narrow<C::DT, C::W>(x[i]);
    if (R::both(u)) *(V*)(row + R::second(u)) = narrow<C::DT, C::W>(x[i] + C::W);
  }
}

// The unit turned (BACK: turned back) by its cosines and sines.
template <class C, bool BACK> __device__ __forceinline__ void turn_unit(int u, const float* c, const float* s, float (&x)[2 * C::W]) {
  if (u >= Row<C>::TURNING) return;
  Chunk<float, C::W> cc, ss;
  if constexpr (C::W > 4) {
#pragma unroll
    for (int i = 0; i < C::W; i += 4) {
      const Chunk<float, 4> a = *(const Chunk<float, 4>*)(c + C::W * u + i), b = *(const Chunk<float, 4>*)(s + C::W * u + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        cc.v[i + j] = a.v[j];
        ss.v[i + j] = b.v[j];
      }
    }
  } else {
    cc = *(const Chunk<float, C::W>*)(c + C::W * u);
    ss = *(const Chunk<float, C::W>*)(s + C::W * u);
  }
#pragma unroll
  for (int i = 0; i < C::W; ++i) {
    const int ia = C::NEIGHBOURS ? 2 * i : i, ib = C::NEIGHBOURS ? 2 * i + 1 : C::W + i;
    const float a = x[ia], b = x[ib], sn = BACK ? -ss.v[i] : ss.v[i];
    x[ia] = a * cc.v[i] - b * sn;
    x[ib] = b * cc.v[i] + a * sn;
  }
}

// The sum over the lanes of a row.
template <class C> __device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = 1; o < C::LANES; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// A row of the tile that starts at token t0: its token, and its place in the queries' or keys' buffer.
template <class C, int H> __device__ __forceinline__ bool place(long t0, int row, int& t, long& at) {
  t = row / H;
  at = ((t0 + t) * H + row % H) * C::D;
  return t < C::TT && t0 + t < C::TOKENS;
}

// The first rows of the tile that are this lane's, on their way.
template <class C, int H, int DT> __device__ __forceinline__ void start(const typename Elem<DT>::type* __restrict__ x, long t0, Units<C, DT>& next) {
  int t;
  long at;
  const bool here = place<C, H>(t0, threadIdx.x / C::LANES, t, at);
  next.load(x + (here ? at : 0), here);
}

// The H heads of each token of the tile, x to y; `next`: its first rows. The rows after are on their way while some are worked on.
template <class C, int H>
__device__ __forceinline__ void rotate_rows(const typename Elem<C::DT>::type* __restrict__ x, typename Elem<C::DT>::type* __restrict__ y,
                                            const float (&gain)[Row<C>::PER][2 * C::W], long t0, const float (*c)[C::F], const float (*s)[C::F],
                                            Units<C, C::DT>& next) {
  typedef Row<C> R;
  constexpr int AT_ONCE = 256 / C::LANES;
  const int lane = threadIdx.x % C::LANES;
  for (int row = threadIdx.x / C::LANES; row < C::TT * H; row += AT_ONCE) {
    float v[R::PER][2 * C::W];
    int t, nt;
    long at, nat;
    const bool here = place<C, H>(t0, row, t, at), more = place<C, H>(t0, row + AT_ONCE, nt, nat);
    next.widen_to(v);
    if (more) next.load(x + nat, true);
    if constexpr (C::NORM) {
      float sum = 0.0f;
#pragma unroll
      for (int u = 0; u < R::PER; ++u)
#pragma unroll
        for (int i = 0; i < 2 * C::W; ++i) sum = __builtin_fmaf(v[u][i], v[u][i], sum);
      const float r = __builtin_amdgcn_rsqf(row_sum<C>(sum) / C::D + C::EPS);
#pragma unroll
      for (int u = 0; u < R::PER; ++u)
#pragma unroll
        for (int i = 0; i < 2 * C::W; ++i) v[u][i] = v[u][i] * r * gain[u][i];
    }
    if (!here) continue;
#pragma unroll
    for (int u = 0; u < R::PER; ++u) turn_unit<C, false>(lane + u * C::LANES, c[t], s[t], v[u]);
    store_row<C>(y + at, v);
  }
}

template <class C>
__device__ __forceinline__ void load_gain(const typename Elem<C::GT>::type* __restrict__ gain, float (&g)[Row<C>::PER][2 * C::W]) {
  if constexpr (C::NORM) {
    Units<C, C::GT> raw;
    raw.load(gain, true);
    raw.widen_to(g);
  }
}

// Queries, keys or both (none: nullptr) of TT tokens to a workgroup.
template <class C>
__device__ __forceinline__ void rotate(const typename Elem<C::DT>::type* __restrict__ q, const typename Elem<C::DT>::type* __restrict__ k,
                                       const int* __restrict__ positions, const float* __restrict__ frequencies, const int* __restrict__ axes,
                                       const typename Elem<C::GT>::type* __restrict__ qgain, const typename Elem<C::GT>::type* __restrict__ kgain,
                                       typename Elem<C::DT>::type* __restrict__ qout, typename Elem<C::DT>::type* __restrict__ kout) {
  typedef Row<C> R;
  __shared__ __attribute__((aligned(16))) float c[C::TT][C::F], s[C::TT][C::F];
  const long t0 = (long)blockIdx.x * C::TT;
  float gain[R::PER][2 * C::W];
  Units<C, C::DT> queries, keys;
  if constexpr (C::HQ > 0) start<C, C::HQ>(q, t0, queries);
  if constexpr (C::HK > 0) start<C, C::HK>(k, t0, keys);
  turns<C>(positions, frequencies, axes, t0, c, s);
  __syncthreads();
  if constexpr (C::HQ > 0) {
    load_gain<C>(qgain, gain);
    rotate_rows<C, C::HQ>(q, qout, gain, t0, c, s, queries);
  }
  if constexpr (C::HK > 0) {
    load_gain<C>(kgain, gain);
    rotate_rows<C, C::HK>(k, kout, gain, t0, c, s, keys);
  }
}

// ---- the gradient ----
//
// With n = x r, r = 1 / sqrt(mean(x^2) + eps) and g the result's gradient turned back: d gain = sum over rows of g n, dx = r (g gain -
// n mean(g gain n)). Each lane keeps its dims' sums of g n over its workgroup's rows; they meet in LDS, the workgroups' in a second
// kernel in order, so that a call's sums do not depend on when its workgroups run.
template <class C, int H>
__device__ __forceinline__ void rotate_rows_grad(const typename Elem<C::DT>::type* __restrict__ dy, const typename Elem<C::DT>::type* __restrict__ x,
                                                 typename Elem<C::DT>::type* __restrict__ dx, const float (&gain)[Row<C>::PER][2 * C::W], long t0,
                                                 const float (*c)[C::F], const float (*s)[C::F], float (&sums)[Row<C>::PER][2 * C::W],
                                                 Units<C, C::DT>& next_g, Units<C, C::DT>& next_x) {
  typedef Row<C> R;
  constexpr int AT_ONCE = 256 / C::LANES;
  const int lane = threadIdx.x % C::LANES;
  for (int row = threadIdx.x / C::LANES; row < C::TT * H; row += AT_ONCE) {
    int t, nt;
    long at, nat;
    if (!place<C, H>(t0, row, t, at)) break;  // (the lanes of a row are here or gone together)
    float g[R::PER][2 * C::W], v[R::PER][2 * C::W];
    next_g.widen_to(g);
    if constexpr (C::NORM) next_x.widen_to(v);
    if (place<C, H>(t0, row + AT_ONCE, nt, nat)) {
      next_g.load(dy + nat, true);
      if constexpr (C::NORM) next_x.load(x + nat, true);
    }
#pragma unroll
    for (int u = 0; u < R::PER; ++u) turn_unit<C, true>(lane + u * C::LANES, c[t], s[t], g[u]);
    if constexpr (C::NORM) {
      float squares = 0.0f, inner = 0.0f;
#pragma unroll
      for (int u = 0; u < R::PER; ++u)
#pragma unroll
        for (int i = 0; i < 2 * C::W; ++i) {
          squares = __builtin_fmaf(v[u][i], v[u][i], squares);
          inner = __builtin_fmaf(g[u][i] * gain[u][i], v[u][i], inner);
        }
      const float r = __builtin_amdgcn_rsqf(row_sum<C>(squares) / C::D + C::EPS);
      const float mean = row_sum<C>(inner) * r / C::D;
#pragma unroll
      for (int u = 0; u < R::PER; ++u)
#pragma unroll
        for (int i = 0; i < 2 * C::W; ++i) {
          const float n = v[u][i] * r;
          sums[u][i] = __builtin_fmaf(g[u][i], n, sums[u][i]);
          g[u][i] = r * __builtin_fmaf(-n, mean, g[u][i] * gain[u][i]);
        }
    }
    if (dx) store_row<C>(dx + at, g);
  }
}

// The lanes' sums of a workgroup, D of them, to `to`.
template <class C> __device__ __forceinline__ void meet(float (&sums)[Row<C>::PER][2 * C::W], float (*lds)[C::D], float* __restrict__ to) {
  typedef Row<C> R;
  const int lane = threadIdx.x % C::LANES, wave = threadIdx.x >> 6;
#pragma unroll
  for (int u = 0; u < R::PER; ++u) {
#pragma unroll
    for (int i = 0; i < 2 * C::W; ++i) {
#pragma unroll
      for (int o = C::LANES; o < 64; o <<= 1) sums[u][i] += __shfl_xor(sums[u][i], o, 64);
    }
    const int unit = lane + u * C::LANES;
    if ((threadIdx.x & 63) < C::LANES && R::has(unit)) {
#pragma unroll
      for (int i = 0; i < C::W; ++i) {
        lds[wave][R::first(unit) + i] = sums[u][i];
        if (R::both(unit)) lds[wave][R::second(unit) + i] = sums[u][C::W + i];
      }
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < C::D; d += 256) to[d] = (lds[0][d] + lds[1][d]) + (lds[2][d] + lds[3][d]);
  __syncthreads();
}

// GROUPS workgroups walk over the tiles; part [GROUPS][2][D]: sums of the queries' gain and of the keys'. Gradients that nobody asked
// for: nullptr (and none of the sums without `part`).
template <class C>
__device__ __forceinline__ void rotate_grad(const typename Elem<C::DT>::type* __restrict__ dq, const typename Elem<C::DT>::type* __restrict__ dk,
                                            const typename Elem<C::DT>::type* __restrict__ q, const typename Elem<C::DT>::type* __restrict__ k,
                                            const int* __restrict__ positions, const float* __restrict__ frequencies, const int* __restrict__ axes,
                                            const typename Elem<C::GT>::type* __restrict__ qgain, const typename Elem<C::GT>::type* __restrict__ kgain,
                                            typename Elem<C::DT>::type* __restrict__ qout, typename Elem<C::DT>::type* __restrict__ kout,
                                            float* __restrict__ part) {
  typedef Row<C> R;
  __shared__ __attribute__((aligned(16))) float c[C::TT][C::F], s[C::TT][C::F], lds[C::NORM ? 4 : 1][C::D];
  float gains[2][R::PER][2 * C::W], sums[2][R::PER][2 * C::W];
  load_gain<C>(qgain, gains[0]);
  load_gain<C>(kgain, gains[1]);
#pragma unroll
  for (int u = 0; u < R::PER; ++u)
#pragma unroll
    for (int i = 0; i < 2 * C::W; ++i) sums[0][u][i] = sums[1][u][i] = 0.0f;
  for (long t0 = (long)blockIdx.x * C::TT; t0 < C::TOKENS; t0 += (long)gridDim.x * C::TT) {
    Units<C, C::DT> gq, xq, gk, xk;
    if constexpr (C::HQ > 0) {
      start<C, C::HQ>(dq, t0, gq);
      if constexpr (C::NORM) start<C, C::HQ>(q, t0, xq);
    }
    if constexpr (C::HK > 0) {
      start<C, C::HK>(dk, t0, gk);
      if constexpr (C::NORM) start<C, C::HK>(k, t0, xk);
    }
    __syncthreads();
    turns<C>(positions, frequencies, axes, t0, c, s);
    __syncthreads();
    if constexpr (C::HQ > 0) rotate_rows_grad<C, C::HQ>(dq, q, qout, gains[0], t0, c, s, sums[0], gq, xq);
    if constexpr (C::HK > 0) rotate_rows_grad<C, C::HK>(dk, k, kout, gains[1], t0, c, s, sums[1], gk, xk);
  }
  if constexpr (C::NORM) {
    if (part) {
      meet<C>(sums[0], lds, part + (long)blockIdx.x * 2 * C::D);
      meet<C>(sums[1], lds, part + ((long)blockIdx.x * 2 + 1) * C::D);
    }
  }
}

// The workgroups' sums, 32 dims and 32 strands of them to a workgroup of 1024; blockIdx.y: queries, keys.
template <class C, int GROUPS>
__device__ __forceinline__ void gain_sums(const float* __restrict__ part, typename Elem<C::GT>::type* __restrict__ qgain,
                                          typename Elem<C::GT>::type* __restrict__ kgain) {
  __shared__ float lds[32][33];
  const int lane = threadIdx.x & 31, d = blockIdx.x * 32 + lane, strand = threadIdx.x >> 5;
  typename Elem<C::GT>::type* const to = blockIdx.y ? kgain : qgain;
  float sum = 0.0f;
  if (d < C::D) {
#pragma unroll 16
    for (int g = strand; g < GROUPS; g += 32) sum += part[((long)g * 2 + blockIdx.y) * C::D + d];
  }
  lds[strand][lane] = sum;
  __syncthreads();
  // a row of lanes each adds up a dim
  sum = lds[lane][strand];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor(sum, o, 64);
  const int mine = blockIdx.x * 32 + strand;
  if (lane == 0 && mine < C::D && to) to[mine] = to_elem<C::GT>(sum);
}

}  // namespace heads
}  // namespace accy
