// Build-time check (compiled by accy_amd/build.py with hipcc --offload-arch=gfx950): instantiates the templates of heads, pages and
// logits with shapes the planner emits, so that a host without a GPU still verifies that they compile for CDNA4. Nothing calls
// these kernels.
#include "common.h"
#include "heads.h"
#include "logits.h"
#include "pages.h"

template <int D_, int DIM, int PAIRS, int WIDTH, int ROW_LANES, bool NEAR>
struct CheckHeads {
  static constexpr int DT = D_, GT = D_, D = DIM, F = PAIRS, HQ = 12, HK = 4, AXES = NEAR ? 3 : 0, W = WIDTH, LANES = ROW_LANES, TT = 2;
  static constexpr bool NEIGHBOURS = NEAR, NORM = true;
  static constexpr long TOKENS = 1001;
  static constexpr float EPS = 1e-6f;
};
template <int D_, long VOCAB, int TOP, int S, int THREADS, int CHUNKS>
struct CheckLogits {
  static constexpr int DT = D_, K = TOP, SPLITS = S, NT = THREADS, U = CHUNKS;
  static constexpr long ROWS = 77, V = VOCAB;
  static constexpr bool ONCE = S == 1;
};
template <long PAGES, long R, bool W = false> struct CheckFork {
  static constexpr bool WIDE = W;
  static constexpr long SEQS = 20, ROWS = R, SLOTS = 9, P = PAGES, T = 64, NEW = 2, ENTRIES = 180, MOVES = 50;
};
struct CheckCopy {
  static constexpr long N = 30, P = 100, BYTES = 8704, PER = 8192;
  static constexpr int W = 16;
  static constexpr bool ONCE = true, CHECK = true, OWNERS = false;
};

typedef CheckHeads<0, 128, 64, 8, 8, false> Bf16Heads;
typedef CheckHeads<2, 96, 32, 4, 16, true> F32Heads;
extern "C" __global__ void __launch_bounds__(256) check_heads(const u16_t* q, const u16_t* k, const int* p, const float* f, const u16_t* g, u16_t* a, u16_t* b) {
  accy::heads::rotate<Bf16Heads>(q, k, p, f, nullptr, g, g, a, b);
}
extern "C" __global__ void __launch_bounds__(256) check_heads_grad(const float* dq, const float* dk, const float* q, const float* k, const int* p, const float* f,
                                                                   const int* x, const float* g, float* a, float* b, float* part) {
  accy::heads::rotate_grad<F32Heads>(dq, dk, q, k, p, f, x, g, g, a, b, part);
}
extern "C" __global__ void __launch_bounds__(1024) check_heads_gain(const float* part, float* a, float* b) { accy::heads::gain_sums<F32Heads, 501>(part, a, b); }

typedef CheckLogits<0, 50257, 20, 1, 256, 7> Bf16Logits;
typedef CheckLogits<2, 32001, 5, 8, 256, 4> F32Logits;
typedef CheckLogits<1, 50257, 0, 1, 512, 13> F16Grad;
typedef CheckLogits<1, 50257, 0, 4, 256, 7> F16Split;
extern "C" __global__ void __launch_bounds__(256) check_log_probs(const u16_t* x, const int* t, float* a, float* b, float* c, int* d) {
  accy::logits::log_probs<Bf16Logits>(x, t, a, b, c, d, nullptr);
}
extern "C" __global__ void __launch_bounds__(256) check_log_probs_split(const float* x, const int* t, float* part) {
  accy::logits::log_probs<F32Logits>(x, t, nullptr, nullptr, nullptr, nullptr, part);
}
extern "C" __global__ void __launch_bounds__(256) check_log_probs_join(const float* x, const int* t, const float* part, float* a, float* b, float* c, int* d) {
  accy::logits::log_probs_join<F32Logits>(x, t, part, a, b, c, d);
}
extern "C" __global__ void __launch_bounds__(512) check_grad(const u16_t* x, const int* t, const float* a, const float* b, u16_t* o) {
  accy::logits::grad_row<F16Grad>(x, t, a, b, o);
}
extern "C" __global__ void __launch_bounds__(256) check_grad_split(const u16_t* x, const int* t, const float* a, const float* b, const float* part, u16_t* o) {
  accy::logits::grad_split<F16Split>(x, t, a, b, part, o);
}

extern "C" __global__ void __launch_bounds__(1024) check_fork(const int* t, const int* l, const int* p, const int* r, const u8_t* h, int* a, int* b, int* c,
                                                              int* d, int* e, int* s) {
  accy::pages::fork<CheckFork<1000, 20>>(t, l, p, r, h, a, b, c, d, e, s, nullptr);
}
extern "C" __global__ void __launch_bounds__(1024) check_fork_large(const int* t, const int* l, const int* p, const int* r, const u8_t* h, int* a, int* b, int* c,
                                                                    int* d, int* e, int* s, int* work) {
  accy::pages::fork<CheckFork<1000000, 2000, true>>(t, l, p, r, h, a, b, c, d, e, s, work);
}
extern "C" __global__ void __launch_bounds__(256) check_fork_rows(const int* t, const int* work, int* a) { accy::pages::fork_rows<CheckFork<1000000, 2000, true>>(t, work, a); }
extern "C" __global__ void __launch_bounds__(1024) check_compact(const int* t, const u8_t* h, int* a, int* b, int* c) {
  accy::pages::compact<CheckFork<1000, 20>>(t, h, a, b, c, nullptr);
}
extern "C" __global__ void __launch_bounds__(256) check_compact_rows(const int* t, const int* to, int* work, int* a) {
  accy::pages::compact_rows<CheckFork<1000, 20, true>>(t, to, work, a);
}
extern "C" __global__ void __launch_bounds__(256) check_copy(const u8_t* from, u8_t* to, const int* s, const int* t, const u8_t* aside, const int* flags) {
  accy::pages::copy<CheckCopy>(from, to, s, t, nullptr, aside, flags);
}
extern "C" __global__ void __launch_bounds__(256) check_put_aside(const u8_t* from, const u8_t* to, const int* s, const int* t, u8_t* aside, int* flags) {
  accy::pages::put_aside<CheckCopy>(from, to, s, t, nullptr, aside, flags);
}
