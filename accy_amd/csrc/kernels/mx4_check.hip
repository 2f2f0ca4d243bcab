// Build-time check (compiled by accy_amd/build.py with hipcc --offload-arch=gfx950): instantiates the
// microscaled 4-bit templates with shapes the planner emits, so that a host without a GPU still
// verifies that they compile for CDNA4. Nothing calls these kernels.
#include "common.h"
#include "gemm.h"
#include "mx4.h"
#include "mx4_contract.h"

struct CheckStore {
  float* c;
  __device__ __forceinline__ void operator()(long, long m, long n, float v) const { c[m * 513 + n] = v; }
};
struct CheckProduct {
  static constexpr long M = 300, N = 513, K = 1056;
  static constexpr int BM = 128, BN = 128, GROUP_M = 8, SPLITS = 2, WK = 0;
};
struct CheckSmall : CheckProduct {
  static constexpr int BM = 32, BN = 32, WK = 4;
};
template <int D, int DIM, int QUERIES, int GROUP, int S>
struct CheckCache {
  static constexpr int DT = D, HD = DIM, H = 8, T = 64, P = 512, Q = QUERIES, G = GROUP, MAXP = 64, SPLITS = S;
  static constexpr long SEQS = 8, TOKENS = 100;
  static constexpr float SL = 0x1.05p-3f;
};

extern "C" __global__ void __launch_bounds__(256) check_mx4_small(const u8_t* a, const u8_t* sa, const u8_t* b, const u8_t* sb, float* c) {
  accy::mx4::contract_direct<CheckSmall>(a, sa, b, sb, CheckStore{c});
}
extern "C" __global__ void __launch_bounds__(256) check_mx4_tile(const u8_t* a, const u8_t* sa, const u8_t* b, const u8_t* sb, float* c) {
  accy::mx4::contract_tile<CheckProduct>(a, sa, b, sb, CheckStore{c});
}
extern "C" __global__ void __launch_bounds__(256) check_mx4_values(const u8_t* c, const u8_t* s, u16_t* o) {
  accy::mx4::values<0, int, 4096>(c, s, o);
}
extern "C" __global__ void __launch_bounds__(256) check_mx4_write(u8_t* c, const float* k, const float* v, const int* s) {
  accy::mx4::cache_write<CheckCache<2, 96, 1, 1, 1>, false>(c, k, v, s, nullptr);
}
extern "C" __global__ void __launch_bounds__(256) check_mx4_read(const u8_t* c, const int* s, u16_t* k, u16_t* v) {
  accy::mx4::cache_read<CheckCache<1, 96, 1, 1, 1>>(c, s, k, v);
}
extern "C" __global__ void __launch_bounds__(256) check_mx4_attend_bf16(const u16_t* q, const u8_t* c, const int* p, const int* l, u16_t* o, float* part) {
  accy::mx4::attend<CheckCache<0, 128, 1, 8, 4>>(q, c, p, l, o, part);
}
extern "C" __global__ void __launch_bounds__(256) check_mx4_attend_f32(const float* q, const u8_t* c, const int* p, const int* l, float* o, float* part) {
  accy::mx4::attend<CheckCache<2, 96, 5, 4, 1>>(q, c, p, l, o, part);
}
extern "C" __global__ void __launch_bounds__(256) check_mx4_join(const float* part, u16_t* o) {
  accy::mx4::attend_join<CheckCache<0, 128, 1, 8, 4>>(part, o);
}
struct CheckShared : CheckCache<0, 128, 2, 4, 2> {
  static constexpr int PREFIXES = 3, PSPLITS = 4, PREFIX_MAXP = 128;
};
extern "C" __global__ void __launch_bounds__(256) check_mx4_attend_shared(const u16_t* q, const u8_t* c, const int* p, const int* l, const int* sp, const int* sl,
                                                                          const int* of, float* part) {
  accy::mx4::attend_shared<CheckShared>(q, c, p, l, sp, sl, of, part);
}
extern "C" __global__ void __launch_bounds__(256) check_mx4_join_shared(const float* part, u16_t* o, const int* of) {
  accy::mx4::attend_join<CheckShared>(part, o, of);
}
