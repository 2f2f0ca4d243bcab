// What the planners of this target's custom calls share (planner_custom.cpp, planner_mx4.cpp, planner_heads.cpp, planner_pages.cpp,
// planner_logits.cpp). The wire carries a custom call's result type, so everything about a call is checked where it is planned.
#pragma once

#include "planner_internal.hpp"

namespace accy {
namespace planning {

[[noreturn]] inline void refuse(const Op& op, const std::string& why) {
  fail(Err::Unsupported, "custom_call " + op.bytes + ": " + why);
}

inline void require(bool ok, const Op& op, const std::string& why) {
  if (!ok) refuse(op, why);
}

// DT of kernels/mx4.h.
inline int element_type(const Op& op, DType d) {
  switch (d) {
    case DType::bf16: return 0;
    case DType::f16: return 1;
    case DType::f32: return 2;
    default: refuse(op, std::string(dtype_name(d)) + " values (bf16, f16 or f32)");
  }
}

inline int64_t last(const Type& t) { return t.rank() ? t.dims.back().extent : 0; }

// The extents of a's leading axes are b's.
inline bool same_rows(const Type& a, const Type& b) {
  if (a.rank() != b.rank()) return false;
  for (size_t i = 0; i + 1 < a.rank(); ++i)
    if (a.dims[i].extent != b.dims[i].extent) return false;
  return true;
}

inline std::string num(int64_t n) { return std::to_string(n); }

}  // namespace planning
}  // namespace accy
