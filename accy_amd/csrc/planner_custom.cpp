// Custom calls of this target, version 1 of "accy.<set>.<name>":
//
//   accy.group(..)      two to four operands as one of another call, which takes four at most; it computes nothing
//   accy.mx4.*          microscaled 4-bit floats (planner_mx4.cpp)
//   accy.heads.*        norms and rotations of heads (planner_heads.cpp)
//   accy.pages.*        page tables and pages of a cache (planner_pages.cpp)
//   accy.logits.*       log probabilities (planner_logits.cpp)
#include "planner_custom.hpp"

namespace accy {
namespace planning {

void Planner::custom(uint32_t v) {
  const Op& op = g_.ops[v];
  auto after = [&](const char* prefix) { return op.bytes.compare(0, std::strlen(prefix), prefix) == 0 ? op.bytes.substr(std::strlen(prefix)) : ""; };
  auto operands = [&](size_t n) { require(op.args.size() == n, op, num((int64_t)n) + " operands"); };
  if (op.index == 1) {
    if (op.bytes == "accy.group") return group(v);
    const std::string mx4 = after("accy.mx4.");
    if (mx4 == "codes" || mx4 == "scales") return operands(1), mx4_quantize(v);
    if (mx4 == "values") return operands(2), mx4_values(v);
    if (mx4 == "contract") return operands(4), mx4_contract(v);
    if (mx4 == "cache_write") return operands(4), mx4_cache_write(v);
    if (mx4 == "cache_keys" || mx4 == "cache_values") return operands(2), mx4_cache_read(v);
    if (mx4 == "attend" || mx4 == "attend_shared") return operands(4), mx4_attend(v);
    if (heads(v)) return;
    const std::string pages = after("accy.pages.");
    if (pages == "copy") return operands(3), pages_copy(v);
    if (pages.compare(0, 5, "fork_") == 0) return operands(4), pages_fork(v);
    if (pages.compare(0, 8, "compact_") == 0) return operands(3), pages_compact(v);
    const std::string logits = after("accy.logits.");
    if (logits == "grad") return operands(4), logits_grad(v);
    if (logits == "token" || logits == "entropy" || logits == "top" || logits == "top_tokens") return operands(2), logits_log_probs(v);
  }
  fail(Err::Unsupported, "custom_call " + op.bytes + " version " + std::to_string(op.index) + " is not supported by the HIP target");
}

// A group is no value: nothing but another custom call may read it.
void Planner::group(uint32_t v) {
  const Op& op = g_.ops[v];
  require(!is_output_[v], op, "a group is no output");
  for (const uint32_t u : users_[v]) require(g_.ops[u].kind == Kind::custom_call, op, "a group is an operand of custom calls only");
  done_[v] = true;
}

std::vector<uint32_t> Planner::grouped(const Op& op, uint32_t a, size_t least, size_t most) const {
  const Op& group = g_.ops[a];
  require(group.kind == Kind::custom_call && group.bytes == "accy.group" && group.index == 1 && group.args.size() >= least && group.args.size() <= most, op,
          "a group of " + num((int64_t)least) + (most > least ? " to " + num((int64_t)most) : "") + " operands");
  return group.args;
}

// The live calls of one set with v's operands (v among them) that `fits` takes, each name once: name -> operation. They are one kernel's. `fits` sees
// them in order, v first.
std::map<std::string, uint32_t> Planner::siblings(uint32_t v, const std::string& prefix, const std::string& suffix, const std::function<bool(const Op&)>& fits) const {
  const Op& op = g_.ops[v];
  std::map<std::string, uint32_t> found;
  for (uint32_t u = v; u < g_.ops.size(); ++u) {
    const Op& uo = g_.ops[u];
    if (!live_[u] || done_[u] || uo.kind != Kind::custom_call || uo.index != 1 || uo.args != op.args) continue;
    if (uo.bytes.size() < prefix.size() + suffix.size() || uo.bytes.compare(0, prefix.size(), prefix) != 0) continue;
    if (uo.bytes.compare(uo.bytes.size() - suffix.size(), suffix.size(), suffix) != 0) continue;
    if (fits && !fits(uo)) continue;
    found.emplace(uo.bytes.substr(prefix.size(), uo.bytes.size() - prefix.size() - suffix.size()), u);
  }
  return found;
}

uint32_t Planner::dense_source(uint32_t v) const {
  while (g_.ops[v].kind == Kind::reshape && slots_.slot_of[v] < 0) v = g_.ops[v].args[0];
  return v;
}

int Planner::dense_slot(uint32_t v) { return materialize(dense_source(v)); }

std::vector<bool> Planner::opaque_caches() const {
  auto call = [](const Op& op, const char* name) { return op.kind == Kind::custom_call && op.bytes == std::string("accy.") + name; };
  std::vector<bool> opaque(g_.ops.size());
  for (size_t v = 0; v < g_.ops.size(); ++v) {
    const Op& op = g_.ops[v];
    opaque[v] = op.kind == Kind::parameter || op.kind == Kind::scan || op.kind == Kind::projection || call(op, "mx4.cache_write") || call(op, "pages.copy");
    for (size_t i = 0; i < op.args.size(); ++i) {
      const bool cache = (i == 0 && (call(op, "mx4.cache_write") || call(op, "mx4.cache_keys") || call(op, "mx4.cache_values") || call(op, "pages.copy"))) ||
                         (i == 1 && (call(op, "mx4.attend") || call(op, "mx4.attend_shared")));
      if (!cache && op.kind != Kind::scan && op.kind != Kind::projection) opaque[op.args[i]] = false;
    }
  }
  return opaque;
}

void Planner::mark_custom_operands() {
  for (uint32_t v = 0; v < g_.ops.size(); ++v) {
    const Op& op = g_.ops[v];
    if (!live_[v] || op.kind != Kind::custom_call) continue;
    // A quantised tensor is evaluated inside the kernel that quantises it.
    if (op.args.size() == 1) continue;
    for (uint32_t a : op.args) {
      const uint32_t s = dense_source(a);
      // (scalar constants, an eps or the size of a page, are read when the call is planned)
      if (is_inlinable(g_.ops[s].kind) && !(g_.ops[s].kind == Kind::constant && g_.ops[s].result.rank() == 0)) needed_[s] = true;
    }
  }
}

// The cache's own buffer may be the result's where the caller hands it in, gets it back, and nothing else of the program
// reads what was in it; else the whole cache is copied first. A result that only another update reads is that one's buffer already. Returns the
// result's slot.
int Planner::updated_cache(uint32_t v) {
  const Op& op = g_.ops[v];
  uint32_t end = v;
  while (!is_output_[end] && users_[end].size() == 1) {
    const uint32_t u = users_[end][0];
    const Op& uo = g_.ops[u];
    const bool update = uo.kind == Kind::custom_call && uo.index == 1 && (uo.bytes == "accy.mx4.cache_write" || uo.bytes == "accy.pages.copy");
    if (!update || uo.args.empty() || uo.args[0] != end || !(uo.result == op.result)) break;
    end = u;
  }
  if (end != v && slots_.slot_of[v] < 0) slots_.slot_of[v] = temp_slot(end);
  const int old = dense_slot(op.args[0]), out = temp_slot(v);
  if (old == out) return out;
  Step copy;
  copy.type = Step::Copy;
  copy.copy.src = old;
  copy.copy.dst = out;
  copy.copy.bytes = op.result.bytes();
  copy.copy.unless_same = true;
  if (copy.copy.bytes) plan_.steps.push_back(copy);
  const SlotInfo &from = plan_.slots[(size_t)old], &to = plan_.slots[(size_t)out];
  if (from.role == SlotInfo::Input && to.role == SlotInfo::Output && g_.ops[op.args[0]].kind == Kind::parameter &&
      users_[op.args[0]].size() == 1 && !is_output_[op.args[0]])
    plan_.updates.push_back({(size_t)from.io_index, (size_t)to.io_index});
  return out;
}

}  // namespace planning
}  // namespace accy
