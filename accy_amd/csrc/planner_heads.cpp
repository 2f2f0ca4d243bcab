// Custom calls on the heads of queries and keys (kernels/heads.h), "accy.heads.<name>" or "accy.heads.<name>_neighbours":
//
//   queries, keys(q, k, rotation, (norm))             as attention takes them, planned as one kernel
//   d_queries, d_keys, d_query_gain, d_key_gain(group(dq, dk), group(q, k), rotation, (norm))
//
// rotation: group(positions, frequencies, (axes)); norm: group(query gain, key gain, eps). q [token .., head, dim], k [token .., kv_head,
// dim] of bf16, f16 or f32.
#include "planner_custom.hpp"

namespace accy {
namespace planning {

bool Planner::heads(uint32_t v) {
  const Op& op = g_.ops[v];
  const std::string prefix = "accy.heads.", tail = "_neighbours";
  if (op.bytes.compare(0, prefix.size(), prefix) != 0) return false;
  std::string what = op.bytes.substr(prefix.size());
  const bool neighbours = what.size() > tail.size() && what.compare(what.size() - tail.size(), tail.size(), tail) == 0;
  if (neighbours) what.resize(what.size() - tail.size());
  const bool grad = what == "d_queries" || what == "d_keys" || what == "d_query_gain" || what == "d_key_gain";
  if (!grad && what != "queries" && what != "keys") return false;
  require(op.args.size() == 3 || op.args.size() == 4, op, "3 or 4 operands");
  const bool norm = op.args.size() == 4;
  std::vector<uint32_t> d, x;
  if (grad) {
    d = grouped(op, op.args[0], 2, 2);
    x = grouped(op, op.args[1], 2, 2);
  } else {
    x = {op.args[0], op.args[1]};
  }
  const std::vector<uint32_t> rotation = grouped(op, op.args[2], 2, 3), norms = norm ? grouped(op, op.args[3], 3, 3) : std::vector<uint32_t>();
  const Type &qt = g_.type(x[0]), &kt = g_.type(x[1]), &pt = g_.type(rotation[0]), &ft = g_.type(rotation[1]);
  const int dt = element_type(op, qt.dtype);
  require(qt.rank() >= 2 && kt.rank() == qt.rank() && kt.dtype == qt.dtype && last(kt) == last(qt), op, "queries and keys of one type are [token .., head, dim]");
  const size_t lead = qt.rank() - 2;
  for (size_t i = 0; i < lead; ++i) require(qt.dims[i].extent == kt.dims[i].extent, op, "queries and keys of the same tokens");
  auto like = [](const Type& a, const Type& b) {
    if (a.dtype != b.dtype || !same_rows(a, b) || last(a) != last(b)) return false;
    return true;
  };
  if (grad) require(like(g_.type(d[0]), qt) && like(g_.type(d[1]), kt), op, "gradients of the results' types");
  const int64_t D = last(qt), F = ft.rank() == 1 ? ft.dims[0].extent : 0;
  require(D >= 2 && D <= 512, op, "2 to 512 dims");
  require(ft.dtype == DType::f32 && F >= 1 && 2 * F <= D, op, "frequencies are f32 [pair], one to dim / 2");
  const bool several = rotation.size() == 3;
  require(pt.dtype == DType::i32 && pt.rank() == lead + (several ? 1 : 0), op, "positions are i32 [token ..], with axes [token .., axis]");
  for (size_t i = 0; i < lead; ++i) require(pt.dims[i].extent == qt.dims[i].extent, op, "a position for every token");
  if (several) {
    const Type& at = g_.type(rotation[2]);
    require(at.dtype == DType::i32 && at.rank() == 1 && at.dims[0].extent == F, op, "axes are i32 [pair]");
    require(last(pt) < (int64_t(1) << 31), op, "2^31 axes or more");
  }
  int gt = dt;
  double eps = 0;
  if (norm) {
    const Type &a = g_.type(norms[0]), &b = g_.type(norms[1]);
    gt = element_type(op, a.dtype);
    require(a.dtype == b.dtype && (a.dtype == qt.dtype || a.dtype == DType::f32), op, "gains of the heads' type or f32");
    require(a.rank() == 1 && b.rank() == 1 && last(a) == D && last(b) == D, op, "gains are [dim]");
    require(g_.type(norms[2]).dtype == DType::f32 && splat_float(norms[2], eps), op, "eps is an f32 constant");
  }
  // The calls with these operands, checked each: one kernel stores what all of them ask for.
  const auto calls = siblings(v, prefix, neighbours ? tail : "");
  int out[4] = {-1, -1, -1, -1};
  const char* const names[] = {grad ? "d_queries" : "queries", grad ? "d_keys" : "keys", "d_query_gain", "d_key_gain"};
  std::vector<uint32_t> made;
  for (int i = 0; i < (grad ? 4 : 2); ++i) {
    const auto call = calls.find(names[i]);
    if (call == calls.end()) continue;
    const Op& uo = g_.ops[call->second];
    if (i >= 2) require(norm, uo, "there is no gain without a norm");
    require(like(uo.result, i == 0 ? qt : i == 1 ? kt : g_.type(norms[(size_t)i - 2])), uo, "the result has its operand's type");
    out[i] = temp_slot(call->second);
    made.push_back(call->second);
  }
  const uint64_t tokens = prod(qt.dims, 0, lead), hq = (uint64_t)qt.dims[lead].extent, hk = (uint64_t)kt.dims[lead].extent;
  const bool sums = out[2] >= 0 || out[3] >= 0;
  require(hq < (1u << 20) && hk < (1u << 20), op, "2^20 heads or more");
  // Without an element nothing is left but sums of nothing.
  const bool empty = tokens == 0 || (hq == 0 && hk == 0);
  if (!empty || sums) {
    // W: as many dims as a lane takes at once, up to 16 bytes.
    int64_t W = qt.dtype == DType::f32 ? 4 : 8;
    while (D % W || F % W) W /= 2;
    const int64_t units = F / W + (D - 2 * F + 2 * W - 1) / (2 * W);
    int64_t lanes = 1;
    while (lanes < 64 && lanes < units) lanes *= 2;
    // Tokens of a workgroup's tile: more than one while tiles are left for every CU, the tile's rows are no more than a few rounds of the workgroup's
    // lanes, and the tile's cosines and sines fit 16 KB. The gradient's workgroups, two to a CU, walk over the tiles (us, tiles at least / rounds / workgroups:
    // 4001 x 15 heads of 96 f32 2048 / 4 / 1024 22.5, 1024 / 4 / 512 23.0, 512 / 8 / 512 20.2, 8192 x 20 x 128 bf16 36.3, 32.8, 31.3, 16000 x 5 x 256
    // bf16 40.7, 34.6, 32.9); without it 1024 / 4, 2048 / 4, 1024 / 8 and 512 / 8 are within 2 % for 8192 x 32 x 128 bf16, 27.3, and 3000 x 32 x 80
    // f32 takes 12.6, 13.9, 12.7, 13.0.
    const int64_t rows = (int64_t)(out[0] >= 0 || grad ? hq : 0) + (int64_t)(out[1] >= 0 || grad ? hk : 0);
    const uint64_t least = grad ? 512 : 1024;
    int64_t tt = 1;
    while (tt < 16 && tokens / (uint64_t)(2 * tt) >= least && 2 * tt * F * 8 <= 16384 && tt * rows < (grad ? 8 : 4) * 256 / lanes) tt *= 2;
    const uint64_t tiles = (tokens + (uint64_t)tt - 1) / (uint64_t)tt;
    const uint64_t groups = grad ? std::max<uint64_t>(1, std::min<uint64_t>(tiles, 512)) : tiles;
    require(launchable(groups, 256), op, "more workgroups than a launch takes");
    const std::string nm = name(grad ? "heads_grad" : "heads", v);
    char e[64];
    std::snprintf(e, sizeof e, "%af", eps);
    std::string eps_text = e;
    if (!std::isfinite(eps)) refuse(op, "eps is a number");
    const std::string head = "#include \"heads\"\nstruct Cfg_" + nm + " {\n  static constexpr int DT = " + num(dt) + ", GT = " + num(gt) + ", D = " + num(D) + ", F = " +
                             num(F) + ", HQ = " + num(grad || out[0] >= 0 ? (int64_t)hq : 0) + ", HK = " + num(grad || out[1] >= 0 ? (int64_t)hk : 0) +
                             ", AXES = " + num(several ? std::max<int64_t>(1, last(pt)) : 0) + ", W = " + num(W) + ", LANES = " + num(lanes) + ", TT = " + num(tt) +
                             ";\n  static constexpr bool NEIGHBOURS = " + (neighbours ? "true" : "false") + ", NORM = " + (norm ? "true" : "false")  +
                             ";\n  static constexpr long TOKENS = " + std::to_string(tokens) + ";\n  static constexpr float EPS = " + eps_text + ";\n};\n";
    require(!several || last(pt) > 0 || tokens == 0, op, "positions without an axis");
    KernelWriter w(g_, slots_, "i64_t");
    std::string args;
    auto read = [&](uint32_t a) { args += w.arg(dense_slot(a), false) + ", "; };
    auto none = [&] { args += "nullptr, "; };
    for (const uint32_t a : d) read(a);
    for (const uint32_t a : x) read(a);
    read(rotation[0]);
    read(rotation[1]);
    if (several) read(rotation[2]);
    else none();
    for (int i = 0; i < 2; ++i) {
      if (norm) read(norms[(size_t)i]);
      else none();
    }
    for (int i = 0; i < 2; ++i) args += (out[i] >= 0 ? w.arg(out[i], true) : std::string("nullptr")) + (i == 0 || grad ? ", " : "");
    int part = -1;
    if (grad) {
      if (sums) part = slots_.add(SlotInfo::Temp, -1, DType::f32, groups * 2 * (uint64_t)D * 4);
      args += sums ? w.arg(part, true) : "nullptr";
    }
    KernelStep k;
    k.source = head + "extern \"C\" __global__ void __launch_bounds__(256) " + nm + "(" + w.params() + ") {\n  accy::heads::" + (grad ? "rotate_grad" : "rotate") +
               "<Cfg_" + nm + ">(" + args + ");\n}\n";
    k.name = nm;
    k.grid[0] = (uint32_t)groups;
    k.block[0] = 256;
    k.klass = "heads";
    k.label = std::string(grad ? "heads_grad:%" : "heads:%") + std::to_string(v);
    push(std::move(k), w);
    if (sums) {
      KernelWriter sw(g_, slots_, "i64_t");
      const std::string p = sw.arg(part, false), a = out[2] >= 0 ? sw.arg(out[2], true) : "nullptr", b = out[3] >= 0 ? sw.arg(out[3], true) : "nullptr";
      KernelStep s;
      s.name = name("heads_gain", v);
      s.source = head + "extern \"C\" __global__ void __launch_bounds__(1024) " + s.name + "(" + sw.params() + ") {\n  accy::heads::gain_sums<Cfg_" + nm + ", " +
                 std::to_string(groups) + ">(" + p + ", " + a + ", " + b + ");\n}\n";
      s.grid[0] = (uint32_t)((D + 31) / 32);
      s.grid[1] = 2;
      s.block[0] = 1024;
      s.klass = "heads";
      s.label = "heads_gain:%" + std::to_string(v);
      push(std::move(s), sw);
    }
  }
  for (const uint32_t u : made) finish(u);
  return true;
}

}  // namespace planning
}  // namespace accy
