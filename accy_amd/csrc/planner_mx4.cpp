// Custom calls of this target: microscaled 4-bit floats (kernels/mx4.h, mx4_contract.h). A program names them "accy.mx4.<name>", version 1:
//
//   codes(x), scales(x)                    x [.., K] -> u8 [.., K / 2] and u8 [.., K / 32], planned as one kernel
//   values(codes, scales)                  -> [.., K]
//   contract(codes, scales, codes, scales) [rows .., K / 2] .. and [columns .., K / 2] .. -> [rows .., columns ..]
//   cache_write(cache, keys, values, slots) -> the cache with the rows of the tokens' slots replaced
//   cache_keys(cache, slots), cache_values  -> [slots .., kv_head, dim]
//   attend(q, cache, pages, lengths)        q [seq, (query,) head, dim] -> the same
//
// Float operands and results are bf16, f16 or f32. The wire carries a custom call's result type, so everything about it is
// checked here.
#include "planner_internal.hpp"

namespace accy {
namespace planning {

namespace {

[[noreturn]] void refuse(const Op& op, const std::string& why) {
  fail(Err::Unsupported, "custom_call " + op.bytes + ": " + why);
}

void require(bool ok, const Op& op, const std::string& why) {
  if (!ok) refuse(op, why);
}

// DT of kernels/mx4.h.
int element_type(const Op& op, DType d) {
  switch (d) {
    case DType::bf16: return 0;
    case DType::f16: return 1;
    case DType::f32: return 2;
    default: refuse(op, std::string(dtype_name(d)) + " values (bf16, f16 or f32)");
  }
}

int64_t last(const Type& t) { return t.rank() ? t.dims.back().extent : 0; }

// The extents of a's leading axes are b's.
bool same_rows(const Type& a, const Type& b) {
  if (a.rank() != b.rank()) return false;
  for (size_t i = 0; i + 1 < a.rank(); ++i)
    if (a.dims[i].extent != b.dims[i].extent) return false;
  return true;
}

// Codes and scales of one tensor: the elements along its blocked axis.
int64_t blocked(const Op& op, const Type& codes, const Type& scales) {
  require(codes.dtype == DType::u8 && scales.dtype == DType::u8, op, "codes and scales are u8");
  require(codes.rank() >= 1 && same_rows(codes, scales), op, "codes and scales of different rows");
  const int64_t k = last(codes) * 2;
  require(k % 32 == 0 && last(scales) == k / 32, op, "K / 2 codes and K / 32 scales to a row, K a multiple of 32");
  return k;
}

std::string num(int64_t n) { return std::to_string(n); }

}  // namespace

void Planner::custom(uint32_t v) {
  const Op& op = g_.ops[v];
  const std::string prefix = "accy.mx4.";
  const std::string what = op.bytes.compare(0, prefix.size(), prefix) == 0 ? op.bytes.substr(prefix.size()) : "";
  auto operands = [&](size_t n) { require(op.args.size() == n, op, num((int64_t)n) + " operands"); };
  if (op.index == 1) {
    if (what == "codes" || what == "scales") return operands(1), mx4_quantize(v);
    if (what == "values") return operands(2), mx4_values(v);
    if (what == "contract") return operands(4), mx4_contract(v);
    if (what == "cache_write") return operands(4), mx4_cache_write(v);
    if (what == "cache_keys" || what == "cache_values") return operands(2), mx4_cache_read(v);
    if (what == "attend") return operands(4), mx4_attend(v);
  }
  fail(Err::Unsupported, "custom_call " + op.bytes + " version " + std::to_string(op.index) + " is not supported by the HIP target");
}

uint32_t Planner::dense_source(uint32_t v) const {
  while (g_.ops[v].kind == Kind::reshape && slots_.slot_of[v] < 0) v = g_.ops[v].args[0];
  return v;
}

int Planner::dense_slot(uint32_t v) { return materialize(dense_source(v)); }

std::vector<bool> Planner::opaque_caches() const {
  auto call = [](const Op& op, const char* name) { return op.kind == Kind::custom_call && op.bytes == std::string("accy.mx4.") + name; };
  std::vector<bool> opaque(g_.ops.size());
  for (size_t v = 0; v < g_.ops.size(); ++v) {
    const Op& op = g_.ops[v];
    opaque[v] = op.kind == Kind::parameter || op.kind == Kind::scan || op.kind == Kind::projection || call(op, "cache_write");
    for (size_t i = 0; i < op.args.size(); ++i) {
      const bool cache = (i == 0 && (call(op, "cache_write") || call(op, "cache_keys") || call(op, "cache_values"))) || (i == 1 && call(op, "attend"));
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
      if (is_inlinable(g_.ops[s].kind)) needed_[s] = true;
    }
  }
}

// ---- codes and scales: eight values per thread, four lanes to a block ----

void Planner::mx4_quantize(uint32_t v) {
  const Op& op = g_.ops[v];
  const uint32_t x = op.args[0];
  const Type& t = g_.type(x);
  element_type(op, t.dtype);
  const int64_t K = last(t);
  require(t.rank() >= 1 && K % 32 == 0, op, "the last axis is a multiple of 32");
  // codes, scales: the first of each
  bool have[2] = {false, false};
  uint32_t id[2] = {0, 0};
  std::vector<uint32_t> made;
  for (uint32_t u = v; u < g_.ops.size(); ++u) {
    const Op& uo = g_.ops[u];
    if (!live_[u] || done_[u] || uo.kind != Kind::custom_call || uo.index != 1 || uo.args != op.args) continue;
    const bool is_codes = uo.bytes == "accy.mx4.codes";
    if (!is_codes && uo.bytes != "accy.mx4.scales") continue;
    if (have[!is_codes]) continue;
    require(uo.result.dtype == DType::u8 && same_rows(uo.result, t) && last(uo.result) == K / (is_codes ? 2 : 32), uo,
            is_codes ? "u8 codes, K / 2 to a row" : "u8 scales, K / 32 to a row");
    have[!is_codes] = true;
    id[!is_codes] = u;
    made.push_back(u);
  }
  // Their values, where the program reads them back, are stored by the same kernel; what only they read is not stored.
  std::vector<std::pair<int, uint32_t>> values;  // element type, operation
  for (uint32_t u = v; have[0] && have[1] && u < g_.ops.size(); ++u) {
    const Op& uo = g_.ops[u];
    if (!live_[u] || done_[u] || uo.kind != Kind::custom_call || uo.index != 1 || uo.bytes != "accy.mx4.values") continue;
    if (uo.args.size() != 2 || uo.args[0] != id[0] || uo.args[1] != id[1]) continue;
    require(same_rows(uo.result, t) && last(uo.result) == K, uo, "the result has the codes' rows and two values for each of their bytes");
    values.push_back({element_type(uo, uo.result.dtype), u});
  }
  auto stored = [&](int which) {
    if (!have[which]) return false;
    if (values.empty() || is_output_[id[which]]) return true;
    for (const uint32_t u : users_[id[which]])
      if (std::none_of(values.begin(), values.end(), [&](const std::pair<int, uint32_t>& x) { return x.second == u; })) return true;
    return false;
  };
  const int codes = stored(0) ? temp_slot(id[0]) : -1, scales = stored(1) ? temp_slot(id[1]) : -1;
  std::vector<int> value_slots;
  for (const auto& x : values) {
    value_slots.push_back(temp_slot(x.second));
    made.push_back(x.second);
  }
  const uint64_t nel = t.elements();
  if (nel) {
    // A thread takes eight values of a workgroup's 2048, next to each other where they are 16 bits wide, else four and, 1024 further on,
    // four more: 16 bytes a lane and whole lines a wave (8192 x 8192 f32 with its values: 91 us, and eight together 110).
    bool apart = t.dtype == DType::f32;
    for (const auto& x : values) apart |= x.first == 2;
    KernelWriter w(g_, slots_, itype(nel));
    std::vector<Dim> outer(t.dims.begin(), t.dims.end() - 1);
    std::ostringstream body;
    for (int half = 0; half < 2; ++half) {
      // Four elements at a time: a leaf read at `rest + c` is one load for the four, non-temporal when this kernel reads each
      // of its elements once.
      const std::string at = !half ? "i0" : apart ? "i1" : "(i0 + 4)";
      std::vector<std::string> coords =
          outer.empty() ? std::vector<std::string>{} : delinearize(std::string("(") + (half && apart ? "i1" : "i0") + " / " + num(K) + ")", outer);
      coords.push_back("c");
      std::string hoisted;
      std::map<std::string, std::string> hoisted_var;
      w.leaf_hook = [&](int s, const std::string& off, DType d, Scope& sc, std::string& out) -> bool {
        std::optional<std::string> base = quad_base(off);
        if (!base) return false;
        const std::string key = num(s) + "|" + off;
        auto hv = hoisted_var.find(key);
        if (hv == hoisted_var.end()) {
          const std::string q = "q" + std::to_string(hoisted_var.size());
          const bool once = plan_.slots[(size_t)s].bytes / dtype_size(d) == nel;
          hoisted += "      " + w.quad_load(s, q, *base, d, once) + "\n";
          hv = hoisted_var.emplace(key, q).first;
        }
        out = w.tmp();
        sc.out << sc.indent << "const " << compute_type(d) << " " << out << " = " << KernelWriter::quad_elem(hv->second, "u", d) << ";\n";
        return true;
      };
      std::ostringstream inner;
      Scope sc(inner, "        ");
      const std::string e = w.value(x, coords, sc);
      body << "    {\n      const I c0 = " << (outer.empty() ? at : at + " % " + num(K)) << ";\n"
           << hoisted << "#pragma unroll\n      for (int u = 0; u < 4; ++u) {\n        const I c = c0 + u;\n"
           << inner.str() << "        " << (apart ? "x[" + num(half) + "][u]" : "x[" + num(4 * half) + " + u]") << " = " << e << ";\n      }\n    }\n";
    }
    w.leaf_hook = nullptr;
    // x's codes, scale and values at element i
    auto store = [&](const std::string& x, const std::string& i) {
      const std::string v = apart ? "4" : "8";
      std::string o = "      const u32_t scale = accy::mx4::block_scale(" + x + "), codes = accy::mx4::encode" + v + "(" + x + ", scale);\n";
      if (codes >= 0) o += "      *(" + std::string(apart ? "u16_t" : "u32_t") + "*)(" + w.arg(codes, true) + " + " + i + " / 2) = codes;\n";
      if (scales >= 0) o += "      if (" + i + " % 32 == 0) " + w.arg(scales, true) + "[" + i + " / 32] = (u8_t)scale;\n";
      if (!values.empty()) o += "      accy::mx4::decode" + v + "(codes, scale, " + x + ");\n";
      for (size_t k = 0; k < values.size(); ++k)
        o += "      accy::mx4::store" + v + "<" + num(values[k].first) + ">(" + w.arg(value_slots[k], true) + " + " + i + ", " + x + ");\n";
      return "    {\n" + o + "    }\n";
    };
    const std::string nm = name("mx4_quantize", v), n = "(I)" + std::to_string(nel);
    std::string loop;
    if (apart) {
      // whole blocks (eight lanes) pass the end or do not
      const bool whole = nel % 2048 == 0;
      loop = "  for (I i0 = (I)blockIdx.x * 2048 + (I)threadIdx.x * 4; i0 < " + n + "; i0 += (I)gridDim.x * 2048) {\n    const I i1 = " +
             (whole ? "i0 + 1024" : "i0 + 1024 < " + n + " ? i0 + 1024 : i0") + ";\n    float x[2][4];\n" + body.str() + store("x[0]", "i0") +
             (whole ? "" : "    if (i1 != i0)\n") + store("x[1]", "i1");
    } else {
      loop = "  for (I i0 = ((I)blockIdx.x * 256 + (I)threadIdx.x) * 8; i0 < " + n + "; i0 += (I)gridDim.x * 2048) {\n    float x[8];\n" + body.str() +
             store("x", "i0");
    }
    std::ostringstream src;
    src << "#include \"mx4\"\n"
        << "extern \"C\" __global__ void __launch_bounds__(256) " << nm << "(" << w.params() << ") {\n  typedef " << w.itype << " I;\n"
        << w.align_hints() << loop << "  }\n}\n";
    KernelStep k;
    k.source = src.str();
    k.name = nm;
    k.grid[0] = grid_for(nel / 8, 256);
    k.block[0] = 256;
    k.klass = "quantize";
    k.label = "quantize:%" + std::to_string(v);
    push(std::move(k), w);
  }
  for (uint32_t u : made) finish(u);
}

void Planner::mx4_values(uint32_t v) {
  const Op& op = g_.ops[v];
  const Type& c = g_.type(op.args[0]);
  const int64_t K = blocked(op, c, g_.type(op.args[1]));
  const int dt = element_type(op, op.result.dtype);
  require(same_rows(op.result, c) && last(op.result) == K, op, "the result has the codes' rows and two values for each of their bytes");
  const uint64_t nel = op.result.elements();
  const int out = temp_slot(v);
  if (nel) {
    const int cs = dense_slot(op.args[0]), ss = dense_slot(op.args[1]);
    KernelWriter w(g_, slots_, itype(nel));
    const std::string a = w.arg(cs, false), b = w.arg(ss, false), o = w.arg(out, true), nm = name("mx4_values", v);
    KernelStep k;
    k.source = "#include \"mx4\"\nextern \"C\" __global__ void __launch_bounds__(256) " + nm + "(" + w.params() + ") {\n  accy::mx4::values<" +
               num(dt) + ", " + w.itype + ", " + std::to_string(nel) + ">(" + a + ", " + b + ", " + o + ");\n}\n";
    k.name = nm;
    k.grid[0] = grid_for(nel / 8, 256);
    k.block[0] = 256;
    k.klass = "quantize";
    k.label = "values:%" + std::to_string(v);
    push(std::move(k), w);
  }
  finish(v);
}

// ---- products ----

void Planner::mx4_contract(uint32_t v) {
  const Op& op = g_.ops[v];
  const Type &at = g_.type(op.args[0]), &bt = g_.type(op.args[2]), &rt = op.result;
  const int64_t K = blocked(op, at, g_.type(op.args[1]));
  require(blocked(op, bt, g_.type(op.args[3])) == K, op, "operands of different K");
  require(K > 0, op, "an empty contraction");
  const DType d = rt.dtype;
  const int dt = element_type(op, d);
  const size_t ra = at.rank() - 1, rb = bt.rank() - 1;
  bool shape = rt.rank() == ra + rb;
  for (size_t i = 0; shape && i < rt.rank(); ++i) shape = rt.dims[i].extent == (i < ra ? at.dims[i] : bt.dims[i - ra]).extent;
  require(shape, op, "the result has the rows of the first operand and then those of the second");
  const int64_t M = (int64_t)prod(at.dims, 0, ra), N = (int64_t)prod(bt.dims, 0, rb);
  if (M == 0 || N == 0) {
    temp_slot(v);
    finish(v);
    return;
  }
  int as = dense_slot(op.args[0]), ss = dense_slot(op.args[1]), bs = dense_slot(op.args[2]), ts = dense_slot(op.args[3]);
  const std::string nm = name("mx4_contract", v), cidx = "m * " + num(N) + "L + n";
  const Mx4Tile tile = mx4_tile(M, N, K);
  const bool split = tile.splits > 1;
  require(tile.bm > 0, op, "more tiles than a launch takes");
  if (!tile.wk && K % 128 != 0) {
    // the tiles read scales a whole step at a time
    const int64_t steps = (K + 127) / 128;
    const int pa = slots_.add(SlotInfo::Temp, -1, DType::u32, (uint64_t)(M * steps) * 4);
    const int pb = slots_.add(SlotInfo::Temp, -1, DType::u32, (uint64_t)(N * steps) * 4);
    KernelWriter w(g_, slots_, "i64_t");
    const std::string a = w.arg(ss, false), b = w.arg(ts, false), x = w.arg(pa, true), y = w.arg(pb, true);
    KernelStep k;
    k.name = name("mx4_pad", v);
    k.source = "#include \"gemm\"\n#include \"mx4\"\n#include \"mx4_contract\"\nstruct Cfg_" + nm + " {\n  static constexpr long M = " + num(M) + ", N = " +
               num(N) + ", K = " + num(K) + ";\n};\nextern \"C\" __global__ void __launch_bounds__(256) " + k.name + "(" + w.params() +
               ") {\n  accy::mx4::pad_scales<Cfg_" + nm + ">(" + a + ", " + b + ", " + x + ", " + y + ");\n}\n";
    k.grid[0] = grid_for((uint64_t)(std::max(M, N) * steps), 256);
    k.grid[1] = 2;
    k.block[0] = 256;
    k.klass = "gemm";
    k.label = "mx4_pad:%" + std::to_string(v);
    push(std::move(k), w);
    ss = pa;
    ts = pb;
  }
  // The kernel that stores the results (the product's own, or the sum of its splits) and what it reads.
  std::unique_ptr<KernelWriter> w;
  auto operands = [&](KernelWriter& k) {
    std::string call;
    for (int s : {as, ss, bs, ts}) call += "(const u8_t*)" + k.arg(s, false) + ", ";
    return call;
  };
  uint32_t target = v;
  std::ostringstream epi;
  // As for every contraction: an elementwise region that ends in one value is the epilogue (see planner_contraction.cpp).
  if (epilogue_target(v, target)) {
    try {
      w.reset(new KernelWriter(g_, slots_, "i64_t"));
      if (!split) operands(*w);
      std::vector<std::string> coords = delinearize("m", std::vector<Dim>(rt.dims.begin(), rt.dims.begin() + (long)ra));
      for (auto& c : delinearize("n", std::vector<Dim>(rt.dims.begin() + (long)ra, rt.dims.end()))) coords.push_back(c);
      w->provide = [&](uint32_t vid, const std::vector<std::string>& c, std::string& out) -> bool {
        if (vid != v) return false;
        if (c != coords) throw NotFusable("contraction value read at another index");
        out = "vv";
        return true;
      };
      Scope sc(epi, "    ");
      const std::string x = w->value(target, coords, sc);
      epi << "    " << w->store(temp_slot(target), cidx, g_.type(target).dtype, x) << "\n";
    } catch (const NotFusable&) {
      target = v;
      w.reset();
      epi.str("");
    }
  }
  if (!w) {
    w.reset(new KernelWriter(g_, slots_, "i64_t"));
    if (!split) operands(*w);
    epi << "    " << w->arg(temp_slot(v), true) << "[" << cidx << "] = accy::mx4::to_elem<" << dt << ">(v);\n";
  }
  const KernelWriter::Members members = w->members();
  const std::string rounded = target != v ? "    const float vv = accy::mx4::rounded<" + num(dt) + ">(v);\n" : "";
  std::ostringstream head;
  head << "#include \"gemm\"\n#include \"mx4\"\n#include \"mx4_contract\"\nstruct Epi_" << nm << " {\n" << members.decls
       << "  __device__ __forceinline__ void operator()(long, long m, long n, float v) const {\n" << rounded << epi.str() << "  }\n};\n"
       << "struct Cfg_" << nm << " {\n  static constexpr long BATCH = 1, M = " << M << ", N = " << N << ", K = " << K << ";\n"
       << "  static constexpr int BM = " << tile.bm << ", BN = " << tile.bn << ", GROUP_M = " << (M > N ? 4 : 8) << ", WK = " << tile.wk
       << ", SPLITS = " << tile.splits << ";\n};\n";
  const std::string own = "Epi_" + nm + "{" + members.inits + "}";
  KernelWriter pw(g_, slots_, "i64_t");
  std::string functor = own, partial_struct;
  KernelWriter& kw = split ? pw : *w;
  const std::string args = operands(kw);
  int part = -1;
  if (split) {
    part = slots_.add(SlotInfo::Temp, -1, DType::f32, (uint64_t)tile.splits * (uint64_t)(M * N) * 4);
    functor = "Part_" + nm + "{" + pw.arg(part, true) + "}";
    partial_struct = "struct Part_" + nm + " {\n  float* __restrict__ p;\n  __device__ __forceinline__ void operator()(long, long m, long n, float v) const {\n    p[blockIdx.z * " +
                     num(M * N) + "L + " + cidx + "] = v;\n  }\n};\n";
  }
  KernelStep k;
  k.block[0] = tile.wk ? 64u * (uint32_t)tile.wk : 256u;
  k.source = head.str() + partial_struct + "extern \"C\" __global__ void __launch_bounds__(" + std::to_string(k.block[0]) + ") " + nm + "(" + kw.params() + ") {\n  accy::mx4::" +
             (tile.wk ? "contract_direct" : "contract_tile") + "<Cfg_" + nm + ">(" + args + functor + ");\n}\n";
  k.name = nm;
  const uint64_t groups = (uint64_t)((M + tile.bm - 1) / tile.bm) * (uint64_t)((N + tile.bn - 1) / tile.bn);
  k.grid[0] = (uint32_t)groups;
  k.grid[2] = (uint32_t)tile.splits;
  k.klass = "gemm";
  k.label = "mx4:%" + std::to_string(v) + (target != v ? "+%" + std::to_string(target) : "");
  k.algorithmic_flops = 2.0 * (double)M * (double)N * (double)K;
  push(std::move(k), kw);
  if (split) {
    KernelStep sum;
    sum.name = name("mx4_sum", v);
    const std::string p = w->arg(part, false);
    sum.source = head.str() + "extern \"C\" __global__ void __launch_bounds__(256) " + sum.name + "(" + w->params() + ") {\n  accy::split::sum<Cfg_" + nm +
                 ">(" + p + ", " + own + ");\n}\n";
    sum.grid[0] = grid_for((uint64_t)(M * N), 256);
    sum.block[0] = 256;
    sum.klass = "gemm";
    sum.label = "mx4_sum:%" + std::to_string(target);
    push(std::move(sum), *w);
  }
  done_[v] = true;
  finish(target);
}

// The kernel, tile and K split of a product: the least of the times estimated for each, in us without a launch (kernels/mx4_contract.h).
// Small tiles are bound by the bytes that a CU takes, 52 KB a us and 0.1 us a workgroup; a workgroup of a large one takes a time per
// step of 128 values that grows with the workgroups at work (two of 128 x 128 to a CU, one of 256 x 256) and the time to store its results.
// Measured (us back to back, 2.4 of them a launch; 128 x 128 / 256 x 256): 512 x 8192 x 2048 8.4 / 17.0, 1024 x 8192 x 2048 16.0 /
// 19.6, 1536 x 8192 x 2048 21.8 / 21.6, 2048 x 8192 x 2048 28.3 / 24.5, 3000 x 8192 x 2048 42 / 48, 4096 x 4096 x 1024 19.4 /
// 18.1, 8192^3 377 / 276; 32 x 32 / 128 x 128: 64 x 8192 x 2048 4.6 / 6.5, 500 x 1000 x 2048 5.0 / 7.0, 200 x 1000 x 8192 7.0 / 15.8,
// 1000 x 1000 x 1024 5.3 / 5.6, 2000 x 1000 x 1024 8.7 / 6.1, 1000 x 4096 x 256 7.9 / 5.7; 128 x 128 in one / split along K (with the
// sum) / 32 x 32: 512 x 2048 x 28672 58 / 33 / 65, 256 x 2048 x 16384 31 / 16.6 / 19.7, 200 x 1000 x 28672 54 / 15.7 / 18.1.
Planner::Mx4Tile Planner::mx4_tile(int64_t M, int64_t N, int64_t K) const {
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t steps = up(K, 128), groups = up(steps, 4);
  Mx4Tile best;
  double least = 0;
  auto offer = [&](const Mx4Tile& t, double cost) {
    if (!launchable((uint64_t)(up(M, t.bm) * up(N, t.bn)), t.wk ? 64u * (unsigned)t.wk : 256u)) return;
    if (best.bm && cost >= least) return;
    best = t;
    least = cost;
  };
  // Four waves along K where their stages leave room for two workgroups on a CU or there is but one for each (1000 x 1000 x 1024 in 32 x
  // 32: four 5.3, two 5.4, one 6.2; 300 x 1000 x 16384 19.7 and 17.4). Larger tiles read less, but fewer of them do (64 x 8192 x 2048: 32 x
  // 32 4.6, 32 x 64 5.3, 64 x 64 7.1).
  const int bm = M <= 16 ? 16 : 32;
  for (const int bn : {16, 32}) {
    Mx4Tile t;
    t.bm = bm;
    t.bn = bn;
    const int64_t wgs = up(M, bm) * up(N, bn), lds = std::min<int64_t>(4, up(K, 1024)) * 4 * (bm + bn) * 128;
    t.wk = wgs > 256 && lds > 80 * 1024 ? 2 : 4;
    const double per_cu = std::max(1.0, (double)wgs / 256);
    offer(t, 0.3 + per_cu * (0.1 + (double)((bm + bn) * K) * 0.53 / 52e3));
  }
  // (a tile's scales are addressed in 32 bits)
  for (const int size : {128, 256}) {
    if (K > (int64_t(1) << 28)) continue;
    const int64_t tiles = up(M, size) * up(N, size), most = size == 128 ? 512 : 256;
    for (int splits = 1; splits <= (opt_.allow_split && size == 128 ? 8 : 1); splits *= 2) {
      if (splits > 1 && up(groups, up(groups, splits)) != splits) continue;
      const double share = (double)(splits > 1 ? up(groups, splits) * 4 : steps);
      auto round = [&](double n) {
        if (size == 128) return 0.9 + 1.8 * std::min(1.0, n / 256) + share * (0.2 + 0.5 * std::max(0.0, n - 256) / 256);
        return 1.0 + 4.0 * n / 256 + share * (0.65 + 0.4 * n / 256);
      };
      const int64_t all = tiles * splits;
      Mx4Tile t;
      t.bm = t.bn = size;
      t.splits = splits;
      offer(t, (double)(all / most) * round((double)most) + (all % most ? round((double)(all % most)) : 0.0) + (K % 128 ? 2.6 : 0.0) +
                   (splits > 1 ? 3.0 + (double)splits * (double)(M * N) * 8.0 / 4e6 : 0.0));
    }
  }
  return best;
}

// ---- the paged cache ----

Planner::Mx4Cache Planner::mx4_cache(const Op& op, uint32_t cache, int64_t heads, int64_t dim) const {
  const Type& t = g_.type(cache);
  require(t.dtype == DType::u8 && t.rank() == 3, op, "a cache is u8 [page, kv_head, bytes]");
  Mx4Cache c;
  c.pages = t.dims[0].extent;
  c.heads = t.dims[1].extent;
  c.dim = dim;
  require(c.heads == heads, op, "the cache holds " + num(c.heads) + " heads, the rows " + num(heads));
  require(dim >= 32 && dim <= 256 && dim % 32 == 0, op, "head dimensions are multiples of 32 up to 256");
  const int64_t row = dim + dim / 16, bytes = t.dims[2].extent;
  c.tokens = bytes / row;
  require(bytes % row == 0 && c.tokens > 0 && c.tokens % 32 == 0, op,
          "a page holds a multiple of 32 tokens of " + num(row) + " bytes, not " + num(bytes) + " bytes");
  require(c.tokens < (1 << 20) && c.pages < (int64_t(1) << 31) / c.tokens, op, "a cache has fewer than 2^31 slots");
  return c;
}

std::string Planner::Mx4Cache::members(DType d) const {
  return "  static constexpr int DT = " + std::string(d == DType::bf16 ? "0" : d == DType::f16 ? "1" : "2") + ", HD = " + num(dim) +
         ", H = " + num(heads) + ", T = " + num(tokens) + ", P = " + num(pages) + ";\n";
}

void Planner::mx4_cache_write(uint32_t v) {
  const Op& op = g_.ops[v];
  const Type &kt = g_.type(op.args[1]), &vt = g_.type(op.args[2]), &st = g_.type(op.args[3]);
  element_type(op, kt.dtype);
  require(kt.rank() >= 2 && kt.dtype == vt.dtype && same_rows(kt, vt) && last(kt) == last(vt), op, "keys and values of one type and shape");
  require(st.dtype == DType::i32 && st.rank() + 2 == kt.rank(), op, "an i32 slot for every token");
  for (size_t i = 0; i < st.rank(); ++i) require(st.dims[i].extent == kt.dims[i].extent, op, "an i32 slot for every token");
  const Mx4Cache c = mx4_cache(op, op.args[0], kt.dims[kt.rank() - 2].extent, last(kt));
  require(op.result == g_.type(op.args[0]), op, "the result has the cache's type");
  const int old = dense_slot(op.args[0]), out = temp_slot(v);
  Step copy;
  copy.type = Step::Copy;
  copy.copy.src = old;
  copy.copy.dst = out;
  copy.copy.bytes = op.result.bytes();
  copy.copy.unless_same = true;
  if (copy.copy.bytes) plan_.steps.push_back(copy);
  // The cache's own buffer may be the result's where the caller hands it in, gets it back, and nothing else of the program
  // reads what was in it.
  const SlotInfo &from = plan_.slots[(size_t)old], &to = plan_.slots[(size_t)out];
  if (from.role == SlotInfo::Input && to.role == SlotInfo::Output && g_.ops[op.args[0]].kind == Kind::parameter &&
      users_[op.args[0]].size() == 1 && !is_output_[op.args[0]])
    plan_.updates.push_back({(size_t)from.io_index, (size_t)to.io_index});
  const uint64_t n = st.elements();
  if (n && c.pages && c.heads) {
    const int ks = dense_slot(op.args[1]), vs = dense_slot(op.args[2]), ss = dense_slot(op.args[3]);
    require(n < (uint64_t(1) << 31), op, "2^31 tokens or more");
    // Looking through the later slots costs every workgroup a pass over the list; a table of each slot's last token two launches
    // (8 heads of 128 bf16: 1000 tokens 3.9 us by the list and 7.7 by the table, 4000 7.0 and 10.1, 8192 13.9 and 14.7, 16384 27.2 and 23.9).
    const bool owners = n > 8192;
    const std::string nm = name("mx4_cache_write", v);
    const std::string head = "#include \"mx4\"\nstruct Cfg_" + nm + " {\n" + c.members(kt.dtype) + "  static constexpr long TOKENS = " +
                             std::to_string(n) + ";\n};\n";
    auto launch = [&](const std::string& kernel, uint64_t groups, const std::string& call, const KernelWriter& w) {
      require(launchable(groups, 256), op, "more workgroups than a launch takes");
      KernelStep k;
      k.source = head + "extern \"C\" __global__ void __launch_bounds__(256) " + kernel + "(" + w.params() + ") {\n  accy::mx4::" + call + ";\n}\n";
      k.name = kernel;
      k.grid[0] = (uint32_t)groups;
      k.block[0] = 256;
      k.klass = "quantize";
      k.label = "cache_write:%" + std::to_string(v);
      push(std::move(k), w);
    };
    int owner = -1;
    if (owners) {
      owner = slots_.add(SlotInfo::Temp, -1, DType::i32, (uint64_t)(c.pages * c.tokens) * 4);
      for (const bool first : {true, false}) {
        KernelWriter w(g_, slots_, "i64_t");
        const std::string s = w.arg(ss, false), o = w.arg(owner, true);
        launch(name("mx4_claim", v), (n + 255) / 256, std::string("claim<Cfg_") + nm + ", " + (first ? "true" : "false") + ">(" + s + ", " + o + ")", w);
      }
    }
    KernelWriter w(g_, slots_, "i64_t");
    const std::string o = w.arg(out, true), a = w.arg(ks, false), b = w.arg(vs, false), s = w.arg(ss, false);
    const int64_t row = c.heads * c.dim / 8, per = row >= 512 ? 1 : 512 / row;  // Write<C>::TW
    launch(nm, (n + (uint64_t)per - 1) / (uint64_t)per, "cache_write<Cfg_" + nm + (owners ? ", true>(" : ", false>(") + o + ", " + a + ", " + b +
               ", " + s + ", " + (owners ? w.arg(owner, false) : std::string("nullptr")) + ")", w);
  }
  finish(v);
}

// Keys and values of the same slots are one kernel, whichever is asked for first.
void Planner::mx4_cache_read(uint32_t v) {
  const Op& op = g_.ops[v];
  const Type &rt = op.result, &st = g_.type(op.args[1]);
  element_type(op, rt.dtype);
  require(st.dtype == DType::i32 && st.rank() + 2 == rt.rank(), op, "i32 slots; the result is [slots .., kv_head, dim]");
  for (size_t i = 0; i < st.rank(); ++i) require(st.dims[i].extent == rt.dims[i].extent, op, "i32 slots; the result is [slots .., kv_head, dim]");
  const Mx4Cache c = mx4_cache(op, op.args[0], rt.dims[rt.rank() - 2].extent, last(rt));
  int out[2] = {-1, -1};  // keys, values
  std::vector<uint32_t> made;
  for (uint32_t u = v; u < g_.ops.size(); ++u) {
    const Op& uo = g_.ops[u];
    if (!live_[u] || done_[u] || uo.kind != Kind::custom_call || uo.index != 1 || uo.args != op.args || !(uo.result == rt)) continue;
    if (uo.bytes != "accy.mx4.cache_keys" && uo.bytes != "accy.mx4.cache_values") continue;
    int& slot = out[uo.bytes == "accy.mx4.cache_values"];
    if (slot >= 0) continue;
    slot = temp_slot(u);
    made.push_back(u);
  }
  if (rt.elements()) {
    const int cs = dense_slot(op.args[0]), ss = dense_slot(op.args[1]);
    KernelWriter w(g_, slots_, "i64_t");
    const std::string a = w.arg(cs, false), s = w.arg(ss, false), nm = name("mx4_cache_read", v);
    std::string to[2];
    for (int i = 0; i < 2; ++i) to[i] = out[i] >= 0 ? w.arg(out[i], true) : "nullptr";
    KernelStep k;
    k.source = "#include \"mx4\"\nstruct Cfg_" + nm + " {\n" + c.members(rt.dtype) + "  static constexpr long TOKENS = " +
               std::to_string(st.elements()) + ";\n};\nextern \"C\" __global__ void __launch_bounds__(256) " + nm + "(" + w.params() +
               ") {\n  accy::mx4::cache_read<Cfg_" + nm + ">(" + a + ", " + s + ", " + to[0] + ", " + to[1] + ");\n}\n";
    k.name = nm;
    k.grid[0] = grid_for(rt.elements() / 8, 256);
    k.block[0] = 256;
    k.klass = "quantize";
    k.label = "cache_read:%" + std::to_string(v);
    push(std::move(k), w);
  }
  for (uint32_t u : made) finish(u);
}

// ---- attention over the cache ----

void Planner::mx4_attend(uint32_t v) {
  const Op& op = g_.ops[v];
  const Type &qt = g_.type(op.args[0]), &ct = g_.type(op.args[1]), &pt = g_.type(op.args[2]), &lt = g_.type(op.args[3]);
  element_type(op, qt.dtype);
  require(op.result.dtype == qt.dtype && same_rows(op.result, qt) && last(op.result) == last(qt), op, "the result has the queries' type");
  require(qt.rank() == 3 || qt.rank() == 4, op, "queries are [seq, (query,) head, dim]");
  require(ct.rank() == 3, op, "a cache is u8 [page, kv_head, bytes]");
  const int64_t seqs = qt.dims[0].extent, Q = qt.rank() == 4 ? qt.dims[1].extent : 1, heads = qt.dims[qt.rank() - 2].extent;
  const int64_t H = ct.dims[1].extent, hd = last(qt);
  require(pt.dtype == DType::i32 && pt.rank() == 2 && pt.dims[0].extent == seqs, op, "pages are i32 [seq, page]");
  require(lt.dtype == DType::i32 && lt.rank() == 1 && lt.dims[0].extent == seqs, op, "lengths are i32 [seq]");
  require(H > 0 && heads % H == 0, op, num(heads) + " query heads over " + num(H) + " key-value heads");
  const int64_t G = heads / H;
  const Mx4Cache c = mx4_cache(op, op.args[1], H, hd);
  const int64_t maxp = pt.dims[1].extent;
  require(maxp < (int64_t(1) << 31) / c.tokens, op, "a sequence has fewer than 2^31 keys");
  const int out = temp_slot(v);
  const uint64_t nel = op.result.elements();
  if (nel) {
    require(Q * G < (int64_t(1) << 24), op, "2^24 query rows of a key-value head or more");
    const int qs = dense_slot(op.args[0]), cs = dense_slot(op.args[1]), ps = dense_slot(op.args[2]), ls = dense_slot(op.args[3]);
    // Outputs and queries are registers of the whole run, and with several queries the outputs before a step as well: two workgroups of a CU
    // where they leave half of 256, else one, whose kernel may take 512 (24 x 8 heads x 4096 keys, four rows of 192 f16 39 us in two, 47 in one,
    // five queries of 160 bf16 34 and 44; five of 192 would spill in two). Three, whose LDS there is up to 128 dims, where one query's kernel
    // fits 168 (a row of 128 f16, which takes 169 unasked, 26.9 us in three and 28.7 in two).
    const int64_t groups = (Q * G + 15) / 16, wgs = seqs * H * groups, parts = qt.dtype == DType::f32 ? 3 : qt.dtype == DType::f16 ? 2 : 1;
    const int64_t held = hd / 4 * (Q > 1 ? 2 : 1) + hd / 8 * parts;
    const int bounds = Q == 1 && hd <= 128 && held <= 64 ? 3 : held < 120 ? 2 : 1;
    // Up to three workgroups share a CU. Fewer sequences and heads than 256 are split along their keys till 512 workgroups are at
    // work (8 x 16 heads x 4096 keys of 128 bf16: 31.5 us in 1, 20.9 in 2, 18.5 in 4, 18.7 in 6 and 8 splits), more of them till
    // uneven lengths even out (48 x 8 x 16000: 155 in 1, 119 to 125 in 2 to 8), each split with four steps of every wave at least.
    const int64_t steps = (maxp * c.tokens + 31) / 32, want = wgs >= 256 ? 1024 : 512;
    const int64_t splits = opt_.allow_split ? std::max<int64_t>(1, std::min<int64_t>({(want + wgs - 1) / wgs, steps / 16, 64})) : 1;
    require(launchable((uint64_t)wgs, 256), op, "more workgroups than a launch takes");
    KernelWriter w(g_, slots_, "i64_t");
    const std::string q = w.arg(qs, false), a = w.arg(cs, false), p = w.arg(ps, false), l = w.arg(ls, false);
    int part = -1;
    if (splits > 1) part = slots_.add(SlotInfo::Temp, -1, DType::f32, (uint64_t)(seqs * H * Q * G * splits * (hd + 4)) * 4);
    const std::string o = splits > 1 ? "nullptr" : w.arg(out, true), pp = splits > 1 ? w.arg(part, true) : "nullptr";
    const std::string nm = name("mx4_attend", v);
    char sl[64];
    std::snprintf(sl, sizeof sl, "%af", (double)(float)(1.4426950408889634 / std::sqrt((double)hd)));
    const std::string head = "#include \"mx4\"\nstruct Cfg_" + nm + " {\n" + c.members(qt.dtype) + "  static constexpr int Q = " + num(Q) +
                             ", G = " + num(G) + ", MAXP = " + num(maxp) + ", SPLITS = " + num(splits) +
                             ";\n  static constexpr long SEQS = " + num(seqs) + ";\n  static constexpr float SL = " + sl + ";\n};\n";
    KernelStep k;
    k.source = head + "extern \"C\" __global__ void __launch_bounds__(256, " + num(bounds) + ") " + nm + "(" + w.params() + ") {\n  accy::mx4::attend<Cfg_" + nm +
               ">(" + q + ", " + a + ", " + p + ", " + l + ", " + o + ", " + pp + ");\n}\n";
    k.name = nm;
    k.grid[0] = (uint32_t)wgs;
    k.grid[1] = (uint32_t)splits;
    k.block[0] = 256;
    k.klass = "attention";
    k.label = "mx4_attend:%" + std::to_string(v);
    k.algorithmic_flops = 4.0 * (double)nel * (double)(maxp * c.tokens);
    push(std::move(k), w);
    if (splits > 1) {
      KernelWriter jw(g_, slots_, "i64_t");
      const std::string jp = jw.arg(part, false), jo = jw.arg(out, true);
      KernelStep j;
      j.name = name("mx4_join", v);
      j.source = head + "extern \"C\" __global__ void __launch_bounds__(256) " + j.name + "(" + jw.params() + ") {\n  accy::mx4::attend_join<Cfg_" +
                 nm + ">(" + jp + ", " + jo + ");\n}\n";
      require(launchable((nel + 255) / 256, 256), op, "more workgroups than a launch takes");
      j.grid[0] = (uint32_t)((nel + 255) / 256);
      j.block[0] = 256;
      j.klass = "attention";
      j.label = "mx4_join:%" + std::to_string(v);
      push(std::move(j), jw);
    }
  }
  finish(v);
}

}  // namespace planning
}  // namespace accy
