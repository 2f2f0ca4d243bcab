// Custom calls on logits (kernels/logits.h), "accy.logits.<name>":
//
//   token, entropy, top, top_tokens(logits, tokens)   f32 [row ..], f32 [row ..], f32 [row .., top], i32 [row .., top]: planned as one
//   grad(logits, tokens, d token, d entropy)          as the logits
//
// logits [row .., vocab] of bf16, f16 or f32; tokens i32 [row ..].
#include "planner_custom.hpp"

namespace accy {
namespace planning {

namespace {

bool rows_only(const Type& t, DType d, const Type& logits) {
  if (t.dtype != d || t.rank() + 1 != logits.rank()) return false;
  for (size_t i = 0; i < t.rank(); ++i)
    if (t.dims[i].extent != logits.dims[i].extent) return false;
  return true;
}

// Logits that the caches do not hold are read, and their gradient written, past them (us without / with the hint: gradients of 1001 x 50257 f16 55.4 / 49.8,
// 512 x 50257 f32 50.6 / 42.8, 2048 x 32000 bf16 52.6 / 50.2; log probabilities 2048 x 50257 bf16 66.1 / 65.1, 1024 x 50257 f32 46.3 / 44.6, but 600
// x 8000 bf16 9.1 / 9.5, 64 x 50257 13.8 / 14.3).
bool past_caches(const Type& logits) { return logits.bytes() >= uint64_t(64) << 20; }

}  // namespace

// Chunks of a row at most: rows of whole chunks start on one, others anywhere.
int64_t Planner::logit_chunks(int64_t vocab, DType d) const {
  const int64_t per = d == DType::f32 ? 4 : 8;
  return vocab % per == 0 ? vocab / per : (vocab + 2 * per - 2) / per;
}

std::string Planner::logit_config(const std::string& nm, int dt, uint64_t rows, int64_t vocab, int64_t k, int64_t splits, int64_t threads, int64_t u, bool once) const {
  return "#include \"logits\"\nstruct Cfg_" + nm + " {\n  static constexpr int DT = " + num(dt) + ", K = " + num(k) + ", SPLITS = " + num(splits) + ", NT = " +
         num(threads) + ", U = " + num(u) + ";\n  static constexpr long ROWS = " + std::to_string(rows) + ", V = " + num(vocab) + ";\n  static constexpr bool ONCE = " + (once ? "true" : "false") + ";\n};\n";
}

// Workgroups of a row: one where there are rows enough, else till four workgroups for every CU are at work, each with a chunk for every
// thread at least; their alternatives fit one list when they are joined.
int64_t Planner::logit_splits(uint64_t rows, int64_t chunks, int64_t k) const {
  if (!opt_.allow_split || rows >= 512) return 1;
  const int64_t want = (int64_t)((1024 + rows - 1) / rows);
  return std::max<int64_t>(1, std::min<int64_t>({want, chunks / 256, 64, k > 0 ? 1024 / k : 64}));
}

void Planner::logits_log_probs(uint32_t v) {
  const Op& op = g_.ops[v];
  const Type &xt = g_.type(op.args[0]), &tt = g_.type(op.args[1]);
  const int dt = element_type(op, xt.dtype);
  require(xt.rank() >= 1 && rows_only(tt, DType::i32, xt), op, "logits are [row .., vocab], tokens i32 [row ..]");
  const int64_t V = last(xt);
  require(V >= 1 && V < (int64_t(1) << 30), op, "1 to 2^30 logits to a row");
  const uint64_t rows = tt.elements();
  // As many alternatives as v asks for, or else the first call that asks for some; calls for another number are kernels of their own.
  int64_t K = 0;
  const auto calls = siblings(v, "accy.logits.", "", [&](const Op& o) {
    if (o.bytes != "accy.logits.top" && o.bytes != "accy.logits.top_tokens") return true;
    if (!K) K = last(o.result);
    return last(o.result) == K;
  });
  int out[4] = {-1, -1, -1, -1};
  const char* const names[] = {"token", "entropy", "top", "top_tokens"};
  std::vector<uint32_t> made;
  for (int i = 0; i < 4; ++i) {
    const auto call = calls.find(names[i]);
    if (call == calls.end()) continue;
    const Type& rt = g_.ops[call->second].result;
    if (i < 2) {
      require(rows_only(rt, DType::f32, xt), g_.ops[call->second], "the result is f32 [row ..]");
    } else {
      require(rt.dtype == (i == 2 ? DType::f32 : DType::i32) && rt.rank() == xt.rank() && same_rows(rt, xt), g_.ops[call->second],
              "the result is f32, of tokens i32, [row .., top]");
      require(last(rt) >= 1 && last(rt) <= 64 && last(rt) <= V, g_.ops[call->second], "1 to 64 alternatives, as many as there are logits");
    }
    out[i] = temp_slot(call->second);
    made.push_back(call->second);
  }
  if (rows) {
    require(launchable(rows, 256), op, "more rows than a launch takes");
    const int xs = dense_slot(op.args[0]), ts = dense_slot(op.args[1]);
    const int64_t chunks = logit_chunks(V, xt.dtype), splits = logit_splits(rows, chunks, K), mine = (chunks + splits - 1) / splits;
    // A thread holds up to four chunks at once and has four more on their way, in as few rounds as they take and as even (us, 256 threads of 4 /
    // 3 / 2 chunks: 2048 x 50257 bf16, 20 alternatives, 58 / 59 / 64, 1024 x 50257 f32 42 / 45 / 50; in an earlier form 256 threads of 4 / 5 / 8 chunks
    // and 512 of 4: 66 / 67 / 71 / 85, 46 / 47 / 50 / 56, 600 x 131072 bf16, five, 53 / 53 / 53 / 59).
    const int64_t rounds = (mine + 256 * 4 - 1) / (256 * 4), u = std::max<int64_t>(1, (mine + 256 * rounds - 1) / (256 * rounds));
    const std::string nm = name("log_probs", v), head = logit_config(nm, dt, rows, V, K, splits, 256, u, past_caches(xt));
    auto results = [&](KernelWriter& w) {
      std::string s;
      for (int i = 0; i < 4; ++i) s += std::string(i ? ", " : "") + (out[i] >= 0 ? w.arg(out[i], true) : std::string("nullptr"));
      return s;
    };
    int part = -1;
    if (splits > 1) part = slots_.add(SlotInfo::Temp, -1, DType::f32, rows * (uint64_t)splits * logit_part(K));
    KernelWriter w(g_, slots_, "i64_t");
    const std::string x = w.arg(xs, false), t = w.arg(ts, false);
    KernelStep k;
    const std::string to = splits > 1 ? "nullptr, nullptr, nullptr, nullptr, " + w.arg(part, true) : results(w) + ", nullptr";
    k.source = head + "extern \"C\" __global__ void __launch_bounds__(256) " + nm + "(" + w.params() + ") {\n  accy::logits::log_probs<Cfg_" + nm + ">(" + x + ", " + t +
               ", " + to + ");\n}\n";
    k.name = nm;
    k.grid[0] = (uint32_t)rows;
    k.grid[1] = (uint32_t)splits;
    k.block[0] = 256;
    k.klass = "row";
    k.label = "log_probs:%" + std::to_string(v);
    push(std::move(k), w);
    if (splits > 1) {
      KernelWriter jw(g_, slots_, "i64_t");
      const std::string jx = jw.arg(xs, false), jt = jw.arg(ts, false), jp = jw.arg(part, false), jr = results(jw);
      KernelStep j;
      j.name = name("log_probs_join", v);
      j.source = head + "extern \"C\" __global__ void __launch_bounds__(256) " + j.name + "(" + jw.params() + ") {\n  accy::logits::log_probs_join<Cfg_" + nm + ">(" + jx +
                 ", " + jt + ", " + jp + ", " + jr + ");\n}\n";
      j.grid[0] = (uint32_t)rows;
      j.block[0] = 256;
      j.klass = "row";
      j.label = "log_probs_join:%" + std::to_string(v);
      push(std::move(j), jw);
    }
  }
  for (const uint32_t u : made) finish(u);
}

void Planner::logits_grad(uint32_t v) {
  const Op& op = g_.ops[v];
  const Type &xt = g_.type(op.args[0]), &tt = g_.type(op.args[1]);
  const int dt = element_type(op, xt.dtype);
  require(xt.rank() >= 1 && rows_only(tt, DType::i32, xt), op, "logits are [row .., vocab], tokens i32 [row ..]");
  for (const int i : {2, 3}) require(rows_only(g_.type(op.args[(size_t)i]), DType::f32, xt), op, "gradients are f32 [row ..]");
  require(op.result.dtype == xt.dtype && same_rows(op.result, xt) && last(op.result) == last(xt), op, "the result has the logits' type");
  const int64_t V = last(xt);
  require(V >= 1 && V < (int64_t(1) << 30), op, "1 to 2^30 logits to a row");
  const uint64_t rows = tt.elements();
  const int out = temp_slot(v);
  if (rows) {
    require(launchable(rows, 1024), op, "more rows than a launch takes");
    int slots[4];
    for (size_t i = 0; i < 4; ++i) slots[i] = dense_slot(op.args[i]);
    const int64_t chunks = logit_chunks(V, xt.dtype);
    // Rows stay in the registers of one workgroup where there are rows for every CU (or they are short), in as few threads as hold them in eight chunks
    // each: 1001 x 50257 f16 55 us with 1024 threads, 58 with 512, 69 with 256. Other rows are read twice, by several workgroups. 22 chunks are as
    // many as 128 registers hold of every type beside what else they do, and so far one reading is the faster one (us, in registers / read twice: 1024 x
    // 139264 bf16, 17 chunks, 110 / 180, 1024 x 151936 127 / 199, 300 x 151936 51 / 58, 1024 x 180215 f16 160 / 250, 512 x 69632 f32 51 / 90, 256 x 90107 38 / 55).
    int64_t threads = 256;
    while (threads < 1024 && (chunks + threads - 1) / threads > 8) threads *= 2;
    const int64_t u = (chunks + threads - 1) / threads;
    const std::string nm = name("log_probs_grad", v);
    auto launch = [&](const std::string& kernel, const std::string& head, const std::string& call, bool first, int part, int64_t nt, int64_t splits) {
      KernelWriter w(g_, slots_, "i64_t");
      std::string args = w.arg(slots[0], false) + ", " + w.arg(slots[1], false);
      if (first) args += ", nullptr, nullptr, nullptr, nullptr, " + w.arg(part, true);
      else {
        for (const int i : {2, 3}) args += ", " + w.arg(slots[i], false);
        if (part >= 0) args += ", " + w.arg(part, false);
        args += ", " + w.arg(out, true);
      }
      KernelStep k;
      k.source = head + "extern \"C\" __global__ void __launch_bounds__(" + num(nt) + ") " + kernel + "(" + w.params() + ") {\n  accy::logits::" + call + "<Cfg_" + nm +
                 ">(" + args + ");\n}\n";
      k.name = kernel;
      k.grid[0] = (uint32_t)rows;
      k.grid[1] = (uint32_t)splits;
      k.block[0] = (uint32_t)nt;
      k.klass = "row";
      k.label = "log_probs_grad:%" + std::to_string(v);
      push(std::move(k), w);
    };
    if (u <= 22 && (rows >= 256 || chunks <= 512)) {
      launch(nm, logit_config(nm, dt, rows, V, 0, 1, threads, u, past_caches(xt)), "grad_row", false, -1, threads, 1);
    } else {
      const int64_t splits = std::max<int64_t>(1, std::min<int64_t>({(int64_t)((1024 + rows - 1) / rows), chunks / 256, 64})), mine = (chunks + splits - 1) / splits;
      const int64_t rounds = (mine + 256 * 4 - 1) / (256 * 4);
      // (one split is written to the parts too: the kernels of a row's sums and of its gradient are two)
      const std::string head = logit_config(nm, dt, rows, V, 0, std::max<int64_t>(2, splits), 256, std::max<int64_t>(1, (mine + 256 * rounds - 1) / (256 * rounds)), false);
      const int part = slots_.add(SlotInfo::Temp, -1, DType::f32, rows * (uint64_t)std::max<int64_t>(2, splits) * logit_part(0));
      launch(name("log_probs_sums", v), head, "log_probs", true, part, 256, std::max<int64_t>(2, splits));
      launch(nm, head, "grad_split", false, part, 256, std::max<int64_t>(2, splits));
    }
  }
  finish(v);
}

// Bytes of a Part: 64-bit keys, then three f32 sums, on 8 bytes.
uint64_t Planner::logit_part(int64_t k) const { return (uint64_t)std::max<int64_t>(1, k) * 8 + 16; }

}  // namespace planning
}  // namespace accy
