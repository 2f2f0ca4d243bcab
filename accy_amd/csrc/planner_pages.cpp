// Custom calls on the pages of a cache (kernels/pages.h), "accy.pages.<name>":
//
//   fork_table, fork_lengths, fork_source, fork_target, fork_left, fork_slots(group(table, lengths), group(parents, room), held, page)
//       table i32 [seq, slot], lengths i32 [seq], parents, room i32 [row], held i1 [page], page an i32 constant -> i32 [row, slot], [row], [row],
//       [row], [], [row] or [row, token]: planned as one kernel
//   compact_table, compact_source, compact_target(table, held, moves)   table i32 [seq, slot], held i1 [page], moves an i32 constant -> as the table,
//       i32 [move] twice
//   copy(cache, source, target)   cache [page, ..], i32 [copy] twice -> the cache
#include "planner_custom.hpp"

namespace accy {
namespace planning {

namespace {

constexpr int64_t kMostPages = int64_t(1) << 24;
constexpr int64_t kLdsPages = int64_t(1) << 17;  // LDS_PAGES of kernels/pages.h

// Entries of tables that one workgroup writes as fast as another launch would (us with a copy of a few pages, one launch / two: 8 x 64 entries
// 12 / 15, 64 x 64 14 / 15, 64 x 256 24 / 15, 128 x 256 42 / 16, 256 x 512 114 / 18).
constexpr uint64_t kOneWorkgroup = 4096;

bool whole_numbers(const Type& t, size_t rank) { return t.dtype == DType::i32 && t.rank() == rank; }

}  // namespace

// An operand that is an i32 constant, -1 where it is none.
int64_t Planner::whole_constant(uint32_t v) const {
  const Op& op = g_.ops[v];
  int32_t n = -1;
  if (op.kind == Kind::constant && op.result.dtype == DType::i32 && op.result.rank() == 0 && op.bytes.size() >= 4) std::memcpy(&n, op.bytes.data(), 4);
  return n;
}

void Planner::pages_fork(uint32_t v) {
  const Op& op = g_.ops[v];
  const std::vector<uint32_t> now = grouped(op, op.args[0], 2, 2), next = grouped(op, op.args[1], 2, 2);
  const Type &tt = g_.type(now[0]), &lt = g_.type(now[1]), &pt = g_.type(next[0]), &rt = g_.type(next[1]), &ht = g_.type(op.args[2]);
  require(whole_numbers(tt, 2) && whole_numbers(lt, 1) && lt.dims[0].extent == tt.dims[0].extent, op, "tables are i32 [seq, slot], lengths i32 [seq]");
  require(whole_numbers(pt, 1) && whole_numbers(rt, 1) && pt.dims[0].extent == rt.dims[0].extent, op, "parents and room are i32 [row]");
  require(ht.dtype == DType::i1 && ht.rank() == 1, op, "held pages are i1 [page]");
  const int64_t page = whole_constant(op.args[3]);
  require(page >= 1 && page < (1 << 20), op, "the size of a page is an i32 constant of 1 to 2^20");
  const int64_t seqs = tt.dims[0].extent, slots = tt.dims[1].extent, rows = pt.dims[0].extent, pages = ht.dims[0].extent;
  require(pages <= kMostPages, op, "more than 2^24 pages");
  require(pages < (int64_t(1) << 31) / page && slots < (int64_t(1) << 31) / page, op, "2^31 slots or more");
  require(slots < (int64_t(1) << 31) && rows < (int64_t(1) << 31) && rows * std::max<int64_t>(1, slots) < (int64_t(1) << 31), op, "2^31 entries or more");
  const auto calls = siblings(v, "accy.pages.fork_");
  const char* const names[] = {"table", "lengths", "source", "target", "left", "slots"};
  std::vector<int> out(6, -1);
  std::vector<uint32_t> made;
  int64_t tokens = 0;  // of a row, whose slots are asked for
  for (size_t i = 0; i < 6; ++i) {
    const auto call = calls.find(names[i]);
    if (i == 5) {
      if (call == calls.end()) break;
      const Type& t = g_.ops[call->second].result;
      require((whole_numbers(t, 1) || whole_numbers(t, 2)) && t.dims[0].extent == rows && (t.rank() == 1 || (last(t) >= 1 && last(t) <= 1024)),
              g_.ops[call->second], "the result is i32 [row] or [row, token], of up to 1024 tokens");
      tokens = t.rank() == 1 ? 1 : last(t);
      out[i] = temp_slot(call->second);
      made.push_back(call->second);
      break;
    }
    const uint64_t bytes = i == 0 ? (uint64_t)(rows * slots) * 4 : i == 4 ? 4 : (uint64_t)rows * 4;
    if (call == calls.end()) {
      out[i] = slots_.add(SlotInfo::Temp, -1, DType::i32, bytes);  // what nobody reads is written all the same
      continue;
    }
    const Type& t = g_.ops[call->second].result;
    const bool fits = i == 0 ? whole_numbers(t, 2) && t.dims[0].extent == rows && t.dims[1].extent == slots
                             : i == 4 ? whole_numbers(t, 0) : whole_numbers(t, 1) && t.dims[0].extent == rows;
    require(fits, g_.ops[call->second], i == 0 ? "the result is i32 [row, slot]" : i == 4 ? "the result is i32 []" : "the result is i32 [row]");
    out[i] = temp_slot(call->second);
    made.push_back(call->second);
  }
  require(std::find(made.begin(), made.end(), v) != made.end(), op, "no result of that name");
  // One workgroup writes small tables itself; of larger ones it leaves what each row takes to workgroups of their own.
  const bool wide = (uint64_t)(rows * slots) > kOneWorkgroup;
  require(launchable((uint64_t)rows, 256) && (slots + 1023) / 1024 < 65536, op, "more workgroups than a launch takes");
  // ForkWork of kernels/pages.h
  const uint64_t words = (uint64_t)(pages + 31) / 32, work = (pages > kLdsPages ? (2 * words + 3) / 4 * 4 : 0) + (wide ? (uint64_t)(rows * (4 + slots)) : 0) +
                                                             (rows > 1024 ? (uint64_t)pages : 0);
  const int table = dense_slot(now[0]), ws = work ? slots_.add(SlotInfo::Temp, -1, DType::i32, work * 4) : -1;
  KernelWriter w(g_, slots_, "i64_t");
  std::string args = w.arg(table, false) + ", ";
  for (const uint32_t a : {now[1], next[0], next[1], op.args[2]}) args += w.arg(dense_slot(a), false) + ", ";
  for (size_t i = 0; i < 6; ++i) args += ((i == 0 && wide) || out[i] < 0 ? std::string("nullptr") : w.arg(out[i], true)) + ", ";
  args += work ? w.arg(ws, true) : "nullptr";
  KernelStep k;
  const std::string nm = name("fork", v);
  const std::string head = "#include \"pages\"\nstruct Cfg_" + nm + " {\n  static constexpr long SEQS = " + num(seqs) + ", ROWS = " + num(rows) + ", SLOTS = " + num(slots) +
                           ", P = " + num(pages) + ", T = " + num(page) + ", NEW = " + num(tokens) + ";\n  static constexpr bool WIDE = " + (wide ? "true" : "false") + ";\n};\n";
  k.source = head + "extern \"C\" __global__ void __launch_bounds__(1024) " + nm + "(" + w.params() + ") {\n  accy::pages::fork<Cfg_" + nm + ">(" + args + ");\n}\n";
  k.name = nm;
  k.block[0] = 1024;
  k.klass = "pages";
  k.label = "fork:%" + std::to_string(v);
  push(std::move(k), w);
  if (wide) {
    KernelWriter rw(g_, slots_, "i64_t");
    const std::string a = rw.arg(table, false), b = rw.arg(ws, false), c = rw.arg(out[0], true);
    KernelStep t;
    t.name = name("fork_rows", v);
    t.source = head + "extern \"C\" __global__ void __launch_bounds__(256) " + t.name + "(" + rw.params() + ") {\n  accy::pages::fork_rows<Cfg_" + nm + ">(" + a + ", " + b +
               ", " + c + ");\n}\n";
    t.grid[0] = (uint32_t)rows;
    t.grid[1] = (uint32_t)((slots + 1023) / 1024);
    t.block[0] = 256;
    t.klass = "pages";
    t.label = "fork_rows:%" + std::to_string(v);
    push(std::move(t), rw);
  }
  for (const uint32_t u : made) finish(u);
}

void Planner::pages_compact(uint32_t v) {
  const Op& op = g_.ops[v];
  const Type &tt = g_.type(op.args[0]), &ht = g_.type(op.args[1]);
  require(whole_numbers(tt, 2), op, "tables are i32 [seq, slot]");
  require(ht.dtype == DType::i1 && ht.rank() == 1, op, "held pages are i1 [page]");
  const int64_t pages = ht.dims[0].extent;
  require(pages <= kMostPages, op, "more than 2^24 pages");
  const auto calls = siblings(v, "accy.pages.compact_");
  const int64_t moves = whole_constant(op.args[2]);
  require(moves >= 0 && moves <= pages, op, "the number of moves is an i32 constant, at most as many as pages");
  int out[3] = {-1, -1, -1};
  const char* const names[] = {"table", "source", "target"};
  std::vector<uint32_t> made;
  for (int i = 0; i < 3; ++i) {
    const auto call = calls.find(names[i]);
    if (call == calls.end()) {
      out[i] = slots_.add(SlotInfo::Temp, -1, DType::i32, i == 0 ? tt.bytes() : (uint64_t)moves * 4);
      continue;
    }
    const Type& t = g_.ops[call->second].result;
    if (i == 0) require(whole_numbers(t, 2) && t.dims[0].extent == tt.dims[0].extent && t.dims[1].extent == tt.dims[1].extent, g_.ops[call->second], "the result is as the table");
    else require(whole_numbers(t, 1) && t.dims[0].extent == moves, g_.ops[call->second], "the result is i32 [move]");
    out[i] = temp_slot(call->second);
    made.push_back(call->second);
  }
  require(std::find(made.begin(), made.end(), v) != made.end(), op, "no result of that name");
  const uint64_t entries = tt.elements(), words = (uint64_t)(pages + 31) / 32;
  const bool wide = entries > kOneWorkgroup;
  const int table = dense_slot(op.args[0]);
  const int ws = pages > kLdsPages || wide ? slots_.add(SlotInfo::Temp, -1, DType::i32, (4 + 3 * words) * 4) : -1;
  KernelWriter w(g_, slots_, "i64_t");
  std::string args = w.arg(table, false) + ", " + w.arg(dense_slot(op.args[1]), false);
  for (int i = 0; i < 3; ++i) args += ", " + (i == 0 && wide ? std::string("nullptr") : w.arg(out[i], true));
  args += ws >= 0 ? ", " + w.arg(ws, true) : ", nullptr";
  KernelStep k;
  const std::string nm = name("compact", v);
  const std::string head = "#include \"pages\"\nstruct Cfg_" + nm + " {\n  static constexpr long ENTRIES = " + std::to_string(entries) + ", P = " + num(pages) + ", MOVES = " +
                           num(moves) + ";\n  static constexpr bool WIDE = " + (wide ? "true" : "false") + ";\n};\n";
  k.source = head + "extern \"C\" __global__ void __launch_bounds__(1024) " + nm + "(" + w.params() + ") {\n  accy::pages::compact<Cfg_" + nm + ">(" + args + ");\n}\n";
  k.name = nm;
  k.block[0] = 1024;
  k.klass = "pages";
  k.label = "compact:%" + std::to_string(v);
  push(std::move(k), w);
  if (wide) {
    KernelWriter rw(g_, slots_, "i64_t");
    const std::string a = rw.arg(table, false), b = rw.arg(out[2], false), c = rw.arg(ws, true), d = rw.arg(out[0], true);
    KernelStep t;
    t.name = name("compact_rows", v);
    t.source = head + "extern \"C\" __global__ void __launch_bounds__(256) " + t.name + "(" + rw.params() + ") {\n  accy::pages::compact_rows<Cfg_" + nm + ">(" + a + ", " +
               b + ", " + c + ", " + d + ");\n}\n";
    t.grid[0] = grid_for(entries / 4, 256);
    t.block[0] = 256;
    t.klass = "pages";
    t.label = "compact_rows:%" + std::to_string(v);
    push(std::move(t), rw);
  }
  for (const uint32_t u : made) finish(u);
}

void Planner::pages_copy(uint32_t v) {
  const Op& op = g_.ops[v];
  const Type &ct = g_.type(op.args[0]), &st = g_.type(op.args[1]), &tt = g_.type(op.args[2]);
  require(ct.rank() >= 1, op, "a cache is [page, ..]");
  require(whole_numbers(st, 1) && whole_numbers(tt, 1) && st.dims[0].extent == tt.dims[0].extent, op, "source and target are i32 [copy]");
  require(op.result == ct, op, "the result has the cache's type");
  const int from = dense_slot(op.args[0]), out = updated_cache(v);
  const int64_t n = st.dims[0].extent, pages = ct.dims[0].extent, bytes = pages ? (int64_t)(ct.bytes() / (uint64_t)pages) : 0;
  if (n && bytes) {
    require(pages < (int64_t(1) << 31), op, "2^31 pages or more");
    // Lists of fork and compact name pages that differ.
    const Op &so = g_.ops[op.args[1]], &to = g_.ops[op.args[2]];
    auto call = [&](const Op& o, const std::string& what) { return o.kind == Kind::custom_call && o.index == 1 && o.bytes == "accy.pages." + what; };
    const bool check = !(so.args == to.args && ((call(so, "fork_source") && call(to, "fork_target")) || (call(so, "compact_source") && call(to, "compact_target"))));
    const bool owners = check && n > 4096;
    int64_t W = 16;
    while (bytes % W) W /= 2;
    // A part of a page to a workgroup (4, 8, 12, 16 KB and whole pages of 34 KB: the same to 2 %). What the caches do not hold anyway goes by them:
    // 2990 pages of 34 KB 42 us, with the hint for loads 36, for stores 33, for both 32; a few pages may be read again at once.
    const bool once = n * bytes >= int64_t(64) << 20;
    const int64_t per = 8192, parts = (bytes + per - 1) / per;
    require(parts < 65536 && launchable((uint64_t)n, 256), op, "more workgroups than a launch takes");
    const std::string nm = name("copy_pages", v);
    const std::string head = "#include \"pages\"\nstruct Cfg_" + nm + " {\n  static constexpr long N = " + num(n) + ", P = " + num(pages) + ", BYTES = " + num(bytes) + ", PER = " +
                             num(per) + ";\n  static constexpr int W = " + num(W) + ";\n  static constexpr bool ONCE = " + (once ? "true" : "false") + ", CHECK = " + (check ? "true" : "false") + ", OWNERS = " +
                             (owners ? "true" : "false") + ";\n};\n";
    const int ss = dense_slot(op.args[1]), ts = dense_slot(op.args[2]);
    const int aside = check ? slots_.add(SlotInfo::Temp, -1, DType::u8, (uint64_t)(n * bytes)) : -1;
    const int flags = check ? slots_.add(SlotInfo::Temp, -1, DType::i32, (uint64_t)n * 4) : -1;
    const int owner = owners ? slots_.add(SlotInfo::Temp, -1, DType::i32, (uint64_t)pages * 4) : -1;
    auto launch = [&](const std::string& kernel, const std::string& call, const KernelWriter& w, uint64_t x, uint64_t y) {
      KernelStep k;
      // The cache's two buffers may be one, and the kernels ask whether they are.
      std::string params = w.params();
      for (size_t at; (at = params.find("__restrict__ ")) != std::string::npos;) params.erase(at, 13);
      k.source = head + "extern \"C\" __global__ void __launch_bounds__(256) " + kernel + "(" + params + ") {\n  accy::pages::" + call + ";\n}\n";
      k.name = kernel;
      k.grid[0] = (uint32_t)x;
      k.grid[1] = (uint32_t)y;
      k.block[0] = 256;
      k.klass = "pages";
      k.label = "copy_pages:%" + std::to_string(v);
      push(std::move(k), w);
    };
    for (const bool first : {true, false}) {
      if (!owners) break;
      KernelWriter w(g_, slots_, "i64_t");
      const std::string s = w.arg(ss, false), t = w.arg(ts, false), o = w.arg(owner, true);
      launch(name("claim_pages", v), std::string("claim<Cfg_") + nm + ", " + (first ? "true" : "false") + ">(" + s + ", " + t + ", " + o + ")", w, (uint64_t)(n + 255) / 256, 1);
    }
    for (const bool last : {false, true}) {
      if (!last && !check) continue;
      KernelWriter w(g_, slots_, "i64_t");
      const std::string a = w.arg(from, false), b = w.arg(out, last), s = w.arg(ss, false), t = w.arg(ts, false), o = owners ? w.arg(owner, false) : "nullptr";
      const std::string i = check ? w.arg(aside, !last) : "nullptr", f = check ? w.arg(flags, !last) : "nullptr";
      launch(last ? nm : name("put_aside", v),
             std::string(last ? "copy" : "put_aside") + "<Cfg_" + nm + ">((const u8_t*)" + a + ", (" + (last ? "" : "const ") + "u8_t*)" + b + ", " + s + ", " + t + ", " + o + ", " +
                 (check ? std::string(last ? "(const u8_t*)" : "(u8_t*)") + i : i) + ", " + f + ")",
             w, (uint64_t)n, (uint64_t)parts);
    }
  }
  finish(v);
}

}  // namespace planning
}  // namespace accy
