// Lowering of the floating point products and what stands around them: a checked descriptor -> kernel source (their
// device library plus the entries that instantiate it) and the launch interface as JSON.
#include <sstream>

#include "unp_internal.hpp"

namespace unp {

extern const char* const kMatmulLibrary;  // unp_matmul.hip, embedded at build time

namespace {

const char* device_type(int32_t k) { return k == UNP_F32 ? "float" : k == UNP_BF16 ? "__bf16" : "_Float16"; }
const char* short_name(int32_t k) {
  switch (k) {
    case UNP_F32: return "f32";
    case UNP_BF16: return "bf16";
    case UNP_F16: return "f16";
    case UNP_FP8_E4M3FN: return "e4m3";
    case UNP_FP8_E5M2: return "e5m2";
    case UNP_I32: return "i32";
    default: return "i64";
  }
}
// The device library's name of an operand's kind.
const char* operand(int32_t k) {
  return k == UNP_BF16 ? "unpm::BF16" : k == UNP_F16 ? "unpm::F16" : k == UNP_FP8_E4M3FN ? "unpm::E4M3" : "unpm::E5M2";
}
bool code_kind(int32_t k) { return k == UNP_FP8_E4M3FN || k == UNP_FP8_E5M2; }
bool float_kind(int32_t k) { return k == UNP_F32 || k == UNP_BF16 || k == UNP_F16; }

std::string source_head(const std::string& name) {
  return "// unpopped-hip kernel `" + name + "` for rocm:gfx950.\n" + kMatmulLibrary + "\n";
}

// What a product's operands, result and groups are; its entries follow from that alone.
struct Product {
  const char *x, *w, *out;
  bool x_turned, w_turned;
  const char* by;  // ALL, ROWS, DEPTH
  int scale_rows;
};

const char* kFewest = "16-byte aligned operands and strides, columns of out along an operand's rows in whole vectors; the least time";

void add_product(Lowered& L, const Product& p, std::ostringstream& src, std::vector<std::string>& when) {
  const std::string types = std::string(p.x) + ", " + p.w + ", " + (p.x_turned ? "true" : "false") + ", " +
                            (p.w_turned ? "true" : "false") + ", " + p.out + ", unpm::" + p.by + ", " +
                            std::to_string(p.scale_rows);
  const std::string params = std::string("(const unpm::u8* x, const unpm::u8* w, const float* xs, const float* ws, const int* starts, ") +
                             p.out + "* out, float* parts, unpm::product_args a)";
  auto add = [&](const char* tail, int tm, int tn, int wm, int wn, int split, int stages, bool direct, const char* cond) {
    Entry e;
    e.symbol = L.name + tail;
    e.threads = 64 * wm * wn * split;
    e.vec = tm;
    e.cols = tn;
    e.k = split;
    e.fast = direct;
    L.entries.push_back(e);
    when.push_back(cond);
    src << "extern \"C\" __global__ void __launch_bounds__(" << e.threads << ") " << e.symbol << params << " {\n  unpm::matmul<"
        << types << ", " << tm << ", " << tn << ", " << wm << ", " << wn << ", " << split << ", " << stages << ", "
        << (direct ? "true" : "false") << ">(x, w, xs, ws, starts, out, parts, a);\n}\n";
  };
  // In the order of their tiles; product_plan says which of them a launch takes.  Few rows: the weights' bytes count, and waves
  // share a tile's steps so that enough loads are on their way.
  if (std::string(p.by) != "DEPTH") {
    add("_one", 16, 16, 1, 1, 8, 4, true, kFewest);
    add("_slim", 32, 32, 1, 2, 4, 3, true, kFewest);
    add("_few", 32, 64, 1, 4, 2, 3, true, kFewest);
    add("_some", 64, 128, 1, 4, 2, 3, true, kFewest);
  }
  add("_tile", 128, 128, 2, 4, 1, 2, true, kFewest);
  Entry wide;
  wide.symbol = L.name + "_wide";
  wide.threads = 512;
  wide.vec = wide.cols = 256;
  wide.fast = true;
  L.entries.push_back(wide);
  when.push_back(kFewest);
  src << "extern \"C\" __global__ void __launch_bounds__(512) " << wide.symbol << params << " {\n  unpm::matmul_wide<" << types
      << ">(x, w, xs, ws, starts, out, parts, a);\n}\n";
  add("_any", 128, 128, 2, 2, 1, 2, false, "otherwise");
  Entry e;
  e.symbol = L.name + "_join";
  L.entries.push_back(e);
  when.push_back("after any of them, where the depth is split");
  src << "extern \"C\" __global__ void __launch_bounds__(256) " << e.symbol << "(const int* starts, " << p.out
      << "* out, const float* parts, unpm::product_args a) {\n  unpm::join<" << p.out << ", unpm::" << p.by
      << ">(starts, out, parts, a);\n}\n";
}

const char* kProductGrid = "a block per tile of out and part of the depth";
const char* kProductWorkspace = "the caller's, by unp_hip_exec_workspace";

}  // namespace

int32_t lower_quant8(const unp_quant8& q, Lowered& L, std::string& why) {
  L = Lowered{};
  if (!float_kind(q.dtype)) return why = "a quantisation of values outside F32, Bf16 and F16", UNP_UNSUPPORTED_DTYPE;
  if (!code_kind(q.kind)) return why = "codes are Fp8E4M3FN or Fp8E5M2", UNP_UNSUPPORTED_DTYPE;
  if (q.block_rows != 1 && q.block_rows != 128) return why = "a block has 1 or 128 rows", UNP_UNSUPPORTED_KERNEL;
  if (q.transpose != 0 && q.transpose != 1) return why = "transpose is 0 or 1", UNP_UNSUPPORTED_KERNEL;
  L.form.kind = UNP_FORM_QUANT8;
  L.form.dtype = q.dtype;
  L.quant8 = q;
  L.name = std::string("unp_quant8_") + short_name(q.dtype) + "_" + short_name(q.kind) + "_b" + std::to_string(q.block_rows) +
           (q.transpose ? "_t" : "");
  std::ostringstream src;
  src << source_head(L.name);
  const bool rows = q.block_rows == 1 && !q.transpose;
  Entry e;
  e.symbol = L.name + "_k";
  e.threads = rows ? 256 : 512;
  L.entries.push_back(e);
  const std::string T = device_type(q.dtype);
  src << "extern \"C\" __global__ void __launch_bounds__(" << e.threads << ") " << e.symbol << "(const " << T
      << "* x, unpm::u8* codes, float* scales, unpm::quant_args a) {\n  unpm::quantise_" << (rows ? "rows<" : "tiles<") << T << ", "
      << operand(q.kind);
  if (!rows) src << ", " << q.block_rows << ", " << (q.transpose ? "true" : "false");
  src << ">(x, codes, scales, a);\n}\n";
  L.source = src.str();
  L.interface_json = form_interface(
      L, "quant8", "\"block_rows\":" + std::to_string(q.block_rows) + ",\"transpose\":" + std::to_string(q.transpose),
      {{"x", "Read", kind_name(q.dtype)}, {"codes", "Write", kind_name(q.kind)}, {"scales", "Write", "F32"},
       {"rows", nullptr, "I64"}, {"cols", nullptr, "I64"}, {"x_row", nullptr, "I64"}, {"code_row", nullptr, "I64"},
       {"scale_row", nullptr, "I64"}},
      rows ? "8 lanes a block of 128 elements" : "a block of lanes per 128 x 128 elements",
      {"always"}, nullptr, "scales as the largest magnitude times an f32 constant, quotients correctly rounded to f32, codes rounded to even: bit-exact");
  return UNP_OK;
}

int32_t lower_matmul8(const unp_matmul8& m, Lowered& L, std::string& why) {
  L = Lowered{};
  if (!code_kind(m.a_kind) || !code_kind(m.b_kind)) return why = "codes are Fp8E4M3FN or Fp8E5M2", UNP_UNSUPPORTED_DTYPE;
  // 32 bits would hold digits that the matrix unit does not keep of codes.
  if (m.out != UNP_BF16 && m.out != UNP_F16) return why = "a product of codes gives Bf16 or F16", UNP_UNSUPPORTED_DTYPE;
  if (m.b_rows != 1 && m.b_rows != 128) return why = "a scale of b has 1 or 128 rows", UNP_UNSUPPORTED_KERNEL;
  if (m.grouped != 0 && m.grouped != 1) return why = "grouped is 0 or 1", UNP_UNSUPPORTED_KERNEL;
  L.form.kind = UNP_FORM_MATMUL8;
  L.form.dtype = m.out;
  L.matmul8 = m;
  L.name = std::string("unp_matmul8_") + short_name(m.a_kind) + "_" + short_name(m.b_kind) + "_" + short_name(m.out) + "_b" +
           std::to_string(m.b_rows) + (m.grouped ? "_grouped" : "");
  std::ostringstream src;
  src << source_head(L.name);
  std::vector<std::string> when;
  add_product(L, {operand(m.a_kind), operand(m.b_kind), device_type(m.out), false, false, m.grouped ? "ROWS" : "ALL", m.b_rows},
              src, when);
  L.source = src.str();
  std::vector<FormParam> ps = {{"a", "Read", kind_name(m.a_kind)}, {"a_scales", "Read", "F32"}, {"b", "Read", kind_name(m.b_kind)},
                               {"b_scales", "Read", "F32"}};
  if (m.grouped) ps.push_back({"starts", "Read", "I32"});
  ps.push_back({"out", "Write", kind_name(m.out)});
  ps.push_back({"workspace", "ReadWrite", "U8"});
  for (const char* s : {"m", "n", "k"}) ps.push_back({s, nullptr, "I64"});
  if (m.grouped) ps.push_back({"groups", nullptr, "I64"});
  for (const char* s : {"a_row", "a_scale_row", "b_row", "b_scale_row"}) ps.push_back({s, nullptr, "I64"});
  if (m.grouped)
    for (const char* s : {"b_group", "b_scale_group"}) ps.push_back({s, nullptr, "I64"});
  for (const char* s : {"out_row", "workspace_bytes"}) ps.push_back({s, nullptr, "I64"});
  L.interface_json = form_interface(L, "matmul8", "\"b_rows\":" + std::to_string(m.b_rows), ps, kProductGrid, when, kProductWorkspace,
                                    "products of 16 codes summed to 2^-13 of their largest, those sums in f32, times both scales and added in f32; one rounding");
  return UNP_OK;
}

int32_t lower_grouped_matmul(const unp_grouped_matmul& m, Lowered& L, std::string& why) {
  L = Lowered{};
  if (m.dtype != UNP_BF16 && m.dtype != UNP_F16) return why = "a grouped product of numbers outside Bf16 and F16", UNP_UNSUPPORTED_DTYPE;
  if (m.out != m.dtype && m.out != UNP_F32) return why = "the result has the operands' type or F32", UNP_UNSUPPORTED_DTYPE;
  if (m.direction != UNP_GROUPED_FORWARD && m.direction != UNP_GROUPED_INPUT && m.direction != UNP_GROUPED_WEIGHT)
    return why = "an unknown direction of a grouped product", UNP_UNSUPPORTED_OP;
  const bool weight = m.direction == UNP_GROUPED_WEIGHT;
  L.form.kind = UNP_FORM_GROUPED_MATMUL;
  L.form.dtype = m.out;
  L.grouped_matmul = m;
  const char* way = weight ? "weight" : m.direction == UNP_GROUPED_INPUT ? "input" : "forward";
  L.name = std::string("unp_grouped_matmul_") + short_name(m.dtype) + "_" + short_name(m.out) + "_" + way;
  std::ostringstream src;
  src << source_head(L.name);
  std::vector<std::string> when;
  add_product(L, {operand(m.dtype), operand(m.dtype), device_type(m.out), weight, m.direction != UNP_GROUPED_FORWARD,
                  weight ? "DEPTH" : "ROWS", 1}, src, when);
  L.source = src.str();
  const char *dt = kind_name(m.dtype), *ot = kind_name(m.out);
  std::vector<FormParam> ps = {{"x", "Read", dt}, {weight ? "y" : "w", "Read", dt}, {"starts", "Read", "I32"}, {"out", "Write", ot},
                               {"workspace", "ReadWrite", "U8"}};
  for (const char* s : {"rows", "n", "k", "groups", "x_row"}) ps.push_back({s, nullptr, "I64"});
  if (weight)
    for (const char* s : {"y_row", "out_group", "out_row"}) ps.push_back({s, nullptr, "I64"});
  else
    for (const char* s : {"w_group", "w_row", "out_row"}) ps.push_back({s, nullptr, "I64"});
  ps.push_back({"workspace_bytes", nullptr, "I64"});
  L.interface_json = form_interface(L, "grouped_matmul", std::string("\"direction\":\"") + way + "\"", ps, kProductGrid, when,
                                    kProductWorkspace, "products and sums in f32; one rounding");
  return UNP_OK;
}

int32_t lower_group_rows(const unp_group_rows& r, Lowered& L, std::string& why) {
  L = Lowered{};
  if (r.index_dtype != UNP_I32 && r.index_dtype != UNP_I64) return why = "ids are I32 or I64", UNP_UNSUPPORTED_DTYPE;
  L.form.kind = UNP_FORM_GROUP_ROWS;
  L.form.dtype = r.index_dtype;
  L.group_rows = r;
  L.name = std::string("unp_group_rows_") + short_name(r.index_dtype);
  L.threads = 512;
  std::ostringstream src;
  src << source_head(L.name);
  const std::string I = r.index_dtype == UNP_I32 ? "int" : "long long";
  for (const char* tail : {"_place", "_count"}) {
    Entry e;
    e.symbol = L.name + tail;
    L.entries.push_back(e);
  }
  src << "extern \"C\" __global__ void __launch_bounds__(512) " << L.entries[0].symbol << "(const " << I
      << "* ids, int* starts, int* rows, int* place, const int* counted, unpm::rows_args a) {\n  unpm::place_rows<" << I
      << ">(ids, starts, rows, place, counted, a);\n}\n";
  src << "extern \"C\" __global__ void __launch_bounds__(512) " << L.entries[1].symbol << "(const " << I
      << "* ids, int* counted, unpm::rows_args a) {\n  unpm::count_rows<" << I << ">(ids, counted, a);\n}\n";
  L.source = src.str();
  L.interface_json = form_interface(
      L, "group_rows", "\"most_groups\":1024",
      {{"ids", "Read", kind_name(r.index_dtype)}, {"starts", "Write", "I32"}, {"rows", "Write", "I32"}, {"place", "Write", "I32"},
       {"workspace", "ReadWrite", "U8"}, {"count", nullptr, "I64"}, {"per", nullptr, "I64"}, {"groups", nullptr, "I64"},
       {"workspace_bytes", nullptr, "I64"}},
      "a block per chunk of ids", {"always", "before it, where there are several chunks"}, kProductWorkspace,
      "whole numbers, in the ids' order: exact");
  return UNP_OK;
}

}  // namespace unp
