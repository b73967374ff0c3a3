// Lowering of the rotary and 4-bit cache forms: a checked descriptor -> kernel source (their device
// library plus the entries that instantiate it) and the launch interface as JSON.
#include <cmath>
#include <sstream>

#include "unp_internal.hpp"

namespace unp {

extern const char* const kCache4Library;  // unp_cache4.hip, embedded at build time

namespace {

const char* device_type(int32_t k) {
  switch (k) {
    case UNP_F32: return "float";
    case UNP_BF16: return "__bf16";
    case UNP_F16: return "_Float16";
    case UNP_I32: return "int";
    case UNP_I64: return "long long";
    default: return nullptr;
  }
}
const char* short_name(int32_t k) {
  switch (k) {
    case UNP_F32: return "f32";
    case UNP_BF16: return "bf16";
    case UNP_F16: return "f16";
    case UNP_I32: return "i32";
    default: return "i64";
  }
}
bool index_ok(int32_t k, std::string& why) {
  if (k == UNP_I32 || k == UNP_I64) return true;
  why = "positions and slots are I32 or I64";
  return false;
}
bool layout_ok(int32_t l, std::string& why) {
  if (l == UNP_ROPE_HALVES || l == UNP_ROPE_PAIRS) return true;
  why = "an unknown rotary layout";
  return false;
}

// One parameter of the interface JSON.
struct Param {
  const char* name;
  const char* role;  // "Read", "Write", "ReadWrite"; null: a scalar
  const char* dtype;
};
std::string interface(const Lowered& L, const char* form, const std::string& fields, const std::vector<Param>& ps,
                      const char* policy, const std::vector<std::string>& when, const char* workspace,
                      const char* note) {
  std::ostringstream j;
  j << "{\"backend\":\"hip\",\"target\":\"rocm:gfx950\",\"form\":\"" << form << "\"," << fields << ",\"params\":[";
  for (size_t i = 0; i < ps.size(); ++i) {
    j << (i ? "," : "") << "{\"name\":\"" << ps[i].name << "\",\"kind\":\"" << (ps[i].role ? "buffer" : "scalar") << "\"";
    if (ps[i].role) j << ",\"role\":\"" << ps[i].role << "\"";
    j << ",\"dtype\":\"" << ps[i].dtype << "\"}";
  }
  j << "],\"launch\":{\"block\":[" << L.threads << ",1,1],\"grid_policy\":\"" << policy << "\"},\"entries\":[";
  for (size_t i = 0; i < L.entries.size(); ++i)
    j << (i ? "," : "") << "{\"symbol\":\"" << L.entries[i].symbol << "\",\"when\":\"" << when[i] << "\"}";
  j << "],\"workspace\":" << (workspace ? std::string("\"") + workspace + "\"" : "null")
    << ",\"compiler_args\":[\"--offload-arch=gfx950\",\"-O3\",\"-std=c++17\",\"-ffp-contract=off\"]"
    << ",\"fidelity_notes\":[\"" << note << "\"]}";
  return j.str();
}

std::string source_head(const std::string& name) {
  return "// unpopped-hip kernel `" + name + "` for rocm:gfx950.\n" + kCache4Library + "\n";
}

const char* kBounds256 = "extern \"C\" __global__ void __launch_bounds__(256) ";

}  // namespace

int32_t lower_rope_table(const unp_rope_table& t, Lowered& L, std::string& why) {
  L = Lowered{};
  if (t.rot < 2 || t.rot % 2 != 0 || t.rot > 4096) return why = "rot is even, 2..4096", UNP_UNSUPPORTED_KERNEL;
  if (t.scaling != UNP_ROPE_NONE && t.scaling != UNP_ROPE_LINEAR && t.scaling != UNP_ROPE_RAMP)
    return why = "an unknown frequency scaling", UNP_UNSUPPORTED_OP;
  auto positive = [](double v) { return std::isfinite(v) && v > 0.0; };
  if (!positive(t.base)) return why = "the base is a positive number", UNP_UNSUPPORTED_KERNEL;
  if (!std::isfinite(t.amplitude)) return why = "the amplitude is a finite number", UNP_UNSUPPORTED_KERNEL;
  if (t.scaling != UNP_ROPE_NONE && !positive(t.factor))
    return why = "the scaling factor is a positive number", UNP_UNSUPPORTED_KERNEL;
  if (t.scaling == UNP_ROPE_RAMP &&
      (!std::isfinite(t.low) || !std::isfinite(t.high) || t.low >= t.high || !positive(t.original)))
    return why = "a ramp needs low < high and a positive original length", UNP_UNSUPPORTED_KERNEL;
  L.form.kind = UNP_FORM_ROPE_TABLE;
  L.form.dtype = UNP_F32;
  L.rope_table = t;
  L.name = "unp_rope_table_r" + std::to_string(t.rot);
  std::ostringstream src;
  src << source_head(L.name);
  std::vector<std::string> when;
  auto add = [&](const char* tail, int v, const char* cond) {
    Entry e;
    e.symbol = L.name + tail;
    e.fast = v > 1;
    e.vec = v;
    L.entries.push_back(e);
    when.push_back(cond);
    src << kBounds256 << e.symbol << "(float* table, long long first, long long count, unp4::stretch s) {\n  unp4::rope_table<"
        << t.rot << ", " << v << ">(table, first, count, s);\n}\n";
  };
  if (t.rot % 4 == 0) add("_v", 2, "a 16-byte aligned table");
  add("_e", 1, "otherwise");
  L.source = src.str();
  L.interface_json = interface(
      L, "rope_table", "\"rot\":" + std::to_string(t.rot),
      {{"table", "Write", "F32"}, {"first", nullptr, "I64"}, {"count", nullptr, "I64"}},
      "pairs by lanes in order; blocks stride over them", when, nullptr,
      "angles, cosines and sines in f64, rounded once to f32");
  return UNP_OK;
}

int32_t lower_rope(const unp_rope& r, Lowered& L, std::string& why) {
  L = Lowered{};
  if (r.dtype != UNP_F32 && r.dtype != UNP_BF16 && r.dtype != UNP_F16)
    return why = "a rotation outside F32, Bf16 and F16", UNP_UNSUPPORTED_DTYPE;
  if (!index_ok(r.index_dtype, why)) return UNP_UNSUPPORTED_DTYPE;
  if (!layout_ok(r.layout, why)) return UNP_UNSUPPORTED_OP;
  if (r.inverse != 0 && r.inverse != 1) return why = "inverse is 0 or 1", UNP_UNSUPPORTED_KERNEL;
  if (r.head_dim < 2 || r.head_dim > 4096 || r.rot < 2 || r.rot % 2 != 0 || r.rot > r.head_dim)
    return why = "head_dim is 2..4096 and rot even, 2..head_dim", UNP_UNSUPPORTED_KERNEL;
  L.form.kind = UNP_FORM_ROPE;
  L.form.dtype = r.dtype;
  L.rope = r;
  const char *T = device_type(r.dtype), *I = device_type(r.index_dtype);
  L.name = std::string("unp_rope_") + short_name(r.dtype) + "_d" + std::to_string(r.head_dim) + "_r" +
           std::to_string(r.rot) + (r.layout == UNP_ROPE_HALVES ? "_halves" : "_pairs") + (r.inverse ? "_inv" : "") +
           "_" + short_name(r.index_dtype);
  std::ostringstream src;
  src << source_head(L.name);
  const int v = r.dtype == UNP_F32 ? 4 : 8;
  std::vector<std::string> when;
  auto add = [&](const char* tail, int vec, const char* cond) {
    Entry e;
    e.symbol = L.name + tail;
    e.fast = vec > 0;
    e.vec = vec;
    L.entries.push_back(e);
    when.push_back(cond);
    src << kBounds256 << e.symbol << "(const " << T << "* x, const " << I << "* positions, const float* table, " << T
        << "* out, unp4::rope_args a) {\n  unp4::rope<" << T << ", " << r.head_dim << ", " << r.rot << ", " << r.layout
        << ", " << (r.inverse ? "true" : "false") << ", " << I << ", " << vec << ">(x, positions, table, out, a);\n}\n";
  };
  if (r.rot / 2 % v == 0 && (r.head_dim - r.rot) % (2 * v) == 0)
    add("_v", v, "16-byte aligned buffers and strides of whole 16-byte vectors");
  add("_e", 0, "otherwise");
  L.source = src.str();
  const char *dt = kind_name(r.dtype), *ix = kind_name(r.index_dtype);
  L.interface_json = interface(
      L, "rope", "\"head_dim\":" + std::to_string(r.head_dim) + ",\"rot\":" + std::to_string(r.rot),
      {{"x", "Read", dt}, {"positions", "Read", ix}, {"table", "Read", "F32"}, {"out", "Write", dt},
       {"tokens", nullptr, "I64"}, {"heads", nullptr, "I64"}, {"x_token", nullptr, "I64"}, {"x_head", nullptr, "I64"},
       {"out_token", nullptr, "I64"}, {"out_head", nullptr, "I64"}, {"table_first", nullptr, "I64"},
       {"table_rows", nullptr, "I64"}},
      "lanes take pairs (vectors of them) in order and stride over the grid", when, nullptr,
      "f32 products and sums, rounded once to the type");
  return UNP_OK;
}

int32_t check_cache4(const unp_cache4& c, std::string& why) {
  if (c.dtype != UNP_BF16 && c.dtype != UNP_F16) return why = "a cache of values outside Bf16 and F16", UNP_UNSUPPORTED_DTYPE;
  if (!index_ok(c.index_dtype, why)) return UNP_UNSUPPORTED_DTYPE;
  if (c.kv_heads < 1 || c.kv_heads > 1024) return why = "kv_heads is 1..1024", UNP_UNSUPPORTED_KERNEL;
  if (c.head_dim < 32 || c.head_dim > 256 || c.head_dim % 32 != 0)
    return why = "head_dim is a multiple of 32, 32..256", UNP_UNSUPPORTED_KERNEL;
  if ((c.group != 32 && c.group != 64 && c.group != 128 && c.group != c.head_dim) || c.group < 1 ||
      c.head_dim % c.group != 0)
    return why = "group is 32, 64, 128 or head_dim, and divides head_dim", UNP_UNSUPPORTED_KERNEL;
  if (c.page != 16 && c.page != 32 && c.page != 64 && c.page != 128 && c.page != 256)
    return why = "page is 16, 32, 64, 128 or 256 tokens", UNP_UNSUPPORTED_KERNEL;
  return UNP_OK;
}

namespace {

std::string cache_name(const unp_cache4& c) {
  return std::string(short_name(c.dtype)) + "_h" + std::to_string(c.kv_heads) + "_d" + std::to_string(c.head_dim) + "_g" +
         std::to_string(c.group) + "_p" + std::to_string(c.page);
}
std::string cache_fields(const unp_cache4& c) {
  return "\"kv_heads\":" + std::to_string(c.kv_heads) + ",\"head_dim\":" + std::to_string(c.head_dim) +
         ",\"group\":" + std::to_string(c.group) + ",\"page\":" + std::to_string(c.page);
}
std::string cache_args(const unp_cache4& c) {
  return std::to_string(c.kv_heads) + ", " + std::to_string(c.head_dim) + ", " + std::to_string(c.group) + ", " +
         std::to_string(c.page);
}
const char* kAlignedWhen = "16-byte aligned keys and values, strides of whole 16-byte vectors";

}  // namespace

int32_t lower_cache4_append(const unp_cache4& c, int32_t rot, int32_t layout, Lowered& L, std::string& why) {
  L = Lowered{};
  if (const int32_t rc = check_cache4(c, why)) return rc;
  if (!layout_ok(layout, why)) return UNP_UNSUPPORTED_OP;
  if (rot < 0 || rot > c.head_dim || rot % 16 != 0)
    return why = "an append rotates 0..head_dim elements, a multiple of 16", UNP_UNSUPPORTED_KERNEL;
  L.form.kind = UNP_FORM_CACHE4_APPEND;
  L.form.dtype = c.dtype;
  L.cache4 = c;
  L.rope.rot = rot;
  const char *T = device_type(c.dtype), *I = device_type(c.index_dtype);
  L.name = "unp_cache4_append_" + cache_name(c) + "_r" + std::to_string(rot) +
           (layout == UNP_ROPE_HALVES ? "_halves_" : "_pairs_") + short_name(c.index_dtype);
  std::ostringstream src;
  src << source_head(L.name);
  for (int aligned = 1; aligned >= 0; --aligned) {
    Entry e;
    e.symbol = L.name + (aligned ? "_v" : "_e");
    e.fast = aligned != 0;
    L.entries.push_back(e);
    src << kBounds256 << e.symbol << "(const " << T << "* k, const " << T << "* v, const " << I
        << "* slots, unsigned* cache, const " << I
        << "* positions, const float* table, unp4::cache_args a) {\n  unp4::append<" << T << ", " << cache_args(c) << ", "
        << rot << ", " << layout << ", " << I << ", " << (aligned ? "true" : "false")
        << ">(k, v, slots, cache, positions, table, a);\n}\n";
  }
  L.source = src.str();
  const char *dt = kind_name(c.dtype), *ix = kind_name(c.index_dtype);
  std::vector<Param> ps = {{"k", "Read", dt}, {"v", "Read", dt}, {"slots", "Read", ix}, {"cache", "ReadWrite", "U8"}};
  if (rot > 0) {
    ps.push_back({"positions", "Read", ix});
    ps.push_back({"table", "Read", "F32"});
  }
  for (const char* s : {"tokens", "pages", "k_token", "k_head", "v_token", "v_head"}) ps.push_back({s, nullptr, "I64"});
  if (rot > 0)
    for (const char* s : {"table_first", "table_rows"}) ps.push_back({s, nullptr, "I64"});
  L.interface_json = interface(L, "cache4_append", cache_fields(c) + ",\"rot\":" + std::to_string(rot), ps,
                               "a word of 8 codes per lane; blocks stride over the heads", {kAlignedWhen, "otherwise"},
                               nullptr, "keys rotated in f64, rounded to f32 and then to their type; codes of correctly rounded quotients");
  return UNP_OK;
}

int32_t lower_cache4_read(const unp_cache4& c, Lowered& L, std::string& why) {
  L = Lowered{};
  if (const int32_t rc = check_cache4(c, why)) return rc;
  L.form.kind = UNP_FORM_CACHE4_READ;
  L.form.dtype = c.dtype;
  L.cache4 = c;
  const char *T = device_type(c.dtype), *I = device_type(c.index_dtype);
  L.name = "unp_cache4_read_" + cache_name(c) + "_" + short_name(c.index_dtype);
  std::ostringstream src;
  src << source_head(L.name);
  for (int aligned = 1; aligned >= 0; --aligned) {
    Entry e;
    e.symbol = L.name + (aligned ? "_v" : "_e");
    e.fast = aligned != 0;
    L.entries.push_back(e);
    src << kBounds256 << e.symbol << "(const " << I << "* slots, const unsigned* cache, " << T << "* k, " << T
        << "* v, unp4::cache_args a) {\n  unp4::read<" << T << ", " << cache_args(c) << ", " << I << ", "
        << (aligned ? "true" : "false") << ">(slots, cache, k, v, a);\n}\n";
  }
  L.source = src.str();
  const char *dt = kind_name(c.dtype), *ix = kind_name(c.index_dtype);
  std::vector<Param> ps = {{"slots", "Read", ix}, {"cache", "Read", "U8"}, {"k", "Write", dt}, {"v", "Write", dt}};
  for (const char* s : {"tokens", "pages", "k_token", "k_head", "v_token", "v_head"}) ps.push_back({s, nullptr, "I64"});
  L.interface_json = interface(L, "cache4_read", cache_fields(c), ps, "a word of 8 codes per lane, striding over the grid",
                               {kAlignedWhen, "otherwise"}, nullptr,
                               "exact integer difference and f32 product; one round-to-nearest-even to the type: bit-exact");
  return UNP_OK;
}

int32_t lower_cache4_attention(const unp_cache4& c, const unp_attention& a, Lowered& L, std::string& why) {
  L = Lowered{};
  if (const int32_t rc = check_cache4(c, why)) return rc;
  if (a.heads < c.kv_heads || a.heads % c.kv_heads != 0 || a.heads / c.kv_heads > 128)
    return why = "heads is kv_heads times 1..128", UNP_UNSUPPORTED_KERNEL;
  if ((a.causal != 0 && a.causal != 1) || (a.lse != 0 && a.lse != 1))
    return why = "causal and lse are 0 or 1", UNP_UNSUPPORTED_KERNEL;
  if (a.scale != 0.0 && !(a.scale >= 0x1p-24 && a.scale <= 0x1p24))
    return why = "the scale is 0 (1 / sqrt(head_dim)) or lies in 2^-24..2^24", UNP_UNSUPPORTED_KERNEL;
  L.form.kind = UNP_FORM_CACHE4_ATTENTION;
  L.form.dtype = c.dtype;
  L.cache4 = c;
  L.attention = a;
  L.attention.scale = a.scale == 0.0 ? 1.0 / std::sqrt((double)c.head_dim) : a.scale;
  const char* T = device_type(c.dtype);
  L.name = "unp_cache4_attention_" + cache_name(c) + "_q" + std::to_string(a.heads) + (a.causal ? "_causal" : "_full") +
           (a.lse ? "_lse" : "");
  std::ostringstream src;
  src << source_head(L.name);
  const std::string same = std::string(T) + ", " + std::to_string(c.kv_heads) + ", " + std::to_string(a.heads) + ", " +
                           std::to_string(c.head_dim);
  const char* lse = a.lse ? "true" : "false";
  // cg groups of columns hold the same 16 / cg rows (few rows); wk waves share a block's rows, or wr have their own.
  auto add = [&](const char* tail, int qt, int cg, int wr, int wk, bool once, int per_simd) {
    Entry e;
    e.symbol = L.name + tail;
    e.threads = 64 * wr * wk;
    e.vec = 16 / cg * qt * wr;  // rows of a block
    e.k = wk * 32 * cg;         // keys of a block's step
    L.entries.push_back(e);
    src << "extern \"C\" __global__ void __launch_bounds__(" << e.threads << ", " << per_simd << ") " << e.symbol
        << "(const " << T
        << "* q, const unsigned* cache, const int* table, const int* starts, const int* lengths, " << T
        << "* out, float* lse, float* ws, float scale, unp4::attention_args a) {\n  unp4::attend<" << same << ", " << c.group
        << ", " << c.page << ", " << (a.causal ? "true" : "false") << ", " << lse << ", " << qt << ", " << cg << ", " << wr
        << ", " << wk << ", " << (once ? "true" : "false") << ">(q, cache, table, starts, lengths, out, lse, ws, scale, a);\n}\n";
  };
  const int gq = a.heads / c.kv_heads;
  // What a wave holds, in registers: the words of a step, the rows, their sums and the words of groups.  The kernels
  // take about 60 more, and two waves of a SIMD have 256 each (a SIMD's one wave of twice the rows took 646 us for
  // prompts that two take 380 for).  A whole head of 192 is at 204: two of its tiles keep up to 50 words in scratch and
  // are mostly the faster (three prompts of up to 4099 tokens x 16 heads over 8 Bf16 280 us, 315 with one, F16 335 and 328;
  // 16 sequences of up to 100 rows over 6000 keys 112 and 168, 128 and 172).
  const int deep = c.head_dim / 32, groups = c.head_dim / c.group, words = c.group / 8, rest = words % 16;
  const int tiles = groups * (words / 16 + (rest > 0));
  const int products = groups * (words / 16 * 8 + (rest == 0 ? 0 : rest <= 4 ? 2 : rest <= 8 ? 4 : 8));
  auto held = [&](int cg, int qt) {
    return 2 * cg * (deep + 4 * tiles) + qt * (4 * deep + 4 * products + (cg == 1 ? 8 * groups : 0)) + 16 * groups;
  };
  // As many groups of columns as leave room for a row each, as far as they fit; two row tiles a wave if they fit.
  int cg = gq <= 4 ? 4 : gq <= 8 ? 2 : 1;
  while (cg > 1 && held(cg, 1) > 176) cg /= 2;
  add("_few", 1, cg, 1, 4, true, held(cg, 1) <= 204 ? 2 : 1);
  // For sequences of several tiles, whose blocks read the same keys: through the caches, and of one row a column where the first
  // shares them (32 heads over 2, 64 sequences of up to 2 and 4 tokens over 3000 keys 22.7 and 29.2 us, past the caches 26.1 and
  // 33.0; heads of 192, groups of 64, up to 16 tokens 140 and 152).
  const int qt = held(1, 2) <= 204 ? 2 : 1, per_simd = held(1, qt) <= 204 ? 2 : 1;
  const bool some = cg > 1 || qt > 1;  // else `_more` has the same tiles
  if (some) add(cg > 1 ? "_some" : "_cached_few", 1, 1, 1, 4, false, held(1, 1) <= 204 ? 2 : 1);
  add("_more", qt, 1, 1, 4, false, per_simd);
  add("_many", qt, 1, 4, 1, false, per_simd);
  Entry e;
  e.symbol = L.name + "_join";
  L.entries.push_back(e);
  src << kBounds256 << e.symbol << "(const int* starts, " << T
      << "* out, float* lse, float* ws, unp4::attention_args a) {\n  unp4::join<" << same << ", " << lse
      << ">(starts, out, lse, ws, a);\n}\n";
  L.source = src.str();
  std::vector<std::string> when = {"a sequence has no more rows of a key/value head, on average, than one of its tiles"};
  if (some) when.push_back("at most one of its tiles, or four over a long context");
  when.push_back("a long context and at most eight of its tiles, or too few blocks of the next");
  when.push_back("otherwise");
  when.push_back("after any of them, where a context is split");
  const char* dt = kind_name(c.dtype);
  std::vector<Param> ps = {{"q", "Read", dt}, {"cache", "Read", "U8"}, {"page_table", "Read", "I32"},
                           {"starts", "Read", "I32"}, {"lengths", "Read", "I32"}, {"out", "Write", dt}};
  if (a.lse) ps.push_back({"lse", "Write", "F32"});
  ps.push_back({"workspace", "ReadWrite", "U8"});
  for (const char* s : {"tokens", "batch", "width", "pages", "q_token", "q_head", "out_token", "out_head", "window",
                        "workspace_bytes"})
    ps.push_back({s, nullptr, "I64"});
  L.interface_json =
      interface(L, "cache4_attention", cache_fields(c) + ",\"heads\":" + std::to_string(a.heads), ps,
                "a block per row tile, part of a context and key/value head",
                when,
                "the caller's, by unp_hip_exec_workspace",
                "scores, softmax statistics and sums in f32, probabilities times value scales as f16 in the products; each output rounded once");
  return UNP_OK;
}

}  // namespace unp
