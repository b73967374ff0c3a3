// unpopped-hip device library of the floating point products (gfx950, wave64): quantisation to 8 bits, products of
// 8-bit codes with scales, products grouped by expert, and the rows of each expert.
//
// The emitter writes these forms' sources as this library + the `extern "C" __global__` entries that
// instantiate its templates, as it does with the fold and scan library for the lifted forms.
//
// Numerics: block scales and quotients in f32, correctly rounded; products of 16-bit numbers and their sums in the matrix
// unit's f32.  Products of 8-bit codes it takes to 2^-13 of the largest of 16 neighbours, and sums those sums in f32; the
// scales and the sums over blocks are f32 multiply-adds.  Each output rounded once.

#if !defined(__HIPCC_RTC__)
#include <hip/hip_runtime.h>
#endif

namespace unpm {

typedef unsigned char u8;
typedef unsigned short u16;
typedef unsigned int u32;
typedef unsigned long long u64;
typedef int i32;
typedef long long i64;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef u32 u32x2 __attribute__((ext_vector_type(2)));
typedef u32 u32x4 __attribute__((ext_vector_type(4)));
typedef i32 i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

#define UNPM_DEV __device__ __forceinline__

enum : int { BF16 = 0, F16 = 1, E4M3 = 2, E5M2 = 3 };

template <class To, class From> UNPM_DEV To bits(const From& x) {
  static_assert(sizeof(To) == sizeof(From), "bits");
  To y;
  __builtin_memcpy(&y, &x, sizeof(To));
  return y;
}
template <int N> UNPM_DEV void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// Every wave's LDS accesses are done, and none of a later one begins before it.
UNPM_DEV void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
UNPM_DEV u32 lds_address(const void* p) { return (u32)(size_t)(lds_void*)p; }
UNPM_DEV i64 least(i64 a, i64 b) { return a < b ? a : b; }
UNPM_DEV u32 more(u32 a, u32 b) { return a > b ? a : b; }
// What every lane of a wave has, in scalar registers.
UNPM_DEV u32 scalar(u32 x) { return __builtin_amdgcn_readfirstlane(x); }
UNPM_DEV i64 uniform(i64 x) {
  return (i64)((u64)(u32)__builtin_amdgcn_readfirstlane((i32)(x >> 32)) << 32 | (u32)__builtin_amdgcn_readfirstlane((i32)x));
}

// ---------------------------------------------------------------------------------------
// Products: out[i][j] = sum over d of x[i][d] * w[j][d], of 16-bit numbers, or of 8-bit codes with an f32 scale for 128
// elements along d.
//
// A block makes a TM x TN tile of out.  A step is 128 bytes along d of every row of both tiles, in LDS; an operand whose
// rows run along out instead (transposed: the gradients') lies there as it does in memory, 64 of its rows a step, and
// is turned by the transposing LDS read.  16 bytes of a row of the tile lie at a slot that its row permutes, so that the 16
// rows that a matrix instruction's lanes read lie in different banks.
//
// w gives the instruction's rows and x its columns: a lane then holds four adjacent columns of one row of out, so it
// stores them at once and a scale of x is one number per tile of 16 x 16.  The products of 128 codes are summed by the
// matrix unit from zero and then added, times both scales, to the f32 sums: four multiply-adds beside the 32 cycles of the
// instruction.
// ---------------------------------------------------------------------------------------
struct product_args {
  i64 m, n, depth;                 // rows and columns of out (by group where the depth is grouped), elements along d
  i64 x_row, w_row, w_group;       // strides in bytes
  i64 xs_row, ws_row, ws_group;    // of the scales, in elements
  i64 out_row, out_group;          // in elements
  i32 groups, tiles_m, tiles_n, parts;
  i32 wide;                        // out takes vectors of 16 bytes: 1, or 2 past the caches
  i32 tail;                        // bytes of a row's last 16 along d that exist, where not all do
  i32 turn, pad;                   // steps by which neighbouring columns of tiles begin apart
};

constexpr u32 OUTSIDE = 0x80000000u;  // an offset past every buffer: loads of it give zeros

UNPM_DEV u32x4 resource(const u8* p) {
  const u64 a = (u64)p;
  return u32x4{scalar((u32)a), scalar((u32)(a >> 32) & 0xFFFFu), OUTSIDE, 0x00020000u};
}
// 16 bytes of each lane from p + offset to LDS, lane after lane from `to` on; zeros where the offset is OUTSIDE.  (Nothing
// else here uses M0, which no clobber list may name.)  A scalar register that a vector instruction wrote, as reading the
// first lane or a spilled register back does, may be read by a load or store five wait states later; within assembly the
// compiler adds none.
UNPM_DEV void load_to_lds(const u8* p, u32 offset, u32 to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(scalar(to)), "v"(offset),
               "s"(resource(p))
               : "memory");
}
UNPM_DEV void load_word_to_lds(const float* p, u32 to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(scalar(to)), "v"(p) : "memory");
}

// 16 bytes at p, aligned or not, of which `there` exist (elements of E bytes), zeros for the others.
template <int E> UNPM_DEV u32x4 fetch16(const u8* p, i64 there) {
  u32x4 x = {0, 0, 0, 0};
  if (there >= 16) {
    __builtin_memcpy(&x, p, 16);
    return x;
  }
#pragma unroll
  for (int i = 0; i < 16; i += E)
    if (i < there) {
      const u32 v = E == 1 ? (u32)p[i] : (u32) * reinterpret_cast<const u16*>(p + i);
      x[i / 4] |= v << (i % 4 * 8);
    }
  return x;
}

// Where the 16 bytes of a tile's row lie: a row of 128 bytes along d has 8 slots, and the slot of a chunk goes by bits 1 to
// 3 of the row (bit 0 is half of the banks).  Then the 16 lanes that one cycle of a read serves, eight rows' chunk g and eight
// others' chunk g + 1, are in different banks.  A transposed row (2 T bytes) moves pairs of slots: the four rows that 16
// lanes read, and the four that lie eight further, are in different banks.
UNPM_DEV int straight_slot(int row, int chunk) { return chunk ^ ((row >> 1) & 7); }
template <int T> UNPM_DEV int turned_slot(int row, int chunk) {
  constexpr int PAIRS = T / 16;
  const int f = PAIRS >= 8 ? (row & 3) | ((row >> 3) & 1) << 2 : row & (PAIRS - 1);
  return chunk ^ (f << 1);
}

// One operand's tile: T rows of out's axis, 128 bytes along d.
template <int KIND, bool TURNED, int T> struct side {
  static constexpr int E = KIND >= E4M3 ? 1 : 2;  // bytes of an element
  static constexpr int D = 128 / E;               // elements of a step
  static constexpr int BYTES = T * 128, UNITS = BYTES / 1024;
  static constexpr int CHUNKS = TURNED ? T * 2 / 16 : 8;  // of a row in LDS
  static_assert(!TURNED || E == 2, "8-bit codes lie along d");
  const u8* p;      // the tile's first element
  i64 row;          // stride in bytes
  i64 there;        // rows of the tile that exist (TURNED: bytes of its columns)

  // Lane `lane` of unit u: the row and the chunk that lie at its 16 bytes.
  static UNPM_DEV int row_of(int u, int lane) { return u * (64 / CHUNKS) + lane / CHUNKS; }
  static UNPM_DEV int chunk_of(int u, int lane) {
    const int r = row_of(u, lane), s = lane % CHUNKS;
    return TURNED ? turned_slot<T>(r, s) : straight_slot(r, s);
  }
  // The offset of the lane's 16 bytes from the step's first; OUTSIDE where its row or column does not exist.  The tile's row
  // (TURNED: chunk of columns) i is number map(i) from p on.
  template <class M> UNPM_DEV u32 offset(int u, int lane, M map) const {
    const int r = TURNED ? row_of(u, lane) : map(row_of(u, lane)), c = TURNED ? map(chunk_of(u, lane)) : chunk_of(u, lane);
    const bool in = TURNED ? c * 16 < there : r < there;
    return in ? (u32)(r * (i32)row + c * 16) : OUTSIDE;
  }
  UNPM_DEV u32 offset(int u, int lane) const {
    return offset(u, lane, [](int i) { return i; });
  }
  // What of the step's length has to be left for the lane's 16 bytes to exist, in bytes or TURNED rows.
  static UNPM_DEV int after(int u, int lane) { return TURNED ? row_of(u, lane) : chunk_of(u, lane) * 16; }
  static UNPM_DEV i64 left(i64 elements) { return TURNED ? elements : elements * E; }
  static UNPM_DEV bool exists(int after, i64 left) { return TURNED ? after < left : after + 16 <= left; }
  // Row r of the last step: the first `bytes` of 16 that do not all exist, which no load to LDS took (it wrote zeros).
  UNPM_DEV void patch(u8* lds, int r, i64 step, i64 elements, int bytes) const {
    if (TURNED || r >= there) return;
    const int c = (int)elements * E / 16;
    const u8* from = at(step) + r * row + c * 16;
    u8* to = lds + r * 128 + straight_slot(r, c) * 16;
#pragma clang loop unroll(disable)
    for (int i = 0; i < bytes; i += E) {
      if constexpr (E == 1)
        to[i] = from[i];
      else
        *reinterpret_cast<u16*>(to + i) = *reinterpret_cast<const u16*>(from + i);
    }
  }
  // 16 bytes (the q-th) of a step that holds those alone, as its first elements along d.
  template <class M> UNPM_DEV void alone(u8* lds, int q, i64 step, i64 elements, M map) const {
    const i64 first = elements * E / 16 * (16 / E);
    u32x4 v = {0, 0, 0, 0};
    const int r = q / CHUNKS, c = q % CHUNKS;
    if constexpr (TURNED) {
      const int from = map(c);
      if (r < elements - first) v = fetch16<E>(at(step) + (first + r) * row + from * 16, there - from * 16);
      *reinterpret_cast<u32x4*>(lds + r * (T * 2) + turned_slot<T>(r, c) * 16) = v;
    } else {
      const int from = map(r);
      if (c == 0 && from < there) v = fetch16<E>(at(step) + from * row + first * E, (elements - first) * E);
      *reinterpret_cast<u32x4*>(lds + r * 128 + straight_slot(r, c) * 16) = v;
    }
  }
  UNPM_DEV const u8* at(i64 step) const { return p + (TURNED ? step * D * row : step * 128); }
  UNPM_DEV u32x4 fetch(int u, int lane, i64 step, i64 elements) const {
    const int r = row_of(u, lane), c = chunk_of(u, lane);
    const i64 bytes = TURNED ? (r < elements ? there - c * 16 : 0) : (r < there ? elements * E - c * 16 : 0);
    return fetch16<E>(at(step) + r * row + c * 16, bytes);
  }

  // The 16 bytes of lane (i, g) for the matrix instruction: half h of the step of tile row first + i.
  static UNPM_DEV u32x4 read(const u8* lds, int first, int h, int lane) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (TURNED) {
      // Four rows of d by 16 columns a read: each lane names 8 bytes of one of them and takes a column.
      u32x4 v;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int d = h * 32 + g * 8 + q * 4 + i / 4, c = first / 8 + i % 4 / 2;
        const u8* a = lds + d * (T * 2) + turned_slot<T>(d, c) * 16 + i % 2 * 8;
        const u32x2 t = bits<u32x2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_void*)a));
        v[2 * q] = t[0];
        v[2 * q + 1] = t[1];
      }
      return v;
    } else {
      return *reinterpret_cast<const u32x4*>(lds + (first + i) * 128 + straight_slot(first + i, h * 4 + g) * 16);
    }
  }
};

template <int KIND> UNPM_DEV f32x4 multiply(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (KIND == BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bits<bf16x8>(a), bits<bf16x8>(b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(bits<f16x8>(a), bits<f16x8>(b), c, 0, 0, 0);
}
// 128 codes of each: the scales of the instruction itself are not used.
template <int KA, int KB> UNPM_DEV f32x4 multiply8(const u32x4 (&a)[2], const u32x4 (&b)[2]) {
  struct both {
    u32x4 v[2];
  };
  const i32x8 x = bits<i32x8>(both{{a[0], a[1]}}), y = bits<i32x8>(both{{b[0], b[1]}});
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, f32x4{0, 0, 0, 0}, KA - E4M3, KB - E4M3, 0, 0, 0, 0);
}

// A block's sum of codes times both scales, added to the sum of blocks.  One multiply-add with the product of the scales serves
// where that is a normal number, as that of scales from 2^-63 up to 2^64 is, and for zeros, infinities and NaN.  Scales beyond
// are rare, but their product may be outside f32 where its product with a sum of up to 2^39 is not: add_far gives the sum their
// exponents and multiplies by the product of their fractions.  The waves of a tile look at the scales that they loaded, and
// a tile with one beyond is made again with add_far once its sums are there.  That gives the same bits where one multiply-add serves
// (and the result is above 2^-124), so a row's do not go by its neighbours' scales.  Looking takes up to 3 % of a launch of
// a few hundred rows (1024 x 4096 x 4096 32.8 us, 31.8 without) and nothing that shows of 8192^3; a choice inside the loop took
// 36 registers more than there are.
UNPM_DEV u32 reach(float scale) { return (u32)(__builtin_amdgcn_frexp_expf(scale) + 62); }  // above 126: beyond
struct parts_of {
  float fraction;  // 1 to 2
  i32 exponent;
};
UNPM_DEV parts_of taken_apart(float scale) {  // of 0 an exponent that no other's makes up for
  return {2.0f * __builtin_amdgcn_frexp_mantf(scale), scale == 0.0f ? -1000 : __builtin_amdgcn_frexp_expf(scale) - 1};
}
UNPM_DEV void add_far(f32x4& sum, const f32x4& p, float a, const f32x4& b) {
  const parts_of x = taken_apart(a);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const parts_of y = taken_apart(b[j]);
    sum[j] = __builtin_fmaf(__builtin_amdgcn_ldexpf(p[j], x.exponent + y.exponent), x.fraction * y.fraction, sum[j]);
  }
  __builtin_amdgcn_sched_barrier(0);  // in fewer registers
}
template <bool B> struct choice {
  static constexpr bool value = B;
};

// Blocks are dealt to the 8 XCDs in turn.  Each takes a run of as many neighbouring tiles as its CUs hold at once, so that
// its L2 holds what they share; the runs of the XCDs lie side by side, so that groups of any size load them alike.
// Tiles are counted in bands of 8 along out's rows.
struct tile_at {
  i64 m, n;
  int part;
};
template <u32 RUN> UNPM_DEV bool tile_of(const product_args& a, u32 tiles_m, tile_at& at) {
  const u32 tiles = tiles_m * (u32)a.tiles_n, all = tiles * (u32)a.parts, b = blockIdx.x;
  if (b >= all) return false;
  const u32 turn = b / (8 * RUN) * (8 * RUN), in = b - turn, rest = all - turn;
  u32 id = turn;
  if (rest >= 8 * RUN) {
    id += in % 8 * RUN + in / 8;
  } else {  // the last turn: runs as equal as they can be
    const u32 each = rest / 8, more = rest % 8, xcd = in % 8;
    id += xcd * each + (xcd < more ? xcd : more) + in / 8;
  }
  const u32 part = id / tiles, t = id % tiles;
  constexpr u32 BAND = 8;
  const u32 per = BAND * (u32)a.tiles_n, band = t / per, of = t % per;
  const u32 first = band * BAND, high = tiles_m - first < BAND ? tiles_m - first : BAND;
  at = {(i64)(first + of % high), (i64)(of / high), (int)part};
  return true;
}

// The rows of group g, whatever the starts are: within 0 .. rows.
UNPM_DEV void group_rows(const i32* starts, int g, i64 rows, i64& r0, i64& r1) {
  r0 = least(starts[g] < 0 ? 0 : starts[g], rows);
  r1 = least(starts[g + 1] < 0 ? 0 : starts[g + 1], rows);
}
// How many tiles of T rows this lane's group has, of the 64 groups from `first` on, and how many those up to it have.  A start
// below an earlier one, of which `floor` is the largest before these, counts as that one: so no row is two groups', each from the
// first start to the largest is one's, and there are no more tiles than the launch has.
struct tiles_upto {
  i32 own, upto;
  i64 r0, r1;
};
template <int T> UNPM_DEV tiles_upto group_tiles(const i32* starts, int groups, i64 rows, int first, i32 floor) {
  const int lane = threadIdx.x & 63;
  const bool in = first + lane < groups;
  tiles_upto t{0, 0, 0, 0};
  if (in) group_rows(starts, first + lane, rows, t.r0, t.r1);
  if (__any(in && (t.r1 < t.r0 || t.r0 < floor))) {
    i32 top = t.r0 < floor ? floor : (i32)t.r0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const i32 v = __shfl_up(top, d);
      if (lane >= d && v > top) top = v;
    }
    t.r0 = top;
    if (t.r1 < top) t.r1 = top;
  }
  t.own = t.r1 > t.r0 ? (i32)((t.r1 - t.r0 + T - 1) / T) : 0;
  t.upto = t.own;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const i32 v = __shfl_up(t.upto, d);
    if (lane >= d) t.upto += v;
  }
  return t;
}
// This block's tile of T rows of the groups that have rows: its place, group and rows, or none.  Every wave finds it alike.
template <int T, u32 RUN>
UNPM_DEV bool find_group(const i32* starts, const product_args& a, tile_at& at, int& group, i64& r0, i64& r1) {
  tiles_upto t = group_tiles<T>(starts, a.groups, a.m, 0, 0);
  const tiles_upto low = t;
  i64 all = __shfl(t.upto, 63);
  for (int first = 64; first < a.groups; first += 64) {
    t = group_tiles<T>(starts, a.groups, a.m, first, __shfl((i32)t.r1, 63));
    all += __shfl(t.upto, 63);
  }
  if (!tile_of<RUN>(a, scalar((u32)all), at)) return false;
  i64 past = 0;
  t = low;
  for (int first = 0;; first += 64) {
    if (first > 0) t = group_tiles<T>(starts, a.groups, a.m, first, __shfl((i32)t.r1, 63));
    const u64 has = __ballot(past + t.upto > at.m);
    if (has) {
      const int l = __builtin_ctzll(has);
      group = first + l;
      const i64 tile = at.m - past - (__shfl(t.upto, l) - __shfl(t.own, l));
      r0 = uniform(__shfl((i32)t.r0, l) + tile * T);
      r1 = uniform(__shfl((i32)t.r1, l));
      return true;
    }
    past += __shfl(t.upto, 63);
    if (first + 64 >= a.groups) return false;
  }
}

// N adjacent columns of out, `there` of which exist; `wide`: out takes vectors of 16 bytes, 2: and is larger than what the
// caches keep (12001 x 8192 results of 16 bits 380 us past them, 394 through; 16 x 8192 x 2048 of 32 bits 482 and 536).
template <class OUT, int N> UNPM_DEV void store_columns(OUT* p, const float (&v)[N], i64 there, i32 wide) {
  constexpr int V = 16 / sizeof(OUT);
  struct alignas(16) vec {
    OUT v[V];
  };
#pragma unroll
  for (int i = 0; i < N; i += V) {
    vec q;
#pragma unroll
    for (int j = 0; j < V; ++j) q.v[j] = (OUT)v[i + j];
    if (wide == 2 && there >= i + V) {
      __builtin_nontemporal_store(bits<u32x4>(q), reinterpret_cast<u32x4*>(p + i));
    } else if (wide && there >= i + V) {
      *reinterpret_cast<vec*>(p + i) = q;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (i + j < there) p[i + j] = q.v[j];
    }
  }
}

enum : int { ALL = 0, ROWS = 1, DEPTH = 2 };  // what the groups divide: nothing, the rows of x and out, the depth

// One block's part of the work.
template <int XK, int WK_, bool XT, bool WT, int BY, int TM, int TN> struct place {
  side<XK, XT, TM> x;
  side<WK_, WT, TN> w;
  const float *xs, *ws;  // scales of the first rows
  i64 xs_last, ws_last;  // the tile's last rows that have scales
  i64 first, last;       // steps
  i64 end, depth;        // elements along d up to this part's end, and in all
  i64 m0, n0, m_there;   // the tile in out
  i64 row0;              // the tile's first row among all rows (of all groups) of the result
};

template <int XK, int WKIND, bool XT, bool WT, int BY, int SB, int TM, int TN, u32 RUN>
UNPM_DEV bool find_place(const u8* x, const u8* w, const float* xs, const float* ws, const i32* starts,
                         const product_args& a, int& part, place<XK, WKIND, XT, WT, BY, TM, TN>& o) {
  constexpr int E = XK >= E4M3 ? 1 : 2, D = 128 / E;
  tile_at t;
  i64 depth = a.depth;
  if constexpr (BY == ROWS) {
    int g;
    i64 r0, r1;
    if (!find_group<TM, RUN>(starts, a, t, g, r0, r1)) return false;
    g = __builtin_amdgcn_readfirstlane(g);
    o.m0 = o.row0 = r0;
    o.m_there = r1 - r0;
    w += g * a.w_group;
    ws += g * a.ws_group;
  } else {
    if (!tile_of<RUN>(a, (u32)a.tiles_m, t)) return false;
    o.m0 = t.m * TM;
    o.row0 = o.m0;
    if constexpr (BY == DEPTH) {
      const u32 each = (u32)a.tiles_m / (u32)a.groups, g = (u32)t.m / each;
      i64 r0, r1;
      group_rows(starts, (int)g, a.depth, r0, r1);
      r0 = uniform(r0);
      r1 = uniform(r1);
      depth = r1 > r0 ? r1 - r0 : 0;
      o.m0 = (t.m - g * each) * TM;
      o.row0 = g * a.m + o.m0;
      x += r0 * a.x_row;
      w += r0 * a.w_row;
    }
    o.m_there = a.m - o.m0;
  }
  part = t.part;
  o.n0 = t.n * TN;
  const i64 n_there = a.n - o.n0;
  if (o.m_there > TM) o.m_there = TM;
  o.x.p = XT ? x + o.m0 * 2 : x + o.m0 * a.x_row;
  o.x.row = a.x_row;
  o.x.there = XT ? o.m_there * 2 : o.m_there;
  o.w.p = WT ? w + o.n0 * 2 : w + o.n0 * a.w_row;
  o.w.row = a.w_row;
  o.w.there = WT ? n_there * 2 : n_there;
  if constexpr (E == 1) {
    o.xs = xs + o.m0 * a.xs_row;
    o.xs_last = o.m_there - 1;
    o.ws = ws + o.n0 / SB * a.ws_row;
    o.ws_last = ((n_there < TN ? n_there : TN) - 1) / SB;
  }
  const i64 steps = (depth + D - 1) / D;
  o.first = steps * part / a.parts;
  o.last = steps * (part + 1) / a.parts;
  o.end = least(depth, o.last * D);
  o.depth = depth;
  return true;
}

// A tile's sums in LDS, [SPLIT][TM][TN] in f32: a row's quads of columns are moved by the row's low bits, so that the 16 rows
// that a wave's sums of a 16 x 16 product lie in are in different banks.
template <int TM, int TN> UNPM_DEV int sum_at(int split, int m, int n) {
  constexpr int Q = TN / 4 < 16 ? TN / 4 : 16;
  return (split * TM + m) * TN + ((n / 4) ^ (m & (Q - 1))) * 4;
}
// From there to out, or where the depth is split to this part's sums: whole rows at a time, as columns written where the
// matrix instruction leaves them would be 32 bytes of each of 16 rows (a launch of 12001 x 8192 results of 16 bits took 468 us,
// 343 without its stores).  Row 0 of the sums is row `first` of the block's tile.
template <class OUT, int BY, int TM, int TN, int SPLIT, int THREADS>
UNPM_DEV void store_sums(const float* sums, OUT* out, float* parts, const product_args& a, int part, i64 row0, i64 m0, i64 n0,
                         i64 m_there, int first) {
  constexpr int V = 16 / sizeof(OUT) < TN ? 16 / sizeof(OUT) : TN;
  for (int q = threadIdx.x; q < TM * TN / V; q += THREADS) {
    const int m = q / (TN / V), n = q % (TN / V) * V;
    const i64 there = a.n - n0 - n;
    if (first + m >= m_there || there <= 0) continue;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      f32x4 t = *reinterpret_cast<const f32x4*>(sums + sum_at<TM, TN>(0, m, n + i));
#pragma unroll
      for (int s = 1; s < SPLIT; ++s) t += *reinterpret_cast<const f32x4*>(sums + sum_at<TM, TN>(s, m, n + i));
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i + j] = t[j];
    }
    if (a.parts > 1) {
      const i64 rows = BY == DEPTH ? a.groups * a.m : a.m, wide = (a.n + 7) / 8 * 8;
      float* p = parts + (part * rows + row0 + first + m) * wide + n0 + n;
#pragma unroll
      for (int i = 0; i < V; i += 4) *reinterpret_cast<f32x4*>(p + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    } else {
      const i64 g = BY == DEPTH ? (row0 - m0) / a.m : 0;
      store_columns<OUT>(out + g * a.out_group + (m0 + first + m) * a.out_row + n0 + n, v, there, a.wide);
    }
  }
}

// WM x WN waves share the tile; SPLIT sets of them take the steps in turn and meet in LDS at the end.  STAGES of
// SPLIT steps lie in LDS at once: DIRECT loads go there without registers, STAGES - 1 ahead of the products.  The others
// take rows of any alignment, strides and lengths through registers.
template <int XK, int WKIND, bool XT, bool WT, class OUT, int BY, int SB, int TM, int TN, int WM, int WN, int SPLIT, int STAGES,
          bool DIRECT>
UNPM_DEV void matmul(const u8* xp, const u8* wp, const float* xsp, const float* wsp, const i32* starts, OUT* out, float* parts,
                     const product_args& a) {
  constexpr int WAVES = WM * WN * SPLIT, E = XK >= E4M3 ? 1 : 2, D = 128 / E;
  constexpr int MT = TM / WM / 16, NT = TN / WN / 16;
  typedef side<XK, XT, TM> xside;
  typedef side<WKIND, WT, TN> wside;
  constexpr int SET = WM * WN;  // waves of a step
  constexpr int STEP = xside::BYTES + wside::BYTES, SCALES = E == 1 ? WAVES * 256 : 0, STAGE = SPLIT * STEP + SCALES;
  constexpr int UNITS = xside::UNITS + wside::UNITS, EACH = UNITS / SET;
  static_assert(UNITS % SET == 0, "whole units a wave");
  static_assert(E == 2 || TM + TN <= SET * 64, "a scale a lane");
  static_assert(SPLIT * TM * TN * 4 <= STAGES * STAGE, "the sums of split steps");
  __shared__ __attribute__((aligned(1024))) u8 lds[STAGES * STAGE];
  __shared__ u32 farthest[WAVES];

  place<XK, WKIND, XT, WT, BY, TM, TN> o;
  int part;
  if (!find_place<XK, WKIND, XT, WT, BY, SB, TM, TN, 64>(xp, wp, xsp, wsp, starts, a, part, o)) return;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int in_set = wave % SET, own = wave / SET, wm = in_set % WM, wn = in_set / WM;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0, 0, 0, 0};

  // This lane's part of a step: every wave loads for the set of waves that multiply it.
  const u8* from[EACH];
  u32 offset[EACH];
  i32 after[EACH];
  const u32 lds0 = lds_address(lds);
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int u = i * SET + in_set;
    if (u < xside::UNITS) {
      from[i] = o.x.p;
      offset[i] = o.x.offset(u, lane);
      after[i] = xside::after(u, lane);
    } else {
      from[i] = o.w.p;
      offset[i] = o.w.offset(u - xside::UNITS, lane);
      after[i] = wside::after(u - xside::UNITS, lane);
    }
  }
  const float* scale = nullptr;
  if constexpr (E == 1) {
    // A scale that no row has is another's: it multiplies rows that are not stored.
    const int f = in_set * 64 + lane, r = f < TM + TN ? f : 0;
    scale = r < TM ? o.xs + least(r, o.xs_last) * a.xs_row : o.ws + least((r - TM) / SB, o.ws_last) * a.ws_row;
  }
  // The steps in order, or from one on that a block's column of tiles sets: blocks that read weights at one place of rows
  // that lie 2^k bytes apart meet in a few memory channels (64 rows by 28672 x 8192 codes 57.2 us, 48.2 from different ones).
  const i32 steps = (i32)(o.last - o.first);
  const i32 turn = steps > 0 ? (i32)((u32)(o.n0 / TN) * (u32)a.turn % (u32)steps) : 0;
  auto issue = [&](i32 stage, int slot) {
    const i32 at = stage * SPLIT + own, l = at + turn;
    const i64 step = o.first + (l >= steps ? l - steps : l);
    const i64 left = at < steps ? o.end - step * D : 0;
    const int base = slot * STAGE + own * STEP;
    const i64 x_off = XT ? step * D * a.x_row : step * 128, w_off = WT ? step * D * a.w_row : step * 128;
    const i32 x_left = (i32)xside::left(least(left, D)), w_left = (i32)wside::left(least(left, D));
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int u = i * SET + in_set;
      const bool isx = u < xside::UNITS;
      if constexpr (DIRECT) {
        const bool in = isx ? xside::exists(after[i], x_left) : wside::exists(after[i], w_left);
        load_to_lds(from[i] + (isx ? x_off : w_off), in ? offset[i] : OUTSIDE, lds0 + base + u * 1024);
      } else {
        const u32x4 y = isx ? o.x.fetch(u, lane, step, left) : o.w.fetch(u - xside::UNITS, lane, step, left);
        *reinterpret_cast<u32x4*>(lds + base + u * 1024 + lane * 16) = y;
      }
    }
    if constexpr (E == 1) {
      // Behind the last step there are zeros, whose scale is another's too.
      const float* p = scale + (at < steps ? step : o.first);
      const int to = slot * STAGE + SPLIT * STEP + wave * 256;
      if constexpr (DIRECT)
        load_word_to_lds(p, lds0 + to);
      else
        *reinterpret_cast<float*>(lds + to + lane * 4) = *p;
    }
  };
  u32 far = 0;  // the farthest of the scales that this wave loaded
  auto compute = [&](int slot, auto again) {
    const u8* xl = lds + slot * STAGE + own * STEP;
    const u8* wl = xl + xside::BYTES;
    if constexpr (E == 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 xf[MT], wf[NT];
#pragma unroll
        for (int m = 0; m < MT; ++m) xf[m] = xside::read(xl, (wm * MT + m) * 16, h, lane);
#pragma unroll
        for (int n = 0; n < NT; ++n) wf[n] = wside::read(wl, (wn * NT + n) * 16, h, lane);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[n][m] = multiply<XK>(wf[n], xf[m], acc[n][m]);
      }
    } else {
      const float* sl = reinterpret_cast<const float*>(lds + slot * STAGE + SPLIT * STEP) + own * SET * 64;
      const float mine = sl[in_set * 64 + lane];
      u32x4 xf[MT][2];
      float xsc[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        xsc[m] = sl[(wm * MT + m) * 16 + (lane & 15)];
#pragma unroll
        for (int h = 0; h < 2; ++h) xf[m][h] = xside::read(xl, (wm * MT + m) * 16, h, lane);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int n0 = (wn * NT + n) * 16;
        u32x4 wf[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) wf[h] = wside::read(wl, n0, h, lane);
        f32x4 wsc;
        if constexpr (SB == 1)
          wsc = *reinterpret_cast<const f32x4*>(sl + TM + n0 + (lane >> 4) * 4);
        else
          wsc[0] = sl[TM + n0];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const f32x4 p = multiply8<WKIND, XK>(wf, xf[m]);
          if constexpr (decltype(again)::value) {
            add_far(acc[n][m], p, xsc[m], SB == 1 ? wsc : f32x4{wsc[0], wsc[0], wsc[0], wsc[0]});
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              acc[n][m][j] = __builtin_fmaf(p[j], xsc[m] * (SB == 1 ? wsc[j] : wsc[0]), acc[n][m][j]);
          }
        }
      }
      if constexpr (!decltype(again)::value) far = more(far, reach(mine));
    }
  };

  const i32 stages = (steps + SPLIT - 1) / SPLIT;
  auto walk = [&](auto again) {
    if (stages == 0) return;
    constexpr int LOADS = EACH + (E == 1);  // of a wave and stage
    // The stage that holds a step whose last 16 bytes do not all exist, which no load to LDS took.
    const i32 cut = DIRECT && a.tail && o.end == o.depth ? (turn > 0 ? steps - 1 - turn : steps - 1) : -1;
    int slot = 0;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(s, s);
    for (i32 s = 0; s < stages; ++s) {
      if constexpr (DIRECT) wait_loads<(STAGES - 2) * LOADS>();
      lds_barrier();
      issue(s + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
      if (cut >= 0 && s == cut / SPLIT) {
        const i64 last = o.last - 1, left = o.end - last * D;
        u8* at = lds + slot * STAGE + cut % SPLIT * STEP;
        for (int r = threadIdx.x; r < TM + TN; r += WAVES * 64) {
          if (r < TM)
            o.x.patch(at, r, last, left, a.tail);
          else
            o.w.patch(at + xside::BYTES, r - TM, last, left, a.tail);
        }
        lds_barrier();
      }
      compute(slot, again);
      slot = slot == STAGES - 1 ? 0 : slot + 1;
    }
    if constexpr (DIRECT) wait_loads<0>();  // LDS is not written after the block's end
  };
  walk(choice<false>{});
  if constexpr (E == 1) {
    if (__any(far > 126)) far = 127;
    if (lane == 0) farthest[wave] = far;
    lds_barrier();
    if (__any(farthest[lane % WAVES] > 126)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0, 0, 0, 0};
      walk(choice<true>{});
      lds_barrier();
    }
  } else {
    lds_barrier();
  }

  float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m)
      *reinterpret_cast<f32x4*>(sums + sum_at<TM, TN>(own, (wm * MT + m) * 16 + (lane & 15), (wn * NT + n) * 16 + (lane >> 4) * 4)) =
          acc[n][m];
  lds_barrier();
  store_sums<OUT, BY, TM, TN, SPLIT, WAVES * 64>(sums, out, parts, a, part, o.row0, o.m0, o.n0, o.m_there, 0);
}

// A wave's 16 x 64 (of 16 bits) or 16 x 32 sums on their way out: 2 KB of LDS that no other wave uses turn the rows that the
// matrix instruction gives a lane's quad of into 128 bytes of eight rows a store, which are whole lines of the caches.  Without
// barriers and of half the bytes it takes 1 us a tile of 256 x 256 less than store_sums does (12001 x 8192 x 2048 by 16
// groups 382 us with that, 378 so; depth 512 95 and 83); for 32 bits, whose rows of 128 bytes leave slower than longer ones,
// it loses (16 x 8192 x 2048 of depth 768 526 and 497).  Lane (i, g) holds columns 4 g .. of each 16 columns' block of row i.
template <class OUT> struct rows_out {
  static constexpr int V = 16 / sizeof(OUT), COLUMNS = 8 * V, BLOCKS = COLUMNS / 16;
  OUT* to;
  i64 stride, m_there, n_there;  // of `to`
  i32 wide;                      // as store_columns takes it

  UNPM_DEV void put(u8* lds, int row, int column, const f32x4 (&v)[BLOCKS], int lane) const {
    const int i = lane & 15, g = lane >> 4;
    asm volatile("" ::: "memory");  // behind the reads of what was here
#pragma unroll
    for (int n = 0; n < BLOCKS; ++n) {
      struct alignas(4 * sizeof(OUT)) quad {
        OUT v[4];
      } q;
#pragma unroll
      for (int j = 0; j < 4; ++j) q.v[j] = (OUT)v[n][j];
      const int c = n * 16 + g * 4;
      *reinterpret_cast<quad*>(lds + i * 128 + straight_slot(i, c / V) * 16 + c % V * sizeof(OUT)) = q;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = k * 8 + lane / 8, n = column + lane % 8 * V;
      const u8* from = lds + r * 128 + straight_slot(r, lane % 8) * 16;
      const i64 there = n_there - n;
      if (row + r >= m_there || there <= 0) continue;
      OUT* p = to + (row + r) * stride + n;
      if (wide && there >= V) {
        const u32x4 q = *reinterpret_cast<const u32x4*>(from);
        if (wide == 2)
          __builtin_nontemporal_store(q, reinterpret_cast<u32x4*>(p));
        else
          *reinterpret_cast<u32x4*>(p) = q;
      } else {
#pragma clang loop unroll(disable)
        for (int j = 0; j < V && j < there; ++j) p[j] = reinterpret_cast<const OUT*>(from)[j];
      }
    }
  }
};

// Tiles of 256 x 256 for much work: eight waves, two on each SIMD, of which one multiplies while the other reads LDS and
// starts loads (the second set runs one barrier behind the first).  A wave has 128 x 64 of the tile as four blocks of 64 x 32,
// one of each pair of halves; the halves of the operands' tiles lie in LDS twice, and as a half has been read by every wave, the
// loads of the same half two steps on go there: four halves or five are on their way at any time.  (X0 is the first 128 rows; W0 the
// first 32 of each 64, so that a wave stores whole lines, or where W lies along out the first 128, as loads take more of a row.)
//   phase  reads     multiplies    loads
//   0      X0 W0 W1  X0 W0, X0 W1  scales two steps on, X1 of the next step
//   1      X1        X1 W1, X1 W0  X0, W0 and W1 of the one after it
// A wave waits for its own loads of what the next phase reads before the barrier that ends its reads: all but those that it
// has started since.  (Four phases of half the products each took 519 us for 8192^3 codes, these 482, and 399 and 387 for 12001 x
// 8192 x 2048 in 16 bits by 16 groups.)  A tile of at most 128 rows, the last of a group, multiplies X0 W0 and X0 W1 in a phase
// each: the first loads scales two steps ahead and W1 of the next, the second X0 and W0 two ahead.
template <int XK, int WKIND, bool XT, bool WT, class OUT, int BY, int SB>
UNPM_DEV void matmul_wide(const u8* xp, const u8* wp, const float* xsp, const float* wsp, const i32* starts, OUT* out, float* parts,
                          const product_args& a) {
  constexpr int E = XK >= E4M3 ? 1 : 2, D = 128 / E;
  typedef side<XK, XT, 128> xside;
  typedef side<WKIND, WT, 128> wside;
  constexpr int HALF = 16384, STAGE = 4 * HALF, SCALES = E == 1 ? 2048 : 0;
  __shared__ __attribute__((aligned(1024))) u8 lds[2 * STAGE + 4 * SCALES];  // the scales of four steps
  __shared__ u32 farthest[8];

  place<XK, WKIND, XT, WT, BY, 256, 256> o;
  int part;
  if (!find_place<XK, WKIND, XT, WT, BY, SB, 256, 256, 32>(xp, wp, xsp, wsp, starts, a, part, o)) return;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave >> 2, wn = wave & 3;
  const u32 lds0 = lds_address(lds);

  // The halves of the operands: X0, X1, W0, W1.  Two loads of a wave each.
  xside xh[2];
  wside w;
  // Row i of half h of W; of one that lies along out, chunk i of 8 columns.
  auto of_half = [](int h) {
    return [h](int i) { return WT ? h * 16 + i : (i >> 5) * 64 + h * 32 + (i & 31); };
  };
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    xh[h].row = a.x_row;
    xh[h].p = XT ? o.x.p + h * 256 : o.x.p + h * 128 * a.x_row;
    xh[h].there = o.x.there - h * (XT ? 256 : 128);
  }
  w.row = a.w_row;
  w.p = o.w.p;
  w.there = o.w.there;
  u32 offset[4][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      offset[h][i] = xh[h].offset(i * 8 + wave, lane);
      offset[2 + h][i] = w.offset(i * 8 + wave, lane, of_half(h));
    }
  const float* scale = nullptr;
  if constexpr (E == 1) {
    const int f = wave * 64 + lane, n = of_half(f >> 7 & 1)(f & 127);  // codes' rows are not turned
    scale = f < 256 ? o.xs + least(f, o.xs_last) * a.xs_row : o.ws + least(n / SB, o.ws_last) * a.ws_row;
  }
  // What of a step has to be left for a lane's 16 bytes to exist is the same for every load of it along d.
  const i32 x_after = xside::after(wave, lane), w_after = wside::after(wave, lane);
  auto issue = [&](int half, i64 step) {
    const bool isx = half < 2;
    // Of W that lies along out only the rows that meet whole 16 bytes of X: the others meet zeros, which times infinity are NaN.
    const i32 there = (i32)(o.end - (o.first + step) * D), left = !isx && WT && !XT ? there & ~(16 / E - 1) : there;
    const u8* p = isx ? xh[half & 1].at(o.first + step) : w.at(o.first + step);
    const u32 to = lds0 + (u32)(step & 1) * STAGE + half * HALF + wave * 1024;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const i32 after = (isx ? x_after + (XT ? i * 32 : 0) : w_after + (WT ? i * 32 : 0));
      const i32 rest = (i32)(isx ? xside::left(left) : wside::left(left));
      load_to_lds(p, (isx ? xside::exists(after, rest) : wside::exists(after, rest)) ? offset[half][i] : OUTSIDE, to + i * 8192);
    }
  };
  auto issue_scales = [&](i64 step) {
    if constexpr (E == 1)
      load_word_to_lds(scale + least(o.first + step, o.last - 1), lds0 + 2 * STAGE + (u32)(step & 3) * SCALES + wave * 256);
  };

  f32x4 acc[2][2][2][4];  // of W half, X half, tile of W, tile of X
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < 32; ++i) (&acc[0][0][0][0])[i] = f32x4{0, 0, 0, 0};
  };
  clear();
  u32 far = 0;  // the farthest of the scales that this wave loaded
  auto look = [&](i64 step) {
    if constexpr (E == 1)
      far = more(far, reach(*reinterpret_cast<const float*>(lds + 2 * STAGE + (u32)(step & 3) * SCALES + wave * 256 + lane * 4)));
  };
  const i64 steps = o.last - o.first;
  const bool low = o.m_there <= 128;
  if (steps > 0) {
    issue_scales(0);
    issue(0, 0);
    issue(2, 0);
    issue(3, 0);
    issue_scales(1);
    if (!low) issue(1, 0);
    issue(0, 1);
    issue(2, 1);
    if (!low) issue(3, 1);
    if (low)
      wait_loads<E == 1 ? 7 : 6>();
    else
      wait_loads<E == 1 ? 9 : 8>();
    lds_barrier();
    if (wm == 1) lds_barrier();

    u32x4 xf[4][2], wf[2][2][2];
    float xsc[4], wsc = 0;  // of the halves at hand
    f32x4 wrow[2];
    auto read_x = [&](const u8* at, const float* scales, int h) {
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int k = 0; k < 2; ++k) xf[m][k] = xside::read(at + h * HALF, wm * 64 + m * 16, k, lane);
      if constexpr (E == 1)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          xsc[m] = scales[h * 128 + wm * 64 + m * 16 + (lane & 15)];
    };
    auto read_w_scales = [&](const float* scales, int h) {
      const float* s = scales + 256 + h * 128 + wn * 32;
      if constexpr (E == 1 && SB == 1)
#pragma unroll
        for (int n = 0; n < 2; ++n) wrow[n] = *reinterpret_cast<const f32x4*>(s + n * 16 + (lane >> 4) * 4);
      if constexpr (E == 1 && SB > 1) wsc = *s;
    };
    auto read_w_codes = [&](const u8* at, int h) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) wf[h][n][k] = wside::read(at + (2 + h) * HALF, wn * 32 + n * 16, k, lane);
    };
    auto read_w = [&](const u8* at, const float* scales, int h) {
      read_w_codes(at, h);
      read_w_scales(scales, h);
    };
    // `next`: where the scales of W's other half are, read as this half's are used up.
    auto products = [&](auto again, int hw, int hx, const float* next = nullptr) {
      __builtin_amdgcn_s_setprio(1);
      if constexpr (E == 2) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int m = 0; m < 4; ++m) acc[hw][hx][n][m] = multiply<XK>(wf[hw][n][k], xf[m][k], acc[hw][hx][n][m]);
      } else {
        // A product's sums are taken up two instructions later, when they are there: three are held, not eight.
        constexpr int LATE = 2;
        f32x4 p[LATE + 1];
        float both[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) both[m] = SB == 1 ? xsc[m] : xsc[m] * wsc;
#pragma unroll
        for (int i = 0; i < 8 + LATE; ++i) {
          if (i < 8) p[i % (LATE + 1)] = multiply8<WKIND, XK>(wf[hw][i / 4], xf[i % 4]);
          __builtin_amdgcn_sched_barrier(0);
          if (i >= LATE) {
            const int n = (i - LATE) / 4, m = (i - LATE) % 4;
            if constexpr (decltype(again)::value) {
              add_far(acc[hw][hx][n][m], p[(i - LATE) % (LATE + 1)], xsc[m], SB == 1 ? wrow[n] : f32x4{wsc, wsc, wsc, wsc});
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                acc[hw][hx][n][m][j] =
                    __builtin_fmaf(p[(i - LATE) % (LATE + 1)][j], SB == 1 ? both[m] * wrow[n][j] : both[m], acc[hw][hx][n][m][j]);
            }
          }
          if constexpr (SB == 1)
            if (next && (i == 3 + LATE || i == 7 + LATE)) {
              const int n = (i - LATE) / 4;
              wrow[n] = *reinterpret_cast<const f32x4*>(next + 256 + (1 - hw) * 128 + wn * 32 + n * 16 + (lane >> 4) * 4);
            }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    };
    auto meet = [&] {
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    auto read_done = [&] {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      meet();
    };
    // A step that lies in LDS for every wave, whatever its scales are.
    auto single = [&](const u8* at, const float* sc) {
      constexpr choice<E == 1> again{};
      read_x(at, sc, 0);
      read_w(at, sc, 0);
      products(again, 0, 0);
      read_w(at, sc, 1);
      products(again, 1, 0);
      read_x(at, sc, 1);
      products(again, 1, 1);
      read_w(at, sc, 0);
      products(again, 0, 1);
    };
    constexpr choice<false> once{};
    for (i64 s = 0; low && s < steps; ++s) {
      const u8* at = lds + (u32)(s & 1) * STAGE;
      const float* sc = reinterpret_cast<const float*>(lds + 2 * STAGE + (u32)(s & 3) * SCALES);
      read_x(at, sc, 0);
      read_w(at, sc, 0);
      issue_scales(s + 2);
      issue(3, s + 1);
      wait_loads<E == 1 ? 7 : 6>();
      read_done();
      products(once, 0, 0);
      meet();
      read_w(at, sc, 1);
      look(s);
      issue(0, s + 2);
      issue(2, s + 2);
      wait_loads<E == 1 ? 7 : 6>();
      read_done();
      products(once, 1, 0);
      meet();
    }
    for (i64 s = 0; !low && s < steps; ++s) {
      const u8* at = lds + (u32)(s & 1) * STAGE;
      const float* sc = reinterpret_cast<const float*>(lds + 2 * STAGE + (u32)(s & 3) * SCALES);
      read_x(at, sc, 0);
      read_w(at, sc, 0);
      read_w_codes(at, 1);
      issue_scales(s + 2);
      issue(1, s + 1);
      wait_loads<E == 1 ? 9 : 8>();
      read_done();
      products(once, 0, 0, sc);
      products(once, 1, 0);
      meet();
      read_x(at, sc, 1);
      look(s);
      issue(0, s + 2);
      issue(2, s + 2);
      issue(3, s + 2);
      wait_loads<E == 1 ? 9 : 8>();
      read_done();
      products(once, 1, 1, sc);
      products(once, 0, 1);
      meet();
    }
    if constexpr (E == 1) {
      if (__any(far > 126)) far = 127;
      if (lane == 0) farthest[wave] = far;
    }
    if (wm == 0) lds_barrier();
    wait_loads<0>();
    if constexpr (E == 1) {
      lds_barrier();
      if (__any(farthest[lane & 7] > 126)) {
        clear();
        for (i64 s = 0; s < steps; ++s) {
          const u32 at = (u32)(s & 1) * STAGE;
          issue_scales(s);
#pragma unroll
          for (int h = 0; h < 4; ++h) issue(h, s);
          wait_loads<0>();
          lds_barrier();
          single(lds + at, reinterpret_cast<const float*>(lds + 2 * STAGE + (u32)(s & 3) * SCALES));
          lds_barrier();
        }
      }
    }
    if (a.tail && o.end == o.depth) {
      // The bytes of the last 16 that exist, which the last step had as zeros: one more step of them alone.
      const i64 last = o.last - 1, left = o.end - last * D;
      lds_barrier();
#pragma clang loop unroll(disable)
      for (int q = threadIdx.x; q < 1024; q += 512) {
        xh[0].alone(lds, q, last, left, [](int i) { return i; });
        xh[1].alone(lds + HALF, q, last, left, [](int i) { return i; });
        w.alone(lds + 2 * HALF, q, last, left, of_half(0));
        w.alone(lds + 3 * HALF, q, last, left, of_half(1));
      }
      if constexpr (E == 1) *reinterpret_cast<float*>(lds + 2 * STAGE + threadIdx.x * 4) = scale[last];
      lds_barrier();
      const float* sc = reinterpret_cast<const float*>(lds + 2 * STAGE);
      single(lds, sc);
    }
  }
  lds_barrier();
  if constexpr (sizeof(OUT) == 2 && !WT) {
    const i64 n0 = o.n0 + wn * 64, m_there = o.m_there - wm * 64;
    u8* own = lds + wave * 2048;
    auto send = [&](auto to) {
      constexpr int BLOCKS = decltype(to)::BLOCKS;
#pragma unroll
      for (int hx = 0; hx < 2; ++hx) {
        if (hx && low) break;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int t = 0; t < 4 / BLOCKS; ++t) {
            f32x4 v[BLOCKS];
#pragma unroll
            for (int i = 0; i < BLOCKS; ++i) v[i] = acc[BLOCKS == 4 ? i / 2 : t][hx][i % 2][m];
            to.put(own, hx * 128 + m * 16, t * 32, v, lane);
          }
      }
    };
    if (a.parts > 1) {
      const i64 wide = (a.n + 7) / 8 * 8;
      send(rows_out<float>{parts + (part * a.m + o.row0 + wm * 64) * wide + n0, wide, m_there, wide - n0, 1});
    } else {
      send(rows_out<OUT>{out + (o.m0 + wm * 64) * a.out_row + n0, a.out_row, m_there, a.n - n0, a.wide});
    }
  } else {
    // A half of X at a time: 128 rows of sums fill what held the steps, and go out as whole rows of 256.
    float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int hx = 0; hx < 2; ++hx) {
      if (hx && low) break;
      lds_barrier();
#pragma unroll
      for (int hw = 0; hw < 2; ++hw)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int m = 0; m < 4; ++m)
            *reinterpret_cast<f32x4*>(sums + sum_at<128, 256>(0, wm * 64 + m * 16 + (lane & 15),
                                                              (WT ? hw * 128 + wn * 32 : wn * 64 + hw * 32) + n * 16 + (lane >> 4) * 4)) = acc[hw][hx][n][m];
      lds_barrier();
      store_sums<OUT, BY, 128, 256, 1, 512>(sums, out, parts, a, part, o.row0, o.m0, o.n0, o.m_there, hx * 128);
    }
  }
}

// The sums of a split depth, part after part.
template <class OUT, int BY>
UNPM_DEV void join(const i32* starts, OUT* out, const float* parts, const product_args& a) {
  const i64 rows = BY == DEPTH ? a.groups * a.m : a.m, units = (a.n + 7) / 8;
  i64 r0 = 0, r1 = rows;
  if constexpr (BY == ROWS) {  // from the first start to the largest
    i32 top = 0;
    for (int i = threadIdx.x & 63; i <= a.groups; i += 64) top = starts[i] > top ? starts[i] : top;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const i32 v = __shfl_xor(top, d);
      top = v > top ? v : top;
    }
    r0 = least(starts[0] < 0 ? 0 : starts[0], rows);
    r1 = least(top, rows);
  }
  for (i64 i = r0 * units + (i64)blockIdx.x * 256 + threadIdx.x; i < r1 * units; i += (i64)gridDim.x * 256) {
    const i64 r = i / units, n = i % units * 8;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int p = 0; p < a.parts; ++p) {
      const f32x4* q = reinterpret_cast<const f32x4*>(parts + (p * rows + r) * units * 8 + n);
      const f32x4 x = q[0], y = n + 4 < a.n ? q[1] : f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] += x[j];
        v[4 + j] += y[j];
      }
    }
    const i64 g = BY == DEPTH ? r / a.m : 0;
    store_columns<OUT>(out + g * a.out_group + (BY == DEPTH ? r - g * a.m : r) * a.out_row + n, v, a.n - n, a.wide);
  }
}

// ---------------------------------------------------------------------------------------
// Quantisation: codes of y = x or its transpose, and the f32 scale of each block of 128 columns and RB rows of y:
// scale = most times the f32 nearest to 1 / largest code, code = y / scale rounded to even from the correctly rounded quotient.
// A block of zeros has the scale 0 and divides as by 1; one that holds a NaN or an infinity has a NaN scale and codes 0.
// Where the scale is a subnormal number of few digits, its rounding may leave quotients past what rounds to the largest code, up
// to half as much again: they take that code (the conversions would make a NaN or an infinity of them).  A scale that rounds to
// 0 leaves codes 0.
//
// Magnitudes are compared as integers (NaN above infinity above every number).  The quotient of two f32 numbers is taken
// from the divisor's reciprocal by one correction (P. Markstein, 1990), right while f32 holds the remainder; the scales where it may not
// divide.  A code is decided at quotients from the smallest tie on, 2^-17 (e5m2; e4m3 2^-10).  Beside it a quotient has steps of
// 2^-41, a scale of 2^e has steps of 2^(e-23), and so the remainder steps of 2^(e-64): f32's smallest, 2^-149, at e = -85.
// ---------------------------------------------------------------------------------------
struct quant_args {
  i64 rows, cols;  // of x
  i64 x_row, code_row, scale_row;
  i32 x_vectors, code_vectors;
};

template <int KIND> UNPM_DEV float largest() { return KIND == E4M3 ? 448.0f : 57344.0f; }
template <int KIND> UNPM_DEV float inverse_largest() { return 1.0f / largest<KIND>(); }

struct step_of {
  float scale, unit, inverse;
  bool divide, none;
};
template <int KIND> UNPM_DEV step_of block_step(u32 most) {
  step_of s;
  s.none = most >= 0x7F800000u;
  s.scale = s.none ? __builtin_nanf("") : bits<float>(most) * inverse_largest<KIND>();
  s.unit = s.scale > 0.0f ? s.scale : 1.0f;
  s.inverse = 1.0f / s.unit;
  s.divide = s.unit < 0x1p-80f;
  return s;
}
// Numbers of one block over its step; where it is none, whatever comes out.  A wave divides or multiplies as one.  Only scales
// that divide may be subnormal.
template <int KIND, int N> UNPM_DEV void quotients(float (&y)[N], const step_of& s) {
  if (__any(s.divide)) {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = __builtin_amdgcn_fmed3f(y[i] / s.unit, -largest<KIND>(), largest<KIND>());
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float q = y[i] * s.inverse;
      y[i] = __builtin_fmaf(-__builtin_fmaf(q, s.unit, -y[i]), s.inverse, q);  // in this order a zero keeps its sign
    }
  }
}
// Four codes as a word.
template <int KIND> UNPM_DEV u32 codes4(float a, float b, float c, float d) {
  if constexpr (KIND == E4M3)
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
  else
    return __builtin_amdgcn_cvt_pk_bf8_f32(c, d, __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false), true);
}
UNPM_DEV u32 magnitude(float x) { return bits<u32>(x) & 0x7FFFFFFFu; }

// 16 bytes of a row from column c on, zeros past the last one (whole: known to be there and aligned).
template <class T> struct alignas(16) vec_of {
  T v[16 / sizeof(T)];
};
template <class T> UNPM_DEV vec_of<T> load_vec(const T* row, i64 c, i64 cols, bool whole) {
  constexpr int V = 16 / sizeof(T);
  if (whole) return *reinterpret_cast<const vec_of<T>*>(row + c);
  vec_of<T> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.v[i] = c + i < cols ? row[c + i] : (T)0.0f;
  return v;
}
template <int W> UNPM_DEV void store_codes(u8* row, i64 c, i64 cols, bool whole, const u32 (&w)[W]) {
  if (whole) {
    struct alignas(4 * W) vec {
      u32 v[W];
    };
    vec v;
#pragma unroll
    for (int i = 0; i < W; ++i) v.v[i] = w[i];
    *reinterpret_cast<vec*>(row + c) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4 * W; ++i)
      if (c + i < cols) row[c + i] = (u8)(w[i / 4] >> (i % 4 * 8));
  }
}
// The largest of 8 neighbouring lanes' numbers: within pairs, within fours, and of the two fours.
UNPM_DEV u32 most_of_8(u32 m) {
  m = more(m, (u32)__builtin_amdgcn_mov_dpp((i32)m, 0xB1, 0xF, 0xF, true));
  m = more(m, (u32)__builtin_amdgcn_mov_dpp((i32)m, 0x4E, 0xF, 0xF, true));
  return more(m, (u32)__builtin_amdgcn_mov_dpp((i32)m, 0x141, 0xF, 0xF, true));
}

// A scale per row and block: 8 lanes hold its 128 elements, 16 bytes of each run of 128 (so a load covers whole lines).
// Memory bounds it: 69 microseconds for 16384 x 8192 16-bit numbers (5.9 TB/s), 68 for a loop that only reads and writes as much.
template <class T, int KIND> UNPM_DEV void quantise_rows(const T* x, u8* codes, float* scales, const quant_args& a) {
  constexpr int V = 16 / sizeof(T), PIECES = 16 / V;
  const i64 blocks = (a.cols + 127) / 128, all = a.rows * blocks;
  const int lane = threadIdx.x & 7;
  for (i64 first = (i64)blockIdx.x * 32; first < all; first += (i64)gridDim.x * 32) {
    const i64 r0 = first >> 31 ? first / blocks : (u32)first / (u32)blocks;
    const u32 b0 = (u32)(first - r0 * blocks) + threadIdx.x / 8, b = b0 % (u32)blocks;
    const i64 r = r0 + b0 / (u32)blocks;
    if (r >= a.rows) break;
    const i64 c = (i64)b * 128 + lane * V;
    // A wave whose blocks are all there loads and stores without a look at each vector: its loads are then in flight together.
    const bool there = __all((i64)b * 128 + 128 <= a.cols), loads = there && a.x_vectors, stores = there && a.code_vectors;
    vec_of<T> v[PIECES];
    if (loads) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) v[p] = load_vec<T>(x + r * a.x_row, c + p * 8 * V, a.cols, true);
    } else {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) v[p] = load_vec<T>(x + r * a.x_row, c + p * 8 * V, a.cols, false);
    }
    float y[PIECES * V];
    u32 most = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      y[j] = (float)v[j / V].v[j % V];
      most = more(most, magnitude(y[j]));
    }
    const step_of s = block_step<KIND>(most_of_8(most));
    quotients<KIND>(y, s);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      u32 w[V / 4];
#pragma unroll
      for (int j = 0; j < V / 4; ++j) {
        const float* z = y + p * V + 4 * j;
        w[j] = s.none ? 0 : codes4<KIND>(z[0], z[1], z[2], z[3]);
      }
      store_codes<V / 4>(codes + r * a.code_row, c + p * 8 * V, a.cols, stores, w);
    }
    if (lane == 0) scales[r * a.scale_row + b] = s.scale;
  }
}

// The other forms: a block takes 128 x 128 elements of x; thread (i, j) R rows from R i on and 8 columns, 16 bytes of each run
// of 16 lanes.  One scale for all of them, or (TURNED) one for each column, whose 128 rows lie along y's row.
// 34.5 microseconds for 8192 x 4096 of 32 bits (4.9 TB/s), 30 for a copy; threads of 8 rows each, half as many, took 35.4.
template <class T, int KIND, int RB, bool TURNED>
UNPM_DEV void quantise_tiles(const T* x, u8* codes, float* scales, const quant_args& a) {
  static_assert(RB == 128 || TURNED, "scales of rows are quantise_rows's");
  constexpr int ROW = 128 + 16;  // of a transposed tile in LDS
  constexpr int THREADS = 512, V = 16 / sizeof(T), PIECES = 8 / V, R = 2048 / THREADS, TEAMS = 128 / R;
  __shared__ u32 tops[TEAMS][128];
  __shared__ __attribute__((aligned(16))) u8 turned[TURNED ? 128 * ROW : 16];
  const i64 across = (a.cols + 127) / 128, all = (a.rows + 127) / 128 * across;
  const int i = threadIdx.x / 16, j = threadIdx.x % 16;
  for (i64 t = blockIdx.x; t < all; t += gridDim.x) {
    const i64 tr = t / across, tc = t % across, r0 = tr * 128 + i * R, c0 = tc * 128 + j * V;
    const bool there = tr * 128 + 128 <= a.rows && tc * 128 + 128 <= a.cols, loads = there && a.x_vectors, stores = there && a.code_vectors;
    vec_of<T> v[R][PIECES];
    if (loads) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int p = 0; p < PIECES; ++p) v[r][p] = load_vec<T>(x + (r0 + r) * a.x_row, c0 + p * 16 * V, a.cols, true);
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
          v[r][p] = load_vec<T>(x + (r0 + r) * a.x_row, r0 + r < a.rows ? c0 + p * 16 * V : a.cols, a.cols, false);
    }
    float y[8][R];  // of a column, then a row
    u32 top[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      top[c] = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        y[c][r] = (float)v[r][c / V].v[c % V];
        top[c] = more(top[c], magnitude(y[c][r]));
      }
    }
    auto column = [&](int c) { return c / V * 16 * V + j * V + c % V; };
    bool none[8];
    if constexpr (RB == 128) {
      u32 most = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) most = more(most, top[c]);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) most = more(most, (u32)__shfl_xor((i32)most, d));
      if ((threadIdx.x & 63) == 0) tops[0][threadIdx.x / 64] = most;
      __syncthreads();
      most = 0;
#pragma unroll
      for (int w = 0; w < THREADS / 64; ++w) most = more(most, tops[0][w]);
      const step_of s = block_step<KIND>(most);
      if (threadIdx.x == 0) scales[(TURNED ? tc : tr) * a.scale_row + (TURNED ? tr : tc)] = s.scale;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        quotients<KIND>(y[c], s);
        none[c] = s.none;
      }
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) tops[i][column(c)] = top[c];
      __syncthreads();
      if (threadIdx.x < 128) {
        u32 most = 0;
#pragma unroll
        for (int k = 0; k < TEAMS; ++k) most = more(most, tops[k][threadIdx.x]);
        tops[0][threadIdx.x] = most;
        if (tc * 128 + threadIdx.x < a.cols) scales[(tc * 128 + threadIdx.x) * a.scale_row + tr] = block_step<KIND>(most).scale;
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const step_of s = block_step<KIND>(tops[0][column(c)]);
        quotients<KIND>(y[c], s);
        none[c] = s.none;
      }
    }
    if constexpr (TURNED) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        struct alignas(R) codes_of {
          u32 v[R / 4];
        } w;
#pragma unroll
        for (int k = 0; k < R / 4; ++k) w.v[k] = none[c] ? 0 : codes4<KIND>(y[c][4 * k], y[c][4 * k + 1], y[c][4 * k + 2], y[c][4 * k + 3]);
        *reinterpret_cast<codes_of*>(turned + column(c) * ROW + i * R) = w;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 1024 / THREADS; ++k) {
        const int c = k * (THREADS / 8) + threadIdx.x / 8, part = threadIdx.x % 8;
        if (tc * 128 + c < a.cols) {
          const u32x4 u = *reinterpret_cast<const u32x4*>(turned + c * ROW + part * 16);
          const u32 w[4] = {u[0], u[1], u[2], u[3]};
          store_codes<4>(codes + (tc * 128 + c) * a.code_row, tr * 128 + part * 16, a.rows, stores, w);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r0 + r < a.rows)
#pragma unroll
          for (int p = 0; p < PIECES; ++p) {
            u32 w[V / 4];
#pragma unroll
            for (int k = 0; k < V / 4; ++k) {
              const int c = p * V + 4 * k;
              w[k] = none[0] ? 0 : codes4<KIND>(y[c][r], y[c + 1][r], y[c + 2][r], y[c + 3][r]);
            }
            store_codes<V / 4>(codes + (r0 + r) * a.code_row, c0 + p * 16 * V, a.cols, stores, w);
          }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------
// The rows of each group: a stable counting sort of n ids below `groups`.  starts[g] is where group g's rows begin, place[i]
// where i went (-1: an id of no group), rows[p] = i / per of the i that went to p (-1 behind the last).
//
// Chunks of ids in order: count() writes each chunk's ids per group, and place() adds up those of the chunks before its own.
// With one chunk, one block does both.  131072 ids of 128 groups take 13 microseconds in 128 chunks, mostly two launches; adding
// the chunks up one after another took 49.  Inside a chunk a wave takes a run of ids, 64 at a time; the lanes of one
// id find each other by its bits, so their order is that of the lanes.
// ---------------------------------------------------------------------------------------
struct rows_args {
  i64 n, chunk;  // ids, ids of a block: a multiple of 64 times the waves
  i32 groups, chunks;
  u32 per, pad;  // ids of a row
};
constexpr int MOST_GROUPS = 1024, SORT_WAVES = 8;

// This wave's run of its block's chunk.
struct run_of {
  i64 first, last;
};
UNPM_DEV run_of wave_run(const rows_args& a) {
  const i64 each = a.chunk / SORT_WAVES, first = blockIdx.x * a.chunk + threadIdx.x / 64 * each;
  return {first, least(first + each, a.n)};
}
// counts[wave][group] of the block's chunk.
template <class I> UNPM_DEV void count_runs(const I* ids, const rows_args& a, i32 (*counts)[MOST_GROUPS]) {
#pragma unroll
  for (int w = 0; w < SORT_WAVES; ++w)
    for (int g = threadIdx.x; g < a.groups; g += SORT_WAVES * 64) counts[w][g] = 0;
  __syncthreads();
  const run_of r = wave_run(a);
  for (i64 i = r.first + (threadIdx.x & 63); i < r.last; i += 64) {
    const I id = ids[i];
    if (id >= 0 && id < a.groups) atomicAdd(&counts[threadIdx.x / 64][(int)id], 1);
  }
  __syncthreads();
}

template <class I> UNPM_DEV void count_rows(const I* ids, i32* counted, const rows_args& a) {
  __shared__ i32 counts[SORT_WAVES][MOST_GROUPS];
  count_runs<I>(ids, a, counts);
  for (int g = threadIdx.x; g < a.groups; g += SORT_WAVES * 64) {
    i32 c = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) c += counts[w][g];
    counted[(i64)blockIdx.x * a.groups + g] = c;
  }
}

template <class I>
UNPM_DEV void place_rows(const I* ids, i32* starts, i32* rows, i32* place, const i32* counted, const rows_args& a) {
  __shared__ i32 counts[SORT_WAVES][MOST_GROUPS];
  __shared__ i32 before[MOST_GROUPS], sums[SORT_WAVES];
  constexpr int THREADS = SORT_WAVES * 64, EACH = MOST_GROUPS / THREADS;
  count_runs<I>(ids, a, counts);
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  // How many ids the groups have in all, and in the chunks before this one.  With several chunks each thread adds up one
  // group's counts of some of them, 16 at a time.
  __shared__ i32 every[MOST_GROUPS];
  const int teams = a.groups < THREADS ? THREADS / a.groups : 1;
  for (int g = t; g < a.groups; g += THREADS) {
    i32 c = 0;
    if (a.chunks == 1) {
#pragma unroll
      for (int w = 0; w < SORT_WAVES; ++w) c += counts[w][g];
    }
    every[g] = c;
    before[g] = 0;
  }
  __syncthreads();
  if (a.chunks > 1 && t < teams * (a.groups < THREADS ? a.groups : THREADS)) {
    const int team = teams > 1 ? t / a.groups : 0;
    for (int g = teams > 1 ? t % a.groups : t; g < a.groups; g += THREADS) {
      i32 c_all = 0, c_ahead = 0;
      for (int c = team; c < a.chunks; c += 16 * teams) {
        i32 v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = c + k * teams < a.chunks ? counted[(c + k * teams) * a.groups + g] : 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          c_all += v[k];
          c_ahead += c + k * teams < (int)blockIdx.x ? v[k] : 0;
        }
      }
      atomicAdd(&every[g], c_all);
      atomicAdd(&before[g], c_ahead);
    }
  }
  __syncthreads();
  // Where they begin: this thread's groups t * EACH ...
  i32 all[EACH], own = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int g = t * EACH + e;
    all[e] = g < a.groups ? every[g] : 0;
    own += all[e];
  }
  i32 upto = own;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const i32 v = __shfl_up(upto, d);
    if (lane >= d) upto += v;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  i32 start = upto - own, total = 0;
#pragma unroll
  for (int w = 0; w < SORT_WAVES; ++w) {
    if (w < wave) start += sums[w];
    total += sums[w];
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int g = t * EACH + e;
    if (g < a.groups) {
      if (blockIdx.x == 0) starts[g] = start;
      before[g] += start;
    }
    start += all[e];
  }
  if (blockIdx.x == 0 && t == 0) starts[a.groups] = total;
  __syncthreads();
  for (int g = t; g < a.groups; g += THREADS) {
    i32 at = before[g];
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      const i32 c = counts[w][g];
      counts[w][g] = at;
      at += c;
    }
  }
  __syncthreads();
  // Positions behind the last row.
  for (i64 p = total + (i64)blockIdx.x * THREADS + t; p < a.n; p += (i64)gridDim.x * THREADS) rows[p] = -1;
  const run_of r = wave_run(a);
  for (i64 first = r.first; first < r.last; first += 64) {
    const i64 i = first + lane;
    const I id = i < r.last ? ids[i] : (I)-1;
    const bool in = id >= 0 && id < a.groups;
    const int g = in ? (int)id : 0;
    u64 same = __ballot(in);
    for (int b = 1; b < a.groups; b *= 2) {
      const u64 set = __ballot((g & b) != 0);
      same &= g & b ? set : ~set;
    }
    if (in) {
      const int rank = __builtin_popcountll(same & ((1ull << lane) - 1));
      const i32 at = counts[wave][g] + rank;
      place[i] = at;
      rows[at] = (i32)((u32)i / a.per);
      // The last of the lanes moves the count on; the wave has read it by then.
      if ((same >> lane) == 1) counts[wave][g] = at + 1;
    } else if (i < r.last) {
      place[i] = -1;
    }
  }
}

}  // namespace unpm
