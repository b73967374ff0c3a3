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
  i32 x_vectors, w_vectors;        // rows of whole 16-byte vectors
  i32 wide;                        // out takes four columns at once
  i32 pad;
};

constexpr u32 OUTSIDE = 0x80000000u;  // an offset past every buffer: loads of it give zeros

UNPM_DEV u32x4 resource(const u8* p) {
  const u64 a = (u64)p;
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((u32)a);
  r[1] = __builtin_amdgcn_readfirstlane((u32)(a >> 32) & 0xFFFFu);
  r[2] = OUTSIDE;
  r[3] = 0x00020000u;
  return r;
}
// 16 bytes of each lane from p + offset to LDS, lane after lane from `to` on; zeros where the offset is OUTSIDE.
UNPM_DEV void load_to_lds(const u8* p, u32 offset, u32 to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset),
               "s"(resource(p))
               : "memory", "m0");
}
UNPM_DEV void load_word_to_lds(const float* p, u32 to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(p) : "memory", "m0");
}

// 16 bytes at p of which `there` exist (elements of E bytes), zeros for the others.
template <int E> UNPM_DEV u32x4 fetch16(const u8* p, i64 there, bool vector) {
  if (vector && there >= 16) return *reinterpret_cast<const u32x4*>(p);
  u32x4 x = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; i += E)
    if (i < there) {
      const u32 v = E == 1 ? (u32)p[i] : (u32) * reinterpret_cast<const u16*>(p + i);
      x[i / 4] |= v << (i % 4 * 8);
    }
  return x;
}

// Where the 16 bytes of a tile's row lie: a row of 128 bytes along d has 8 slots, the slot of a chunk goes by the row's
// low bits and those above them.  A transposed row (2 T bytes) moves pairs of slots: the four rows that 16 lanes read, and
// the four that lie eight further, are in different banks.
UNPM_DEV int straight_slot(int row, int chunk) { return chunk ^ ((row ^ (row >> 3)) & 7); }
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
  bool vectors;

  // Lane `lane` of unit u: the row and the chunk that lie at its 16 bytes.
  static UNPM_DEV int row_of(int u, int lane) { return u * (64 / CHUNKS) + lane / CHUNKS; }
  static UNPM_DEV int chunk_of(int u, int lane) {
    const int r = row_of(u, lane), s = lane % CHUNKS;
    return TURNED ? turned_slot<T>(r, s) : straight_slot(r, s);
  }
  // The offset of the lane's 16 bytes from the step's first; OUTSIDE where its row or column does not exist.
  UNPM_DEV u32 offset(int u, int lane) const {
    const int r = row_of(u, lane), c = chunk_of(u, lane);
    const bool in = TURNED ? c * 16 < there : r < there;
    return in ? (u32)(r * (i32)row + c * 16) : OUTSIDE;
  }
  // What of the step's length has to be left for the lane's 16 bytes to exist, in bytes or TURNED rows.
  static UNPM_DEV int after(int u, int lane) { return TURNED ? row_of(u, lane) : chunk_of(u, lane) * 16; }
  static UNPM_DEV i64 left(i64 elements) { return TURNED ? elements : elements * E; }
  UNPM_DEV const u8* at(i64 step) const { return p + (TURNED ? step * D * row : step * 128); }
  UNPM_DEV u32x4 fetch(int u, int lane, i64 step, i64 elements) const {
    const int r = row_of(u, lane), c = chunk_of(u, lane);
    const i64 bytes = TURNED ? (r < elements ? there - c * 16 : 0) : (r < there ? elements * E - c * 16 : 0);
    return fetch16<E>(at(step) + r * row + c * 16, bytes, vectors);
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

// Blocks are dealt to the 8 XCDs in turn: each takes a run of the tiles, so that its L2 holds what they share, in bands of
// 8 tiles along out's rows.
struct tile_at {
  i64 m, n;
  int part;
};
UNPM_DEV tile_at tile_of(const product_args& a) {
  const u32 b = blockIdx.x, blocks = gridDim.x, each = blocks / 8, rest = blocks % 8, xcd = b % 8;
  const u32 id = xcd * each + (xcd < rest ? xcd : rest) + b / 8;
  const u32 tiles = (u32)a.tiles_m * (u32)a.tiles_n, part = id / tiles, t = id % tiles;
  constexpr u32 BAND = 8;
  const u32 per = BAND * (u32)a.tiles_n, band = t / per, in = t % per;
  const u32 first = band * BAND, high = (u32)a.tiles_m - first < BAND ? (u32)a.tiles_m - first : BAND;
  return {(i64)(first + in % high), (i64)(in / high), (int)part};
}

// The rows of group g, whatever the starts are: within 0 .. rows.
UNPM_DEV void group_rows(const i32* starts, int g, i64 rows, i64& r0, i64& r1) {
  r0 = least(starts[g] < 0 ? 0 : starts[g], rows);
  r1 = least(starts[g + 1] < 0 ? 0 : starts[g + 1], rows);
}
// Tile t of T rows of the groups that have rows: its group and rows, or no such tile.  Every lane of a wave asks alike.
template <int T> UNPM_DEV bool find_group(const i32* starts, int groups, i64 rows, i64 t, int& group, i64& r0, i64& r1) {
  const int lane = threadIdx.x & 63;
  i64 past = 0;
  for (int first = 0; first < groups; first += 64) {
    i64 s0 = 0, s1 = 0;
    if (first + lane < groups) group_rows(starts, first + lane, rows, s0, s1);
    const i32 own = s1 > s0 ? (i32)((s1 - s0 + T - 1) / T) : 0;
    i32 upto = own;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const i32 v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    const u64 has = __ballot(past + upto > t);
    if (has) {
      const int l = __builtin_ctzll(has);
      group = first + l;
      const i64 tile = t - past - (__shfl(upto, l) - __shfl(own, l));
      r0 = __shfl((i32)s0, l) + tile * T;
      r1 = __shfl((i32)s1, l);
      return true;
    }
    past += __shfl(upto, 63);
  }
  return false;
}

template <class OUT> UNPM_DEV void store4(OUT* p, const f32x4& v, i64 there, bool wide) {
  struct alignas(4 * sizeof(OUT)) quad {
    OUT v[4];
  };
  quad q;
#pragma unroll
  for (int j = 0; j < 4; ++j) q.v[j] = (OUT)v[j];
  if (wide && there >= 4) {
    *reinterpret_cast<quad*>(p) = q;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < there) p[j] = q.v[j];
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
  i64 end;               // elements along d of this part
  i64 m0, n0, m_there;   // the tile in out
  i64 row0;              // the tile's first row among all rows (of all groups) of the result
};

template <int XK, int WKIND, bool XT, bool WT, int BY, int SB, int TM, int TN>
UNPM_DEV bool find_place(const u8* x, const u8* w, const float* xs, const float* ws, const i32* starts,
                         const product_args& a, int& part, place<XK, WKIND, XT, WT, BY, TM, TN>& o) {
  constexpr int E = XK >= E4M3 ? 1 : 2, D = 128 / E;
  const tile_at t = tile_of(a);
  part = t.part;
  i64 depth = a.depth;
  o.n0 = t.n * TN;
  if constexpr (BY == DEPTH) {
    const int g = (int)(t.m / ((a.m + TM - 1) / TM));
    const i64 tm = t.m % ((a.m + TM - 1) / TM);
    i64 r0, r1;
    group_rows(starts, g, a.depth, r0, r1);
    depth = r1 > r0 ? r1 - r0 : 0;
    o.m0 = tm * TM;
    o.m_there = a.m - o.m0;
    o.row0 = g * a.m + o.m0;
    x += r0 * a.x_row;
    w += r0 * a.w_row;
  } else if constexpr (BY == ROWS) {
    int g;
    i64 r0, r1;
    if (!find_group<TM>(starts, a.groups, a.m, t.m, g, r0, r1)) return false;
    o.m0 = o.row0 = r0;
    o.m_there = r1 - r0;
    w += g * a.w_group;
    ws += g * a.ws_group;
  } else {
    o.m0 = o.row0 = t.m * TM;
    o.m_there = a.m - o.m0;
  }
  const i64 n_there = a.n - o.n0;
  if (o.m_there > TM) o.m_there = TM;
  o.x.p = XT ? x + o.m0 * 2 : x + o.m0 * a.x_row;
  o.x.row = a.x_row;
  o.x.there = XT ? o.m_there * 2 : o.m_there;
  o.x.vectors = a.x_vectors;
  o.w.p = WT ? w + o.n0 * 2 : w + o.n0 * a.w_row;
  o.w.row = a.w_row;
  o.w.there = WT ? n_there * 2 : n_there;
  o.w.vectors = a.w_vectors;
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
  return true;
}

// The sums of one 16 x 16 tile to out or, where the depth is split, to this part's sums.
template <class OUT, int BY>
UNPM_DEV void put(OUT* out, float* parts, const product_args& a, int part, i64 row0, i64 m0, i64 n0, i64 m_there, int m, int n,
                  const f32x4& v) {
  const i64 n_there = a.n - n0 - n;
  if (m >= m_there || n_there <= 0) return;
  if (a.parts > 1) {
    const i64 rows = BY == DEPTH ? a.groups * a.m : a.m, wide = (a.n + 3) / 4 * 4;
    *reinterpret_cast<f32x4*>(parts + (part * rows + row0 + m) * wide + n0 + n) = v;
  } else {
    const i64 g = BY == DEPTH ? (row0 - m0) / a.m : 0;
    store4<OUT>(out + g * a.out_group + (m0 + m) * a.out_row + n0 + n, v, n_there, a.wide);
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
  constexpr int STEP = xside::BYTES + wside::BYTES, SCALES = E == 1 ? WAVES * 256 : 0, STAGE = SPLIT * STEP + SCALES;
  constexpr int UNITS = xside::UNITS + wside::UNITS, EACH = SPLIT * UNITS / WAVES;
  static_assert(SPLIT * UNITS % WAVES == 0, "whole units a wave");
  static_assert(E == 2 || SPLIT * (TM + TN) <= WAVES * 64, "a scale a lane");
  static_assert(SPLIT * TM * TN * 4 <= STAGES * STAGE, "the sums of split steps");
  __shared__ __attribute__((aligned(1024))) u8 lds[STAGES * STAGE];

  place<XK, WKIND, XT, WT, BY, TM, TN> o;
  int part;
  if (!find_place<XK, WKIND, XT, WT, BY, SB, TM, TN>(xp, wp, xsp, wsp, starts, a, part, o)) return;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave % WM, wn = wave / WM % WN, own = wave / (WM * WN);
  f32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0, 0, 0, 0};

  // This lane's part of a stage.
  u32 offset[EACH];
  i32 after[EACH];
  const u32 lds0 = lds_address(lds);
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int u = (i * WAVES + wave) % UNITS;
    if (u < xside::UNITS) {
      offset[i] = o.x.offset(u, lane);
      after[i] = xside::after(u, lane);
    } else {
      offset[i] = o.w.offset(u - xside::UNITS, lane);
      after[i] = wside::after(u - xside::UNITS, lane);
    }
  }
  const float* scale = nullptr;
  int scale_step = 0;
  if constexpr (E == 1) {
    // A scale that no row has, or a step behind the last, is another's: it multiplies zeros, or rows that are not stored.
    const int f = wave * 64 + lane, r = f % (TM + TN);
    scale_step = f / (TM + TN) < SPLIT ? f / (TM + TN) : 0;
    scale = r < TM ? o.xs + least(r, o.xs_last) * a.xs_row : o.ws + least((r - TM) / SB, o.ws_last) * a.ws_row;
  }
  auto issue = [&](i64 stage, int slot) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int v = i * WAVES + wave, u = v % UNITS;
      const i64 step = o.first + stage * SPLIT + v / UNITS, left = o.end - step * D;
      const int at = slot * STAGE + v * 1024;
      if constexpr (DIRECT) {
        const bool isx = u < xside::UNITS;
        const i64 rest = isx ? xside::left(left) : wside::left(left);
        const u8* p = isx ? o.x.at(step) : o.w.at(step);
        load_to_lds(p, after[i] < rest ? offset[i] : OUTSIDE, lds0 + at);
      } else {
        const u32x4 y = u < xside::UNITS ? o.x.fetch(u, lane, step, left) : o.w.fetch(u - xside::UNITS, lane, step, left);
        *reinterpret_cast<u32x4*>(lds + at + lane * 16) = y;
      }
    }
    if constexpr (E == 1) {
      const float* p = scale + least(o.first + stage * SPLIT + scale_step, o.last - 1);
      const int at = slot * STAGE + SPLIT * STEP + wave * 256;
      if constexpr (DIRECT)
        load_word_to_lds(p, lds0 + at);
      else
        *reinterpret_cast<float*>(lds + at + lane * 4) = *p;
    }
  };
  auto compute = [&](int slot) {
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
      const float* sl = reinterpret_cast<const float*>(lds + slot * STAGE + SPLIT * STEP) + own * (TM + TN);
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
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[n][m][j] = __builtin_fmaf(p[j], xsc[m] * (SB == 1 ? wsc[j] : wsc[0]), acc[n][m][j]);
        }
      }
    }
  };

  const i64 stages = (o.last - o.first + SPLIT - 1) / SPLIT;
  if (stages > 0) {
    constexpr int LOADS = EACH + (E == 1);  // of a wave and stage
    int slot = 0;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(s, s);
    for (i64 s = 0; s < stages; ++s) {
      if constexpr (DIRECT) wait_loads<(STAGES - 2) * LOADS>();
      lds_barrier();
      issue(s + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
      compute(slot);
      slot = slot == STAGES - 1 ? 0 : slot + 1;
    }
    if constexpr (DIRECT) wait_loads<0>();  // LDS is not written after the block's end
  }

  if constexpr (SPLIT > 1) {
    lds_barrier();
    float* sums = reinterpret_cast<float*>(lds);  // [SPLIT][TM][TN]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m)
        *reinterpret_cast<f32x4*>(sums + (own * TM + (wm * MT + m) * 16 + (lane & 15)) * TN + (wn * NT + n) * 16 + (lane >> 4) * 4) =
            acc[n][m];
    lds_barrier();
    for (int q = threadIdx.x; q < TM * TN / 4; q += WAVES * 64) {
      const int m = q / (TN / 4), n = q % (TN / 4) * 4;
      f32x4 v = *reinterpret_cast<const f32x4*>(sums + m * TN + n);
#pragma unroll
      for (int s = 1; s < SPLIT; ++s) v += *reinterpret_cast<const f32x4*>(sums + (s * TM + m) * TN + n);
      put<OUT, BY>(out, parts, a, part, o.row0, o.m0, o.n0, o.m_there, m, n, v);
    }
  } else {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m)
        put<OUT, BY>(out, parts, a, part, o.row0, o.m0, o.n0, o.m_there, (wm * MT + m) * 16 + (lane & 15),
                     (wn * NT + n) * 16 + (lane >> 4) * 4, acc[n][m]);
  }
}

// The sums of a split depth, part after part.
template <class OUT, int BY>
UNPM_DEV void join(const i32* starts, OUT* out, const float* parts, const product_args& a) {
  const i64 rows = BY == DEPTH ? a.groups * a.m : a.m, quads = (a.n + 3) / 4;
  i64 r0 = 0, r1 = rows;
  if constexpr (BY == ROWS) {
    i64 skip;
    group_rows(starts, 0, rows, r0, skip);
    group_rows(starts, a.groups - 1, rows, skip, r1);
  }
  for (i64 i = r0 * quads + (i64)blockIdx.x * 256 + threadIdx.x; i < r1 * quads; i += (i64)gridDim.x * 256) {
    const i64 r = i / quads, n = i % quads * 4;
    f32x4 v = *reinterpret_cast<const f32x4*>(parts + r * quads * 4 + n);
    for (int p = 1; p < a.parts; ++p) v += *reinterpret_cast<const f32x4*>(parts + (p * rows + r) * quads * 4 + n);
    const i64 g = BY == DEPTH ? r / a.m : 0;
    store4<OUT>(out + g * a.out_group + (r - g * a.m * (BY == DEPTH)) * a.out_row + n, v, a.n - n, a.wide);
  }
}

// ---------------------------------------------------------------------------------------
// Quantisation: codes of y = x or its transpose, and the f32 scale of each block of 128 columns and RB rows of y:
// scale = most / largest code, code = y / scale rounded to even, both quotients correctly rounded.  A block of zeros has the
// scale 0 and divides as by 1; one that holds a NaN or an infinity has a NaN scale and codes 0.
//
// Magnitudes are compared as integers (NaN above infinity above every number).  The quotient of two f32 numbers is taken
// from the divisor's reciprocal by one correction (P. Markstein, 1990), exact while the remainder is a normal number;
// the scales where it may not be divide.
// ---------------------------------------------------------------------------------------
struct quant_args {
  i64 rows, cols;  // of x
  i64 x_row, code_row, scale_row;
  i32 x_vectors, code_vectors;
};

template <int KIND> UNPM_DEV float largest() { return KIND == E4M3 ? 448.0f : 57344.0f; }

struct step_of {
  float scale, unit, inverse;
  bool divide, none;
};
template <int KIND> UNPM_DEV step_of block_step(u32 most) {
  step_of s;
  s.none = most >= 0x7F800000u;
  s.scale = s.none ? __builtin_nanf("") : bits<float>(most) / largest<KIND>();
  s.unit = s.scale > 0.0f ? s.scale : 1.0f;
  s.inverse = 1.0f / s.unit;
  s.divide = s.unit < 0x1p-90f;
  return s;
}
UNPM_DEV float quotient(float y, const step_of& s) {
  if (s.none) return 0.0f;
  if (s.divide) return y / s.unit;
  const float q = y * s.inverse;
  return __builtin_fmaf(-__builtin_fmaf(q, s.unit, -y), s.inverse, q);  // in this order a zero keeps its sign
}
// Four codes as a word.
template <int KIND> UNPM_DEV u32 codes4(float a, float b, float c, float d) {
  if constexpr (KIND == E4M3)
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
  else
    return __builtin_amdgcn_cvt_pk_bf8_f32(c, d, __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false), true);
}
UNPM_DEV u32 magnitude(float x) { return bits<u32>(x) & 0x7FFFFFFFu; }
UNPM_DEV u32 more(u32 a, u32 b) { return a > b ? a : b; }

// N elements of a row from column c on, zeros past the last one.
template <class T, int N> UNPM_DEV void load_row(const T* row, i64 c, i64 cols, bool vectors, float (&y)[N]) {
  if (vectors && c + N <= cols) {
    constexpr int V = 16 / sizeof(T);
    struct alignas(16) vec {
      T v[V];
    };
#pragma unroll
    for (int i = 0; i < N; i += V) {
      const vec v = *reinterpret_cast<const vec*>(row + c + i);
#pragma unroll
      for (int j = 0; j < V; ++j) y[i + j] = (float)v.v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = c + i < cols ? (float)row[c + i] : 0.0f;
  }
}
template <int W> UNPM_DEV void store_codes(u8* row, i64 c, i64 cols, bool vectors, const u32 (&w)[W]) {
  if (vectors && c + 4 * W <= cols) {
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

// A scale per row and block: 8 lanes hold its 128 elements, 16 each.
template <class T, int KIND> UNPM_DEV void quantise_rows(const T* x, u8* codes, float* scales, const quant_args& a) {
  const i64 blocks = (a.cols + 127) / 128, all = a.rows * blocks;
  const int lane = threadIdx.x & 7;
  for (i64 i = ((i64)blockIdx.x * 256 + threadIdx.x) / 8; i < all; i += (i64)gridDim.x * 32) {
    const i64 r = i / blocks, b = i % blocks, c = b * 128 + lane * 16;
    float y[16];
    load_row<T, 16>(x + r * a.x_row, c, a.cols, a.x_vectors, y);
    u32 most = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) most = more(most, magnitude(y[j]));
#pragma unroll
    for (int d = 1; d < 8; d *= 2) most = more(most, (u32)__shfl_xor((i32)most, d));
    const step_of s = block_step<KIND>(most);
    u32 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = codes4<KIND>(quotient(y[4 * j], s), quotient(y[4 * j + 1], s), quotient(y[4 * j + 2], s), quotient(y[4 * j + 3], s));
    store_codes<4>(codes + r * a.code_row, c, a.cols, a.code_vectors, w);
    if (lane == 0) scales[r * a.scale_row + b] = s.scale;
  }
}

// The other forms: a block takes 128 x 128 elements of x; thread (i, j) rows 8 i .. 8 i + 7 and columns 8 j .. 8 j + 7.
// One scale for all of them, or (TURNED) one for each column, whose 128 rows lie along y's row.
template <class T, int KIND, int RB, bool TURNED>
UNPM_DEV void quantise_tiles(const T* x, u8* codes, float* scales, const quant_args& a) {
  static_assert(RB == 128 || TURNED, "scales of rows are quantise_rows's");
  constexpr int ROW = 128 + 16;  // of a transposed tile in LDS
  __shared__ u32 tops[16][128];
  __shared__ __attribute__((aligned(16))) u8 turned[TURNED ? 128 * ROW : 16];
  const i64 across = (a.cols + 127) / 128, all = (a.rows + 127) / 128 * across;
  const int i = threadIdx.x / 16, j = threadIdx.x % 16;
  for (i64 t = blockIdx.x; t < all; t += gridDim.x) {
    const i64 tr = t / across, tc = t % across, r0 = tr * 128 + i * 8, c0 = tc * 128 + j * 8;
    float y[8][8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r0 + r < a.rows) {
        load_row<T, 8>(x + (r0 + r) * a.x_row, c0, a.cols, a.x_vectors, y[r]);
      } else {
#pragma unroll
        for (int c = 0; c < 8; ++c) y[r][c] = 0.0f;
      }
    }
    u32 top[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      top[c] = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) top[c] = more(top[c], magnitude(y[r][c]));
    }
    if constexpr (RB == 128) {
      u32 most = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) most = more(most, top[c]);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) most = more(most, (u32)__shfl_xor((i32)most, d));
      if ((threadIdx.x & 63) == 0) tops[0][threadIdx.x / 64] = most;
      __syncthreads();
      most = more(more(tops[0][0], tops[0][1]), more(tops[0][2], tops[0][3]));
      const step_of s = block_step<KIND>(most);
      if (threadIdx.x == 0) scales[(TURNED ? tc : tr) * a.scale_row + (TURNED ? tr : tc)] = s.scale;
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int c = 0; c < 8; ++c) y[r][c] = quotient(y[r][c], s);
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) tops[i][j * 8 + c] = top[c];
      __syncthreads();
      if (threadIdx.x < 128) {
        u32 most = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) most = more(most, tops[k][threadIdx.x]);
        tops[0][threadIdx.x] = most;
        if (tc * 128 + threadIdx.x < a.cols) scales[(tc * 128 + threadIdx.x) * a.scale_row + tr] = block_step<KIND>(most).scale;
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const step_of s = block_step<KIND>(tops[0][j * 8 + c]);
#pragma unroll
        for (int r = 0; r < 8; ++r) y[r][c] = quotient(y[r][c], s);
      }
    }
    if constexpr (TURNED) {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        *reinterpret_cast<u32x2*>(turned + (j * 8 + c) * ROW + i * 8) =
            u32x2{codes4<KIND>(y[0][c], y[1][c], y[2][c], y[3][c]), codes4<KIND>(y[4][c], y[5][c], y[6][c], y[7][c])};
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = k * 32 + threadIdx.x / 8, part = threadIdx.x % 8;
        if (tc * 128 + c < a.cols) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(turned + c * ROW + part * 16);
          const u32 w[4] = {v[0], v[1], v[2], v[3]};
          store_codes<4>(codes + (tc * 128 + c) * a.code_row, tr * 128 + part * 16, a.rows, a.code_vectors, w);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r0 + r < a.rows) {
          const u32 w[2] = {codes4<KIND>(y[r][0], y[r][1], y[r][2], y[r][3]), codes4<KIND>(y[r][4], y[r][5], y[r][6], y[r][7])};
          store_codes<2>(codes + (r0 + r) * a.code_row, c0, a.cols, a.code_vectors, w);
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
// With one chunk, one block does both.  Inside a chunk a wave takes a run of ids, 64 at a time; the lanes of one
// id find each other by its bits, so their order is that of the lanes.
// ---------------------------------------------------------------------------------------
struct rows_args {
  i64 n, per, chunk;  // ids, ids of a row, ids of a block: a multiple of 64 times the waves
  i32 groups, chunks;
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
  for (int g = threadIdx.x; g < SORT_WAVES * MOST_GROUPS; g += SORT_WAVES * 64) (&counts[0][0])[g] = 0;
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
  // This thread's groups t * EACH ..: how many ids they have in all, and in the chunks before this one.
  i32 all[EACH], ahead[EACH], own = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int g = t * EACH + e;
    all[e] = ahead[e] = 0;
    if (g < a.groups) {
      if (a.chunks > 1) {
        for (int c = 0; c < a.chunks; ++c) {
          const i32 v = counted[(i64)c * a.groups + g];
          all[e] += v;
          ahead[e] += c < (int)blockIdx.x ? v : 0;
        }
      } else {
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) all[e] += counts[w][g];
      }
    }
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
      before[g] = start + ahead[e];
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
      rows[at] = (i32)(i / a.per);
      // The last of the lanes moves the count on; the wave has read it by then.
      if ((same >> lane) == 1) counts[wave][g] = at + 1;
    } else if (i < r.last) {
      place[i] = -1;
    }
  }
}

}  // namespace unpm
