// unpopped-hip device library of the rotary and 4-bit cache forms (gfx950, wave64).
//
// The emitter writes these forms' sources as this library + the `extern "C" __global__` entries that
// instantiate its templates, as it does with the fold and scan library for the lifted forms.
//
// Numerics: angles, cosines and sines in f64; the rotation in f32 (f64 ahead of a quantisation, whose
// borders it decides); scores, softmax statistics and sums in f32; each output rounded once.

#if !defined(__HIPCC_RTC__)
#include <hip/hip_runtime.h>
#endif

namespace unp4 {

typedef unsigned char u8;
typedef unsigned short u16;
typedef unsigned int u32;
typedef unsigned long long u64;
typedef int i32;
typedef long long i64;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef u32 u32x4 __attribute__((ext_vector_type(4)));

#define UNP4_DEV __device__ __forceinline__

enum : int { SCALE_NONE = 0, SCALE_LINEAR = 1, SCALE_RAMP = 2 };
enum : int { HALVES = 0, PAIRS = 1 };

template <class T, int N> struct alignas(sizeof(T) * N) vec {
  T v[N];
};
template <class T, int N> UNP4_DEV vec<T, N> load(const T* p) { return *reinterpret_cast<const vec<T, N>*>(p); }
template <class T, int N> UNP4_DEV void store(T* p, const vec<T, N>& x) { *reinterpret_cast<vec<T, N>*>(p) = x; }
// A store past the caches, for what this launch does not read again.
template <class T, int N> UNP4_DEV void store_stream(T* p, const vec<T, N>& x) {
  constexpr int W = sizeof(x) / 4;
  if constexpr (W % 4 == 0) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      u32x4 y;
      __builtin_memcpy(&y, reinterpret_cast<const char*>(&x) + 4 * i, 16);
      __builtin_nontemporal_store(y, reinterpret_cast<u32x4*>(p) + i / 4);
    }
  } else if constexpr (W == 2) {
    u64 y;
    __builtin_memcpy(&y, &x, 8);
    __builtin_nontemporal_store(y, reinterpret_cast<u64*>(p));
  } else {
    store<T, N>(p, x);
  }
}

// ---------------------------------------------------------------------------------------
// Position tables: [count][ROT / 2][cos, sin] of position first + row.
//
// 64-bit arithmetic beside a write of what it makes: 262144 x 64 pairs take 30 us, a plain write of them 21, and the VALU
// issues in 60% of the cycles.  The product of position and frequency is taken in turns (frequency / 2 pi), whose whole and
// quarter part go off exactly, and on the remaining eighth of a turn either side sine and cosine are their series to x^11
// and x^10 (off by less than 2^-33, rounded to 2^-24 after).  A lane makes V adjacent pairs; a block computes the ROT / 2
// frequencies once, into LDS.
// ---------------------------------------------------------------------------------------
struct stretch {
  int kind;
  double log_base, factor, low, high, original, amplitude;
};

template <int ROT>
UNP4_DEV double frequency(int i, const stretch& s) {
  double f = exp(-2.0 * i / ROT * s.log_base);
  if (s.kind == SCALE_LINEAR) f /= s.factor;
  if (s.kind == SCALE_RAMP) {
    const double r = s.original * f / 6.283185307179586476925;
    const double b = fmin(1.0, fmax(0.0, (r - s.low) / (s.high - s.low)));
    f *= b + (1.0 - b) / s.factor;
  }
  return f;
}

// The cosine and sine of `turns` turns.
UNP4_DEV void turn_of(double turns, double& cs, double& sn) {
  const double part = turns - rint(turns), quarter = rint(part * 4.0);
  const double x = fma(quarter, -0.25, part) * 6.283185307179586476925, y = x * x;
  double a = -1.0 / 39916800.0, b = -1.0 / 3628800.0;
  a = fma(a, y, 1.0 / 362880.0);
  b = fma(b, y, 1.0 / 40320.0);
  a = fma(a, y, -1.0 / 5040.0);
  b = fma(b, y, -1.0 / 720.0);
  a = fma(a, y, 1.0 / 120.0);
  b = fma(b, y, 1.0 / 24.0);
  a = fma(a, y, -1.0 / 6.0);
  b = fma(b, y, -0.5);
  a = fma(a * y, x, x);
  b = fma(b, y, 1.0);
  const int q = (int)quarter;  // -2 .. 2
  cs = q & 1 ? a : b;
  sn = q & 1 ? b : a;
  cs = q == 1 || q == 2 || q == -2 ? -cs : cs;
  sn = q == -1 || q == 2 || q == -2 ? -sn : sn;
}

template <int ROT, int V>
UNP4_DEV void rope_table(float* out, i64 first, i64 count, const stretch& s) {
  constexpr int H = ROT / 2, U = H / V;
  __shared__ double f[H];
  for (int i = threadIdx.x; i < H; i += 256) f[i] = frequency<ROT>(i, s) * 0.15915494309189533576888;
  __syncthreads();
  // Rows and units of V pairs in order; a step adds whole rows and a rest, so only the first divides.
  const i64 at = (i64)blockIdx.x * 256 + threadIdx.x, step = (i64)gridDim.x * 256, dr = step / U;
  const int du = (int)(step - dr * U);
  i64 row = at / U;
  for (int unit = (int)(at - row * U);; row += dr, unit += du) {
    if (unit >= U) {
      unit -= U;
      ++row;
    }
    if (row >= count) return;
    vec<float, 2 * V> y;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      double cs, sn;
      turn_of((double)(first + row) * f[unit * V + i], cs, sn);
      y.v[2 * i] = (float)(cs * s.amplitude);
      y.v[2 * i + 1] = (float)(sn * s.amplitude);
    }
    store_stream<float, 2 * V>(out + row * ROT + unit * 2 * V, y);
  }
}

// ---------------------------------------------------------------------------------------
// Rotation of heads.
//
// (x0, x1) -> (x0 c - x1 s, x1 c + x0 s), the sine negated for the inverse.  It reads and writes each
// element once: a stream.  A unit of the vector entry is V pairs (two 16-byte loads and stores) or 2V
// elements that are only copied; the plain entry takes a pair or a copied element at a time (16384 tokens x 40 heads of 100,
// all of it rotated, 135 us, 2.0 TB/s; of 80, of which 20, 187 us).  An output larger than half of the last-level cache is
// stored past the caches: 16384 tokens x 40 heads x 128 bf16 65.2 us against 67.3 (5.3 TB/s, a plain copy 6.35), but
// 4001 x 24 x 128 f32 (49 MB) 19.6 against 17.4.
// ---------------------------------------------------------------------------------------
struct rope_args {
  i64 tokens, x_token, x_head, out_token, out_head, first, rows;
  int heads, units;  // units of a head: the rotated ones, and the copied ones unless x and out are one
  int past, pad;     // store past the caches
};

template <bool INV> UNP4_DEV void turn(float& a, float& b, float c, float s) {
  if (INV) s = -s;
  const float x0 = a, x1 = b;
  a = fmaf(x0, c, -(x1 * s));
  b = fmaf(x1, c, x0 * s);
}

template <class T, int V> UNP4_DEV void put_unit(T* p, const vec<T, V>& x, int past) {
  if (past)
    store_stream<T, V>(p, x);
  else
    store<T, V>(p, x);
}

template <class T, int D, int ROT, int LAYOUT, bool INV, class I, int V>
UNP4_DEV void rope(const T* x, const I* positions, const float* table, T* out, const rope_args& a) {
  constexpr int RU = V > 0 ? ROT / 2 / (V > 0 ? V : 1) : ROT / 2;  // rotated units of a head
  const i64 per = (i64)a.heads * a.units;
  // Items (token, head, unit) in order; a step adds whole tokens and a rest, so only the first divides.
  const i64 at0 = (i64)blockIdx.x * 256 + threadIdx.x, step = (i64)gridDim.x * 256;
  i64 token = at0 / per, rest = at0 - token * per;
  const i64 dt = step / per, dr = step - dt * per;
  for (; token < a.tokens; token += dt, rest += dr) {
    if (rest >= per) {
      rest -= per;
      if (++token >= a.tokens) break;
    }
    const i64 row = (i64)((u64)(i64)positions[token] - (u64)a.first);  // any position, without overflow
    if ((u64)row >= (u64)a.rows) continue;
    const int head = (int)((u32)rest / (u32)a.units), unit = (int)rest - head * a.units;
    const T* xp = x + token * a.x_token + head * a.x_head;
    T* op = out + token * a.out_token + head * a.out_head;
    const float* cs = table + row * ROT;
    if constexpr (V > 0) {
      if (unit < RU) {
        const int p0 = LAYOUT == HALVES ? unit * V : 2 * unit * V, p1 = LAYOUT == HALVES ? p0 + ROT / 2 : p0 + V;
        vec<T, V> u = load<T, V>(xp + p0), w = load<T, V>(xp + p1);
        f32x4 t[V / 2];
        for (int i = 0; i < V / 2; ++i) t[i] = *reinterpret_cast<const f32x4*>(cs + 2 * unit * V + 4 * i);
        for (int i = 0; i < V; ++i) {
          const float c = t[i / 2][2 * (i & 1)], s = t[i / 2][2 * (i & 1) + 1];
          T& e0 = LAYOUT == HALVES ? u.v[i] : (i < V / 2 ? u.v[2 * i] : w.v[2 * i - V]);
          T& e1 = LAYOUT == HALVES ? w.v[i] : (i < V / 2 ? u.v[2 * i + 1] : w.v[2 * i + 1 - V]);
          float f0 = (float)e0, f1 = (float)e1;
          turn<INV>(f0, f1, c, s);
          e0 = (T)f0;
          e1 = (T)f1;
        }
        put_unit(op + p0, u, a.past);
        put_unit(op + p1, w, a.past);
      } else {
        const int p = ROT + (unit - RU) * 2 * V;
        const vec<T, V> u = load<T, V>(xp + p), w = load<T, V>(xp + p + V);
        put_unit(op + p, u, a.past);
        put_unit(op + p + V, w, a.past);
      }
    } else {
      if (unit < RU) {
        const int p0 = LAYOUT == HALVES ? unit : 2 * unit, p1 = LAYOUT == HALVES ? unit + ROT / 2 : 2 * unit + 1;
        float f0 = (float)xp[p0], f1 = (float)xp[p1];
        turn<INV>(f0, f1, cs[2 * unit], cs[2 * unit + 1]);
        op[p0] = (T)f0;
        op[p1] = (T)f1;
      } else {
        op[ROT + unit - RU] = xp[ROT + unit - RU];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// The cache's records: P tokens of one head (key codes, value codes, key words, value words).
// ---------------------------------------------------------------------------------------
template <int D, int GROUP, int P> struct record {
  static constexpr int W = D / 8, G = D / GROUP;       // words and groups of a token
  static constexpr int KEYS = 0, VALUES = P * W;       // in words
  static constexpr int KPAR = 2 * P * W, VPAR = KPAR + G * P;
  static constexpr int WORDS = VPAR + G * P;
  static UNP4_DEV int key(int t, int w) { return KEYS + t * W + (w & 3) * (D / 32) + (w >> 2); }
  static UNP4_DEV int value(int t, int w) { return VALUES + ((t >> 2) * W + w) * 4 + (t & 3); }
  static UNP4_DEV int kpar(int t, int g) { return KPAR + g * P + t; }
  static UNP4_DEV int vpar(int t, int g) { return VPAR + g * P + t; }
};

UNP4_DEV float scale_of(u32 word) { return (float)__builtin_bit_cast(_Float16, (u16)word); }
UNP4_DEV float zero_of(u32 word) { return (float)(word >> 16); }

// Lanes that hold the words of one head: the next power of two, so that a group's lanes are neighbours.
constexpr int lanes_of(int words) {
  int n = 1;
  while (n < words) n *= 2;
  return n;
}

struct cache_args {
  i64 tokens, slots, k_token, k_head, v_token, v_head, first, rows;  // slots: of the cache
};

// Eight adjacent elements of a head.
template <class T, bool ALIGNED> UNP4_DEV void load8(const T* p, T (&x)[8]) {
  if (ALIGNED) {
    const vec<T, 8> u = load<T, 8>(p);
    for (int i = 0; i < 8; ++i) x[i] = u.v[i];
  } else {
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
}

// The maximum over N neighbouring lanes, N a power of two up to 32, by lane permutations within a row of 16 and, for 32,
// an exchange of two rows.
template <int CTRL> UNP4_DEV float permuted(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
}
template <int N> UNP4_DEV float lane_max(float x) {
  if (N > 1) x = fmaxf(x, permuted<0xB1>(x));   // pairs
  if (N > 2) x = fmaxf(x, permuted<0x4E>(x));   // fours
  if (N > 4) x = fmaxf(x, permuted<0x141>(x));  // eights, mirrored: each four is one value by now
  if (N > 8) x = fmaxf(x, permuted<0x140>(x));  // the row, mirrored
  if (N > 16) {
    const auto y = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(u32, x), __builtin_bit_cast(u32, x), false, false);
    x = fmaxf(__builtin_bit_cast(float, (u32)y[0]), __builtin_bit_cast(float, (u32)y[1]));
  }
  return x;
}

// Heads of the items that a block takes: a wave's lanes hold the words of one head for several tokens, four in a row
// first, whose words lie together in the cache.
template <int H, int W> struct items {
  static constexpr int L = lanes_of(W), BLOCK = 256 / L;
  i64 token;
  int head, w;
  bool key;
  static UNP4_DEV i64 count(i64 tokens) { return (tokens + 3) / 4 * (8 * H); }
  UNP4_DEV explicit items(i64 at) {
    const i64 four = at / (8 * H);
    const int in = (int)(at - four * (8 * H)), which = in / 4;
    token = four * 4 + in % 4;
    head = which % H;
    key = which < H;
    w = threadIdx.x % L;
  }
};

// ---------------------------------------------------------------------------------------
// Append: a lane holds one word's 8 elements of a key or a value head; a group's range is reduced over
// its lanes.  It reads the keys and values once and writes a quarter of that: a stream, if the arithmetic keeps out of
// its way.  It does not quite: 16384 tokens x 8 heads x 128 bf16 take 42 us, of which the exact rotation is 7, with the VALU
// issuing in 70% of the cycles (a plain copy of these bytes 15).  Four tokens are taken together, whose value words lie
// together.
//
// The codes are those of exact arithmetic on the rotated keys.  The rotation's products of a 16-bit element and a 32-bit
// cosine are exact in f64, so the rotated key is rounded to 53 bits, to 24 and to its type, however the sum is contracted: a key
// in 32 bits, as a program that rotates before it appends has it, then one in the cache's type.  A quotient
// y / s of two 11-bit numbers that is no tie between two codes is at least 2^-13 from one ((2 y - (2 n + 1) s) / 2 s is
// a multiple of y's or s's last place), and y times a reciprocal good to 2^-23 is off by less than 2^-17: it rounds
// as the quotient does, and only where some lane's comes within 2^-16 of a tie the wave divides.
// ---------------------------------------------------------------------------------------
template <class T, int H, int D, int GROUP, int P, int ROT, int LAYOUT, class I, bool ALIGNED>
UNP4_DEV void append(const T* k, const T* v, const I* slots, u32* cache, const I* positions, const float* table,
                     const cache_args& a) {
  typedef record<D, GROUP, P> R;
  typedef items<H, R::W> It;
  const i64 n = It::count(a.tokens);
  for (i64 at = (i64)blockIdx.x * It::BLOCK + threadIdx.x / It::L; at < n; at += (i64)gridDim.x * It::BLOCK) {
    const It it(at);
    if (it.token >= a.tokens) continue;  // the same in every lane of the item, as below
    const int w = it.w;
    const bool live = w < R::W, turns = ROT > 0 && it.key && 8 * w < ROT;
    const bool second = LAYOUT == HALVES && 8 * w >= ROT / 2;  // of the pairs' elements
    const int i0 = second ? 8 * w - ROT / 2 : 8 * w;
    // The elements are on their way before the slot says whether they go anywhere.
    T x[8], o[8];  // o: the pairs' other elements
    const T* p = it.key ? k + it.token * a.k_token + it.head * a.k_head : v + it.token * a.v_token + it.head * a.v_head;
    if (live) load8<T, ALIGNED>(p + 8 * w, x);
    if (LAYOUT == HALVES && turns) load8<T, ALIGNED>(p + (second ? i0 : i0 + ROT / 2), o);
    const i64 slot = (i64)slots[it.token];
    const i64 row = ROT > 0 ? (i64)((u64)(i64)positions[it.token] - (u64)a.first) : 0;  // any position, without overflow
    if ((u64)slot >= (u64)a.slots || (ROT > 0 && (u64)row >= (u64)a.rows)) continue;
    float y[8];
    float lo = 0.0f, hi = 0.0f, not_finite = 0.0f;
    if (live) {
      if (turns) {
        const float* cs = table + row * ROT;
        if (LAYOUT == HALVES) {
          for (int i = 0; i < 8; ++i) {
            const double c = cs[2 * (i0 + i)], s = cs[2 * (i0 + i) + 1];
            const double r = (double)(float)x[i] * c + (second ? 1.0 : -1.0) * ((double)(float)o[i] * s);
            x[i] = (T)(float)r;
          }
        } else {
          for (int i = 0; i < 4; ++i) {
            const double c = cs[8 * w + 2 * i], s = cs[8 * w + 2 * i + 1];
            const double x0 = (float)x[2 * i], x1 = (float)x[2 * i + 1];
            x[2 * i] = (T)(float)(x0 * c - x1 * s);
            x[2 * i + 1] = (T)(float)(x1 * c + x0 * s);
          }
        }
      }
      for (int i = 0; i < 8; ++i) {
        y[i] = (float)x[i];
        lo = fminf(lo, y[i]);
        hi = fmaxf(hi, y[i]);
        not_finite = fmaf(y[i], 0.0f, not_finite);  // 0, or no number
      }
      // A NaN or an infinity of either sign opens the range to infinity.
      hi = not_finite == 0.0f ? hi : __builtin_inff();
    }
    constexpr int GL = GROUP == D ? It::L : GROUP / 8;  // lanes of a group
    lo = -lane_max<GL>(-lo);
    hi = lane_max<GL>(hi);
    const _Float16 sh = (_Float16)((hi - lo) / 15.0f);
    const bool finite = (float)sh < __builtin_inff();
    const float s = finite && (float)sh > 0.0f ? (float)sh : 1.0f;
    const float inv = __builtin_amdgcn_rcpf(s);
    const float t0 = -lo * inv;
    float q[8], z = rintf(t0), near = fabsf(fabsf(t0 - z) - 0.5f);  // near: the least distance to a tie
    if (__any(near < 0x1p-16f)) z = rintf(-lo / s);
    z = finite ? __builtin_amdgcn_fmed3f(z, 0.0f, 15.0f) : 0.0f;
    if (!live) continue;
    near = 1.0f;
    for (int i = 0; i < 8; ++i) {
      const float t = y[i] * inv;
      q[i] = rintf(t);
      near = fminf(near, fabsf(fabsf(t - q[i]) - 0.5f));
    }
    if (__any(near < 0x1p-16f))
      for (int i = 0; i < 8; ++i) q[i] = rintf(y[i] / s);
    u32 word = 0;
    for (int i = 0; i < 8; ++i) word |= (u32)__builtin_amdgcn_fmed3f(q[i] + z, 0.0f, 15.0f) << (4 * i);
    if (!finite) word = 0;
    const int t = (int)(slot % P);
    u32* rec = cache + ((slot / P) * H + it.head) * (i64)R::WORDS;
    rec[it.key ? R::key(t, w) : R::value(t, w)] = word;
    if ((8 * w) % GROUP == 0) {
      const u32 bits = finite ? __builtin_bit_cast(u16, sh) : 0x7E00u;
      rec[it.key ? R::kpar(t, 8 * w / GROUP) : R::vpar(t, 8 * w / GROUP)] = bits | (u32)z << 16;
    }
  }
}

// ---------------------------------------------------------------------------------------
// Read back: a lane per word; a slot outside the cache gives zeros.  Bound by its stores, which go past the caches: 16384
// tokens x 8 heads x 128 bf16 17 us, 5 TB/s.
// ---------------------------------------------------------------------------------------
template <class T, int H, int D, int GROUP, int P, class I, bool ALIGNED>
UNP4_DEV void read(const I* slots, const u32* cache, T* k, T* v, const cache_args& a) {
  typedef record<D, GROUP, P> R;
  typedef items<H, R::W> It;
  const i64 n = It::count(a.tokens);
  for (i64 at = (i64)blockIdx.x * It::BLOCK + threadIdx.x / It::L; at < n; at += (i64)gridDim.x * It::BLOCK) {
    const It it(at);
    const int w = it.w;
    if (it.token >= a.tokens || w >= R::W) continue;
    const i64 slot = (i64)slots[it.token];
    vec<T, 8> o;
    if (slot >= 0 && slot < a.slots) {
      const int t = (int)(slot % P), g = 8 * w / GROUP;
      const u32* rec = cache + ((slot / P) * H + it.head) * (i64)R::WORDS;
      const u32 word = rec[it.key ? R::key(t, w) : R::value(t, w)];
      const u32 par = rec[it.key ? R::kpar(t, g) : R::vpar(t, g)];
      for (int i = 0; i < 8; ++i)
        o.v[i] = (T)(((float)(word >> (4 * i) & 15u) - zero_of(par)) * scale_of(par));
    } else {
      for (int i = 0; i < 8; ++i) o.v[i] = (T)0.0f;
    }
    T* p = (it.key ? k + it.token * a.k_token + it.head * a.k_head : v + it.token * a.v_token + it.head * a.v_head) + 8 * w;
    if (ALIGNED) {
      store_stream<T, 8>(p, o);
    } else {
      for (int i = 0; i < 8; ++i) p[i] = o.v[i];
    }
  }
}

// ---------------------------------------------------------------------------------------
// Attention over the cache.
//
// A wave holds QT x 16 / CG rows of a sequence (its tokens times the query heads of one key/value head) and walks
// the keys in steps of 32 CG, all in registers:
//   * S' = K Q' by mfma 16x16x32 f16, keys as rows and query rows as columns.  A key word's nibbles are used
//     as they lie: masked to bits 0..3 or 4..7 of a 16-bit half they are the subnormal f16 numbers n 2^-24
//     and n 2^-20, so 8 codes cost 5 operations, and the queries carry the powers of two (exactly: each row is
//     scaled to f16's range, bf16's 8 bits fit in f16's 11).  The group's scale and zero point are applied to the
//     f32 result: s (sum q n - zero sum q).  The unit adds 32 products in 24 bits from the largest one's on, a subnormal
//     number counting as one of 2^-14 there: less than 2^-14 of the row's largest element is dropped of a product.
//   * Few rows (a decode step) would leave most columns empty, and the softmax's cost is the lanes'.  So CG groups
//     of columns hold the same rows and each keeps the scores of its own 16 of 16 CG keys: columns of one row are
//     parts of its context, joined at the end as the waves are.
//   * softmax over the columns: a lane holds 8 keys of one column, so its maximum needs two exchanges, and
//     only when some score passes the running one by 2^4.9: p is held as 2^11 p in f16, which ends at 2^16
//     (moving at 2^0.9, with 2^15 p, cost a prompt 8%: the sums are multiplied anew each time).
//   * O' += V' P' with the value words as rows: sum p s (n - zero) is the product of n with p s less the sum of p s zero.
//     The nibbles are two bits up, n 2^-22 and n 2^-18, and the zero points normal numbers, so that no more is dropped of a
//     product than 2^-16 (odd elements 2^-20, zero points 2^-21) of the step's largest p s: less than 2^-11 of the largest
//     scale over all steps.  As they lie it is four times that, and all of one sign: one token over 200000 keys was off by
//     1.72e-3 in Bf16 and is by 1.66e-3 (its rounding alone 1.64e-3), over 65536 in F16 3.6e-4 and 2.5e-4, for 3% of a
//     prompt's time.  Key codes two bits up cost 1% more and gave nothing.
//     p s is rounded to f16 (both sums take it as rounded), s in a unit that puts the scales that the wave's rows see
//     between 2^-14 and 1, exactly: then what p s loses below f16's normal numbers is less than 2^-20 of the smallest
//     scale.  Where the scales lie further apart than that, the wave begins anew: p s is made in
//     f32, and each step of a row and group rounds it in a unit of its own (the check cost a prompt nothing; 32 sequences of
//     up to 400 x 32 rows take 269 us, 434 with scales too far apart, 296 with every fifth of them 0).
//     The scores are, lane by lane, the operand that this product needs when its key (g, i) of 4 x 8 is key
//     16 CG (i / 4) + 4 g + i % 4; a lane reads four tokens' words of 8 elements at once and pairs of tokens of one
//     element are made by byte permutes, so nothing goes through LDS.
//
// What bounds it: a decode step its reads (64 single tokens x 8 heads over up to 16384 keys 140 us, 5.4 TB/s, a plain read
// 7.07; one over 262144 keys 53, 5.7 TB/s), a prompt the VALU's issue (9847 tokens x 32 heads of three sequences, causal,
// 362 us one after another, 769 TFLOP/s: 78% of the cycles issue VALU or matrix instructions, about 310 for 32 rows and 32
// keys; 412-425 on a card that was idle before).
// ---------------------------------------------------------------------------------------
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct attention_args {
  i64 tokens, batch, width, pages, q_token, q_head, out_token, out_head, window;
  int slots, splits, by_token;  // row tiles, parts of a context, and how tiles are numbered (tile_of)
  int q_wide, out_wide;         // rows of whole 16-byte vectors
};

constexpr float kHold = 11.0f, kSlack = 4.9f;
// exp2((score - maximum) factor + kHold) is one product and sum with the rounded maximum * factor - kHold, off by up to
// 2^-25 of it in log2: below 2^12 that is 2^-13, past 2^21 it would pass f16's end.  Beyond kFar the maximum is subtracted first,
// for an operation more a score.
constexpr float kFar = 0x1p12f;

// The maximum and the sum over the four lanes of a column (lane, lane ^ 16, lane ^ 32, lane ^ 48).
UNP4_DEV float column_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(u32, x), __builtin_bit_cast(u32, x), false, false);
  x = fmaxf(__builtin_bit_cast(float, (u32)a[0]), __builtin_bit_cast(float, (u32)a[1]));
  a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(u32, x), __builtin_bit_cast(u32, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (u32)a[0]), __builtin_bit_cast(float, (u32)a[1]));
}
UNP4_DEV float column_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(u32, x), __builtin_bit_cast(u32, x), false, false);
  x = __builtin_bit_cast(float, (u32)a[0]) + __builtin_bit_cast(float, (u32)a[1]);
  a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(u32, x), __builtin_bit_cast(u32, x), false, false);
  return __builtin_bit_cast(float, (u32)a[0]) + __builtin_bit_cast(float, (u32)a[1]);
}

// The halves of a word as f16, for products that take them as they are: a zero point n of 0..15 is the subnormal n 2^-24.
UNP4_DEV float low_half(u32 w) { return (float)__builtin_bit_cast(_Float16, (u16)w); }
UNP4_DEV float high_half(u32 w) { return (float)__builtin_bit_cast(_Float16, (u16)(w >> 16)); }
// The low, or high, halves of two words.
UNP4_DEV u32 low_halves(u32 a, u32 b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
UNP4_DEV u32 high_halves(u32 a, u32 b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// The maximum of each half over the wave.
typedef u16 u16x2 __attribute__((ext_vector_type(2)));
template <int CTRL> UNP4_DEV u16x2 half_max(u16x2 x) {
  const u32 w = __builtin_bit_cast(u32, x);
  return __builtin_elementwise_max(x, __builtin_bit_cast(u16x2, __builtin_amdgcn_update_dpp(w, w, CTRL, 0xF, 0xF, false)));
}
UNP4_DEV u16x2 wave_max(u16x2 x) {
  u32 w = __builtin_bit_cast(u32, x);
  auto y = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  x = __builtin_elementwise_max(__builtin_bit_cast(u16x2, (u32)y[0]), __builtin_bit_cast(u16x2, (u32)y[1]));
  w = __builtin_bit_cast(u32, x);
  y = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  x = __builtin_elementwise_max(__builtin_bit_cast(u16x2, (u32)y[0]), __builtin_bit_cast(u16x2, (u32)y[1]));
  return half_max<0x140>(half_max<0x141>(half_max<0x4E>(half_max<0xB1>(x))));  // pairs, fours, eights, the row
}

UNP4_DEV int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// Memory that this launch does not write, read at a place all lanes share: a scalar load, which does not queue
// behind the vector loads in flight.
typedef const __attribute__((address_space(4))) i32* uniform_ints;

// The sequence and tile of a tile number, by one wave.  Tiles are numbered so that a sequence's number is known
// from its start alone: its first is start * GQ / R + b (its rows fill at most one tile more than they span), or its
// first token (by_token: a token's GQ rows fit one tile).
struct tile {
  int seq, start, rows, length, at;  // rows: tokens of the sequence; at: the tile's number in it, or seq < 0
};
template <int GQ, int R>
UNP4_DEV tile tile_of(const i32* starts, const i32* lengths, const attention_args& a, int slot) {
  const int lane = threadIdx.x & 63, tokens = (int)a.tokens;
  auto start_of = [&](i64 b) {
    const int s = starts[b];
    return s < 0 ? 0 : s > tokens ? tokens : s;
  };
  auto first_of = [&](int s, i64 b) { return a.by_token ? (i64)s : (i64)s * GQ / R + b; };
  i64 lo = 0, hi = a.batch;
  for (;;) {  // the last b of lo .. hi - 1 whose first tile is at most slot
    const i64 step = (hi - lo + 63) / 64, b = lo + lane * step;
    const bool in = b < hi;
    const int s = start_of(in ? b : lo), e = start_of((in ? b : lo) + 1), n = lengths[in ? b : lo];
    const int count = __popcll(__ballot(in && first_of(s, b) <= slot));
    if (count == 0) return {-1, 0, 0, 0, 0};
    lo += (count - 1) * step;
    if (step == 1) {
      const int st = __builtin_amdgcn_readlane(s, count - 1), en = __builtin_amdgcn_readlane(e, count - 1);
      tile t{(int)lo, st, en - st, __builtin_amdgcn_readlane(n, count - 1), (int)(slot - first_of(st, lo))};
      if (t.at < 0 || (i64)t.at * R >= (i64)t.rows * GQ) t.seq = -1;
      return t;
    }
    hi = lo + step < hi ? lo + step : hi;
  }
}

template <int N> struct size {
  static constexpr int value = N;
};

// N adjacent elements of a row from their sums.
template <class T, int N> UNP4_DEV void put(T* p, const float (&o)[N], float by, bool wide) {
  vec<T, N> y;
#pragma unroll
  for (int i = 0; i < N; ++i) y.v[i] = (T)(by == 0.0f ? 0.0f : o[i] * by);
  if (wide) {
    store<T, N>(p, y);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = y.v[i];
  }
}
// w[r] of part g of a column and w[g] of part r change places, for all four r and g (lanes 16 apart).
template <int M> UNP4_DEV void transpose(u32 (&w)[4][M]) {
#pragma unroll
  for (int i = 0; i < M; ++i) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const auto y = __builtin_amdgcn_permlane32_swap(w[r][i], w[r + 2][i], false, false);
      w[r][i] = y[0];
      w[r + 2][i] = y[1];
    }
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      const auto y = __builtin_amdgcn_permlane16_swap(w[r][i], w[r + 1][i], false, false);
      w[r][i] = y[0];
      w[r + 1][i] = y[1];
    }
  }
}
// What a row's sums are multiplied with: a row that sees nothing gives 0.
UNP4_DEV float share_of(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
// top: the maximum in log2, to which p is held as 2^kHold p.
UNP4_DEV float log_sum(float top, float l) {
  return l == 0.0f ? -__builtin_inff() : (top - kHold + __log2f(l)) * 0.693147180559945309f;
}

template <class T> struct is_half {
  static constexpr bool value = false;
};
template <> struct is_half<_Float16> {
  static constexpr bool value = true;
};

// Adjacent words; ONCE: what this launch reads once (a sequence's rows fill one tile) goes past the caches (64 single tokens
// over up to 16384 keys took 154 us through them, 141 past them).
typedef u32 u32x2 __attribute__((ext_vector_type(2)));
template <class V, bool ONCE> UNP4_DEV V words_at(const u32* p) {
  const V* v = reinterpret_cast<const V*>(p);
  return ONCE ? __builtin_nontemporal_load(v) : *v;
}
template <int N, bool ONCE> UNP4_DEV void load_words(const u32* p, u32 (&to)[N]) {
  if constexpr (!ONCE) {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = p[i];
  } else if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 y = words_at<u32x4, true>(p + i);
      to[i] = y[0], to[i + 1] = y[1], to[i + 2] = y[2], to[i + 3] = y[3];
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const u32x2 y = words_at<u32x2, true>(p + i);
      to[i] = y[0], to[i + 1] = y[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = words_at<u32, true>(p + i);
  }
}

template <class T, int H, int QH, int D, int GROUP, int P, bool CAUSAL, bool LSE, int QT, int CG, bool ONCE> struct attention {
  static_assert(QT == 1 || CG == 1, "columns are shared by one row tile");
  typedef record<D, GROUP, P> R;
  static constexpr int GQ = QH / H, W = R::W, G = R::G, KJ = D / 32, JG = GROUP / 32;
  static constexpr int NB = 2 * CG, KEYS = 16 * NB, ROWS = 16 / CG;  // blocks of 16 keys, keys of a step; rows of a tile
  static constexpr int NP = KEYS > P ? KEYS / P : 1;                 // pages of a step
  // Value tiles: 16 rows of N adjacent elements each.  A group's words in tiles of 16 words, then one of the rest,
  // whose words go to several rows where they are few.
  static constexpr int GW = GROUP / 8, FULL = GW / 16, REST = GW % 16, TG = FULL + (REST ? 1 : 0), NT = G * TG;
  static constexpr int NREST = REST == 0 ? 0 : REST <= 4 ? 2 : REST <= 8 ? 4 : 8;
  static constexpr int NEG = FULL * 8 + NREST, NE = G * NEG;  // matrix products of 16 elements for a group, a head
  static constexpr int nibbles(int t) { return t % TG < FULL ? 8 : NREST; }
  static constexpr int product(int t, int e) { return t / TG * NEG + t % TG * 8 + e; }

  struct keys {
    u32 k[KJ];
  };
  struct values {
    u32x4 v[NT];
  };
  int lane, c, g;  // c: the row a lane gives and the column it holds, g: its part of the depth
  int own;         // the column's group: which 16 of 16 CG keys it keeps
  // The nibbles' masks in registers: as literals each takes an operation more.
  // mask0, mask1: nibbles at bits 0 and 4 of a half; mask2, mask6: at bits 2 and 6.
  u32 mask0, mask1, mask2, mask6;
  f16x8 q[QT][KJ];
  float qsum[QT][G], factor[QT];  // of this lane's column; qsum 2^24 times, as zeros are held; factor: raw scores to log2
  float m[QT];                    // running maximum
  bool far;                       // some maximum is beyond 2^kFar in log2 (all lanes agree)
  f32x4 l[QT];                    // the sum of p, in l[0] (EXACT_SUM: this lane's part of it until the end)
  // The value scales that the wave's rows saw so far, the same in all lanes: their f16 bits, but for zeros, are from `low` (in
  // both halves) to `span` above it, and `unit`, a power of two, puts them between 2^-14 and 1.
  _Float16 unit;
  u32 low, span;
  f32x4 o[QT][NE];
  // The sums of p s zero by group: this lane's parts, or (one group of columns, few of elements) a product whose rows
  // are all the same.
  static constexpr bool ZERO_PRODUCT = CG == 1 && G <= 2;
  // F16 outputs: p s is rounded once (bf16's rounding hides that p and then p s are), and the sum of p is of what was not
  // rounded, as the log-sum-exp's is; otherwise it is a product with ones, of p as rounded.
  static constexpr bool FINE = is_half<T>::value, EXACT_SUM = LSE || FINE;
  float zs[QT][G];
  f32x4 zp[QT][ZERO_PRODUCT ? G : 1];
  int end[QT], begin[QT];  // keys that the column sees

  UNP4_DEV void clear() {
    unit = (_Float16)0x1p14f;
    low = span = 0;  // no scales yet
    far = false;
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      m[x] = -__builtin_inff();
      l[x] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        zs[x][gi] = 0.0f;
        if (ZERO_PRODUCT) zp[x][ZERO_PRODUCT ? gi : 0] = f32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int e = 0; e < NE; ++e) o[x][e] = f32x4{0, 0, 0, 0};
    }
  }
  // Rows first .. first + QT ROWS - 1 (token * GQ + head of the group) of a sequence.
  UNP4_DEV void rows(const T* qp, const attention_args& a, const tile& t, int kv, int first, float scale, int cap) {
    asm("s_mov_b32 %0, 0x000f000f" : "=s"(mask0));
    asm("s_mov_b32 %0, 0x00f000f0" : "=s"(mask1));
    asm("s_mov_b32 %0, 0x003c003c" : "=s"(mask2));
    asm("s_mov_b32 %0, 0x03c003c0" : "=s"(mask6));
    clear();
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      const int r = first + x * 16 + c % ROWS;
      const bool in = r < t.rows * GQ;
      const int token = in ? r / GQ : 0, head = kv * GQ + (in ? r % GQ : 0);
      const T* p = qp + (i64)(t.start + token) * a.q_token + (i64)head * a.q_head;
      T raw[KJ][8];
      if (a.q_wide) {
#pragma unroll
        for (int j = 0; j < KJ; ++j) load8<T, true>(p + j * 32 + g * 8, raw[j]);
      } else {
#pragma unroll
        for (int j = 0; j < KJ; ++j) load8<T, false>(p + j * 32 + g * 8, raw[j]);
      }
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          raw[j][i] = in ? raw[j][i] : (T)0.0f;
          top = fmaxf(top, fabsf((float)raw[j][i]));
        }
      top = column_max(top);
      // The power of two that puts the largest element into 2^13 .. 2^14: odd nibbles weigh 16 times as much, so
      // their elements are scaled down by 16.
      int up = top > 0.0f && top < __builtin_inff() ? 13 - (int)((__builtin_bit_cast(u32, top) >> 23) & 255) + 127 : 0;
      up = up > 100 ? 100 : up;  // at least -114
      const float mul = __builtin_bit_cast(float, (u32)(up + 127) << 23);
#pragma unroll
      for (int gi = 0; gi < G; ++gi) qsum[x][gi] = 0.0f;
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = (i >> 1) + 4 * (i & 1);  // the element at place i of a word's operand
          const _Float16 y = (_Float16)((float)raw[j][d] * ((d & 1) ? mul * 0.0625f : mul));
          q[x][j][i] = y;
          qsum[x][j / JG] += (float)y * ((d & 1) ? 16.0f : 1.0f);
        }
      }
#pragma unroll
      for (int gi = 0; gi < G; ++gi) qsum[x][gi] = column_sum(qsum[x][gi]);
      // Where this ends at 2^127, two scores that differ at all are further apart than exp reaches either way.
      factor[x] = fminf(scale * 1.4426950408889634f * 0x1p24f * __builtin_bit_cast(float, (u32)(127 - up) << 23), 0x1p127f);
      const int last = CAUSAL ? t.length - t.rows + token + 1 : t.length;
      end[x] = in ? (last < cap ? last : cap) : 0;
      begin[x] = CAUSAL && a.window > 0 && a.window < last ? last - (int)a.window : 0;
    }
  }

  // The keys of steps at, at + by, .. below last, each loaded while the one before is multiplied.  lo, hi: the keys
  // from lo on and below hi that every column sees.
  struct stream {
    const u32* cache;
    uniform_ints table;  // the sequence's pages
    int kv, at, by, last, cap, lo, hi, pages;
    // The step being loaded, and the page numbers of both and of the one after as they lie in the table: what is made
    // of a number a step after its load does not wait for it.
    int next, id[NP], ahead[NP], far[NP];
    keys k[NB];
    values v[NB];
    u32x4 kp[2][G], vp[2][G];  // the words of the keys that this lane's column keeps
    UNP4_DEV void number(int step, int (&to)[NP]) const {  // cap > 0
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int key = step * KEYS + k * P;
        to[k] = table[(u32)(key < cap ? key : cap - 1) / P];
      }
    }
    UNP4_DEV bool good(int step, int b, const int (&id)[NP]) const {
      return step * KEYS + 16 * b < cap && (u32)id[b * 16 / P] < (u32)pages;
    }
    UNP4_DEV const u32* record_of(int b, const int (&id)[NP]) const {
      const int page = id[b * 16 / P];
      return cache + ((i64)((u32)page < (u32)pages ? page : 0) * H + kv) * (i64)R::WORDS;
    }
  };
  UNP4_DEV void load_keys(stream& s, int step, const int (&id)[NP]) const {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const u32* p = s.record_of(b, id) + R::KEYS + (step * KEYS + 16 * b) % P * W + (c * W + g * KJ);
      load_words<KJ, ONCE>(p, s.k[b].k);
    }
  }
  // The first of the column's keys of half h in their record's words: the record, plus their place.
  UNP4_DEV const u32* own_words(const stream& s, int h, int step, const int (&id)[NP]) const {
    auto place = [&](int b) { return s.record_of(b, id) + (step * KEYS + 16 * b) % P; };
    const u32* p = place(h * CG);
    if (P >= 16 * CG) return p + 16 * own;  // one page holds them all
#pragma unroll
    for (int b = 1; b < CG; ++b) p = own == b ? place(h * CG + b) : p;
    return p;
  }
  UNP4_DEV void load_key_words(stream& s, int step, const int (&id)[NP]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32* p = own_words(s, h, step, id) + g * 4;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) s.kp[h][gi] = *reinterpret_cast<const u32x4*>(p + R::kpar(0, gi));
    }
  }
  UNP4_DEV void load_value_words(stream& s, int step, const int (&id)[NP]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32* p = own_words(s, h, step, id) + g * 4;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) s.vp[h][gi] = *reinterpret_cast<const u32x4*>(p + R::vpar(0, gi));
    }
  }
  UNP4_DEV void load_values(stream& s, int step, const int (&id)[NP]) const {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const u32* p = s.record_of(b, id) + R::VALUES + (step * KEYS + 16 * b) % P * W;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int w = t % TG * 16 + c * nibbles(t) / 8;
        s.v[b].v[t] = words_at<u32x4, ONCE>(p + (g * W + t / TG * GW + (w < GW ? w : GW - 1)) * 4);
      }
    }
  }
  UNP4_DEV void open(stream& s) {
    lane = threadIdx.x & 63;
    c = lane & 15;
    g = lane >> 4;
    own = c / ROWS;
    if (s.at >= s.last) return;
    s.next = s.at + s.by < s.last ? s.at + s.by : s.at;
    s.number(s.at, s.id);
    s.number(s.next, s.ahead);
    load_keys(s, s.at, s.id);
    load_key_words(s, s.at, s.id);
    load_value_words(s, s.at, s.id);
    load_values(s, s.at, s.id);
  }

  UNP4_DEV f16x8 key_operand(u32 x) const {
    const u32 y = x >> 8;
    const u32x4 b = {x & mask0, x & mask1, y & mask0, y & mask1};
    return __builtin_bit_cast(f16x8, b);
  }
  // Value tile t of two blocks: out[e] is the operand of element e of each row's N.
  template <int N> UNP4_DEV void value_operands(const values& v0, const values& v1, int t, f16x8 (&out)[N]) const {
    u32 part[N][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u32 wa = k < 2 ? v0.v[t][2 * k] : v1.v[t][2 * k - 4], wb = k < 2 ? v0.v[t][2 * k + 1] : v1.v[t][2 * k - 3];
      if (N < 8) {  // this row's nibbles of the word
        wa >>= (c * N) % 8 * 4;
        wb >>= (c * N) % 8 * 4;
      }
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const u32 x = __builtin_amdgcn_perm(wb, wa, e ? 0x07060302u : 0x05040100u), x2 = x << 2, y = x >> 6;
        part[e][k] = x2 & mask2;
        part[e + 1][k] = x2 & mask6;
        if (N > 2) {
          part[e + 2 < N ? e + 2 : 0][k] = y & mask2;
          part[e + 3 < N ? e + 3 : 0][k] = y & mask6;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
      out[e] = __builtin_bit_cast(f16x8, u32x4{part[e][0], part[e][1], part[e][2], part[e][3]});
  }
  template <int N> UNP4_DEV void multiply_values(const stream& s, int t, int b, const f16x8 (&p)[QT][G]) {
    f16x8 va[N];
    value_operands<N>(s.v[b], s.v[CG + b], t, va);
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
      for (int x = 0; x < QT; ++x)
        o[x][product(t, e)] =
            __builtin_amdgcn_mfma_f32_16x16x32_f16(va[e], p[x][t / TG], o[x][product(t, e)], 0, 0, 0);
  }

  // Whether a value scale of a step lies outside the known range, by its bits; with ZEROS one of 0 does not.
  template <bool ZEROS> UNP4_DEV bool outside(const f16x2 (&vs)[G][4]) const {
    u16x2 most = {0, 0};
#pragma unroll
    for (int gi = 0; gi < G; ++gi)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const u16x2 b = __builtin_bit_cast(u16x2, vs[gi][k]), over = b - __builtin_bit_cast(u16x2, low);
        most = __builtin_elementwise_max(most, ZEROS ? over * __builtin_elementwise_min(b, u16x2{1, 1}) : over);
      }
    return most[0] > span || most[1] > span;
  }
  // Takes a step's value scales (under a mask those of keys that some row sees) into the known range, by their bits.  Gives what
  // the sums are multiplied with as their unit changes: 0 where no unit holds the range.
  UNP4_DEV float widen(const f16x2 (&vs)[G][4], bool mask, u32 seen) {
    u16x2 top = {0, 0}, bottom = {0, 0};  // bottom: 2^16 less the smallest, 0 for none
#pragma unroll
    for (int gi = 0; gi < G; ++gi)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        u16x2 b = __builtin_bit_cast(u16x2, __builtin_bit_cast(u32, vs[gi][k]) & 0x7FFF7FFFu);
        // No unit makes an infinity or a NaN a number.
        b *= __builtin_elementwise_min(__builtin_elementwise_sub_sat(u16x2{0x7C00, 0x7C00}, b), u16x2{1, 1});
        if (mask) b *= u16x2{(u16)(seen >> (2 * k) & 1), (u16)(seen >> (2 * k + 1) & 1)};
        top = __builtin_elementwise_max(top, b);
        bottom = __builtin_elementwise_max(bottom, (u16x2)(u16x2{0, 0} - b));
      }
    const u16x2 ends = wave_max(__builtin_elementwise_max(u16x2{top[0], bottom[0]}, u16x2{top[1], bottom[1]}));
    const u32 both = (u32)uniform(__builtin_bit_cast(int, ends)), most = both & 0xFFFFu, least = 0x10000u - (both >> 16);
    if (most == 0) return 1.0f;
    // A bit of room above and two below, so that later scales seldom pass the range.
    const u32 known = low + span & 0xFFFFu, next = ((most >> 10) + 1) << 10 | 0x3FFu;
    const u32 end = most <= known ? known : next < 0x7BFFu ? next : 0x7BFFu;
    const int exponent = (int)(end >> 10);  // of `end`, 15 too large: 2^14 over it times `end` is below 1
    const u32 limit = exponent >= 14 ? (u32)(exponent - 13) << 10 : exponent >= 4 ? 1u << (exponent - 4) : 0u;  // 2^-14 in it
    u32 from = least > 0xC00u ? least - 0x800u : 1u;
    from = from > limit ? from : least < limit ? least : limit;
    from = span != 0 && (low & 0xFFFFu) < from ? low & 0xFFFFu : from;
    if (from < limit) return 0.0f;
    low = from | from << 16;
    span = end - from;
    unit = (_Float16)__builtin_bit_cast(float, (u32)(141 - exponent) << 23);
    return __builtin_bit_cast(float, (u32)(127 + (int)(known >> 10) - exponent) << 23);
  }

  // The sums of a row tile and group into another unit.
  UNP4_DEV void rescale(int x, int gi, float by) {
    if (ZERO_PRODUCT)
      zp[x][ZERO_PRODUCT ? gi : 0] *= by;
    else
      zs[x][gi] *= by;
#pragma unroll
    for (int e = 0; e < NEG; ++e) o[x][gi * NEG + e] *= by;
  }
  // p s of a step whose scales have no common unit: in f32, then in the one that puts the column's largest into 2^10 .. 2^11
  // (2^15 at most: below that no p s of a maximal p and any scale is lost).  The sums go into it too; gives the way back.
  UNP4_DEV float alone(int x, int gi, const float (&y)[8], const f16x2 (&scale)[4], u32 seen, u32x4& p) {
    float w[8], top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = seen >> i & 1 ? y[i] * (float)scale[i / 2][i % 2] : 0.0f;
      top = fmaxf(top, fabsf(w[i]));
    }
    const int up = 137 - (int)(__builtin_bit_cast(u32, column_max(fminf(top, 0x1p40f))) >> 23);  // 10 less the exponent
    const float to = __builtin_bit_cast(float, (u32)(127 + (up < 15 ? up : 15)) << 23);
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = __builtin_bit_cast(u32, f16x2{(_Float16)(w[2 * k] * to), (_Float16)(w[2 * k + 1] * to)});
    rescale(x, gi, to);
    return 1.0f / to;
  }

  // Without APART: a step whose scales have no unit in common with those before is the last (the walk's sums do not count).
  // The loop keeps its one exit so: from a second one the compiler would have all loads land before each step.
  template <bool APART> UNP4_DEV void step(stream& s) {
    const int k0 = s.at * KEYS, after = s.next + s.by < s.last ? s.next + s.by : s.next;
    s.number(after, s.far);
    bool whole = k0 >= s.lo && k0 + KEYS <= s.hi;
#pragma unroll
    for (int k = 0; k < NP; ++k) whole &= (u32)s.id[k] < (u32)s.pages;
    const bool masked = !whole;
    float sc[QT][8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        f32x4 mine[QT];
#pragma unroll
        for (int b = 0; b < CG; ++b) {
          f16x8 ka[JG];
          f32x4 acc[QT];
#pragma unroll
          for (int j = 0; j < JG; ++j) ka[j] = key_operand(s.k[h * CG + b].k[gi * JG + j]);
#pragma unroll
          for (int x = 0; x < QT; ++x) acc[x] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < JG; ++j)
#pragma unroll
            for (int x = 0; x < QT; ++x)
              acc[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[j], q[x][gi * JG + j], acc[x], 0, 0, 0);
#pragma unroll
          for (int x = 0; x < QT; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[x][i] = b == 0 || own == b ? acc[x][i] : mine[x][i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const u32 w = s.kp[h][gi][i];
#pragma unroll
          for (int x = 0; x < QT; ++x) {
            const float d = fmaf(-high_half(w), qsum[x][gi], mine[x][i]);
            sc[x][4 * h + i] = fmaf(d, low_half(w), gi == 0 ? 0.0f : sc[x][4 * h + i]);
          }
        }
      }
    load_keys(s, s.next, s.ahead);
    load_key_words(s, s.next, s.ahead);
    u32 seen[QT];  // which of its 8 keys each of this lane's columns sees
    if (masked) {
      asm volatile("; a branch: not worth computing for every step");
#pragma unroll
      for (int x = 0; x < QT; ++x) seen[x] = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bool there = s.good(s.at, h * CG, s.id);
#pragma unroll
        for (int b = 1; b < CG; ++b) there = own == b ? s.good(s.at, h * CG + b, s.id) : there;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = k0 + 16 * (h * CG + own) + 4 * g + i;
#pragma unroll
          for (int x = 0; x < QT; ++x) {
            const bool sees = there && key < end[x] && key >= begin[x];
            sc[x][4 * h + i] = sees ? sc[x][4 * h + i] : -__builtin_inff();
            if (sees) seen[x] |= 1u << (4 * h + i);
          }
        }
      }
    }
    // The running maxima and the scales' range; p of a row against an old maximum may reach 2^kSlack.
    float top[QT];
    bool up = false;
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      top[x] = sc[x][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top[x] = fmaxf(top[x], sc[x][i]);
      up |= (top[x] - m[x]) * factor[x] > kSlack;
    }
    f16x2 vs[G][4];  // the scales of keys 2k, 2k + 1
#pragma unroll
    for (int gi = 0; gi < G; ++gi)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        vs[gi][k] = __builtin_bit_cast(f16x2, low_halves(s.vp[k / 2][gi][2 * (k % 2)], s.vp[k / 2][gi][2 * (k % 2) + 1]));
    float by = 1.0f;
    bool past = !APART && outside<false>(vs);
    if (__any(up || past)) {
      if (!APART) past = outside<true>(vs);
      if (__any(past)) {
        by = widen(vs, masked, masked ? seen[0] | seen[QT - 1] : 0xFFu);
        s.last = by == 0.0f ? s.at : s.last;
      }
      if (__any(up || past)) {
        bool beyond = false;
#pragma unroll
        for (int x = 0; x < QT; ++x) {
          const float next = fmaxf(m[x], column_max(top[x]));
          const float keep = m[x] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m[x] - next) * factor[x]);
          m[x] = next;
          beyond |= next != -__builtin_inff() && !(fabsf(next * factor[x]) <= kFar);
          l[x] *= keep;
#pragma unroll
          for (int gi = 0; gi < G; ++gi) rescale(x, gi, keep * by);
        }
        far = __any(beyond);
      }
    }
    if (far) {
      asm volatile("; a branch: not worth computing for every step");
#pragma unroll
      for (int x = 0; x < QT; ++x)
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[x][i] -= m[x] == -__builtin_inff() ? 0.0f : m[x];
    }
    u32x4 zero[G];
#pragma unroll
    for (int gi = 0; gi < G; ++gi)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (!APART) vs[gi][k] *= unit;
        // A zero point n as the normal number n 2^-9.
        const u32 z = high_halves(s.vp[k / 2][gi][2 * (k % 2)], s.vp[k / 2][gi][2 * (k % 2) + 1]) & mask0;
        zero[gi][k] = __builtin_bit_cast(u32, __builtin_bit_cast(f16x2, z) * f16x2{(_Float16)0x1p15f, (_Float16)0x1p15f});
      }
    const f16x8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
    u32x4 p[QT][G];
    float back[QT][G];  // APART: from a row's own unit
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      const float off = m[x] == -__builtin_inff() ? 0.0f : far ? kHold : fmaf(-m[x], factor[x], kHold);
      f16x8 e, fine[G];
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = __builtin_amdgcn_exp2f(fmaf(sc[x][i], factor[x], off));
        if (EXACT_SUM) l[x][0] += y[i];
        e[i] = (_Float16)y[i];
        if (FINE && !APART)
#pragma unroll
          for (int gi = 0; gi < G; ++gi) fine[gi][i] = (_Float16)fmaf(y[i], (float)vs[gi][i / 2][i % 2], 0.0f);
      }
      if (!EXACT_SUM) l[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, e, l[x], 0, 0, 0);
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        if (APART) back[x][gi] = alone(x, gi, y, vs[gi], masked ? seen[x] : 0xFFu, p[x][gi]);
#pragma unroll
        for (int k = 0; k < 4 && !APART; ++k)
          p[x][gi][k] = __builtin_bit_cast(u32, FINE ? f16x2{fine[gi][2 * k], fine[gi][2 * k + 1]}
                                                     : f16x2{e[2 * k], e[2 * k + 1]} * vs[gi][k]);
        if (!APART && masked) {  // a scale that is no number does not reach the columns that do not see its key
          asm volatile("; a branch: not worth computing for every step");
#pragma unroll
          for (int k = 0; k < 4; ++k)
            p[x][gi][k] &= (seen[x] >> (2 * k) & 1 ? 0xFFFFu : 0u) | (seen[x] >> (2 * k + 1) & 1 ? 0xFFFF0000u : 0u);
        }
        if (ZERO_PRODUCT) {
          f32x4& z = zp[x][ZERO_PRODUCT ? gi : 0];
          z = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, zero[gi]), __builtin_bit_cast(f16x8, p[x][gi]),
                                                     z, 0, 0, 0);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            zs[x][gi] = fmaf(low_half(p[x][gi][k]), low_half(zero[gi][k]), zs[x][gi]);
            zs[x][gi] = fmaf(high_half(p[x][gi][k]), high_half(zero[gi][k]), zs[x][gi]);
          }
        }
      }
    }
    load_value_words(s, s.next, s.ahead);
#pragma unroll
    for (int b = 0; b < CG; ++b) {
      // A column keeps its own keys: the others' products with it are with zeros.
      f16x8 mine[QT][G];
#pragma unroll
      for (int x = 0; x < QT; ++x)
#pragma unroll
        for (int gi = 0; gi < G; ++gi) {
          u32x4 w = p[x][gi];
          if (CG > 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = own == b ? w[i] : 0u;
          mine[x][gi] = __builtin_bit_cast(f16x8, w);
        }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (FULL > 0)
          if (t % TG < FULL) multiply_values<8>(s, t, b, mine);
        if constexpr (REST > 0)
          if (t % TG >= FULL) multiply_values<NREST>(s, t, b, mine);
      }
    }
    if (APART)
#pragma unroll
      for (int x = 0; x < QT; ++x)
#pragma unroll
        for (int gi = 0; gi < G; ++gi) rescale(x, gi, back[x][gi]);
    load_values(s, s.next, s.ahead);
    s.at += s.by;
    s.next = after;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      s.id[k] = s.ahead[k];
      s.ahead[k] = s.far[k];
    }
  }

  UNP4_DEV void walk(stream& s) {
    const int first = s.at, last = s.last;
    while (s.at < s.last) step<false>(s);
    if (__builtin_expect(s.last != last, 0)) {
      // Scales too far apart for one unit, which a cache seldom holds: anew, each step of a row and group in its own.
      s.at = first;
      s.last = last;
      clear();
      unit = (_Float16)1.0f;
      open(s);
      while (s.at < s.last) step<true>(s);
    }
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      if (EXACT_SUM) l[x][0] = column_sum(l[x][0]);
#pragma unroll
      for (int gi = 0; gi < G; ++gi) zs[x][gi] = ZERO_PRODUCT ? zp[x][ZERO_PRODUCT ? gi : 0][0] : column_sum(zs[x][gi]);
    }
  }
  // The sum of p v for element e of row g * 4 + r of tile t.
  UNP4_DEV float sum_of(int x, int t, int e, int r) const {
    return (o[x][product(t, e)][r] * ((e & 1) ? 0x1p18f : 0x1p22f) - zs[x][t / TG] * 0x1p9f) * (1.0f / (float)unit);
  }

  // Row x's elements times `by` to p, as U.  A lane's four runs of N elements of a tile lie together, so stores of one
  // run each would touch 64 places N elements wide; after a transposition four lanes' runs do (a prompt's output
  // took 170 us without it, of which 16 are its bytes).
  template <class U, int N> UNP4_DEV void write_tile(int x, int t, U* p, float by, bool there, bool wide) const {
    constexpr int M = sizeof(U) * N / 4;
    u32 w[4][M];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      vec<U, N> y;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float v = sum_of(x, t, e, r) * by;
        y.v[e] = (U)(by == 0.0f ? 0.0f : v);
      }
      __builtin_memcpy(w[r], &y, sizeof(y));
    }
    transpose<M>(w);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = t % TG * 128 + (r * 4 + g) * N;
      if (!there || d >= GROUP) continue;
      vec<U, N> y;
      __builtin_memcpy(&y, w[r], sizeof(y));
      U* to = p + t / TG * GROUP + d;
      if (wide) {
        store_stream<U, N>(to, y);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) to[e] = y.v[e];
      }
    }
  }
  template <class U> UNP4_DEV void write(int x, U* p, float by, bool there, bool wide) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (FULL > 0)
        if (t % TG < FULL) write_tile<U, 8>(x, t, p, by, there, wide);
      if constexpr (REST > 0)
        if (t % TG >= FULL) write_tile<U, NREST>(x, t, p, by, there, wide);
    }
  }

  // f(size<N>, t, r, d): every run of N adjacent elements d .. of the lane's columns.
  template <int N, class F> UNP4_DEV void runs(int t, F f) const {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = t % TG * 128 + (g * 4 + r) * N;
      if (t % TG * 128 + 16 * N <= GROUP || d < GROUP) f(size<N>{}, t, r, t / TG * GROUP + d);
    }
  }
  template <class F> UNP4_DEV void each(F f) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (FULL > 0)
        if (t % TG < FULL) runs<8>(t, f);
      if constexpr (REST > 0)
        if (t % TG >= FULL) runs<NREST>(t, f);
    }
  }
};

// A context's parts in the workspace: [part][token][head] of (maximum in log2, sum), then of D sums.
template <int QH, int D> struct parts {
  static UNP4_DEV float* stat(float* ws, const attention_args& a, i64 part, i64 row, int head) {
    return ws + ((part * a.tokens + row) * QH + head) * 2;
  }
  static UNP4_DEV float* sums(float* ws, const attention_args& a, i64 part, i64 row, int head) {
    const i64 stats = (a.splits * a.tokens * QH * 2 + 3) / 4 * 4;  // the sums stay aligned to 16 bytes
    return ws + stats + ((part * a.tokens + row) * QH + head) * D;
  }
};

// A block: WR waves of QT x 16 rows each or, for few rows, WK waves of the same QT x 16 / CG rows that take the steps in
// turn and are joined through LDS.  Blocks are numbered with the heads innermost (consecutive blocks go to different
// XCDs: with 8 heads each XCD's L2 holds one head's keys), then the parts of a context, then the tiles, last ones
// first: under a causal mask those have the most keys.
template <class T, int H, int QH, int D, int GROUP, int P, bool CAUSAL, bool LSE, int QT, int CG, int WR, int WK, bool ONCE>
UNP4_DEV void attend(const T* q, const u32* cache, const i32* table, const i32* starts, const i32* lengths, T* out,
                     float* lse, float* ws, float scale, const attention_args& a) {
  typedef attention<T, H, QH, D, GROUP, P, CAUSAL, LSE, QT, CG, ONCE> A;
  constexpr int GQ = QH / H, WAVE_ROWS = QT * A::ROWS, ROWS = WAVE_ROWS * WR;
  const int wave = uniform(threadIdx.x >> 6);
  const int kv = blockIdx.x % H, part = (int)(blockIdx.x / H) % a.splits;
  const tile t = tile_of<GQ, ROWS>(starts, lengths, a, a.slots - 1 - (int)(blockIdx.x / H) / a.splits);
  if (t.seq < 0) return;
  const i64 room = a.width * P;
  const int cap = t.length < 0 ? 0 : t.length < room ? t.length : (int)room;
  const int first_row = t.at * ROWS + (WR > 1 ? wave * WAVE_ROWS : 0), all_rows = t.rows * GQ;
  // Keys that the wave's first and last rows see: some column sees keys from .. to, all see lo .. hi.
  const int last_row = (first_row + WAVE_ROWS < all_rows ? first_row + WAVE_ROWS : all_rows) - 1;
  int from = 0, to = cap, lo = 0, hi = cap;
  if (CAUSAL) {
    const i64 near = (i64)t.length - t.rows + first_row / GQ + 1, far = (i64)t.length - t.rows + last_row / GQ + 1;
    to = far < 0 ? 0 : far < cap ? (int)far : cap;
    hi = near < 0 ? 0 : near < cap ? (int)near : cap;
    if (a.window > 0) {
      from = near > a.window ? (int)(near - a.window) : 0;
      lo = far > a.window ? (int)(far - a.window) : 0;
    }
  }
  if (last_row < first_row) to = 0;
  // This part's steps.
  const int step0 = from / A::KEYS, steps = to > from ? (to + A::KEYS - 1) / A::KEYS - step0 : 0;
  const int each = (steps + a.splits - 1) / a.splits;
  A w;
  typename A::stream s;
  s.cache = cache;
  s.table = (uniform_ints)(u64)(table + (i64)t.seq * a.width);
  s.kv = kv;
  s.at = step0 + (int)min((i64)steps, (i64)part * each) + (WK > 1 ? wave : 0);
  s.by = WK;
  s.last = step0 + (int)min((i64)steps, (i64)(part + 1) * each);
  s.cap = cap;
  s.lo = lo;
  s.hi = hi;
  s.pages = (int)a.pages;
  w.open(s);  // the first keys are on their way while the rows are read
  w.rows(q, a, t, kv, first_row, scale, cap);
  w.walk(s);
  if constexpr (WK > 1 || CG > 1) {
    // Join the waves and groups of columns: the rows' maxima and sums, then their elements, each scaled to the
    // common maximum; a row tile at a time.
    static_assert(WR == 1, "a block joins the parts of its waves' rows");
    __shared__ float stat[WK * CG][A::ROWS][2];
    __shared__ float sums[WK * CG][A::ROWS][D + 4];
    const int mine = wave * CG + w.own, r0 = w.c % A::ROWS;
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      if (x > 0) __syncthreads();
      if (w.g == 0) {
        stat[mine][r0][0] = w.m[x] * w.factor[x];
        stat[mine][r0][1] = w.l[x][0];
      }
      w.each([&](auto n, int tl, int r, int d) {
#pragma unroll
        for (int e = 0; e < decltype(n)::value; ++e) sums[mine][r0][d + e] = w.sum_of(x, tl, e, r);
      });
      __syncthreads();
      const int at = first_row + x * A::ROWS, n = all_rows - at < A::ROWS ? all_rows - at : A::ROWS;
      for (int i = threadIdx.x; i < n * (D / 4); i += 64 * WK) {
        const int row = i / (D / 4), d = i % (D / 4) * 4;
        float top = -__builtin_inff(), l = 0.0f;
#pragma unroll
        for (int v = 0; v < WK * CG; ++v) top = fmaxf(top, stat[v][row][0]);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < WK * CG; ++v) {
          const float keep = __builtin_amdgcn_exp2f(stat[v][row][0] - base);
          l = fmaf(stat[v][row][1], keep, l);
          o += *reinterpret_cast<const f32x4*>(&sums[v][row][d]) * keep;
        }
        const int token = t.start + (at + row) / GQ, head = kv * GQ + (at + row) % GQ;
        if (a.splits > 1) {
          if (d == 0) store<float, 2>(parts<QH, D>::stat(ws, a, part, token, head), {top, l});
          if (l != 0.0f) *reinterpret_cast<f32x4*>(parts<QH, D>::sums(ws, a, part, token, head) + d) = o;
        } else {
          const float y[4] = {o[0], o[1], o[2], o[3]};
          put<T, 4>(out + token * a.out_token + head * a.out_head + d, y, share_of(l), a.out_wide);
          if (LSE && d == 0) lse[(i64)token * QH + head] = log_sum(top, l);
        }
      }
    }
  } else {
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      const int row = first_row + x * 16 + w.c;
      const bool there = row < all_rows, split = a.splits > 1;
      const int token = t.start + (there ? row / GQ : 0), head = kv * GQ + (there ? row % GQ : 0);
      const float top = w.m[x] * w.factor[x], l = w.l[x][0];
      if (there && w.g == 0) {
        if (split) store<float, 2>(parts<QH, D>::stat(ws, a, part, token, head), {top, l});
        if (LSE && !split) lse[(i64)token * QH + head] = log_sum(top, l);
      }
      if (split)
        w.template write<float>(x, parts<QH, D>::sums(ws, a, part, token, head), 1.0f, there && l != 0.0f, true);
      else
        w.template write<T>(x, out + token * a.out_token + head * a.out_head, share_of(l), there, a.out_wide);
    }
  }
}

// The last sequence whose start is at most `row`, or -1 where no sequence has the row.
UNP4_DEV i64 sequence_of(const i32* starts, i64 batch, i64 row) {
  i64 lo = 0, hi = batch;
  while (hi - lo > 1) {
    const i64 mid = (lo + hi) >> 1;
    if (starts[mid] <= row) lo = mid; else hi = mid;
  }
  return starts[lo] > row || row >= starts[lo + 1] ? -1 : lo;
}

// The parts of split contexts: a lane holds four elements.  Few parts: as many rows and heads a block as its lanes hold, each
// lane takes all parts, their loads in flight at once (22720 rows of 64 elements in 2 parts: 8 us, with a block each
// 27).  Many parts: a block per row and head, whose groups of lanes take parts in turn: with a lane for all parts of its
// elements, 64 parts took 52 us.
constexpr int kMostParts = 128, kFewParts = 8;
template <class T, int H, int QH, int D, bool LSE>
UNP4_DEV void join(const i32* starts, T* out, float* lse, float* ws, const attention_args& a) {
  constexpr int L = D / 4, GROUPS = 256 / L;
  __shared__ float weight[kMostParts];
  __shared__ f32x4 part[GROUPS][L];
  const int lane = threadIdx.x & 63, group = threadIdx.x / L, d = threadIdx.x % L * 4;
  if (a.splits <= kFewParts) {
    const i64 item = (i64)blockIdx.x * GROUPS + group, row = item / QH;
    const int head = (int)(item % QH);
    if (group >= GROUPS || row >= a.tokens) return;
    f32x2 st[kFewParts];
    f32x4 v[kFewParts];
#pragma unroll
    for (int s = 0; s < kFewParts; ++s) {
      const int part = s < a.splits ? s : 0;
      st[s] = *reinterpret_cast<const f32x2*>(parts<QH, D>::stat(ws, a, part, row, head));
      v[s] = *reinterpret_cast<const f32x4*>(parts<QH, D>::sums(ws, a, part, row, head) + d);
    }
    if (sequence_of(starts, a.batch, row) < 0) return;
    float top = -__builtin_inff(), l = 0.0f;
#pragma unroll
    for (int s = 0; s < kFewParts; ++s) top = s < a.splits ? fmaxf(top, st[s][0]) : top;
    const float base = top == -__builtin_inff() ? 0.0f : top;
    f32x4 o = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < kFewParts; ++s) {
      if (s >= a.splits || st[s][1] == 0.0f) continue;  // a part without keys wrote no sums
      const float keep = __builtin_amdgcn_exp2f(st[s][0] - base);
      l = fmaf(st[s][1], keep, l);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(v[s][i], keep, o[i]);
    }
    const float y[4] = {o[0], o[1], o[2], o[3]};
    put<T, 4>(out + row * a.out_token + head * a.out_head + d, y, share_of(l), a.out_wide);
    if (LSE && d == 0) lse[row * QH + head] = log_sum(top, l);
    return;
  }
  const i64 row = blockIdx.x / QH;
  const int head = (int)(blockIdx.x % QH);
  // The parts' maxima and sums, in every wave; rows that no sequence names have none.
  f32x2 st[kMostParts / 64];
#pragma unroll
  for (int i = 0; i < kMostParts / 64; ++i) {
    const int s = i * 64 + lane;
    st[i] = s < a.splits ? *reinterpret_cast<const f32x2*>(parts<QH, D>::stat(ws, a, s, row, head))
                         : f32x2{-__builtin_inff(), 0.0f};
  }
  if (sequence_of(starts, a.batch, row) < 0) return;
  float top = -__builtin_inff(), l = 0.0f;
#pragma unroll
  for (int i = 0; i < kMostParts / 64; ++i) top = fmaxf(top, st[i][0]);
  for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
  const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
  for (int i = 0; i < kMostParts / 64; ++i) {
    const float keep = __builtin_amdgcn_exp2f(st[i][0] - base);
    // A part without keys wrote no sums.
    if (threadIdx.x < 64) weight[i * 64 + lane] = st[i][1] == 0.0f ? -1.0f : keep;
    l = fmaf(st[i][1], keep, l);
  }
  for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x);
  __syncthreads();
  f32x4 o = {0, 0, 0, 0};
  if (group < GROUPS) {
#pragma unroll 8
    for (int s = group; s < a.splits; s += GROUPS) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(parts<QH, D>::sums(ws, a, s, row, head) + d);
      const float w = weight[s];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = w >= 0.0f ? fmaf(v[i], w, o[i]) : o[i];
    }
    part[group][d / 4] = o;
  }
  __syncthreads();
  if (group != 0) return;
  const int used = a.splits < GROUPS ? a.splits : GROUPS;
  for (int i = 1; i < used; ++i) o += part[i][d / 4];
  const float y[4] = {o[0], o[1], o[2], o[3]};
  put<T, 4>(out + row * a.out_token + head * a.out_head + d, y, share_of(l), a.out_wide);
  if (LSE && d == 0) lse[row * QH + head] = log_sum(top, l);
}

}  // namespace unp4
