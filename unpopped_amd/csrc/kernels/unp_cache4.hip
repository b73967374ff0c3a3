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

// ---------------------------------------------------------------------------------------
// Position tables: [count][ROT / 2][cos, sin] of position first + row.
//
// One pair per lane and step; a block computes the ROT / 2 frequencies once, into LDS.
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

template <int ROT>
UNP4_DEV void rope_table(float* out, i64 first, i64 count, const stretch& s) {
  constexpr int H = ROT / 2;
  __shared__ double f[H];
  for (int i = threadIdx.x; i < H; i += 256) f[i] = frequency<ROT>(i, s);
  __syncthreads();
  const i64 n = count * H;
  for (i64 at = (i64)blockIdx.x * 256 + threadIdx.x; at < n; at += (i64)gridDim.x * 256) {
    const i64 row = at / H;
    double sn, cs;
    sincos((double)(first + row) * f[at - row * H], &sn, &cs);
    store<float, 2>(out + 2 * at, {(float)(cs * s.amplitude), (float)(sn * s.amplitude)});
  }
}

// ---------------------------------------------------------------------------------------
// Rotation of heads.
//
// (x0, x1) -> (x0 c - x1 s, x1 c + x0 s), the sine negated for the inverse.  It reads and writes each
// element once: a stream.  A unit of the vector entry is V pairs (two 16-byte loads and stores) or 2V
// elements that are only copied; the plain entry takes a pair or a copied element at a time.
// ---------------------------------------------------------------------------------------
struct rope_args {
  i64 tokens, x_token, x_head, out_token, out_head, first, rows;
  int heads, units;  // units of a head: the rotated ones, and the copied ones unless x and out are one
};

template <bool INV> UNP4_DEV void turn(float& a, float& b, float c, float s) {
  if (INV) s = -s;
  const float x0 = a, x1 = b;
  a = fmaf(x0, c, -(x1 * s));
  b = fmaf(x1, c, x0 * s);
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
    const i64 row = (i64)positions[token] - a.first;
    if (row < 0 || row >= a.rows) continue;
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
        store<T, V>(op + p0, u);
        store<T, V>(op + p1, w);
      } else {
        const int p = ROT + (unit - RU) * 2 * V;
        const vec<T, V> u = load<T, V>(xp + p), w = load<T, V>(xp + p + V);
        store<T, V>(op + p, u);
        store<T, V>(op + p + V, w);
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

// ---------------------------------------------------------------------------------------
// Append: a lane holds one word's 8 elements of a key or a value head; a group's range is reduced over
// its lanes.  The rotation's products of a 16-bit element and a 32-bit cosine are exact in f64, so the
// rotated key is rounded once to 53 bits and once to its type: its code does not depend on how the sum
// is contracted.  The quotients are correctly rounded f32 divisions; a quotient of an 11-bit by an 11-bit
// number that is no tie is too far from one (2^-20 of it) for f32 to round onto it, so the codes are those of
// exact arithmetic.
// ---------------------------------------------------------------------------------------
template <class T, int H, int D, int GROUP, int P, int ROT, int LAYOUT, class I, bool ALIGNED>
UNP4_DEV void append(const T* k, const T* v, const I* slots, u32* cache, const I* positions, const float* table,
                     const cache_args& a) {
  typedef record<D, GROUP, P> R;
  constexpr int L = lanes_of(R::W), IB = 256 / L;
  const int w = threadIdx.x % L;
  const i64 n = a.tokens * (2 * H);
  for (i64 at = (i64)blockIdx.x * IB + threadIdx.x / L; at < n; at += (i64)gridDim.x * IB) {
    const i64 token = at / (2 * H);
    const int which = (int)(at - token * (2 * H)), head = which % H;
    const bool key = which < H;
    const i64 slot = (i64)slots[token];
    if (slot < 0 || slot >= a.slots) continue;  // the same in every lane of the item
    i64 row = 0;
    if (ROT > 0) {
      row = (i64)positions[token] - a.first;
      if (row < 0 || row >= a.rows) continue;
    }
    const bool live = w < R::W;
    float y[8];
    float lo = 0.0f, hi = 0.0f;
    if (live) {
      const T* p = key ? k + token * a.k_token + head * a.k_head : v + token * a.v_token + head * a.v_head;
      T x[8];
      load8<T, ALIGNED>(p + 8 * w, x);
      if (ROT > 0 && key && 8 * w < ROT) {
        const float* cs = table + row * ROT;
        if (LAYOUT == HALVES) {
          const bool second = 8 * w >= ROT / 2;
          const int i0 = second ? 8 * w - ROT / 2 : 8 * w;
          T o[8];  // the pairs' other elements
          load8<T, ALIGNED>(p + (second ? i0 : i0 + ROT / 2), o);
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
        // A NaN or an infinity of either sign opens the range to infinity.
        hi = fmaxf(hi, fabsf(y[i]) < __builtin_inff() ? y[i] : __builtin_inff());
      }
    }
    constexpr int GL = GROUP == D ? L : GROUP / 8;  // lanes of a group
    for (int m = 1; m < GL; m *= 2) {
      lo = fminf(lo, __shfl_xor(lo, m));
      hi = fmaxf(hi, __shfl_xor(hi, m));
    }
    const _Float16 sh = (_Float16)((hi - lo) / 15.0f);
    const bool finite = (float)sh < __builtin_inff();
    const float s = finite && (float)sh > 0.0f ? (float)sh : 1.0f;
    const float z = finite ? fminf(15.0f, fmaxf(0.0f, rintf(-lo / s))) : 0.0f;
    if (!live) continue;
    u32 word = 0;
    for (int i = 0; i < 8; ++i) {
      const float c = finite ? fminf(15.0f, fmaxf(0.0f, rintf(y[i] / s) + z)) : 0.0f;
      word |= (u32)c << (4 * i);
    }
    const int t = (int)(slot % P);
    u32* rec = cache + ((slot / P) * H + head) * (i64)R::WORDS;
    rec[key ? R::key(t, w) : R::value(t, w)] = word;
    if ((8 * w) % GROUP == 0) {
      const u32 bits = finite ? __builtin_bit_cast(u16, sh) : 0x7E00u;
      rec[key ? R::kpar(t, 8 * w / GROUP) : R::vpar(t, 8 * w / GROUP)] = bits | (u32)z << 16;
    }
  }
}

// ---------------------------------------------------------------------------------------
// Read back: a lane per word; a slot outside the cache gives zeros.
// ---------------------------------------------------------------------------------------
template <class T, int H, int D, int GROUP, int P, class I, bool ALIGNED>
UNP4_DEV void read(const I* slots, const u32* cache, T* k, T* v, const cache_args& a) {
  typedef record<D, GROUP, P> R;
  const i64 n = a.tokens * (2 * H) * R::W;
  for (i64 at = (i64)blockIdx.x * 256 + threadIdx.x; at < n; at += (i64)gridDim.x * 256) {
    const i64 item = at / R::W, token = item / (2 * H);
    const int w = (int)(at - item * R::W), which = (int)(item - token * (2 * H)), head = which % H;
    const bool key = which < H;
    const i64 slot = (i64)slots[token];
    vec<T, 8> o;
    if (slot >= 0 && slot < a.slots) {
      const int t = (int)(slot % P), g = 8 * w / GROUP;
      const u32* rec = cache + ((slot / P) * H + head) * (i64)R::WORDS;
      const u32 word = rec[key ? R::key(t, w) : R::value(t, w)];
      const u32 par = rec[key ? R::kpar(t, g) : R::vpar(t, g)];
      for (int i = 0; i < 8; ++i)
        o.v[i] = (T)(((float)(word >> (4 * i) & 15u) - zero_of(par)) * scale_of(par));
    } else {
      for (int i = 0; i < 8; ++i) o.v[i] = (T)0.0f;
    }
    T* p = (key ? k + token * a.k_token + head * a.k_head : v + token * a.v_token + head * a.v_head) + 8 * w;
    if (ALIGNED) {
      store<T, 8>(p, o);
    } else {
      for (int i = 0; i < 8; ++i) p[i] = o.v[i];
    }
  }
}

// ---------------------------------------------------------------------------------------
// Attention over the cache.
// ---------------------------------------------------------------------------------------
struct attention_args {
  i64 tokens, batch, width, pages, q_token, q_head, out_token, out_head, window;
};

// The sequence of a row: the b with starts[b] <= row < starts[b + 1], or -1.
UNP4_DEV i64 sequence_of(const i32* starts, i64 batch, i64 row) {
  i64 lo = 0, hi = batch;  // the last b with starts[b] <= row lies in lo .. hi - 1
  while (hi - lo > 1) {
    const i64 mid = (lo + hi) >> 1;
    if (starts[mid] <= row) lo = mid; else hi = mid;
  }
  return starts[lo] <= row && row < starts[lo + 1] ? lo : -1;
}

// One wave per row and head: 64 keys a step, one per lane, with a running maximum and sum; then each lane
// adds up its own elements of the output.
template <class T, int H, int QH, int D, int GROUP, int P, bool CAUSAL, bool LSE>
UNP4_DEV void attend(const T* q, const u32* cache, const i32* table, const i32* starts, const i32* lengths, T* out,
                     float* lse, float scale, const attention_args& a) {
  typedef record<D, GROUP, P> R;
  constexpr int E = (D + 63) / 64;
  __shared__ float qs[D], ps[64];
  __shared__ const u32* recs[64];
  const int lane = threadIdx.x;
  for (i64 at = blockIdx.x; at < a.tokens * QH; at += gridDim.x) {
    const i64 row = at / QH;
    const int head = (int)(at - row * QH), kv = head / (QH / H);
    const i64 b = sequence_of(starts, a.batch, row);
    if (b < 0) continue;
    const i64 length = lengths[b];
    i64 end = length, begin = 0;
    if (CAUSAL) {
      end = length - starts[b + 1] + row + 1;
      if (a.window > 0 && end > a.window) begin = end - a.window;
    }
    if (end > a.width * P) end = a.width * P;
    __syncthreads();
    for (int d = lane; d < D; d += 64) qs[d] = (float)q[row * a.q_token + head * a.q_head + d] * scale;
    __syncthreads();
    float m = -__builtin_inff(), sum = 0.0f, o[E];
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    for (i64 j0 = begin; j0 < end; j0 += 64) {
      const i64 j = j0 + lane;
      const i32 page = j < end ? table[b * a.width + j / P] : -1;
      const bool seen = page >= 0 && page < a.pages;
      const u32* rec = seen ? cache + ((i64)page * H + kv) * (i64)R::WORDS : nullptr;
      const int t = (int)(j % P);
      float s = -__builtin_inff();
      if (seen) {
        s = 0.0f;
        for (int w = 0; w < R::W; ++w) {
          const u32 word = rec[R::key(t, w)], par = rec[R::kpar(t, 8 * w / GROUP)];
          const float z = zero_of(par);
          float part = 0.0f;
          for (int i = 0; i < 8; ++i) part = fmaf(qs[8 * w + i], (float)(word >> (4 * i) & 15u) - z, part);
          s = fmaf(part, scale_of(par), s);
        }
      }
      float top = s;
      for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
      const float next = fmaxf(m, top);
      const float base = next > -__builtin_inff() ? next : 0.0f;
      const float p = expf(s - base), keep = expf(m - base);
      float total = p;
      for (int x = 1; x < 64; x *= 2) total += __shfl_xor(total, x);
      sum = fmaf(sum, keep, total);
      m = next;
      for (int e = 0; e < E; ++e) o[e] *= keep;
      __syncthreads();
      ps[lane] = p;
      recs[lane] = rec;
      __syncthreads();
      for (int i = 0; i < 64; ++i) {
        const u32* r = recs[i];
        if (!r) continue;
        const int ti = (int)((j0 + i) % P);
        for (int e = 0; e < E; ++e) {
          const int d = lane + 64 * e;
          if (D % 64 != 0 && d >= D) continue;
          const u32 word = r[R::value(ti, d / 8)], par = r[R::vpar(ti, d / GROUP)];
          o[e] = fmaf(ps[i], ((float)(word >> (4 * (d & 7)) & 15u) - zero_of(par)) * scale_of(par), o[e]);
        }
      }
    }
    for (int e = 0; e < E; ++e) {
      const int d = lane + 64 * e;
      if (D % 64 == 0 || d < D)
        out[row * a.out_token + head * a.out_head + d] = (T)(sum == 0.0f ? 0.0f : o[e] / sum);
    }
    if (LSE && lane == 0) lse[row * QH + head] = sum == 0.0f ? -__builtin_inff() : m + logf(sum);
  }
}

}  // namespace unp4
