// Token rules on logits: penalties for tokens a row's history holds, a bias, a grammar mask -- and what is read from the
// ruled values: the values themselves (apply), a token (choose), a given token's log-probability and its gradients.
//
//   c = how often the row's history holds v
//   x1 = c > 0 ? (x > 0 ? x / rho : x * rho) : x;  x2 = x1 - frequency c - presence [c > 0];  x3 = x2 + bias[v]
//   x4 = allowed(state, v) ? x3 : -inf;            p = softmax(x4 / T)
//
// Kernels, by size.
//   map    (apply, gradients) and sum (what a softmax needs): a row is cut into segments of up to 2048 tokens, one wave each,
//          64 lanes x 16 bytes a step, four steps in flight.  Rows of one segment are decided by their wave on the spot.
//   join   the other rows: segments leave (sum, maximum); a workgroup a row adds them, finds the ONE segment the
//          token is in and searches it again.
//   group  up to 128 tokens: a group of lanes a row, eight tokens a lane, everything in one launch.
//   col    gradients with a bias shared by the rows: its sum over rows in registers.
// Counts: a workgroup counts the history's tokens that fall into its segments in LDS (integer atomics: their order does not
// matter).
//
// Bounds.  apply and log p move the logits once each way and are bound by memory: 256 x 131072 bf16 under all rules 31 us
// (137 MB, 4.4 TB/s), log p of 4096 x 65536 bf16 99 + 10 us, its gradients 179 us (1.07 GB, 6.0 TB/s).  A drawn batch is
// bound by its sums of doubles: 512 x 131072 bf16 under all rules 102 us for 41 M wave instructions -- 39 per element, 15 of
// them the exp, 10 its value and masks, the rest counting and reductions -- where the bytes alone would take 29 us; + 16 us
// join.  The same batch taken greedily: 57 us for 25 M (24 per element; without rules 25 us for 10.6 M) + 13 us join.
//
// Numbers.  A token the history does not hold has the value x + b, one fp32 rounding; a counted one is computed in double
// and rounded once.  Decisions do not rest on that rounding: rounding is monotone, so the largest exact value is among the
// elements whose rounded value is the largest; those few are compared as doubles.  A drawn token is decided where a running
// sum over the whole vocabulary crosses u Z: weights and sums are doubles, with an exp2 of 4e-14.  (131072 tokens, normal logits
// of deviation 2.7, T 0.5 to 1.5: fp32 weights would decide up to 0.8 rows in a thousand otherwise, fp32 sums of them 10 to
// 27, and a bound of the weights' error leaves 4 to 17 % of the rows open to a second pass; fp32 operations are hardly quicker,
// 4.7 cycles a wave against 5.4.)
// A low temperature magnifies what the rounding dropped: against the largest value as rounded, a weight 2^((x4 - ref) k) may
// be 2^1000 or 0 where it is 1.  So doubles are summed against the exact largest value, and a segment whose largest |x4| k is
// no ordinary one (`ordinary`: beyond 2^-400 .. 2^900, a T below 0.02 for a logit of 13) is summed in doubles throughout, token
// by token, as is its gradient (512 x 131072 bf16 with penalties: greedy 53 us, at T 0.01 125); within these bounds the rounding
// of the other tokens moves a log p of fp32 sums by at most 900 ln2 2^-24 = 4e-5.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "elem.h"
#include "rules.h"

namespace {

constexpr double LOG2E = 1.4426950408889634074;
constexpr double LN2 = 0.69314718055994530942;
constexpr double TEMP_MIN = 1e-37, TEMP_MAX = 1e37;       // k and 1 / k are ordinary floats

// what a wave knows about its row
struct RowP {
  double rho, inv_rho, freq, pres, temp, k;      // k = log2(e) / T
  const uint8_t* mask;            // packed bits of the row's grammar state, or NULL: everything allowed
  const float* bias;              // or NULL
  const char* hist;               // the row's history
  int n_hist;
  bool fine;                      // the temperature is one (TEMP_MIN .. TEMP_MAX); else the row is NaN, as for a NaN logit
};

// 1 / v to the last bits for an ordinary v: the hardware's approximation and two Newton steps
__device__ __forceinline__ double reciprocal(double v) {
  double r = __builtin_amdgcn_rcp(v);
  r = fma(fma(-v, r, 1.0), r, r);
  return fma(fma(-v, r, 1.0), r, r);
}

// one setting for all rows: its quotients are formed on the host
struct Rules : dvae_rules {
  double inv_rho, k;
};

__device__ __forceinline__ RowP row_params(const Rules& q, long long r) {
  RowP p;
  p.rho = q.repetition;
  p.inv_rho = q.inv_rho;
  if (q.repetition_rows) {
    p.rho = q.repetition_rows[r];
    p.inv_rho = reciprocal(p.rho);
  }
  p.freq = q.frequency_rows ? (double)q.frequency_rows[r] : q.frequency;
  p.pres = q.presence_rows ? (double)q.presence_rows[r] : q.presence;
  p.temp = q.temperature;
  p.k = q.k;
  if (q.temperature_rows) {
    p.temp = q.temperature_rows[r];
    p.k = LOG2E * reciprocal(p.temp);
  }
  p.fine = p.temp >= TEMP_MIN && p.temp <= TEMP_MAX;
  p.bias = q.bias ? q.bias + r * q.bias_ld : nullptr;
  p.mask = nullptr;
  if (q.mask) {
    const int s = q.state[r];
    // a state outside the table: no mask
    if (s >= 0 && s < q.states) p.mask = reinterpret_cast<const uint8_t*>(q.mask + (size_t)s * q.mask_words);
  }
  p.n_hist = 0;
  p.hist = nullptr;
  if (q.history) {
    int n = q.history_len;
    if (q.lengths) n = max(0, min(n, q.lengths[r]));
    p.n_hist = n;
    p.hist = static_cast<const char*>(q.history) + (r / q.rows_per_history) * q.history_ld * (q.history_i64 ? 8 : 4);
  }
  return p;
}

// the same for a path that hardly ever runs, read there: the steps before it need no registers for what only it uses
__device__ __forceinline__ RowP params_anew(const Rules& q, long long r) {
  asm volatile("" : "+s"(r));
  return row_params(q, r);
}

__device__ __forceinline__ long long hist_at(const RowP& p, int i64, int i) {
  return i64 ? reinterpret_cast<const long long*>(p.hist)[i] : (long long)reinterpret_cast<const int*>(p.hist)[i];
}

// f(token) for the history's tokens from `from` on, `lane` of `width` threads; N loads in flight, whatever the length
template <int N, typename F>
__device__ __forceinline__ void for_history(const RowP& p, int i64, int from, int lane, int width, F f) {
  for (int i = from + lane; i < p.n_hist; i += N * width) {
    long long t[N];
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (i + u * width < p.n_hist) t[u] = hist_at(p, i64, i + u * width);
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (i + u * width < p.n_hist) f(t[u]);
  }
}

// the value of a token that the history holds c > 0 times.  x / rho as x (1 / rho) with one correction step: as good as
// the division (equal quotients stay equal, so ties stay ties) at four operations
__device__ __forceinline__ double counted64(const RowP& p, float x, uint32_t c, float b) {
  const double xd = x;
  double v = xd * p.inv_rho;
  v = fma(fma(-v, p.rho, xd), p.inv_rho, v);
  v = __builtin_amdgcn_classf(x, 0x180) ? v : xd * p.rho;      // positive and finite (+inf: the correction is inf - inf)
  v = fma(-p.freq, (double)c, v);        // one operation everywhere: two kernels compute a value and have to agree
  v -= p.pres;
  return v + (double)b;
}

// NaN if either is: a NaN among the allowed values has to reach the result
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ double max_nan(double a, double b) { return a > b || a != a ? a : b; }

__device__ __forceinline__ float wave_max_nan(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max_nan(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o));
  return v;
}

// 2^(d k) in double for d k from -1000 (`low` = -1000 / k; what lies below counts as 2^-1000) to 1000: a = d k = n + f,
// |f| <= 1/2; n by adding 1.5 2^52, which leaves it in the low bits; 2^f as 1 + f q(f), q the polynomial that
// meets (2^f - 1) / f in the nine Chebyshev nodes of [-1/2, 1/2] (off by at most 3.7e-14 of the result, exact at 0);
// n goes into the exponent by an integer addition.
// 15 operations of full rate: the accurate exp of the math library and its branches took three times as long.
__device__ __forceinline__ double exp2_fast(double d, double k, double low) {
  constexpr double SHIFT = 6755399441055744.0;
  d = fmax(d, low);
  const double t = fma(d, k, SHIFT);
  const double f = fma(d, k, -(t - SHIFT));
  double y = 1.0203121138901363e-07;
  y = fma(y, f, 1.325522487892511e-06);
  y = fma(y, f, 1.525268684597521e-05);
  y = fma(y, f, 0.00015403455852451678);
  y = fma(y, f, 0.0013333558179043376);
  y = fma(y, f, 0.009618129159402562);
  y = fma(y, f, 0.055504108664760424);
  y = fma(y, f, 0.2402265069581299);
  y = fma(y, f, 0.6931471805599453);
  y = fma(y, f, 1.0);
  return __hiloint2double(__double2hiint(y) + (__double2loint(t) << 20), __double2loint(y));
}

// the same, 0 below 2^-1000 and NaN for NaN
__device__ __forceinline__ double exp2_64(double d, double k) {
  const double a = d * k;
  const double w = exp2_fast(a < -1000.0 ? 0.0 : d, k, -INFINITY);
  return a != a ? a : a < -1000.0 ? 0.0 : w;
}

// exp2_64 for loops that hardly ever run: the coefficients come from memory one by one, so that the kernel's ordinary steps
// do not pay for their registers
__constant__ double EXP2_C[] = {1.0203121138901363e-07, 1.325522487892511e-06, 1.525268684597521e-05, 0.00015403455852451678,
                                0.0013333558179043376, 0.009618129159402562, 0.055504108664760424, 0.2402265069581299,
                                0.6931471805599453, 1.0};
__device__ __forceinline__ double exp2_rare(double d, double k) {
  const double a = d * k;
  if (!(a >= -1000.0)) return a != a ? a : 0.0;
  const double n = rint(a), f = fma(d, k, -n);
  double y = EXP2_C[0];
#pragma unroll 1
  for (int i = 1; i < 10; ++i) y = fma(y, f, EXP2_C[i]);
  return ldexp(y, (int)n);
}

// log Z for Z > 0 in double: Z = 2^n c, c in [sqrt 1/2, sqrt 2), log c = 2 atanh t, t = (c - 1) / (c + 1), |t| < 0.172; the
// first term left out of the series is t^18 / 19 of the result (9e-16).  A third of the math library's operations.
__device__ __forceinline__ double log_64(double z) {
  int n;
  double c = frexp(z, &n);
  if (c < 0.70710678118654752) { c += c; --n; }
  const double t = (c - 1.0) * reciprocal(c + 1.0), u = t * t;
  double s = 1.0 / 17.0;
  s = fma(s, u, 1.0 / 15.0);
  s = fma(s, u, 1.0 / 13.0);
  s = fma(s, u, 1.0 / 11.0);
  s = fma(s, u, 1.0 / 9.0);
  s = fma(s, u, 1.0 / 7.0);
  s = fma(s, u, 1.0 / 5.0);
  s = fma(s, u, 1.0 / 3.0);
  s = fma(s, u, 1.0);
  return fma((double)n, LN2, 2.0 * t * s);
}

// whether 2^(m k) and what is near it have their places in the exponents of a double, and the part of m that a rounding to fp32
// drops does not show in it
__device__ __forceinline__ bool ordinary(float m, float k) {
  const float a = m * k;
  return a > -400.f && a < 900.f;
}

// whether the row's values may lie between two floats: those of a bias or a history
__device__ __forceinline__ bool inexact(const Rules& q, const RowP& p) { return p.bias || (q.history && q.history_len); }

// what a segment leaves for the join
struct Seg {
  double s;       // sum of 2^((x4 - ref) k); ref: 0 for an ordinary maximum of a draw (reference()), else top
  double top;     // maximum (NaN when an allowed value is): as rounded to fp32, but exact where it is no ordinary one
};

enum { M_APPLY = 0, M_SUM = 1, M_GREEDY = 2, M_DRAW = 3, M_BWD = 4 };

template <int MODE>
__device__ __forceinline__ double reference(double top, double k) {
  return MODE == M_DRAW && ordinary((float)top, (float)k) ? 0.0 : top;
}

constexpr int SEG_MAX = 4096;   // tokens of a segment at most: the counts of a workgroup's 4 segments are 32 KB of 16 bits

// what a row's decision reads and leaves
struct RowOut {
  const float* uniforms;         // DRAW
  const int* next;               // next state of (state, token), or NULL
  const long long* given;        // SUM, BWD: the given tokens
  long long* tokens;             // GREEDY / DRAW
  float* logprob;
  double* stat;                  // SUM, BWD: [rows][2] = the reference of Z and 1 / Z, kept for the backward pass
  int* state_out;
};

struct SegArgs {
  Rules q;
  RowOut o;
  int nseg, seg_len;            // segments of a row, their tokens (a multiple of 64 x 16 bytes)
  int wgs_per_row;              // workgroups of a row (ROWWAVE: unused)
  void* out; long long out_ld;  // APPLY / BWD (NULL: the bias gradient only)
  Seg* seg;                     // sums: a segment's (ROWWAVE: unused)
  const float* d_logprob;       // BWD
  float* d_bias_rows;           // BWD: gradient of a bias of its own per row, [rows][vocab], or NULL
};

// counts of 4 segments: u16 pairs in 32-bit words while a history has fewer than 65536 tokens, else 32 bits each
template <int HIST> struct Counts;
template <> struct Counts<1> { static constexpr int PER_WORD = 2; };
template <> struct Counts<2> { static constexpr int PER_WORD = 1; };

template <int HIST>
__device__ __forceinline__ uint32_t count_at(const uint32_t* lds, int d) {
  if (HIST == 1) return (lds[d >> 1] >> ((d & 1) * 16)) & 0xffffu;
  return lds[d];
}

// adds the history's tokens in [v0, v0 + span) to lds and, if there is one, marks them in the bitmap; `lane` of `width`
// threads
template <int HIST>
__device__ __forceinline__ void count_history(const RowP& p, int i64, long long v0, int span, uint32_t* lds, uint32_t* bits,
                                              int lane, int width) {
  const auto add = [&](long long token) {
    const long long t = token - v0;
    if ((unsigned long long)t < (unsigned long long)span) {
      const int d = (int)t;
      if (HIST == 1) atomicAdd(&lds[d >> 1], (d & 1) ? 0x10000u : 1u);
      else atomicAdd(&lds[d], 1u);
      if (bits) atomicOr(&bits[d >> 5], 1u << (d & 31));
    }
  };
  if (p.n_hist > 4 * width) for_history<8>(p, i64, 0, lane, width, add);
  else for_history<4>(p, i64, 0, lane, width, add);
}

// A step of a wave: 64 x EV tokens, from v on in this lane.  WHOLE: inside the vocabulary in every lane, as every step but a
// row's last is.
struct Loaded { u32x4 raw; uint32_t keep; };       // keep, bit e: allowed (and inside the vocabulary)

template <int T, bool WHOLE>
__device__ __forceinline__ Loaded load_step(const RowP& p, const char* lrow, int v, int V) {
  constexpr int EV = Elem<T>::EV, BYTES = 16 / EV;
  Loaded l;
  l.keep = (1u << EV) - 1;
  if (WHOLE || v + EV <= V) {
    l.raw = *reinterpret_cast<const u32x4_u*>(lrow + (size_t)v * BYTES);
  } else {
    l.raw = u32x4{0, 0, 0, 0};
    l.keep = v < V ? (1u << (V - v)) - 1 : 0u;
#pragma unroll
    for (int e = 0; e < EV; ++e)
      if (v + e < V) {
        if (T == DVAE_F32) l.raw[e] = reinterpret_cast<const uint32_t*>(lrow)[v + e];
        else l.raw[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(lrow)[v + e] << ((e & 1) * 16);
      }
  }
  if (p.mask && (WHOLE || v < V)) {
    const uint32_t byte = p.mask[v >> 3];
    l.keep &= EV == 8 ? byte : byte >> (v & 4);
  }
  return l;
}

// bias of the step's tokens, 0 past the vocabulary
template <int EV, bool WHOLE>
__device__ __forceinline__ void load_bias(const float* bias, int v, int V, float (&b)[EV]) {
  if (WHOLE || v + EV <= V) {
#pragma unroll
    for (int e = 0; e < EV; e += 4) {
      const f32x4_u t = *reinterpret_cast<const f32x4_u*>(bias + v + e);
      b[e] = t[0]; b[e + 1] = t[1]; b[e + 2] = t[2]; b[e + 3] = t[3];
    }
  } else {
#pragma unroll
    for (int e = 0; e < EV; ++e) b[e] = v + e < V ? bias[v + e] : 0.f;
  }
}

template <int T, bool WHOLE>
__device__ __forceinline__ void store_step(typename Elem<T>::type* orow, int v, int V, const float (&y)[Elem<T>::EV]) {
  constexpr int EV = Elem<T>::EV;
  typename Elem<T>::type o[EV];
#pragma unroll
  for (int e = 0; e < EV; ++e) o[e] = Elem<T>::cast(y[e]);
  if (WHOLE || v + EV <= V) {
    u32x4 w;
    __builtin_memcpy(&w, o, 16);
    // streamed: results do not push logits out of the cache (a training pass over 4096 x 65536 bf16 299 -> 289 us; streamed
    // loads as well 282, but where logits fit the cache they cost: 301 x 50021 fp32 kernels 66 -> 83 us)
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4_u*>(orow + v));
  } else {
#pragma unroll
    for (int e = 0; e < EV; ++e)
      if (v + e < V) orow[v + e] = o[e];
  }
}

// A segment's steps: D of the whole ones in flight (each in registers of its own: moving a load from one to another would
// wait for it), then the partial one, if there is one.  begin() before the history is counted, so that the loads travel
// meanwhile; f(loaded, v, whole) for each step.
template <int T, int D>
struct Steps {
  static constexpr int EV = Elem<T>::EV, STEP = 64 * EV;
  Loaded l[D];
  int full, v, end;                // v: this lane's first token
  __device__ __forceinline__ void begin(const RowP& p, const char* lrow, int v0, int stop, int lane, int V) {
    full = (stop - v0) / STEP;
    v = v0 + lane * EV;
    end = stop;
#pragma unroll
    for (int j = 0; j < D; ++j)
      if (j < full) l[j] = load_step<T, true>(p, lrow, v + j * STEP, V);
  }
  template <typename F>
  __device__ __forceinline__ void run(const RowP& p, const char* lrow, int V, F f) {
    int at = v;
    for (int g = 0; g < full; g += D) {
#pragma unroll
      for (int j = 0; j < D; ++j)
        if (g + j < full) {
          const Loaded in = l[j];
          if (g + j + D < full) l[j] = load_step<T, true>(p, lrow, at + D * STEP, V);
          f(in, at, std::true_type{});
          at += STEP;
        }
    }
    if (at < end) f(load_step<T, false>(p, lrow, at, V), at, std::false_type{});
  }
};

// The values under the rules.  Forbidden places: x = -inf and b = 0 before anything is computed, so that nothing they hold
// shows.  Counted tokens are few: one test for the whole step, then one branch each.
template <int T, int HIST>
struct Ruled {
  typedef Elem<T> E;
  static constexpr int EV = E::EV;
  static constexpr int CW = HIST == 1 ? EV / 2 : HIST == 2 ? EV : 1;
  float x[EV], s[EV];
  uint32_t cw[CW];
  uint32_t any;                 // nonzero: the history holds one of the step's tokens in this lane

  __device__ __forceinline__ uint32_t count(int e) const {
    if (HIST == 1) return (cw[e >> 1] >> ((e & 1) * 16)) & 0xffffu;
    return HIST == 2 ? cw[e] : 0u;
  }
  // cnt: the counts from this lane's first token on
  template <typename W>
  __device__ __forceinline__ Ruled(const RowP& p, const Loaded& in, const uint32_t* cnt, int v, int V, W) {
    constexpr bool WHOLE = W::value;
    const auto on = [&](int e) { return (uint32_t)((int)(in.keep << (31 - e)) >> 31); };
#pragma unroll
    for (int e = 0; e < EV; ++e) x[e] = E::at(in.raw, e);
    if (p.mask || !WHOLE) {
#pragma unroll
      for (int e = 0; e < EV; ++e) x[e] = __uint_as_float((__float_as_uint(x[e]) & on(e)) | (0xff800000u & ~on(e)));
    }
    any = 0;
    if (HIST) {
#pragma unroll
      for (int i = 0; i < CW; ++i) { cw[i] = cnt[i]; any |= cw[i]; }
    }
    float b[EV];
    if (p.bias) {
      load_bias<EV, WHOLE>(p.bias, v, V, b);
      if (p.mask) {
#pragma unroll
        for (int e = 0; e < EV; ++e) b[e] = __uint_as_float(__float_as_uint(b[e]) & on(e));
      }
#pragma unroll
      for (int e = 0; e < EV; ++e) s[e] = x[e] + b[e];
    } else {
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        b[e] = 0.f;
        s[e] = x[e];
      }
    }
    if (HIST && any) {
#pragma unroll
      for (int e = 0; e < EV; ++e)
        if (count(e)) {
          s[e] = (in.keep >> e) & 1 ? (float)counted64(p, x[e], count(e), b[e]) : -INFINITY;
        }
    }
  }
};

// a row's part of the gradient: y = -g / T p, + g / T at the given token
struct Bwd {
  float m, coef, spread, kf, up, down;
  int tok;
  bool zero;                      // an ignored row, or one whose rules leave nothing
  bool far;                       // no ordinary maximum: struct Far instead
  __device__ __forceinline__ Bwd() {}
  __device__ __forceinline__ Bwd(const SegArgs& a, const RowP& p, long long row) {
    const long long t = a.o.given[row];
    m = (float)a.o.stat[2 * row];
    kf = (float)p.k;
    coef = (float)((double)a.d_logprob[row] * (p.k * LN2));
    spread = -coef * (float)a.o.stat[2 * row + 1];
    up = (float)p.rho;
    down = (float)p.inv_rho;
    zero = t < 0 || t >= a.q.vocab || m == -INFINITY;
    tok = zero ? 0 : (int)t;
    far = inexact(a.q, p) && fabsf(m) < INFINITY && !ordinary(m, kf);
  }
  // d values of the step's tokens, from v on
  template <typename R, int EV>
  __device__ __forceinline__ void values(const R& r, uint32_t keep, int v, float (&y)[EV]) const {
    // forbidden places have the weight 0 by themselves
#pragma unroll
    for (int e = 0; e < EV; ++e) y[e] = spread * __builtin_amdgcn_exp2f((r.s[e] - m) * kf);
    const unsigned at = (unsigned)(tok - v);
    if (at < EV) {
#pragma unroll
      for (int e = 0; e < EV; ++e) y[e] += at == e ? coef : 0.f;
    }
    if (zero || !(fabsf(spread) < INFINITY) || at < EV) {      // no gradient, a NaN or infinite one, a forbidden token
#pragma unroll
      for (int e = 0; e < EV; ++e)
        if (zero || !((keep >> e) & 1)) y[e] = 0.f;
    }
  }
  // d values -> d logits
  template <typename R, int EV>
  __device__ __forceinline__ void slope(const R& r, float (&y)[EV]) const {
    if (r.any) {
#pragma unroll
      for (int e = 0; e < EV; ++e)
        if (r.count(e)) y[e] *= r.x[e] > 0.f ? down : up;
    }
  }
};

// a counted token's loads (none waits for another), and its value
struct Counted { float x, b; uint32_t c; bool kept; };
template <int T, int HIST>
__device__ __forceinline__ Counted load_counted(const Rules& q, const RowP& p, const char* lrow, const uint32_t* cnt, int v0,
                                                int d) {
  const int v = v0 + d;
  Counted t;
  t.x = Elem<T>::one(lrow, v);
  t.b = p.bias ? p.bias[v] : 0.f;
  t.kept = !p.mask || ((p.mask[v >> 3] >> (v & 7)) & 1);
  t.c = HIST ? count_at<HIST ? HIST : 1>(cnt, d) : 0u;
  return t;
}
template <int T>
__device__ __forceinline__ double counted_value(const RowP& p, const Counted& t) {
  return t.kept ? counted64(p, t.x, t.c, t.b) : -INFINITY;
}

// the value of a token, counted or not
template <int T>
__device__ __forceinline__ double any_value(const RowP& p, const Counted& t) {
  if (!t.kept) return -INFINITY;
  return t.c ? counted64(p, t.x, t.c, t.b) : (double)t.x + (double)t.b;
}

// ---- rows whose maximum is no ordinary one: token by token in doubles, a few in flight.  What lies `exponents` below the maximum
// (and by more than any rounding) is passed over after an fp32 sum and a comparison: nearly everything, at low temperatures.
__device__ __forceinline__ float far_reach(float m, float k, float exponents) {
  return m - (exponents / k + fabsf(m) * 0x1p-21f);
}

// the exact maximum of n tokens from v0 on and the sum of their weights against it, over a wave; weights below 2^-200 of the
// largest are left out
template <int T, int HIST, int N>
__device__ __forceinline__ void far_sum(const Rules& q, const RowP& p, const char* lrow, const uint32_t* cnt, int v0, int n,
                                        int lane, float m, double& top, double& sum) {
  const float reach = far_reach(m, (float)p.k, 200.f);
  double best = -INFINITY, s = 0.0;
#pragma unroll 1
  for (int d = lane; d < n; d += 64 * N) {
    Counted t[N];
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (d + 64 * u < n) t[u] = load_counted<T, HIST>(q, p, lrow, cnt, v0, d + 64 * u);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (d + 64 * u >= n || !t[u].kept || (!t[u].c && t[u].x + t[u].b < reach)) continue;
      const double y = any_value<T>(p, t[u]);
      const double w = exp2_rare(-fabs(y - best), p.k);
      s = y > best ? fma(s, w, 1.0) : s + w;
      best = fmax(best, y);
    }
  }
  top = wave_max(best);
  sum = wave_sum(best > -INFINITY ? s * exp2_rare(best - top, p.k) : 0.0);
}

// the gradients of a far row
struct Far {
  double top, iz, g;
  float reach;
  __device__ __forceinline__ Far(const SegArgs& a, const RowP& p, long long row, const Bwd& b) {
    top = a.o.stat[2 * row];
    iz = a.o.stat[2 * row + 1];
    g = (double)a.d_logprob[row] * (p.k * LN2);
    // 2^-400 of an ordinary g is no float; a NaN or infinite one shows everywhere
    reach = fabs(g) < INFINITY ? far_reach(b.m, b.kf, 400.f) : -INFINITY;
  }
  // d value of token v
  template <int T>
  __device__ __forceinline__ float value(const RowP& p, const Bwd& b, const Counted& t, int v) const {
    if (!t.kept || b.zero || (!t.c && t.x + t.b < reach && v != b.tok)) return 0.f;
    return (float)(g * ((v == b.tok ? 1.0 : 0.0) - exp2_rare(any_value<T>(p, t) - top, p.k) * iz));
  }
  static __device__ __forceinline__ float slope(const Bwd& b, const Counted& t, float y) {
    return t.c ? y * (t.x > 0.f ? b.down : b.up) : y;
  }
};

// APPLY and BWD: a value written for every logit
template <int T, int HIST, int MODE, bool ROWWAVE>
__global__ __launch_bounds__(256) void rules_map_kernel(SegArgs a) {
  typedef Elem<T> E;
  constexpr int EV = E::EV;
  extern __shared__ uint32_t lds[];          // counts of the workgroup's 4 segments
  const Rules& q = a.q;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long row = ROWWAVE ? (long long)blockIdx.x * 4 + wave : blockIdx.x / a.wgs_per_row;
  const int seg = ROWWAVE ? 0 : (blockIdx.x % a.wgs_per_row) * 4 + wave;
  const bool live = row < q.rows && seg < a.nseg;
  const int V = q.vocab;
  const int v0 = live ? seg * a.seg_len : 0;
  const RowP p = row_params(q, row < q.rows ? row : q.rows - 1);
  const int end = min(v0 + a.seg_len, V);
  const char* lrow = static_cast<const char*>(q.logits) + row * q.ld * (long long)sizeof(typename E::type);
  Steps<T, 4> steps;
  if (live) steps.begin(p, lrow, v0, end, lane, V);
  const uint32_t* cnt = lds;
  if (HIST) {
    const int words = 4 * a.seg_len / Counts<HIST ? HIST : 1>::PER_WORD;
    for (int i = threadIdx.x * 4; i < words; i += 1024) *reinterpret_cast<u32x4*>(&lds[i]) = u32x4{0, 0, 0, 0};
    __syncthreads();
    if (ROWWAVE) {
      if (live) count_history<HIST>(p, q.history_i64, 0, V, lds + wave * (words / 4), nullptr, lane, 64);
    } else {
      const int first = (seg - wave) * a.seg_len;
      count_history<HIST>(p, q.history_i64, first, min(4 * a.seg_len, V - first), lds, nullptr, threadIdx.x, 256);
    }
    __syncthreads();
    cnt = lds + wave * (words / 4);
  }
  if (!live) return;
  constexpr int PER = HIST ? Counts<HIST ? HIST : 1>::PER_WORD : 1;

  typename E::type* orow = static_cast<typename E::type*>(a.out) + row * a.out_ld;
  Bwd b;
  if (MODE == M_BWD) {
    b = Bwd(a, p, row);
    if (__builtin_expect(b.far, 0)) {
      const Far far(a, p, row, b);
#pragma unroll 1
      for (int d = lane; d < end - v0; d += 256) {
        Counted t[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (d + 64 * u < end - v0) t[u] = load_counted<T, HIST>(q, p, lrow, cnt, v0, d + 64 * u);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int v = v0 + d + 64 * u;
          if (v >= end) continue;
          const float y = far.template value<T>(p, b, t[u], v);
          if (a.d_bias_rows) a.d_bias_rows[row * V + v] = y;
          if (a.out) orow[v] = E::cast(far.slope(b, t[u], y));
        }
      }
      return;
    }
  }
  steps.run(p, lrow, V, [&](const Loaded& in, int v, auto whole) {
    const Ruled<T, HIST> r(p, in, cnt + (v - v0) / PER, v, V, whole);
    float y[EV];
#pragma unroll
    for (int e = 0; e < EV; ++e) y[e] = r.s[e];
    if (MODE == M_BWD) {
      b.values(r, in.keep, v, y);
      if (a.d_bias_rows) {
#pragma unroll
        for (int e = 0; e < EV; ++e)
          if (v + e < V) a.d_bias_rows[row * V + v + e] = y[e];
      }
      if (!a.out) return;
      b.slope(r, y);
    }
    store_step<T, decltype(whole)::value>(orow, v, V, y);
  });
}

// value of one token in 64 bits, -inf where the grammar forbids it
template <int T>
__device__ __forceinline__ double token_value(const Rules& q, const RowP& p, long long row, int v, uint32_t c) {
  if (p.mask && !((p.mask[v >> 3] >> (v & 7)) & 1)) return -INFINITY;
  const float x = Elem<T>::one(q.logits, row * q.ld + v), b = p.bias ? p.bias[v] : 0.f;
  return c ? counted64(p, x, c, b) : (double)x + (double)b;
}

// what the running sum has to exceed; from u = 1 on nothing does (and the last token with a weight is taken)
__device__ __forceinline__ double edge_of(float u, double Z) { return u < 1.f ? fmax((double)u, 0.0) * Z : INFINITY; }

// a row's results: its token, `at` the token's value, Z the row's sum against the reference `top` (its maximum); `rounded`: the
// weights in Z are those of values rounded to fp32
template <int MODE>
__device__ __forceinline__ void end_row(const Rules& q, const RowOut& o, const RowP& p, long long row, long long tok,
                                        double at, double top, bool ok, double Z, bool rounded) {
  const bool have = tok >= 0 && tok < q.vocab;
  float lp;
  if (MODE == M_SUM && !have) lp = 0.f;                   // an ignored row
  else if (top == -INFINITY) lp = -INFINITY;              // the rules leave nothing
  else if (!ok || !have) lp = NAN;                        // NaN or +inf among the allowed values (or a NaN u)
  else {
    // the token's own weight as its value has it (where it is most of Z, log p is that of the others' share and never above 0):
    // w e^d - w = w (d + d^2 / 2), |d| <= 4e-5
    const double near = (float)at, d = (at - near) * (p.k * LN2);
    double z = Z;
    if (rounded && at != near && near > -INFINITY) z += exp2_64(near - top, p.k) * fma(0.5 * d, d, d);
    lp = (float)((at - top) * (p.k * LN2) - log_64(z));
  }
  o.logprob[row] = lp;
  if (MODE == M_SUM) {
    o.stat[2 * row] = top == -INFINITY || ok ? top : NAN;
    o.stat[2 * row + 1] = ok ? reciprocal(Z) : NAN;
  } else {
    o.tokens[row] = tok;
    if (o.state_out) {
      const int s = q.state[row];
      o.state_out[row] = tok >= 0 && s >= 0 && s < q.states ? o.next[(size_t)s * q.vocab + tok] : s;
    }
  }
}

constexpr int LIST = 512;       // counted tokens of a segment that are listed; more are looked up bit by bit

// A segment's maximum and sum of weights.  Tokens that the history holds are left out of the steps (one more bit mask) and
// taken afterwards, a lane each: they are few, and the steps stay free of branches.
// DRAW: sums of doubles, against 0 as reference -- an exponent of a double has room for every ordinary row.  Else fp32 sums,
// against a reference of the lane's own that moves when a value exceeds it by 2^8 (an exponent of 8 is still exact to 2^-20).
// Where the maximum is no ordinary one and either kind of sum would show it, the segment is summed again in doubles, token by
// token, against its exact maximum.
// Waves a SIMD: as many as the steps' registers leave without spilling (with the token-by-token sum left to itself the compiler
// takes more registers for it than the steps do, a wave less: 512 x 131072 bf16 greedy under all rules 66.6 -> 69.3 us).
constexpr int sum_waves(int T, int HIST, int MODE, bool ROWWAVE) {
  if (MODE == M_DRAW) return T == DVAE_F32 && !ROWWAVE ? 5 : 4;
  return HIST && ROWWAVE && T != DVAE_F32 ? 6 : 7;
}
template <int T, int HIST, int MODE, bool ROWWAVE>
__global__ __launch_bounds__(256, sum_waves(T, HIST, MODE, ROWWAVE)) void rules_sum_kernel(SegArgs a) {
  constexpr bool DRAW = MODE == M_DRAW;
  typedef Elem<T> E;
  constexpr int EV = E::EV;
  extern __shared__ uint32_t lds[];          // counts of the 4 segments, a bit for each token, lists of the counted ones
  const Rules& q = a.q;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long row = ROWWAVE ? (long long)blockIdx.x * 4 + wave : blockIdx.x / a.wgs_per_row;
  const int seg = ROWWAVE ? 0 : (blockIdx.x % a.wgs_per_row) * 4 + wave;
  const bool live = row < q.rows && seg < a.nseg;
  const int V = q.vocab;
  const int v0 = live ? seg * a.seg_len : 0;
  const RowP p = row_params(q, row < q.rows ? row : q.rows - 1);
  const int end = min(v0 + a.seg_len, V);
  const char* lrow = static_cast<const char*>(q.logits) + row * q.ld * (long long)sizeof(typename E::type);
  Steps<T, DRAW ? 2 : 4> steps;
  if (live) steps.begin(p, lrow, v0, end, lane, V);
  const uint32_t *cnt = lds, *seen = lds;
  if (HIST) {
    const int words = 4 * a.seg_len / Counts<HIST ? HIST : 1>::PER_WORD, marks = 4 * a.seg_len / 32;
    uint32_t* bits = lds + words;
    for (int i = threadIdx.x * 4; i < words + marks; i += 1024) *reinterpret_cast<u32x4*>(&lds[i]) = u32x4{0, 0, 0, 0};
    __syncthreads();
    if (ROWWAVE) {
      if (live) count_history<HIST>(p, q.history_i64, 0, V, lds + wave * (words / 4), bits + wave * (marks / 4), lane, 64);
    } else {
      const int first = (seg - wave) * a.seg_len;
      count_history<HIST>(p, q.history_i64, first, min(4 * a.seg_len, V - first), lds, bits, threadIdx.x, 256);
    }
    __syncthreads();
    cnt = lds + wave * (words / 4);
    seen = bits + wave * (marks / 4);
  }
  if (!live) return;
  const float kf = (float)p.k;

  float m = -INFINITY, z = 0.f;
  float ref = -3.402823466e38f, lim = ref;           // fp32 sums: the lane's reference, and where it moves
  const float room = 8.f * (float)(p.temp * LN2);
  double zd = 0.0;
  const double low = -1000.0 * LN2 * p.temp;        // -1000 / k

  // the segment's counted tokens as a list (in a fixed order); the first 64 are loaded ahead of the steps, which hide the way
  const int counts = HIST ? 4 * a.seg_len / Counts<HIST ? HIST : 1>::PER_WORD + a.seg_len / 8 : 0;
  uint16_t* list = reinterpret_cast<uint16_t*>(lds + counts) + wave * LIST;
  int held = 0;
  Counted first_held{};
  if (HIST) {
    const int words = a.seg_len / 32;
    uint32_t w0 = lane < words ? seen[lane] : 0u, w1 = lane + 64 < words ? seen[lane + 64] : 0u;
    int at = __popc(w0) + __popc(w1);
    const int own = at;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(at, o);
      if (lane >= o) at += t;
    }
    held = __shfl(at, 63);
    if (held <= LIST) {
      at -= own;
      for (; w0; w0 &= w0 - 1) list[at++] = (uint16_t)(lane * 32 + __ffs(w0) - 1);
      for (; w1; w1 &= w1 - 1) list[at++] = (uint16_t)((lane + 64) * 32 + __ffs(w1) - 1);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (lane < held) first_held = load_counted<T, HIST>(q, p, lrow, cnt, v0, list[lane]);
    }
  }
  const auto take = [&](float mx) {
    m = max_nan(m, mx);
    if (!DRAW && mx > lim) {
      z *= __builtin_amdgcn_exp2f((ref - mx) * kf);
      ref = mx;
      lim = ref + room;
    }
  };
  const auto weigh = [&](double y) { zd += exp2_fast(y, p.k, low); };
  steps.run(p, lrow, V, [&](Loaded in, int v, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    if (HIST) {
      const uint32_t byte = reinterpret_cast<const uint8_t*>(seen)[(v - v0) >> 3];
      in.keep &= ~(EV == 8 ? byte : byte >> (v & 4));
    }
    float x[EV], s[EV];
#pragma unroll
    for (int e = 0; e < EV; ++e) x[e] = E::at(in.raw, e);
    const auto on = [&](int e) { return (uint32_t)((int)(in.keep << (31 - e)) >> 31); };
    if (HIST || p.mask || !WHOLE) {
#pragma unroll
      for (int e = 0; e < EV; ++e) x[e] = __uint_as_float((__float_as_uint(x[e]) & on(e)) | (0xff800000u & ~on(e)));
    }
    if (p.bias) {
      float b[EV];
      load_bias<EV, WHOLE>(p.bias, v, V, b);
      if (HIST || p.mask) {
#pragma unroll
        for (int e = 0; e < EV; ++e) b[e] = __uint_as_float(__float_as_uint(b[e]) & on(e));
      }
#pragma unroll
      for (int e = 0; e < EV; ++e) s[e] = x[e] + b[e];
      if (DRAW) {
#pragma unroll
        for (int e = 0; e < EV; ++e) weigh((double)x[e] + (double)b[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < EV; ++e) s[e] = x[e];
      if (DRAW) {
#pragma unroll
        for (int e = 0; e < EV; ++e) weigh((double)x[e]);
      }
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < EV; ++e) mx = max_nan(mx, s[e]);
    take(mx);
    if (!DRAW) {
#pragma unroll
      for (int e = 0; e < EV; ++e) z += __builtin_amdgcn_exp2f((s[e] - ref) * kf);
    }
  });
  if (HIST) {
    // 5 to 9 registers less in the steps, a wave more or none spilled; a draw of halves has the room (512 x 131072 112 us, 114 so)
    const RowP late = DRAW && T != DVAE_F32 ? p : params_anew(q, row);
    const auto one = [&](double y) {
      take((float)y);
      if (DRAW) weigh(y);
      else z += __builtin_amdgcn_exp2f(((float)y - ref) * kf);
    };
    if (held <= LIST) {
      if (lane < held) one(counted_value<T>(late, first_held));
      for (int i = lane + 64; i < held; i += 256) {          // four in flight
        Counted t[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + 64 * u < held) t[u] = load_counted<T, HIST>(q, p, lrow, cnt, v0, list[i + 64 * u]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + 64 * u < held) one(counted_value<T>(late, t[u]));
      }
    } else {
      for (int w = lane; w < a.seg_len / 32; w += 64)
        for (uint32_t left = seen[w]; left; left &= left - 1)
          one(counted_value<T>(late, load_counted<T, HIST>(q, p, lrow, cnt, v0, w * 32 + __ffs(left) - 1)));
    }
  }
  m = wave_max_nan(m);
  const bool finite = m > -INFINITY && m < INFINITY;
  const bool far = finite && (DRAW || inexact(q, p)) && !ordinary(m, DRAW ? (float)p.k : kf);
  Seg r;
  r.s = 0.0; r.top = m;
  if (__builtin_expect(far, 0)) {
    const RowP p = params_anew(q, row);
    far_sum<T, HIST, 4>(q, p, lrow, cnt, v0, end - v0, lane, m, r.top, r.s);
  } else if (finite) {
    r.s = DRAW ? wave_sum(zd) : (double)wave_sum(z * __builtin_amdgcn_exp2f((ref - m) * kf));
  }
  if (!ROWWAVE) {
    if (lane == 0) a.seg[row * a.nseg + seg] = r;
    return;
  }
  // a row of one segment: its wave decides it
  const bool ok = finite && p.fine;
  const double Z = ok ? r.s * exp2_64(reference<MODE>(r.top, p.k) - r.top, p.k) : 0.0;
  long long tok = -1;
  const auto count = [&](int v) { return HIST ? count_at<HIST ? HIST : 1>(cnt, v) : 0u; };
  // values of EV tokens, -inf where there is none
  const auto values = [&](int v, double (&y)[EV]) {
    const Loaded in = load_step<T, false>(p, lrow, v, V);
    float b[EV];
    if (p.bias) load_bias<EV, false>(p.bias, v, V, b);
#pragma unroll
    for (int e = 0; e < EV; ++e) {
      y[e] = -INFINITY;
      if (!((in.keep >> e) & 1)) continue;
      const uint32_t c = count(v + e);
      const float be = p.bias ? b[e] : 0.f;
      y[e] = c ? counted64(p, E::at(in.raw, e), c, be) : (double)E::at(in.raw, e) + (double)be;
    }
  };
  if (MODE == M_SUM) {
    tok = a.o.given[row];
  } else if (ok && MODE == M_GREEDY) {
    double best = -INFINITY;
    int idx = INT32_MAX;
    for (int v = lane * EV; v < end; v += 64 * EV) {
      double y[EV];
      values(v, y);
#pragma unroll
      for (int e = 0; e < EV; ++e)
        if (y[e] > best) { best = y[e]; idx = v + e; }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const double b2 = __shfl_xor(best, o);
      const int i2 = __shfl_xor(idx, o);
      if (b2 > best || (b2 == best && i2 < idx)) { best = b2; idx = i2; }
    }
    if (idx < V) tok = idx;
  } else if (ok && MODE == M_DRAW) {
    const float u = a.o.uniforms[row];
    if (u == u) {
      const double edge = edge_of(u, Z);
      double before = 0.0;
      int last = -1;
      for (int first = 0; first < end && tok < 0; first += 64 * EV) {
        const int v = first + lane * EV;
        double w[EV], sum = 0.0;
        if (v < end) values(v, w);
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          w[e] = v < end ? exp2_64(w[e] - r.top, p.k) : 0.0;
          sum += w[e];
          if (w[e] > 0.0) last = v + e;
        }
        double run = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const double t = __shfl_up(run, o);
          if (lane >= o) run += t;
        }
        const double all = __shfl(run, 63);
        run = before + (run - sum);
        int hit = INT32_MAX;
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          run += w[e];
          if (w[e] > 0.0 && run > edge && hit == INT32_MAX) hit = v + e;
        }
        const unsigned long long over = __ballot(hit != INT32_MAX);
        if (over) tok = __shfl(hit, __ffsll(over) - 1);
        before += all;
      }
      if (tok < 0) {                       // u >= 1, or by rounding: the last token with a weight
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o));
        tok = last;
      }
    }
  }
  if (lane) return;
  const bool have = tok >= 0 && tok < V;
  const double at = have ? token_value<T>(q, p, row, (int)tok, count((int)tok)) : 0.0;
  end_row<MODE>(q, a.o, p, row, tok, at, r.top, ok, Z, !DRAW && !far);
}

// ---------------------------------------------------------------------------------------------------------------
// join: one workgroup a row
// ---------------------------------------------------------------------------------------------------------------
struct JoinArgs {
  Rules q;
  RowOut o;
  int nseg, seg_len;
  const Seg* seg;
};

template <typename X, typename F>
__device__ __forceinline__ X block_reduce(X v, X* sh, F f) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return f(f(sh[0], sh[1]), f(sh[2], sh[3]));
}

// inclusive scan over the 256 threads; returns the thread's exclusive prefix, `total` the sum of all
__device__ __forceinline__ double block_prefix(double v, double* sh, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) sh[wave] = x;
  __syncthreads();
  double before = 0.0;
  for (int w = 0; w < wave; ++w) before += sh[w];
  total = sh[0] + sh[1] + sh[2] + sh[3];
  return before + (x - v);
}

constexpr int HIST_STAGE = 4096;       // tokens of a history that the join keeps in LDS

// One workgroup a row.  What it reads depends on what it has read (partials, then the segment they point to), so the
// loads that do not -- the history, a given token's logit -- are begun first, and the partials stay in registers.
template <int T, int MODE>
__global__ __launch_bounds__(256) void rules_join_kernel(JoinArgs a) {
  constexpr bool SEARCH = MODE != M_SUM;
  __shared__ double shd[4];
  __shared__ float shf[4];
  __shared__ int shi[4];
  __shared__ double pick_before;
  __shared__ int hist[SEARCH ? HIST_STAGE : 1];
  __shared__ uint32_t cnt[SEARCH ? SEG_MAX : 1];      // counts of the segment that is searched
  const Rules& q = a.q;
  const long long row = blockIdx.x;
  const int V = q.vocab, tid = threadIdx.x, n = a.seg_len;
  const RowP p = row_params(q, row);
  const Seg* seg = a.seg + row * a.nseg;
  const char* lrow = static_cast<const char*>(q.logits) + row * q.ld * (long long)sizeof(typename Elem<T>::type);

  // contiguous shares, so that running sums follow the vocabulary's order
  const int per = (a.nseg + 255) / 256;
  const int i0 = min(tid * per, a.nseg), i1 = min(i0 + per, a.nseg);
  Seg mine;
  mine.s = 0.0; mine.top = -INFINITY;
  if (i0 < i1) mine = seg[i0];

  const float uf = MODE == M_DRAW ? a.o.uniforms[row] : 0.f;
  long long tok = -1;
  double given_y = 0.0;
  int c = 0;
  if (SEARCH) {
    RowP staged = p;
    staged.n_hist = min(p.n_hist, HIST_STAGE);
    int at = tid;
    for_history<8>(staged, q.history_i64, 0, tid, 256, [&](long long t) {
      hist[at] = t >= 0 && t < V ? (int)t : -1;
      at += 256;
    });
  } else {
    tok = a.o.given[row];
    if (tok >= 0 && tok < V) {
      for_history<8>(p, q.history_i64, 0, tid, 256, [&](long long t) { c += t == tok; });
      if (p.n_hist) c = block_reduce(c, shi, [](int x, int y) { return x + y; });
      given_y = token_value<T>(q, p, row, (int)tok, c);
    }
  }

  float m = (float)mine.top;
  for (int i = i0 + 1; i < i1; ++i) m = max_nan(m, (float)seg[i].top);
  m = block_reduce(m, shf, [](float x, float y) { return max_nan(x, y); });
  const bool ok = m > -INFINITY && m < INFINITY && p.fine, plain = ordinary(m, (float)p.k);
  double top = m;
  if (ok && !plain) {                  // the exact one (a reduction of doubles takes half a microsecond more)
    top = mine.top;
    for (int i = i0 + 1; i < i1; ++i) top = fmax(top, seg[i].top);
    top = block_reduce(top, shd, [](double x, double y) { return fmax(x, y); });
  }
  // (a segment below 2^-990 of the largest weight counts as 0: what a draw picks has tokens whose own weights, cut at 2^-1000,
  // are none)
  const auto scaled = [&](const Seg& s) {
    return (s.top - top) * p.k >= -990.0 ? s.s * exp2_64(reference<MODE>(s.top, p.k) - top, p.k) : 0.0;
  };
  double z0 = 0.0, z = 0.0;
  if (ok) {
    z0 = scaled(mine);
    z = z0;
    for (int i = i0 + 1; i < i1; ++i) z += scaled(seg[i]);
  }
  double Z;
  const double before = block_prefix(z, shd, Z);

  const bool rounded = MODE != M_DRAW && plain;
  const auto finish = [&](long long t, double y) { end_row<MODE>(q, a.o, p, row, t, y, top, ok, Z, rounded); };
  if (MODE == M_SUM) {
    if (tid == 0) finish(tok, given_y);
    return;
  }
  if (!ok || uf != uf) {
    if (tid == 0) finish(-1, 0.0);
    return;
  }
  // counts of the tokens [v0, v0 + n)
  const auto count = [&](int v0) {
    for (int i = tid; i < n; i += 256) cnt[i] = 0;
    __syncthreads();
    const int staged = min(p.n_hist, HIST_STAGE);
#pragma unroll 4
    for (int i = tid; i < staged; i += 256) {
      const int t = hist[i], d = t - v0;
      if (t >= 0 && d >= 0 && d < n) atomicAdd(&cnt[d], 1u);
    }
    for_history<8>(p, q.history_i64, HIST_STAGE, tid, 256, [&](long long t) {
      const long long d = t - v0;
      if ((unsigned long long)d < (unsigned long long)n) atomicAdd(&cnt[(int)d], 1u);
    });
    __syncthreads();
  };

  if (MODE == M_GREEDY) {
    // the segments whose maximum rounds to the row's (hardly ever more than one), and in them the elements that do: among
    // those the largest one, then the lowest index
    double best = -INFINITY;
    int idx = INT32_MAX;
    int from = 0;
    while (true) {
      int g = (float)mine.top == m && i0 >= from ? i0 : INT32_MAX;
      for (int i = i0 + 1; i < i1; ++i)
        if (i >= from && i < g && (float)seg[i].top == m) g = i;
      g = block_reduce(g, shi, [](int x, int y) { return min(x, y); });
      if (g == INT32_MAX) break;
      from = g + 1;
      const int v0 = g * n;
      count(v0);
      for (int e = tid; e < n && v0 + e < V; e += 1024) {
        Counted t[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (e + 256 * u < n && v0 + e + 256 * u < V) t[u] = load_counted<T, 2>(q, p, lrow, cnt, v0, e + 256 * u);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int v = v0 + e + 256 * u;
          if (e + 256 * u >= n || v >= V) continue;
          const double y = any_value<T>(p, t[u]);
          if ((float)y != m) continue;
          if (y > best || (y == best && v < idx)) { best = y; idx = v; }
        }
      }
      __syncthreads();
    }
    const double most = block_reduce(best, shd, [](double x, double y) { return fmax(x, y); });
    const int t = block_reduce(best == most ? idx : INT32_MAX, shi, [](int x, int y) { return min(x, y); });
    if (t == INT32_MAX) {                // (the sum pass computed the same values: one of them is the maximum)
      if (tid == 0) finish(-1, 0.0);
    } else if (idx == t) {
      finish(t, best);
    }
    return;
  }

  // the segment where the running sum passes u Z; beyond the end (u >= 1, or rounding): the last one with a weight
  const double edge = edge_of(uf, Z);
  int first = INT32_MAX, last = -1;
  double first_before = 0.0, last_before = 0.0, run = before;
  for (int i = i0; i < i1; ++i) {
    const double w = i == i0 ? z0 : scaled(seg[i]);
    if (w > 0.0) { last = i; last_before = run; }
    if (w > 0.0 && run + w > edge && first == INT32_MAX) { first = i; first_before = run; }
    run += w;
  }
  const int f = block_reduce(first, shi, [](int x, int y) { return min(x, y); });
  int g = f;
  if (f == INT32_MAX) g = block_reduce(last, shi, [](int x, int y) { return max(x, y); });
  if (g < 0) {      // no weight at all: not with a finite maximum
    if (tid == 0) finish(-1, 0.0);
    return;
  }
  if (g >= i0 && g < i1) {
    pick_before = f != INT32_MAX ? first_before : last_before;
  }
  const int v0 = g * n;
  count(v0);
  // weights of the segment's tokens: a quarter for each wave, in strips of 64 tokens
  constexpr int STRIPS = SEG_MAX / 256;
  const int strips = n / 256, lane = tid & 63, wave = tid >> 6;
  const int d0 = wave * (n / 4) + lane;
  Counted tokens[STRIPS];
#pragma unroll
  for (int e = 0; e < STRIPS; ++e)
    if (e < strips && v0 + d0 + e * 64 < V) tokens[e] = load_counted<T, 2>(q, p, lrow, cnt, v0, d0 + e * 64);
  double w[STRIPS], sum = 0.0;
#pragma unroll
  for (int e = 0; e < STRIPS; ++e) {
    w[e] = 0.0;
    if (e < strips && v0 + d0 + e * 64 < V) w[e] = exp2_64(any_value<T>(p, tokens[e]) - top, p.k);
    sum += w[e];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  __syncthreads();
  if (lane == 0) shd[wave] = sum;
  __syncthreads();
  double at = pick_before;
  int in = -1;
  for (int i = 0; i < 4; ++i) {
    if (shd[i] > 0.0 && at + shd[i] > edge) { in = i; break; }
    at += shd[i];
  }
  if (in < 0) {      // by rounding, or u >= 1: the last token with a weight
    int tail = -1;
#pragma unroll
    for (int e = 0; e < STRIPS; ++e)
      if (w[e] > 0.0) tail = d0 + e * 64;
    tail = block_reduce(tail, shi, [](int x, int y) { return max(x, y); });
    if (tail < 0) {
      if (tid == 0) finish(-1, 0.0);
    } else if (tail >= d0 && ((tail - d0) & 63) == 0 && tail < wave * (n / 4) + n / 4) {
      finish(v0 + tail, token_value<T>(q, p, row, v0 + tail, cnt[tail]));
    }
    return;
  }
  if (wave != in) return;
  int hit = INT32_MAX, tail = -1;
#pragma unroll
  for (int g = 0; g < STRIPS; g += 4) {             // four strips' running sums at once: a step of one waits for its shuffles
    if (g < strips && hit == INT32_MAX) {
      double run[4] = {w[g], w[g + 1], w[g + 2], w[g + 3]};
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        double t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = __shfl_up(run[j], o);
#pragma unroll
        for (int j = 0; j < 4; ++j) run[j] += lane >= o ? t[j] : 0.0;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned long long over = __ballot(w[g + j] > 0.0 && at + run[j] > edge), any = __ballot(w[g + j] > 0.0);
        if (hit == INT32_MAX) {
          if (any) tail = (g + j) * 64 + 63 - __clzll(any);
          if (over) hit = (g + j) * 64 + __ffsll(over) - 1;
        }
        at += __shfl(run[j], 63);
      }
    }
  }
  // (sums of another order may end a rounding short of the edge: then the wave's last token with a weight)
  const int d = wave * (n / 4) + (hit != INT32_MAX ? hit : tail);
  if (((d - d0) & 63) == 0) finish(v0 + d, token_value<T>(q, p, row, v0 + d, cnt[d]));
}

// ---------------------------------------------------------------------------------------------------------------
// vocabularies of up to 128 tokens: a group of W lanes a row (a power of two), eight tokens a lane, one launch that ends each
// row -- everything in double, sums and searches by shuffles inside the group.  Eight tokens a lane, because what a row costs
// once (its settings, log, decision) takes a whole wave's time however few lanes share it: 100000 x 8 drawn after seven tokens
// of history 8.5 us with a lane a row, 15.6 us with eight.  Against a wave a row: 100000 x 65 bf16 drawn 43 / 160 us, applied 45 /
// 59 us, but 20000 x 300 fp32 40 / 32 and 37 / 15 us.
// ---------------------------------------------------------------------------------------------------------------
constexpr int GROUP_TOKENS = 8, GROUP_VOCAB = 128;

struct GroupArgs {
  Rules q;
  RowOut o;
  int w;                          // lanes of a row
  const float* d_logprob; void* out; long long out_ld; float* d_bias; float* part;             // APPLY, BWD
};

template <int T, int MODE>
__global__ __launch_bounds__(256) void rules_group_kernel(GroupArgs a) {
  typedef Elem<T> E;
  constexpr int EV = E::EV, K = GROUP_TOKENS;
  __shared__ float acc_sh[MODE == M_BWD ? 4 : 1][MODE == M_BWD ? GROUP_VOCAB : 1];
  const Rules& q = a.q;
  const int W = a.w, V = q.vocab;
  const int lane = threadIdx.x & (W - 1), v0 = lane * K;
  const int groups = 256 / W;
  float acc[K];
#pragma unroll
  for (int j = 0; j < K; ++j) acc[j] = 0.f;
  for (long long row = (long long)blockIdx.x * groups + threadIdx.x / W; row < q.rows; row += (long long)gridDim.x * groups) {
    const RowP p = row_params(q, row);
    const char* lrow = static_cast<const char*>(q.logits) + row * q.ld * (long long)sizeof(typename E::type);
    float x[K], b[K];
    uint32_t keep = v0 >= V ? 0u : v0 + K <= V ? 0xffu : (1u << (V - v0)) - 1;
    if (v0 + K <= V) {
#pragma unroll
      for (int i = 0; i < K / EV; ++i) {
        const u32x4 raw = *reinterpret_cast<const u32x4_u*>(lrow + (size_t)v0 * sizeof(typename E::type) + 16 * i);
#pragma unroll
        for (int e = 0; e < EV; ++e) x[i * EV + e] = E::at(raw, e);
      }
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j) x[j] = v0 + j < V ? E::one(lrow, v0 + j) : 0.f;
    }
    if (p.mask && v0 < V) keep &= p.mask[lane];
#pragma unroll
    for (int j = 0; j < K; ++j) b[j] = p.bias && v0 + j < V ? p.bias[v0 + j] : 0.f;
    // counts: bytes of a register (a history has at most 255 tokens here)
    uint64_t c = 0;
    for_history<4>(p, q.history_i64, 0, 0, 1, [&](long long t) {
      const unsigned long long d = (unsigned long long)(t - v0);
      c += d < K ? 1ull << (8 * (d & 7)) : 0ull;
    });
    const auto count = [&](int j) { return (uint32_t)(c >> (8 * j)) & 0xffu; };
    double y[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      y[j] = -INFINITY;
      if ((keep >> j) & 1) y[j] = count(j) ? counted64(p, x[j], count(j), b[j]) : (double)x[j] + (double)b[j];
    }
    if (MODE == M_APPLY || MODE == M_BWD) {
      float out[K];
      if (MODE == M_BWD) {
        const double top = a.o.stat[2 * row];
        const long long tok = a.o.given[row];
        const bool zero = tok < 0 || tok >= V || top == -INFINITY;
        const double coef = (double)a.d_logprob[row] * (p.k * LN2), iz = a.o.stat[2 * row + 1];
#pragma unroll
        for (int j = 0; j < K; ++j) {
          double g = 0.0;
          if (!zero && ((keep >> j) & 1)) g = coef * ((v0 + j == tok ? 1.0 : 0.0) - exp2_64(y[j] - top, p.k) * iz);
          const float gf = (float)g;
          if (a.part) acc[j] += gf;
          else if (a.d_bias && v0 + j < V) a.d_bias[row * V + v0 + j] = gf;
          if (count(j)) g *= x[j] > 0.f ? p.inv_rho : p.rho;
          out[j] = (float)g;
        }
      } else {
#pragma unroll
        for (int j = 0; j < K; ++j) out[j] = (float)y[j];
      }
      if (MODE == M_BWD && !a.out) continue;
      typename E::type* orow = static_cast<typename E::type*>(a.out) + row * a.out_ld;
      typename E::type o[K];
#pragma unroll
      for (int j = 0; j < K; ++j) o[j] = E::cast(out[j]);
      if (v0 + K <= V) {
#pragma unroll
        for (int i = 0; i < K / EV; ++i) {
          u32x4 w;
          __builtin_memcpy(&w, o + i * EV, 16);
          *reinterpret_cast<u32x4_u*>(orow + v0 + i * EV) = w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (v0 + j < V) orow[v0 + j] = o[j];
      }
      continue;
    }
    double top = y[0];
#pragma unroll
    for (int j = 1; j < K; ++j) top = max_nan(top, y[j]);
    for (int o = W >> 1; o > 0; o >>= 1) top = max_nan(top, __shfl_xor(top, o));
    if ((float)top == -INFINITY) top = -INFINITY;      // beyond fp32 is forbidden, as in longer rows
    const bool ok = top > -INFINITY && (float)top < INFINITY && p.fine;
    double w[K], sum = 0.0;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      w[j] = ok && ((keep >> j) & 1) ? exp2_64(y[j] - top, p.k) : 0.0;
      sum += w[j];
    }
    double run = sum;                                 // running sum of the lanes, in the vocabulary's order
    for (int o = 1; o < W; o <<= 1) {
      const double t = __shfl_up(run, o, W);
      if (lane >= o) run += t;
    }
    const double Z = __shfl(run, W - 1, W);
    int tok = -1;
    if (MODE == M_SUM) {
      const long long t = a.o.given[row];
      tok = t >= 0 && t < V ? (int)t : -1;
    } else if (ok && MODE == M_GREEDY) {
      double best = -INFINITY;
      int idx = INT32_MAX;
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (y[j] > best) { best = y[j]; idx = v0 + j; }
      for (int o = W >> 1; o > 0; o >>= 1) {
        const double b2 = __shfl_xor(best, o);
        const int i2 = __shfl_xor(idx, o);
        if (b2 > best || (b2 == best && i2 < idx)) { best = b2; idx = i2; }
      }
      tok = idx < V ? idx : -1;
    } else if (ok && MODE == M_DRAW) {
      const float u = a.o.uniforms[row];
      const double edge = edge_of(u, Z);
      double at = run - sum;
      int hit = INT32_MAX, last = -1;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        at += w[j];
        if (w[j] > 0.0) {
          last = v0 + j;
          if (at > edge && hit == INT32_MAX) hit = v0 + j;
        }
      }
      for (int o = W >> 1; o > 0; o >>= 1) {
        hit = min(hit, __shfl_xor(hit, o));
        last = max(last, __shfl_xor(last, o));
      }
      tok = u != u ? -1 : hit != INT32_MAX ? hit : last;      // beyond the end (u >= 1): the last token with a weight
    }
    double at = 0.0;
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (v0 + j == tok) at = y[j];
    at = __shfl(at, tok >= 0 ? tok / K : 0, W);
    if (lane == 0) end_row<MODE>(q, a.o, p, row, tok, at, top, ok, Z, false);
  }
  if (MODE == M_BWD) {
    if (!a.part) return;
    // the workgroup's share of the bias gradient, in a fixed order: the wave's groups, then the waves
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      for (int o = W; o < 64; o <<= 1) acc[j] += __shfl_xor(acc[j], o);
      if ((threadIdx.x & 63) < W) acc_sh[wave][v0 + j] = acc[j];
    }
    __syncthreads();
    for (int v = threadIdx.x; v < V; v += 256)
      a.part[(size_t)blockIdx.x * V + v] = (acc_sh[0][v] + acc_sh[1][v]) + (acc_sh[2][v] + acc_sh[3][v]);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// gradients with a bias shared by the rows: a workgroup owns 256 EV columns and a share of the rows, each of its waves
// every fourth of them, so that the bias gradient's sum over rows stays in registers and no row costs a barrier (a wave
// counts its row's history by itself); shares are added in a fixed order by a second launch
// ---------------------------------------------------------------------------------------------------------------
struct ColArgs {
  SegArgs s;
  float* part;           // [shares][vocab]
  int rows_per_share;
};

constexpr int COL_STEPS = 4;

template <int T, int HIST>
__global__ __launch_bounds__(256, T == DVAE_F32 && HIST < 2 ? 4 : 2) void rules_bwd_col_kernel(ColArgs ca) {
  typedef Elem<T> E;
  constexpr int EV = E::EV, STEP = 64 * EV, SPAN = COL_STEPS * STEP, PER = HIST ? Counts<HIST ? HIST : 1>::PER_WORD : 1;
  __shared__ uint32_t lds[4 * SPAN];              // counts of each wave's row, then each wave's sums
  __shared__ float turn[4][STEP];
  const SegArgs& a = ca.s;
  const Rules& q = a.q;
  const int V = q.vocab, v0 = blockIdx.x * SPAN, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long r0 = (long long)blockIdx.y * ca.rows_per_share;
  const long long r1 = min(r0 + ca.rows_per_share, q.rows);
  uint32_t* cnt = lds + wave * (SPAN / PER);
  float acc[COL_STEPS][EV];
#pragma unroll
  for (int j = 0; j < COL_STEPS; ++j)
#pragma unroll
    for (int e = 0; e < EV; ++e) acc[j][e] = 0.f;
  const auto sync = [] {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  const auto count = [&](const RowP& p) {
    if (!HIST) return;
    for (int i = lane * 4; i < SPAN / PER; i += 256) *reinterpret_cast<u32x4*>(&cnt[i]) = u32x4{0, 0, 0, 0};
    sync();
    count_history<HIST ? HIST : 1>(p, q.history_i64, v0, min(SPAN, V - v0), cnt, nullptr, lane, 64);
    sync();
  };
  bool some_far = false;
  for (long long row = r0 + wave; row < r1; row += 4) {
    const RowP p = row_params(q, row);
    const Bwd b(a, p, row);
    const char* lrow = static_cast<const char*>(q.logits) + row * q.ld * (long long)sizeof(typename E::type);
    typename E::type* orow = static_cast<typename E::type*>(a.out) + row * a.out_ld;
    Loaded in[COL_STEPS];
#pragma unroll
    for (int j = 0; j < COL_STEPS; ++j) {
      const int v = v0 + j * STEP + lane * EV;
      if (v0 + (j + 1) * STEP <= V) in[j] = load_step<T, true>(p, lrow, v, V);
      else in[j] = load_step<T, false>(p, lrow, v, V);
    }
    if (__builtin_expect(b.far, 0)) {
      some_far = true;
      continue;
    }
    count(p);
#pragma unroll
    for (int j = 0; j < COL_STEPS; ++j) {
      const int d = j * STEP + lane * EV, v = v0 + d;
      const auto step = [&](auto whole) {
        const Ruled<T, HIST> r(p, in[j], cnt + d / PER, v, V, whole);
        float y[EV];
        b.values(r, in[j].keep, v, y);
#pragma unroll
        for (int e = 0; e < EV; ++e) acc[j][e] += y[e];
        if (!a.out) return;
        b.slope(r, y);
        store_step<T, decltype(whole)::value>(orow, v, V, y);
      };
      if (v0 + (j + 1) * STEP <= V) step(std::true_type{});
      else if (v < V) step(std::false_type{});
    }
  }
  if (__builtin_expect(some_far, 0)) {
#pragma unroll 1
    for (long long row = r0 + wave; row < r1; row += 4) {
      const RowP p = row_params(q, row);
      const Bwd b(a, p, row);
      if (!b.far) continue;
      const char* lrow = static_cast<const char*>(q.logits) + row * q.ld * (long long)sizeof(typename E::type);
      typename E::type* orow = static_cast<typename E::type*>(a.out) + row * a.out_ld;
      const Far far(a, p, row, b);
      count(p);
#pragma unroll 1
      for (int i = 0; i < COL_STEPS; ++i) {         // tokens side by side, then to the lanes that add them up
#pragma unroll 1
        for (int c = lane; c < STEP; c += 256) {
          Counted t[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (v0 + i * STEP + c + 64 * u < V) t[u] = load_counted<T, HIST>(q, p, lrow, cnt, v0, i * STEP + c + 64 * u);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int v = v0 + i * STEP + c + 64 * u;
            const float y = v < V ? far.template value<T>(p, b, t[u], v) : 0.f;
            if (a.out && v < V) orow[v] = E::cast(far.slope(b, t[u], y));
            turn[wave][c + 64 * u] = y;
          }
        }
        sync();
#pragma unroll
        for (int j = 0; j < COL_STEPS; ++j)
#pragma unroll
          for (int e = 0; e < EV; ++e) acc[j][e] += i == j ? turn[wave][lane * EV + e] : 0.f;
        sync();
      }
    }
  }
  __syncthreads();
  float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int j = 0; j < COL_STEPS; ++j)
#pragma unroll
    for (int e = 0; e < EV; ++e) sums[wave * SPAN + j * STEP + lane * EV + e] = acc[j][e];
  __syncthreads();
  for (int d = threadIdx.x; d < SPAN && v0 + d < V; d += 256)
    ca.part[(size_t)blockIdx.y * V + v0 + d] = (sums[d] + sums[SPAN + d]) + (sums[2 * SPAN + d] + sums[3 * SPAN + d]);
}

// 16 columns a workgroup, 16 threads a column: shares in a fixed order
__global__ __launch_bounds__(256) void rules_bias_sum_kernel(const float* __restrict__ part, int shares, int V,
                                                             float* __restrict__ d_bias) {
  __shared__ float sh[16][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, v = blockIdx.x * 16 + c;
  float s = 0.f;
  if (v < V) {
#pragma unroll 4
    for (int i = r; i < shares; i += 16) s += part[(size_t)i * V + v];
  }
  sh[r][c] = s;
  __syncthreads();
  if (r || v >= V) return;
  for (int i = 1; i < 16; ++i) s += sh[i][c];
  d_bias[v] = s;
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
constexpr long long MAX_BLOCKS = (1ll << 24) - 1;     // blocks x 256 threads stay below 2^32

struct Plan { int seg_len, nseg, wgs_per_row; bool row_wave; long long blocks; };

Rules with_constants(const dvae_rules& q) {
  Rules r;
  static_cast<dvae_rules&>(r) = q;
  r.repetition = std::max(q.repetition, 1e-200);               // below it every quotient is beyond fp32, and 1 / rho has to be finite
  r.inv_rho = 1.0 / r.repetition;
  r.k = LOG2E / q.temperature;
  return r;
}

Plan plan_of(const dvae_rules& q) {
  Plan p;
  const int step = 64 * (16 / elem_bytes(q.dtype));      // tokens of a wave's step
  // segments as long as 4096 waves (four for each SIMD) leave them: few rows are spread over the whole card
  // (a workgroup counts the whole history, so a long one asks for long segments: 512 x 131072 bf16 drawn after 8192 tokens 189 us
  // with 4096 tokens, 237 with 2048, after 65535 666 and 1012; 32-bit counts take twice the room)
  const int cap = q.history && q.history_len > 4096 && q.history_len < 65536 ? SEG_MAX : 2048;
  p.seg_len = step;
  while (p.seg_len < cap && p.seg_len < q.vocab && q.rows * ((q.vocab + p.seg_len - 1) / p.seg_len) > 4096) p.seg_len *= 2;
  p.nseg = (int)(((long long)q.vocab + p.seg_len - 1) / p.seg_len);
  p.row_wave = p.nseg == 1;
  p.wgs_per_row = (p.nseg + 3) / 4;
  p.blocks = p.row_wave ? (q.rows + 3) / 4 : q.rows * p.wgs_per_row;
  return p;
}

template <int T, int HIST, int MODE>
void launch_seg(const SegArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)p.blocks), block(256);
  // counts of 4 segments and, for sums, a bit for each token and the lists: 38 KB at most
  unsigned lds = HIST ? 16u * p.seg_len / Counts<HIST ? HIST : 1>::PER_WORD : 0u;
  if constexpr (MODE == M_APPLY || MODE == M_BWD) {
    if (p.row_wave) hipLaunchKernelGGL((rules_map_kernel<T, HIST, MODE, true>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((rules_map_kernel<T, HIST, MODE, false>), grid, block, lds, st, a);
  } else {
    if (HIST) lds += p.seg_len / 2 + 4 * LIST * 2;
    if (p.row_wave) hipLaunchKernelGGL((rules_sum_kernel<T, HIST, MODE, true>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((rules_sum_kernel<T, HIST, MODE == M_DRAW ? M_DRAW : M_SUM, false>), grid, block, lds, st, a);
  }
}

template <int T, int MODE>
void pick_hist(const SegArgs& a, const Plan& p, hipStream_t st) {
  if (!a.q.history || a.q.history_len == 0) launch_seg<T, 0, MODE>(a, p, st);
  else if (a.q.history_len < 65536) launch_seg<T, 1, MODE>(a, p, st);
  else launch_seg<T, 2, MODE>(a, p, st);
}

template <int MODE>
int run_seg(SegArgs& a, const Plan& p, hipStream_t st) {
  a.nseg = p.nseg; a.seg_len = p.seg_len; a.wgs_per_row = p.wgs_per_row;
  switch (a.q.dtype) {
    case DVAE_F32: pick_hist<DVAE_F32, MODE>(a, p, st); break;
    case DVAE_BF16: pick_hist<DVAE_BF16, MODE>(a, p, st); break;
    default: pick_hist<DVAE_F16, MODE>(a, p, st);
  }
  DVAE_LAUNCH_CHECK();
  return DVAE_OK;
}

// sums of all segments, then the rows' decisions (ROWWAVE: in the same launch)
template <int MODE>
int run_join(SegArgs& s, hipStream_t st) {
  const Plan p = plan_of(s.q);
  DVAE_TRY(run_seg<MODE>(s, p, st));
  if (p.row_wave) return DVAE_OK;
  JoinArgs a{};
  a.q = s.q; a.o = s.o; a.nseg = p.nseg; a.seg_len = p.seg_len; a.seg = s.seg;
  const dim3 grid((unsigned)a.q.rows), block(256);
  switch (a.q.dtype) {
    case DVAE_F32: hipLaunchKernelGGL((rules_join_kernel<DVAE_F32, MODE>), grid, block, 0, st, a); break;
    case DVAE_BF16: hipLaunchKernelGGL((rules_join_kernel<DVAE_BF16, MODE>), grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL((rules_join_kernel<DVAE_F16, MODE>), grid, block, 0, st, a);
  }
  DVAE_LAUNCH_CHECK();
  return DVAE_OK;
}

// every lane of a group reads the whole history: short ones, the shorter the more lanes do (a wave that counts in LDS reads it
// once; bytes hold counts up to 255)
bool is_small(const dvae_rules& q) {
  return q.vocab <= GROUP_VOCAB && (!q.history || q.history_len <= (q.vocab <= 64 ? 255 : 32));
}

bool needs_segments(const dvae_rules& q) { return !is_small(q) && !plan_of(q).row_wave; }

int group_lanes(const dvae_rules& q) {
  int w = 1;
  while (w * GROUP_TOKENS < q.vocab) w <<= 1;
  return w;
}

long long group_blocks(const dvae_rules& q) {
  const int groups = 256 / group_lanes(q);
  return (q.rows + groups - 1) / groups;
}

template <int MODE>
int run_group(GroupArgs& a, long long blocks, hipStream_t st) {
  a.w = group_lanes(a.q);
  const dim3 grid((unsigned)blocks), block(256);
  switch (a.q.dtype) {
    case DVAE_F32: hipLaunchKernelGGL((rules_group_kernel<DVAE_F32, MODE>), grid, block, 0, st, a); break;
    case DVAE_BF16: hipLaunchKernelGGL((rules_group_kernel<DVAE_BF16, MODE>), grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL((rules_group_kernel<DVAE_F16, MODE>), grid, block, 0, st, a);
  }
  DVAE_LAUNCH_CHECK();
  return DVAE_OK;
}

int bias_shares(const dvae_rules& q) {
  if (is_small(q)) return (int)std::min<long long>(group_blocks(q), 1024);
  const int span = 64 * COL_STEPS * (16 / elem_bytes(q.dtype));
  const long long cols = ((long long)q.vocab + span - 1) / span;
  return (int)std::min<long long>((q.rows + 3) / 4, std::max<long long>(1, 1024 / cols));
}

}  // namespace

int rules_check(const dvae_rules& q, const char* who) {
  DVAE_REQUIRE(q.rows >= 0 && q.vocab >= 1, "%s: rows >= 0 and vocab >= 1", who);
  DVAE_REQUIRE(q.dtype == DVAE_F32 || q.dtype == DVAE_BF16 || q.dtype == DVAE_F16, "%s: dtype %d", who, q.dtype);
  DVAE_REQUIRE(q.logits || q.rows == 0, "%s: null logits", who);
  DVAE_REQUIRE(q.rows <= 1 || q.ld >= q.vocab, "%s: rows of logits overlap (ld %lld < vocab %d)", who, q.ld, q.vocab);
  DVAE_REQUIRE(q.vocab <= (1 << 27), "%s: vocab %d above 2^27", who, q.vocab);
  DVAE_REQUIRE(q.repetition_rows || (q.repetition > 0.0 && std::isfinite(q.repetition)), "%s: repetition must be positive", who);
  DVAE_REQUIRE(q.frequency_rows || std::isfinite(q.frequency), "%s: frequency must be finite", who);
  DVAE_REQUIRE(q.presence_rows || q.presence > -INFINITY, "%s: presence must be above -inf", who);
  DVAE_REQUIRE(q.temperature_rows || (q.temperature >= TEMP_MIN && q.temperature <= TEMP_MAX),
               "%s: temperature must be in [1e-37, 1e37]", who);
  if (q.history) {
    DVAE_REQUIRE(q.history_len >= 0 && q.history_ld >= 0, "%s: negative history length", who);
    DVAE_REQUIRE(q.rows_per_history >= 1, "%s: rows_per_history must be at least 1", who);
  }
  if (q.mask) {
    DVAE_REQUIRE(q.state && q.states >= 1, "%s: a mask needs the rows' states", who);
    DVAE_REQUIRE(q.mask_words >= (q.vocab + 31) / 32, "%s: mask rows hold %d words, vocab %d needs %d", who, q.mask_words,
                 q.vocab, (q.vocab + 31) / 32);
  }
  const Plan p = plan_of(q);
  DVAE_REQUIRE(p.blocks <= MAX_BLOCKS && q.rows <= MAX_BLOCKS, "%s: %lld rows of %d tokens are too many for one call", who,
               q.rows, q.vocab);
  return DVAE_OK;
}

extern "C" size_t dvae_rules_ws_bytes(const dvae_rules* q) {
  if (!q || q->rows <= 0 || q->vocab < 1) return 0;
  const size_t segs = !needs_segments(*q) ? 0 : (size_t)q->rows * plan_of(*q).nseg * sizeof(Seg);
  const size_t bias = q->bias && q->bias_ld == 0 ? (size_t)bias_shares(*q) * q->vocab * sizeof(float) : 0;
  return std::max(segs, bias);
}

extern "C" int dvae_rules_apply(const dvae_rules* q, void* out, long long out_ld, void* stream) {
  DVAE_REQUIRE(q, "rules_apply: null pointer");
  DVAE_TRY(rules_check(*q, "rules_apply"));
  if (q->rows == 0) return DVAE_OK;
  DVAE_REQUIRE(out, "rules_apply: null pointer");
  DVAE_REQUIRE(q->rows <= 1 || out_ld >= q->vocab, "rules_apply: rows of out overlap (ld %lld < vocab %d)", out_ld, q->vocab);
  if (is_small(*q)) {
    GroupArgs m{};
    m.q = with_constants(*q); m.out = out; m.out_ld = out_ld;
    return run_group<M_APPLY>(m, group_blocks(*q), (hipStream_t)stream);
  }
  SegArgs a{};
  a.q = with_constants(*q);
  const Plan p = plan_of(*q);
  a.out = out; a.out_ld = out_ld;
  return run_seg<M_APPLY>(a, p, (hipStream_t)stream);
}

extern "C" int dvae_rules_choose(const dvae_rules* q, const float* uniforms, const int* next, long long* tokens,
                                 float* logprob, int* state_out, void* ws, void* stream) {
  DVAE_REQUIRE(q, "rules_choose: null pointer");
  DVAE_TRY(rules_check(*q, "rules_choose"));
  if (q->rows == 0) return DVAE_OK;
  DVAE_REQUIRE(tokens && logprob && (ws || !needs_segments(*q)), "rules_choose: null pointer");
  DVAE_REQUIRE((next == nullptr) == (state_out == nullptr), "rules_choose: next and state_out go together");
  DVAE_REQUIRE(!next || q->mask, "rules_choose: next states need a grammar mask");
  RowOut o{};
  o.uniforms = uniforms; o.next = next; o.tokens = tokens; o.logprob = logprob; o.state_out = state_out;
  hipStream_t st = (hipStream_t)stream;
  if (is_small(*q)) {
    GroupArgs m{};
    m.q = with_constants(*q); m.o = o;
    return uniforms ? run_group<M_DRAW>(m, group_blocks(*q), st) : run_group<M_GREEDY>(m, group_blocks(*q), st);
  }
  SegArgs a{};
  a.q = with_constants(*q); a.o = o; a.seg = (Seg*)ws;
  return uniforms ? run_join<M_DRAW>(a, st) : run_join<M_GREEDY>(a, st);
}

extern "C" int dvae_rules_logprob(const dvae_rules* q, const long long* tokens, float* logprob, double* stat, void* ws,
                                  void* stream) {
  DVAE_REQUIRE(q, "rules_logprob: null pointer");
  DVAE_TRY(rules_check(*q, "rules_logprob"));
  if (q->rows == 0) return DVAE_OK;
  DVAE_REQUIRE(tokens && logprob && stat && (ws || !needs_segments(*q)), "rules_logprob: null pointer");
  RowOut o{};
  o.given = tokens; o.logprob = logprob; o.stat = stat;
  if (is_small(*q)) {
    GroupArgs m{};
    m.q = with_constants(*q); m.o = o;
    return run_group<M_SUM>(m, group_blocks(*q), (hipStream_t)stream);
  }
  SegArgs a{};
  a.q = with_constants(*q); a.o = o; a.seg = (Seg*)ws;
  return run_join<M_SUM>(a, (hipStream_t)stream);
}

extern "C" int dvae_rules_logprob_bwd(const dvae_rules* q, const long long* tokens, const double* stat,
                                      const float* d_logprob, void* d_logits, long long d_ld, float* d_bias, void* ws,
                                      void* stream) {
  DVAE_REQUIRE(q, "rules_logprob_bwd: null pointer");
  DVAE_TRY(rules_check(*q, "rules_logprob_bwd"));
  hipStream_t st = (hipStream_t)stream;
  DVAE_REQUIRE(!d_bias || q->bias, "rules_logprob_bwd: d_bias without a bias");
  const bool shared = d_bias && q->bias_ld == 0;
  if (q->rows == 0) {
    if (shared) hipLaunchKernelGGL(rules_bias_sum_kernel, dim3(cdiv(q->vocab, 16)), dim3(256), 0, st, nullptr, 0, q->vocab,
                                   d_bias);
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
  }
  DVAE_REQUIRE(tokens && stat && d_logprob && (d_logits || d_bias) && (ws || !shared), "rules_logprob_bwd: null pointer");
  DVAE_REQUIRE(!d_logits || q->rows <= 1 || d_ld >= q->vocab, "rules_logprob_bwd: rows of d_logits overlap (ld %lld < vocab %d)", d_ld,
               q->vocab);
  const int shares = bias_shares(*q);
  const auto sum_shares = [&]() -> int {
    hipLaunchKernelGGL(rules_bias_sum_kernel, dim3(cdiv(q->vocab, 16)), dim3(256), 0, st, (const float*)ws, shares, q->vocab,
                       d_bias);
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
  };
  if (is_small(*q)) {
    GroupArgs m{};
    m.q = with_constants(*q); m.o.given = tokens; m.o.stat = const_cast<double*>(stat); m.d_logprob = d_logprob;
    m.out = d_logits; m.out_ld = d_ld; m.d_bias = shared ? nullptr : d_bias; m.part = shared ? (float*)ws : nullptr;
    DVAE_TRY(run_group<M_BWD>(m, shared ? shares : group_blocks(*q), st));
    return shared ? sum_shares() : DVAE_OK;
  }
  const Plan p = plan_of(*q);
  SegArgs a{};
  a.q = with_constants(*q); a.out = d_logits; a.out_ld = d_ld; a.o.given = tokens;
  a.o.stat = const_cast<double*>(stat); a.d_logprob = d_logprob;
  a.d_bias_rows = shared ? nullptr : d_bias;
  if (!shared) return run_seg<M_BWD>(a, p, st);
  ColArgs c{};
  c.s = a;
  c.part = (float*)ws;
  c.rows_per_share = (int)((q->rows + shares - 1) / shares);
  const dim3 grid((unsigned)cdiv(q->vocab, 64 * COL_STEPS * (16 / elem_bytes(q->dtype))), (unsigned)shares);
  const int hist = !q->history || q->history_len == 0 ? 0 : q->history_len < 65536 ? 1 : 2;
#define COL(T)                                                                                              \
  do {                                                                                                      \
    if (hist == 1) hipLaunchKernelGGL((rules_bwd_col_kernel<T, 1>), grid, dim3(256), 0, st, c);             \
    else if (hist) hipLaunchKernelGGL((rules_bwd_col_kernel<T, 2>), grid, dim3(256), 0, st, c);             \
    else hipLaunchKernelGGL((rules_bwd_col_kernel<T, 0>), grid, dim3(256), 0, st, c);                       \
  } while (0)
  switch (q->dtype) {
    case DVAE_F32: COL(DVAE_F32); break;
    case DVAE_BF16: COL(DVAE_BF16); break;
    default: COL(DVAE_F16);
  }
#undef COL
  DVAE_LAUNCH_CHECK();
  return sum_shares();
}
