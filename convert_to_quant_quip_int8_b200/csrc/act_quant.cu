// Producers of quantized activations: plain fp8 quantization, the
// root-mean-square norm of a residual stream, and the gate of a gated
// feed-forward, each straight to 8-bit codes and scales.
//
//   plain  y = x
//   norm   h = round_T(x + residual),  y = h (mean(h^2) + eps)^-1/2 w
//   gated  y = act(gate) up
//   codes  per row or per (row, 128 columns): maximum, scale, rounding
//
// y never leaves the registers, so each input byte is read once and each output
// byte written once: HBM bounds the large cases, launch latency the small ones.
// A lane holds eight neighbouring columns; 16 lanes are one block of 128.
#include <cstdint>

#include "f8.cuh"

namespace qi8 {
namespace {
namespace aq {

struct Args {
  const void *x, *second;  // second: residual, or up; may be null
  const void* weight;
  void *q, *scale, *sum;
  int64_t ld_x, ld_second, ld_q, ld_sum;
  int64_t rows, n, blocks;
  float eps, inv_n;
  int weight_dtype, mode;
  bool vec, vec_weight, vec_q, vec_sum;
  bool whole() const { return n % 8 == 0 && vec && vec_q && (!weight || vec_weight) && (!sum || vec_sum); }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// 2 units in the last place
__device__ __forceinline__ float2 exp2_of(float2 x) {
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(x.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(x.y));
  return e;
}

// x / (1 + 2^m), given m - 7.  Quotient and denominator are taken 2^-7 times, since
// __fdividef returns 0 for denominators above 2^126 while the result is a normal number
// up to m = 132.6: so it is 0 only where it would be none.  (x under 2^-119 loses its
// last bits instead.)  This is coarser than fp32 has to be: m's constant and its value
// are rounded once each, which counts |m| ln 2 times, exp2 and the division are off by
// 2 units each, in all at most (16 + 2 |m| ln 2) 2^-24 of the result: 1.6e-6 at x = -5, 8e-6
// at x = -60, where a code is off by up to 2^-4 (e4m3) or 2^-8 (int8).  A second word of m
// would cost as many instructions as exp2 itself.
constexpr float SWISH_SHIFT = 7.0f, SWISH_SCALE = 0.0078125f;
__device__ __forceinline__ float2 swish(float2 x, float2 m) {
  const float2 e = __fadd2_rn(exp2_of(m), both(SWISH_SCALE));
  x = __fmul2_rn(x, both(SWISH_SCALE));
  return make_float2(__fdividef(x.x, e.x), __fdividef(x.y, e.y));
}

// x Phi(x) = max(x, 0) - |x| h, h = Phi(-|x|) = exp(-x^2 / 2) R(|x|).  R, half the
// scaled complementary error function of |x| / sqrt(2), falls like 1 / |x|: t times a
// polynomial in t = 1 / (1 + 0.27 |x|), fitted here by least squares weighted
// towards the largest relative error, which is 4.2e-8 up to |x| = 10.  In fp32 h is off
// by 6.2e-7 of itself up to |x| = 3 and 7.5e-6 at 12 if exp2 and the division were exact
// (the rounding of x^2 counts x^2 / 2 times), with them by at most (32 + 2 x^2) 2^-24, and
// x Phi(x) by 2e-7 of x.  erff has two cases, of which a warp meets both: 4096 x 10240
// took 58 us with it.
__device__ __forceinline__ float2 gelu(float2 x) {
  const float2 u = make_float2(fabsf(x.x), fabsf(x.y));
  const float2 d = __ffma2_rn(u, both(0.27f), both(1.0f));
  const float2 t = make_float2(__fdividef(1.0f, d.x), __fdividef(1.0f, d.y));
  float2 r = both(0.0288554337f);
  r = __ffma2_rn(r, t, both(-0.125953481f));
  r = __ffma2_rn(r, t, both(0.168642223f));
  r = __ffma2_rn(r, t, both(-0.0678447261f));
  r = __ffma2_rn(r, t, both(0.106836453f));
  r = __ffma2_rn(r, t, both(0.0724932477f));
  r = __ffma2_rn(r, t, both(0.101690575f));
  r = __ffma2_rn(r, t, both(0.107560746f));
  r = __ffma2_rn(r, t, both(0.107719541f));
  const float2 e = exp2_of(__fmul2_rn(__fmul2_rn(u, u), both(-0.72134752f)));  // -log2(e) / 2
  const float2 h = __fmul2_rn(e, __fmul2_rn(r, t));
  return __ffma2_rn(make_float2(-u.x, -u.y), h, make_float2(fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f)));
}

// y = act(g) * up
template <int ACT>
__device__ __forceinline__ F8x gate(const F8x& g, const F8x& up) {
  F8x y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = g.v[i];
    float2 a;
    if constexpr (ACT == QI8_ACT_SILU) {
      a = swish(x, __ffma2_rn(x, both(-1.4426950408889634f), both(-SWISH_SHIFT)));  // -log2(e)
    } else if constexpr (ACT == QI8_ACT_GELU) {
      a = gelu(x);
    } else {
      // 0.5 x (1 + tanh(u)) = x / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3)
      const float2 c = __ffma2_rn(__fmul2_rn(x, x), both(-0.10294324f), both(-2.3022082f));
      a = swish(x, __ffma2_rn(x, c, both(-SWISH_SHIFT)));
    }
    y.v[i] = __fmul2_rn(a, up.v[i]);
  }
  return y;
}

template <typename W, bool WHOLE>
__device__ __forceinline__ F8x weight_as(const Args& p, int64_t col) {
  Eight<W> e;
  const W* w = static_cast<const W*>(p.weight);
  if (WHOLE ? col < p.n : p.vec_weight && col + 8 <= p.n) e.load(w + col);
  else if (WHOLE) e.clear();
  else e.load_some(w, col, p.n);
  return e.get();
}
template <bool WHOLE>
__device__ __forceinline__ F8x load_weight(const Args& p, int64_t col) {
  if (p.weight_dtype == QI8_BF16) return weight_as<__nv_bfloat16, WHOLE>(p, col);
  return p.weight_dtype == QI8_F16 ? weight_as<__half, WHOLE>(p, col) : weight_as<float, WHOLE>(p, col);
}

// What is done to the two inputs of a column before any step over the row.
enum { PLAIN, NORM, GATED_SILU, GATED_GELU, GATED_TANH };

template <typename T, int OP>
__device__ __forceinline__ F8x combine(const Args& p, const Eight<T>& a, const Eight<T>& b) {
  F8x y = a.get();
  if constexpr (OP == NORM) {
    if (p.second) {
      const F8x r = b.get();
#pragma unroll
      for (int i = 0; i < 4; ++i) y.v[i] = __fadd2_rn(y.v[i], r.v[i]);
      if constexpr (sizeof(T) == 2) {
        Eight<T> e;
        e.set(y);
        y = e.get();
      }
    }
  } else if constexpr (OP != PLAIN) {
    y = gate<OP == GATED_SILU ? QI8_ACT_SILU : OP == GATED_GELU ? QI8_ACT_GELU : QI8_ACT_GELU_TANH>(y, b.get());
  }
  return y;
}

// `N` pieces of a row of each input, `step` columns apart, zero past the end: all
// loads are issued before the first is used.
// LATE: rows that are not WHOLE are shifted in get(), which holds twice the registers
// (gates with one scale per row: 2000 x 4099 takes 19 us so and 32 with shifts in
// load(); the norm, whose registers are short, gains nothing).
template <typename T, int OP, int N, bool WHOLE, bool LATE = false>
struct Raw {
  static constexpr bool LOOSE = !WHOLE && LATE;
  std::conditional_t<LOOSE, Loose<T>, Eight<T>> u[N], v[N];

  __device__ __forceinline__ void load(const Args& p, int64_t row, int64_t col, int step) {
    const T* a = static_cast<const T*>(p.x) + row * p.ld_x + col;
    const T* b = static_cast<const T*>(p.second) + row * p.ld_second + col;
    const bool two = OP != PLAIN && p.second;
    const int64_t left = p.n - col;  // columns from the first piece on
    if constexpr (LOOSE) {
#pragma unroll
      for (int i = 0; i < N; ++i) u[i].load(a - col, col + i * step, p.n);
      if (two)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i].load(b - col, col + i * step, p.n);
    } else if constexpr (WHOLE) {
#pragma unroll
      for (int i = 0; i < N; ++i) i * step < left ? u[i].load(a + i * step) : u[i].clear();
      if (two)
#pragma unroll
        for (int i = 0; i < N; ++i) i * step < left ? v[i].load(b + i * step) : v[i].clear();
    } else if (p.vec && (N - 1) * step + 8 <= left) {
#pragma unroll
      for (int i = 0; i < N; ++i) u[i].load(a + i * step);
      if (two)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i].load(b + i * step);
    } else if (!p.vec && col >= 8 && (N - 1) * step + 16 <= left) {
#pragma unroll
      for (int i = 0; i < N; ++i) u[i].load_shifted(a + i * step);
      if (two)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i].load_shifted(b + i * step);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        u[i].load_some(a + i * step, 0, left - i * step);
        if (two) v[i].load_some(b + i * step, 0, left - i * step);
      }
    }
  }
  // of the row that was loaded last
  __device__ __forceinline__ void get(const Args& p, int64_t row, int64_t col, int step, F8x (&y)[N]) const {
    if constexpr (LOOSE) {
      const T* a = static_cast<const T*>(p.x) + row * p.ld_x;
      const T* b = static_cast<const T*>(p.second) + row * p.ld_second;
#pragma unroll
      for (int i = 0; i < N; ++i)
        y[i] = combine<T, OP>(p, u[i].get(a, col + i * step, p.n), v[i].get(b, col + i * step, p.n));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = combine<T, OP>(p, u[i], v[i]);
    }
  }
};
template <typename T, int OP, bool WHOLE, int N>
__device__ __forceinline__ void row_values(const Args& p, int64_t row, int64_t col, int step, F8x (&y)[N]) {
  Raw<T, OP, N, WHOLE> raw;
  raw.load(p, row, col, step);
  raw.get(p, row, col, step, y);
}

template <typename T, bool WHOLE>
__device__ __forceinline__ void store_sum(const Args& p, int64_t row, int64_t col, const F8x& h) {
  Eight<T> e;
  e.set(h);
  T* to = static_cast<T*>(p.sum) + row * p.ld_sum;
  if constexpr (WHOLE) {
    if (col < p.n) e.store(to + col);
  } else {
    e.store_some(to, col, p.n, p.vec_sum);
  }
}

__device__ __forceinline__ float squares(const F8x& h, float ss) {
  float2 s = make_float2(ss, 0.0f);
#pragma unroll
  for (int i = 0; i < 4; ++i) s = __ffma2_rn(h.v[i], h.v[i], s);
  return s.x + s.y;
}
__device__ __forceinline__ F8x normed(const Args& p, F8x h, float rstd, const F8x& w) {
  h = scaled(h, rstd);
  if (p.weight)
#pragma unroll
    for (int i = 0; i < 4; ++i) h.v[i] = __fmul2_rn(h.v[i], w.v[i]);
  return h;
}

// Sums (or maxima) over the `warps` warps of a row, which meet at a barrier of their
// own.  Calls take turns with two sets of words: a set is written again only behind
// the barrier of the call in between.
template <typename V, typename F>
__device__ __forceinline__ V over_row(V v, V* shared, int row_in_block, int warps, F&& f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (warps == 1) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) shared[threadIdx.x >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(row_in_block + 1), "r"(warps * 32) : "memory");
  v = lane < warps ? shared[row_in_block * warps + lane] : V(0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float add_f(float a, float b) { return a + b; }
__device__ __forceinline__ uint32_t max_u(uint32_t a, uint32_t b) { return max(a, b); }

// A row whose squares pass fp32's range is summed again with values 2^-80 of theirs
// (the largest becomes 2^48), one whose squares vanish with 2^95 times its values
// (these are 2^-54 to 2^45 then).  That is looked for where eps does not cover them.
constexpr float SMALLER = 8.271806125530277e-25f;  // 2^-80
constexpr float LARGER = 3.961408125713217e28f;    // 2^95
constexpr float EPS_COVERS = 1e-20f, VANISHED = 7.888609052210118e-31f;  // 2^-100

// What the values of a row with this sum of squares are multiplied by before they are
// squared again; 1: nothing.
__device__ __forceinline__ float again_with(const Args& p, float ss) {
  return isinf(ss) ? SMALLER : ss < VANISHED && p.eps < EPS_COVERS ? LARGER : 1.0f;
}
// 1 / root mean square of values times `factor`
__device__ __forceinline__ float root(const Args& p, float ss, float factor) {
  const float m = fmaf(ss, p.inv_n, p.eps * factor * factor);
  float r = rsqrtf(m);
  if (m > 0.0f && m < 3e38f) r *= fmaf(-0.5f * m * r, r, 1.5f);  // one step of Newton's: half a unit
  return r;
}

// The maxima of neighbouring blocks, two at a time: scale bytes are as good as the
// maxima themselves, and two fit a word.  m: of each chunk's eight columns.
template <int N>
__device__ __forceinline__ void block_codes(const uint32_t (&m)[N], uint32_t (&code)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    uint32_t c = f8_scale_code(m[i]) | (i + 1 < N ? f8_scale_code(m[i + 1 < N ? i + 1 : i]) << 16 : 0u);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, c, o);
      asm("max.u16x2 %0, %0, %1;" : "+r"(c) : "r"(other));
    }
    code[i] = c & 0xffffu;
    if (i + 1 < N) code[i + 1 < N ? i + 1 : i] = c >> 16;
  }
}

// N pieces of a row, `step` columns apart, to codes and scales.  top: the row's
// maximum (QI8_Q_TOKEN).
template <bool WHOLE, int N>
__device__ __forceinline__ void emit_row(const Args& p, const F8x (&y)[N], int64_t row, int64_t col0, int step,
                                         uint32_t top) {
  uint8_t* q = static_cast<uint8_t*>(p.q) + row * p.ld_q;
  if (p.mode == QI8_Q_FP8) {
    uint32_t m[N], code[N];
#pragma unroll
    for (int i = 0; i < N; ++i) m[i] = amax_bits(y[i]);
    block_codes(m, code);
    uint8_t* scale = static_cast<uint8_t*>(p.scale) + row * p.blocks;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t col = col0 + i * step;
      if (col >= p.n) continue;
      store_codes<WHOLE>(q, col, p.n, f8_codes(y[i], f8_inverse(code[i])), p.vec_q);
      if ((threadIdx.x & 15) == 0) scale[col / F8_BLOCK] = (uint8_t)code[i];
    }
  } else {
    float* scale = static_cast<float*>(p.scale) + row * (p.mode == QI8_Q_TOKEN ? 1 : p.blocks);
    float s = 0.0f, inv = 0.0f;
    if (p.mode == QI8_Q_TOKEN) {
      s = i8_scale(top, 1e-30f);
      inv = __frcp_rn(s);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t col = col0 + i * step;
      if (p.mode == QI8_Q_BLOCK) {
        s = i8_scale(max16(amax_bits(y[i])), 1e-8f);
        inv = __frcp_rn(s);
      }
      if (col >= p.n) continue;
      store_codes<WHOLE>(q, col, p.n, i8_codes(y[i], inv), p.vec_q);
      if (p.mode == QI8_Q_TOKEN ? col == 0 : (threadIdx.x & 15) == 0) scale[p.mode == QI8_Q_TOKEN ? 0 : col / F8_BLOCK] = s;
    }
  }
}

// Whole rows in registers: `warps` warps hold one, eight columns per lane and
// chunk, and a thread block holds as many rows as fit.  Blocks stay and go on to
// other rows, whose loads are under way while these are reduced and stored: 4096 x
// 4096 bf16 with a residual takes 21.6 us so (5.4 TB/s), 27 with a block for each row.
constexpr int ROW_THREADS = 512;

template <typename T, int OP, int CHUNKS, bool WHOLE>
__global__ void __launch_bounds__(ROW_THREADS) row_kernel(const __grid_constant__ Args p, const int warps) {
  __shared__ float sums[2][32], again[2][32];
  __shared__ uint32_t tops[2][32];
  const int mine = (threadIdx.x >> 5) / warps, step = warps * 256;
  const int64_t col0 = (threadIdx.x - mine * warps * 32) * 8, per = (blockDim.x >> 5) / warps;
  const int64_t stride = gridDim.x * per;
  int64_t row = blockIdx.x * per + mine;
  wait_for_last_kernel();
  if (row >= p.rows) return;
  constexpr bool LATE = OP != NORM;
  Raw<T, OP, CHUNKS, WHOLE, LATE> raw;
  if (WHOLE || !LATE) raw.load(p, row, col0, step);
  F8x w[CHUNKS];
  if (OP == NORM && p.weight)
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) w[c] = load_weight<WHOLE>(p, col0 + c * step);
  for (int turn = 0; row < p.rows; row += stride, turn ^= 1) {
    F8x y[CHUNKS];
    if (!WHOLE && LATE) raw.load(p, row, col0, step);
    raw.get(p, row, col0, step, y);
    if ((WHOLE || !LATE) && row + stride < p.rows) raw.load(p, row + stride, col0, step);
    if constexpr (OP == NORM) {
      float ss = 0.0f;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) ss = squares(y[c], ss);
      if (p.sum)
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) store_sum<T, WHOLE>(p, row, col0 + c * step, y[c]);
      ss = over_row(ss, sums[turn], mine, warps, add_f);
      const float factor = again_with(p, ss);
      if (factor != 1.0f) {  // the whole row
        ss = 0.0f;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          y[c] = scaled(y[c], factor);
          ss = squares(y[c], ss);
        }
        ss = over_row(ss, again[turn], mine, warps, add_f);
      }
      const float rstd = root(p, ss, factor);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) y[c] = normed(p, y[c], rstd, w[c]);
    }
    uint32_t top = 0;
    if (p.mode == QI8_Q_TOKEN) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) top = max(top, amax_bits(y[c]));
      top = over_row(top, tops[turn], mine, warps, max_u);
    }
    emit_row<WHOLE>(p, y, row, col0, step, top);
  }
}

// Rows too long for that are read again for each step (from L2, mostly).
constexpr int LONG_THREADS = 1024;

template <typename T, int OP>
__global__ void __launch_bounds__(LONG_THREADS) long_row_kernel(const __grid_constant__ Args p) {
  __shared__ float sums[32], again[32];
  __shared__ uint32_t tops[32];
  constexpr int STEP = LONG_THREADS * 8;
  const int64_t row = blockIdx.x, col0 = threadIdx.x * 8;
  wait_for_last_kernel();
  float factor = 1.0f, rstd = 1.0f;
  F8x y[1];
  if constexpr (OP == NORM) {
    float ss = 0.0f;
    for (int64_t col = col0; col < p.n; col += STEP) {
      row_values<T, OP, false>(p, row, col, STEP, y);
      ss = squares(y[0], ss);
      if (p.sum) store_sum<T, false>(p, row, col, y[0]);
    }
    ss = over_row(ss, sums, 0, LONG_THREADS / 32, add_f);
    factor = again_with(p, ss);  // the same for all threads
    if (factor != 1.0f) {
      ss = 0.0f;
      for (int64_t col = col0; col < p.n; col += STEP) {
        row_values<T, OP, false>(p, row, col, STEP, y);
        ss = squares(scaled(y[0], factor), ss);
      }
      ss = over_row(ss, again, 0, LONG_THREADS / 32, add_f);
    }
    rstd = root(p, ss, factor);
  }
  auto final_values = [&](int64_t col) {
    row_values<T, OP, false>(p, row, col, STEP, y);
    if constexpr (OP == NORM) {
      F8x w;
      if (p.weight) w = load_weight<false>(p, col);
      y[0] = normed(p, scaled(y[0], factor), rstd, w);
    }
  };
  uint32_t m = 0;
  if (p.mode == QI8_Q_TOKEN) {
    for (int64_t col = col0; col < p.n; col += STEP) {
      final_values(col);
      m = max(m, amax_bits(y[0]));
    }
    m = over_row(m, tops, 0, LONG_THREADS / 32, max_u);
  }
  for (int64_t first = 0; first < p.n; first += STEP) {  // the warp's lanes together
    const int64_t col = first + col0;
    if (col < p.n) final_values(col);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i) y[0].v[i] = make_float2(0.0f, 0.0f);
    emit_row<false>(p, y, row, col, 0, m);
  }
}

// No step over whole rows: 16 lanes per block of 128 columns.  A warp takes 2 *
// STEPS neighbouring blocks of one row.
constexpr int THREADS = 256;

template <typename T, int OP, int STEPS, bool WHOLE>
__global__ void __launch_bounds__(THREADS) block_kernel(const __grid_constant__ Args p, const unsigned groups) {
  const int lane = threadIdx.x & 31;
  const unsigned unit = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  const unsigned row = unit / groups;
  if (row >= p.rows) return;
  const int64_t col0 = (int64_t)(unit - row * groups) * (STEPS * 256) + lane * 8;
  wait_for_last_kernel();
  F8x y[STEPS];
  row_values<T, OP, WHOLE>(p, row, col0, 256, y);
  emit_row<WHOLE>(p, y, row, col0, 256, 0);
}

template <typename T, int OP, int STEPS>
int launch_blocks(const Args& p, cudaStream_t st) {
  const int64_t groups = (p.blocks + 2 * STEPS - 1) / (2 * STEPS), units = p.rows * groups;
  QI8_REQUIRE(units < (1ll << 32) - THREADS, QI8_ESHAPE, "%lld rows of %lld", (long long)p.rows, (long long)p.n);
  const dim3 grid((unsigned)((units + THREADS / 32 - 1) / (THREADS / 32)));
  return launch_early("block_kernel launch",
                      p.whole() ? block_kernel<T, OP, STEPS, true> : block_kernel<T, OP, STEPS, false>, grid, THREADS, 0, 1,
                      st, p, (unsigned)groups);
}

template <typename T, int OP, int CHUNKS>
int launch_rows(const Args& p, cudaStream_t st) {
  const int warps = (int)((p.n + 256 * CHUNKS - 1) / (256 * CHUNKS));
  const int per = warps >= 8 ? 1 : 8 / warps;  // rows per thread block
  const bool whole = p.whole();
  auto kern = whole ? row_kernel<T, OP, CHUNKS, true> : row_kernel<T, OP, CHUNKS, false>;
  static int resident[2][64][ROW_THREADS / 32 + 1];  // blocks per SM, by device and warps
  int dev = 0, blocks = 0;
  QI8_CUDA(cudaGetDevice(&dev));
  if (dev < 64) blocks = resident[whole][dev][warps * per];
  if (blocks == 0) {
    QI8_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kern, warps * per * 32, 0));
    if (dev < 64) resident[whole][dev][warps * per] = blocks;
  }
  const int64_t groups = (p.rows + per - 1) / per, most = (int64_t)blocks * sm_count();
  return launch_early("row_kernel launch", kern, dim3((unsigned)(groups < most ? groups : most)), warps * per * 32, 0, 1, st,
                      p, warps);
}

template <typename T, int OP>
int launch_type(const Args& p, cudaStream_t st) {
  if constexpr (OP != NORM) {
    if (p.mode != QI8_Q_TOKEN)
      // Two steps per warp from 4096 blocks of 128 columns on: 4096 x 10240 SiLU takes 39.7
      // us so and 41.1 with one, GELU 45.0 and 51.4, 16 x 10240 1.54 and 1.47.
      return p.rows * p.blocks < 4096 ? launch_blocks<T, OP, 1>(p, st) : launch_blocks<T, OP, 2>(p, st);
  }
  if constexpr (OP != PLAIN) {
    // Two chunks per lane from 2048 columns on (4096 x 2048 takes the same either way,
    // 4096 x 4096 gains 4 %, 8192 x 256 would take twice as long); four need the registers
    // of half as many blocks: only where two do not reach.
    if (p.n <= 2048) return launch_rows<T, OP, 1>(p, st);
    if (p.n <= 8192) return launch_rows<T, OP, 2>(p, st);
    if constexpr (sizeof(T) == 2)
      if (p.n <= 16384) return launch_rows<T, OP, 4>(p, st);
    return launch_early("long_row_kernel launch", long_row_kernel<T, OP>, dim3((unsigned)p.rows), LONG_THREADS, 0, 1, st,
                        p);
  }
  return QI8_OK;
}

template <int OP>
int launch(const Args& p, int dtype, cudaStream_t st) {
  if (p.rows == 0 || p.n == 0) return QI8_OK;
  QI8_REQUIRE(p.rows < (1ll << 31) && p.n < (1ll << 31), QI8_ESHAPE, "%lld rows of %lld", (long long)p.rows,
              (long long)p.n);
  switch (dtype) {
    case QI8_BF16: return launch_type<__nv_bfloat16, OP>(p, st);
    case QI8_F16: return launch_type<__half, OP>(p, st);
    default: return launch_type<float, OP>(p, st);
  }
}

bool is_float(int dtype) { return dtype == QI8_BF16 || dtype == QI8_F16 || dtype == QI8_F32; }

}  // namespace aq
}  // namespace

using namespace aq;

int quant_rows_f8(const void* x, int x_dtype, int64_t rows, int64_t n, int64_t ld_x, uint8_t* q, int64_t ld_q,
                  uint8_t* scale, cudaStream_t st) {
  Args p{};
  p.x = x;
  p.ld_x = ld_x;
  p.q = q;
  p.ld_q = ld_q;
  p.scale = scale;
  p.rows = rows;
  p.n = n;
  p.blocks = f8_blocks(n);
  p.mode = QI8_Q_FP8;
  p.vec = rows_aligned(x, ld_x, elem_size(x_dtype), 16);
  p.vec_q = rows_aligned(q, ld_q, 1, 8);
  return launch<PLAIN>(p, x_dtype, st);
}

}  // namespace qi8

using namespace qi8;

extern "C" int qi8_quant_rows_f8(const void* x, int x_dtype, int64_t rows, int64_t n, int64_t ld_x, uint8_t* q_out,
                                 int64_t ld_q, uint8_t* scale_out, void* stream) {
  QI8_REQUIRE(device_ok(), QI8_EUNSUPPORTED, "no sm_100 device current");
  QI8_REQUIRE(aq::is_float(x_dtype), QI8_EDTYPE, "input dtype %d: bf16, f16 or f32", x_dtype);
  QI8_REQUIRE(rows >= 0 && n >= 0 && ld_x >= n && ld_q >= n, QI8_ESHAPE, "%lld rows of %lld, row strides %lld and %lld",
              (long long)rows, (long long)n, (long long)ld_x, (long long)ld_q);
  if (rows == 0 || n == 0) return QI8_OK;
  QI8_REQUIRE(x && q_out && scale_out, QI8_EINVAL, "null pointer");
  return quant_rows_f8(x, x_dtype, rows, n, ld_x, q_out, ld_q, scale_out, static_cast<cudaStream_t>(stream));
}

// What the two producers with a choice of output check alike.
static int check_output(int dtype, int64_t rows, int64_t n, int mode, int64_t ld_q) {
  QI8_REQUIRE(device_ok(), QI8_EUNSUPPORTED, "no sm_100 device current");
  QI8_REQUIRE(aq::is_float(dtype), QI8_EDTYPE, "input dtype %d: bf16, f16 or f32", dtype);
  QI8_REQUIRE(mode == QI8_Q_TOKEN || mode == QI8_Q_BLOCK || mode == QI8_Q_FP8, QI8_EINVAL, "output mode %d", mode);
  QI8_REQUIRE(rows >= 0 && n >= 0 && ld_q >= n, QI8_ESHAPE, "%lld rows of %lld, row stride of the codes %lld",
              (long long)rows, (long long)n, (long long)ld_q);
  QI8_REQUIRE(mode != QI8_Q_BLOCK || n % F8_BLOCK == 0, QI8_ESHAPE,
              "Last dimension must be divisible by block_size=%d, got %lld", F8_BLOCK, (long long)n);
  return QI8_OK;
}

extern "C" int qi8_rms_norm_quant(const void* x, int x_dtype, int64_t rows, int64_t n, int64_t ld_x,
                                  const void* residual, int64_t ld_residual, const void* weight, int weight_dtype,
                                  double eps, int mode, void* q_out, int64_t ld_q, void* scale_out, void* sum_out,
                                  int64_t ld_sum, void* stream) {
  if (int rc = check_output(x_dtype, rows, n, mode, ld_q)) return rc;
  QI8_REQUIRE(ld_x >= n && (!residual || ld_residual >= n) && (!sum_out || ld_sum >= n), QI8_ESHAPE,
              "row strides %lld, %lld and %lld for rows of %lld", (long long)ld_x, (long long)ld_residual,
              (long long)ld_sum, (long long)n);
  QI8_REQUIRE(eps == 0.0 || (eps >= 1e-37 && eps < 1e30), QI8_EINVAL, "eps %g: 0, or from 1e-37 to 1e30", eps);
  QI8_REQUIRE(!weight || aq::is_float(weight_dtype), QI8_EDTYPE, "weight dtype %d: bf16, f16 or f32", weight_dtype);
  if (rows == 0 || n == 0) return QI8_OK;
  QI8_REQUIRE(x && q_out && scale_out, QI8_EINVAL, "null pointer");
  const int size = elem_size(x_dtype);
  aq::Args p{};
  p.x = x;
  p.ld_x = ld_x;
  p.second = residual;
  p.ld_second = ld_residual;
  p.weight = weight;
  p.weight_dtype = weight_dtype;
  p.q = q_out;
  p.ld_q = ld_q;
  p.scale = scale_out;
  p.sum = sum_out;
  p.ld_sum = ld_sum;
  p.rows = rows;
  p.n = n;
  p.blocks = f8_blocks(n);
  p.eps = (float)eps;
  p.inv_n = (float)(1.0 / (double)n);
  p.mode = mode;
  p.vec = rows_aligned(x, ld_x, size, 16) && (!residual || rows_aligned(residual, ld_residual, size, 16));
  p.vec_weight = aligned16(weight);
  p.vec_q = rows_aligned(q_out, ld_q, 1, 8);
  p.vec_sum = sum_out && rows_aligned(sum_out, ld_sum, size, 16);
  return aq::launch<aq::NORM>(p, x_dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int qi8_gated_quant(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, int dtype, int64_t rows,
                               int64_t n, int act, int mode, void* q_out, int64_t ld_q, void* scale_out, void* stream) {
  if (int rc = check_output(dtype, rows, n, mode, ld_q)) return rc;
  QI8_REQUIRE(ld_gate >= n && ld_up >= n, QI8_ESHAPE, "row strides %lld and %lld for rows of %lld", (long long)ld_gate,
              (long long)ld_up, (long long)n);
  QI8_REQUIRE(act == QI8_ACT_SILU || act == QI8_ACT_GELU || act == QI8_ACT_GELU_TANH, QI8_EINVAL, "activation %d", act);
  if (rows == 0 || n == 0) return QI8_OK;
  QI8_REQUIRE(gate && up && q_out && scale_out, QI8_EINVAL, "null pointer");
  const int size = elem_size(dtype);
  aq::Args p{};
  p.x = gate;
  p.ld_x = ld_gate;
  p.second = up;
  p.ld_second = ld_up;
  p.q = q_out;
  p.ld_q = ld_q;
  p.scale = scale_out;
  p.rows = rows;
  p.n = n;
  p.blocks = f8_blocks(n);
  p.mode = mode;
  p.vec = rows_aligned(gate, ld_gate, size, 16) && rows_aligned(up, ld_up, size, 16);
  p.vec_q = rows_aligned(q_out, ld_q, 1, 8);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return act == QI8_ACT_SILU ? aq::launch<aq::GATED_SILU>(p, dtype, st)
         : act == QI8_ACT_GELU ? aq::launch<aq::GATED_GELU>(p, dtype, st) : aq::launch<aq::GATED_TANH>(p, dtype, st);
}
