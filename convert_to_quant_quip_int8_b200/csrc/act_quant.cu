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
  float eps;
  int weight_dtype, mode;
  bool vec, vec_weight, vec_q, vec_sum;
};

// x 2^t / (1 + 2^t) ... as x / (1 + 2^-t): 0 where 2^-t passes fp32, as it should be
// (MUFU's exp2 and reciprocal: 2 and 1 units in the last place)
__device__ __forceinline__ float2 swish(float2 x, float2 minus_t) {
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(minus_t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(minus_t.y));
  e = __fadd2_rn(e, make_float2(1.0f, 1.0f));
  return make_float2(__fdividef(x.x, e.x), __fdividef(x.y, e.y));
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// y = act(g) * up
template <int ACT>
__device__ __forceinline__ F8x gate(const F8x& g, const F8x& up) {
  F8x y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = g.v[i];
    float2 a;
    if constexpr (ACT == QI8_ACT_SILU) {
      a = swish(x, __fmul2_rn(x, both(-1.4426950408889634f)));  // -log2(e)
    } else if constexpr (ACT == QI8_ACT_GELU) {
      a = make_float2(gelu_erf(x.x), gelu_erf(x.y));
    } else {
      // 0.5 x (1 + tanh(u)) = x / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3)
      const float2 c = __ffma2_rn(__fmul2_rn(x, x), both(-0.10294324f), both(-2.3022082f));
      a = swish(x, __fmul2_rn(x, c));
    }
    y.v[i] = __fmul2_rn(a, up.v[i]);
  }
  return y;
}

// A block of columns to codes and a scale; m: the maximum of what shares the
// scale, as bits.  `first`: this lane writes the scale at index s.
__device__ __forceinline__ void emit(const Args& p, const F8x& y, uint32_t m, int64_t row, int64_t col, bool first,
                                     int64_t s) {
  uint8_t* q = static_cast<uint8_t*>(p.q) + row * p.ld_q;
  if (p.mode == QI8_Q_FP8) {
    const uint32_t code = f8_scale_code(m);
    store_codes(q, col, p.n, f8_codes(y, f8_inverse(code)), p.vec_q);
    if (first) static_cast<uint8_t*>(p.scale)[s] = (uint8_t)code;
  } else {
    const float sc = i8_scale(m, p.mode == QI8_Q_BLOCK ? 1e-8f : 1e-30f);
    store_codes(q, col, p.n, i8_codes(y, __frcp_rn(sc)), p.vec_q);
    if (first) static_cast<float*>(p.scale)[s] = sc;
  }
}

template <typename W>
__device__ __forceinline__ F8x weight_as(const Args& p, int64_t col) {
  Eight<W> e;
  const W* w = static_cast<const W*>(p.weight);
  if (p.vec_weight && col + 8 <= p.n) e.load(w + col);
  else e.load_some(w, col, p.n);
  return e.get();
}
__device__ __forceinline__ F8x load_weight(const Args& p, int64_t col) {
  if (p.weight_dtype == QI8_BF16) return weight_as<__nv_bfloat16>(p, col);
  return p.weight_dtype == QI8_F16 ? weight_as<__half>(p, col) : weight_as<float>(p, col);
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

// `N` pieces of a row, `step` columns apart, zero past the end: all loads are
// issued before the first is used.
template <typename T, int OP, int N>
__device__ __forceinline__ void row_values(const Args& p, int64_t row, int64_t col, int step, F8x (&y)[N]) {
  const T* a = static_cast<const T*>(p.x) + row * p.ld_x;
  const T* b = static_cast<const T*>(p.second) + row * p.ld_second;
  const bool two = OP != PLAIN && p.second;
  Eight<T> u[N], v[N];
  if (p.vec && col + (N - 1) * step + 8 <= p.n) {
#pragma unroll
    for (int i = 0; i < N; ++i) u[i].load(a + col + i * step);
    if (two)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i].load(b + col + i * step);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      u[i].load_some(a, col + i * step, p.n);
      if (two) v[i].load_some(b, col + i * step, p.n);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = combine<T, OP>(p, u[i], v[i]);
}

template <typename T>
__device__ __forceinline__ void store_sum(const Args& p, int64_t row, int64_t col, const F8x& h) {
  Eight<T> e;
  e.set(h);
  e.store(static_cast<T*>(p.sum) + row * p.ld_sum, col, p.n, p.vec_sum);
}

__device__ __forceinline__ float squares(const F8x& h, float ss, float by) {
  float2 s = make_float2(ss, 0.0f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __fmul2_rn(h.v[i], both(by));
    s = __ffma2_rn(t, t, s);
  }
  return s.x + s.y;
}
__device__ __forceinline__ F8x normed(const Args& p, F8x h, float rstd, const F8x& w) {
  h = scaled(h, rstd);
  if (p.weight)
#pragma unroll
    for (int i = 0; i < 4; ++i) h.v[i] = __fmul2_rn(h.v[i], w.v[i]);
  return h;
}

// Sums (or maxima) over the `warps` warps of a row.  Each call takes shared words
// of its own, so that none waits for the reads of the one before.
template <typename V, typename F>
__device__ __forceinline__ V over_row(V v, V* shared, int first_warp, int warps, F&& f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (warps == 1) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) shared[warp] = v;
  __syncthreads();
  v = shared[first_warp + (lane < warps ? lane : 0)];
  V rest = lane < warps ? v : V(0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) rest = f(rest, __shfl_xor_sync(0xffffffffu, rest, o));
  return rest;
}
__device__ __forceinline__ float add_f(float a, float b) { return a + b; }
__device__ __forceinline__ uint32_t max_u(uint32_t a, uint32_t b) { return max(a, b); }

// A row whose squares pass fp32's range is summed again with values 2^-80 of
// theirs: the largest becomes 2^48.
constexpr float SMALLER = 8.271806125530277e-25f;  // 2^-80

__device__ __forceinline__ float root(const Args& p, float ss, bool smaller) {
  if (smaller) return __frsqrt_rn(__fdiv_rn(ss, (float)p.n)) * SMALLER;  // eps would vanish beside it
  return __frsqrt_rn(__fdiv_rn(ss, (float)p.n) + p.eps);
}

// Whole rows in registers: `warps` warps hold one, eight columns per lane and
// chunk, and a thread block holds as many rows as fit.
constexpr int ROW_THREADS = 512;

template <typename T, int OP, int CHUNKS>
__global__ void __launch_bounds__(ROW_THREADS) row_kernel(const __grid_constant__ Args p, const int warps) {
  __shared__ float sums[2][32];
  __shared__ uint32_t tops[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mine = warp / warps, first_warp = mine * warps, step = warps * 256;
  const int t = threadIdx.x - first_warp * 32;
  const int64_t col0 = t * 8, per = (blockDim.x >> 5) / warps;
  int64_t row = blockIdx.x * per + mine;
  const bool live = row < p.rows;
  if (!live) row = p.rows - 1;  // takes part in the barriers
  wait_for_last_kernel();
  F8x y[CHUNKS];
  row_values<T, OP>(p, row, col0, step, y);
  if constexpr (OP == NORM) {
    F8x w[CHUNKS];  // loads that wait behind the reduction's barrier
    if (p.weight)
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) w[c] = load_weight(p, col0 + c * step);
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) ss = squares(y[c], ss, 1.0f);
    if (p.sum && live)
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) store_sum<T>(p, row, col0 + c * step, y[c]);
    ss = over_row(ss, sums[0], first_warp, warps, add_f);
    const bool smaller = isinf(ss);
    if (__syncthreads_or(smaller)) {
      float s2 = 0.0f;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) s2 = squares(y[c], s2, SMALLER);
      s2 = over_row(s2, sums[1], first_warp, warps, add_f);
      if (smaller) ss = s2;
    }
    const float rstd = root(p, ss, smaller);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) y[c] = normed(p, y[c], rstd, w[c]);
  }
  uint32_t m = 0;
  if (p.mode == QI8_Q_TOKEN) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) m = max(m, amax_bits(y[c]));
    m = over_row(m, tops, first_warp, warps, max_u);
  }
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int64_t col = col0 + c * step;
    const uint32_t top = p.mode == QI8_Q_TOKEN ? m : max16(amax_bits(y[c]));
    if (!live || col >= p.n) continue;
    if (p.mode == QI8_Q_TOKEN) emit(p, y[c], top, row, col, c == 0 && t == 0, row);
    else emit(p, y[c], top, row, col, (lane & 15) == 0, row * p.blocks + col / F8_BLOCK);
  }
}

// Rows too long for that are read again for each step (from L2, mostly).
constexpr int LONG_THREADS = 1024;

template <typename T, int OP>
__global__ void __launch_bounds__(LONG_THREADS) long_row_kernel(const __grid_constant__ Args p) {
  __shared__ float sums[2][32];
  __shared__ uint32_t tops[32];
  constexpr int STEP = LONG_THREADS * 8;
  const int64_t row = blockIdx.x, col0 = threadIdx.x * 8;
  wait_for_last_kernel();
  float rstd = 1.0f;
  F8x y[1];
  if constexpr (OP == NORM) {
    float ss = 0.0f;
    for (int64_t col = col0; col < p.n; col += STEP) {
      row_values<T, OP>(p, row, col, STEP, y);
      ss = squares(y[0], ss, 1.0f);
      if (p.sum) store_sum<T>(p, row, col, y[0]);
    }
    ss = over_row(ss, sums[0], 0, LONG_THREADS / 32, add_f);
    const bool smaller = isinf(ss);  // the same for all threads
    if (smaller) {
      ss = 0.0f;
      for (int64_t col = col0; col < p.n; col += STEP) {
        row_values<T, OP>(p, row, col, STEP, y);
        ss = squares(y[0], ss, SMALLER);
      }
      ss = over_row(ss, sums[1], 0, LONG_THREADS / 32, add_f);
    }
    rstd = root(p, ss, smaller);
  }
  auto final_values = [&](int64_t col) {
    row_values<T, OP>(p, row, col, STEP, y);
    if constexpr (OP == NORM) {
      F8x w;
      if (p.weight) w = load_weight(p, col);
      y[0] = normed(p, y[0], rstd, w);
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
    const uint32_t top = p.mode == QI8_Q_TOKEN ? m : max16(col < p.n ? amax_bits(y[0]) : 0);
    if (col >= p.n) continue;
    if (p.mode == QI8_Q_TOKEN) emit(p, y[0], top, row, col, col == 0, row);
    else emit(p, y[0], top, row, col, (threadIdx.x & 15) == 0, row * p.blocks + col / F8_BLOCK);
  }
}

// No step over whole rows: 16 lanes per block of 128 columns.  A warp takes 2 *
// STEPS neighbouring blocks of one row.
constexpr int THREADS = 256;

template <typename T, int OP, int STEPS>
__global__ void __launch_bounds__(THREADS) block_kernel(const __grid_constant__ Args p, const unsigned groups) {
  const int lane = threadIdx.x & 31;
  const unsigned unit = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  const unsigned row = unit / groups;
  if (row >= p.rows) return;
  const int64_t col0 = (int64_t)(unit - row * groups) * (STEPS * 256) + lane * 8;
  wait_for_last_kernel();
  F8x y[STEPS];
  row_values<T, OP>(p, row, col0, 256, y);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int64_t col = col0 + i * 256;
    const uint32_t top = max16(amax_bits(y[i]));
    if (col < p.n) emit(p, y[i], top, row, col, (lane & 15) == 0, row * p.blocks + col / F8_BLOCK);
  }
}

template <typename T, int OP, int STEPS>
int launch_blocks(const Args& p, cudaStream_t st) {
  const int64_t groups = (p.blocks + 2 * STEPS - 1) / (2 * STEPS), units = p.rows * groups;
  QI8_REQUIRE(units < (1ll << 32) - THREADS, QI8_ESHAPE, "%lld rows of %lld", (long long)p.rows, (long long)p.n);
  return launch_early("block_kernel launch", block_kernel<T, OP, STEPS>,
                      dim3((unsigned)((units + THREADS / 32 - 1) / (THREADS / 32))), THREADS, 0, 1, st, p,
                      (unsigned)groups);
}

template <typename T, int OP, int CHUNKS>
int launch_rows(const Args& p, cudaStream_t st) {
  const int warps = (int)((p.n + 256 * CHUNKS - 1) / (256 * CHUNKS));
  const int per = warps >= 8 ? 1 : 8 / warps;  // rows per thread block
  return launch_early("row_kernel launch", row_kernel<T, OP, CHUNKS>, dim3((unsigned)((p.rows + per - 1) / per)),
                      warps * per * 32, 0, 1, st, p, warps);
}

template <typename T, int OP>
int launch_type(const Args& p, cudaStream_t st) {
  if constexpr (OP != NORM) {
    // few units: one step each spreads them over more SMs
    if (p.mode != QI8_Q_TOKEN)
      return p.blocks < 4 || p.rows * p.blocks < 4 * 8 * 148 * 4 ? launch_blocks<T, OP, 1>(p, st)
                                                                 : launch_blocks<T, OP, 2>(p, st);
  }
  if constexpr (OP != PLAIN) {
    if (p.n <= 1024) return launch_rows<T, OP, 1>(p, st);
    if (p.n <= 8192) return launch_rows<T, OP, 2>(p, st);
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
  QI8_REQUIRE(eps >= 0.0 && eps < 1e30, QI8_EINVAL, "eps %g", eps);
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
