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
  double eps;
  int weight_dtype, act, mode;
  bool vec, vec_weight, vec_q, vec_sum;
};

// g / (1 + exp(-t)).  An exp beyond fp32 makes it 0, as it should be.
__device__ __forceinline__ float swish(float g, float t) { return __fdividef(g, 1.0f + expf(-t)); }

// One activation for eight columns: y = act(y) * up
__device__ __forceinline__ void gate(float (&y)[8], const float (&up)[8], int act) {
  if (act == QI8_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = swish(y[i], y[i]) * up[i];
  } else if (act == QI8_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = gelu_erf(y[i]) * up[i];
  } else {
    // 0.5 g (1 + tanh(u)) = g / (1 + exp(-2 u)), u = sqrt(2 / pi) (g + 0.044715 g^3)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = swish(y[i], 1.5957691216057308f * fmaf(0.044715f * y[i] * y[i], y[i], y[i])) * up[i];
  }
}

// A block of columns to codes and a scale; m: the maximum of what shares the
// scale, as bits.  `first`: this lane writes the scale at index s.
__device__ __forceinline__ void emit(const Args& p, const float (&y)[8], uint32_t m, int64_t row, int64_t col, bool first,
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

__device__ __forceinline__ void load_weight(const Args& p, int64_t col, float (&w)[8]) {
  if (p.weight_dtype == QI8_F32) {
    Eight<float> e;
    e.load(static_cast<const float*>(p.weight), col, p.n, p.vec_weight);
    e.get(w);
  } else if (p.weight_dtype == QI8_BF16) {
    Eight<__nv_bfloat16> e;
    e.load(static_cast<const __nv_bfloat16*>(p.weight), col, p.n, p.vec_weight);
    e.get(w);
  } else {
    Eight<__half> e;
    e.load(static_cast<const __half*>(p.weight), col, p.n, p.vec_weight);
    e.get(w);
  }
}

// Eight columns' worth of y before the norm's factor (norm: h), zero past the end.
template <typename T, bool NORM>
__device__ __forceinline__ void row_values(const Args& p, int64_t row, int64_t col, float (&y)[8]) {
  Eight<T> e, f;
  e.load(static_cast<const T*>(p.x) + row * p.ld_x, col, p.n, p.vec);
  if (p.second) f.load(static_cast<const T*>(p.second) + row * p.ld_second, col, p.n, p.vec);
  e.get(y);
  if (p.second) {
    float b[8];
    f.get(b);
    if constexpr (NORM) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = Elem<T>::to_f32(Elem<T>::from_f32(y[i] + b[i]));
    } else {
      gate(y, b, p.act);
    }
  }
}

template <typename T>
__device__ __forceinline__ void store_sum(const Args& p, int64_t row, int64_t col, const float (&h)[8]) {
  Eight<T> e;
  e.set(h);
  e.store(static_cast<T*>(p.sum) + row * p.ld_sum, col, p.n, p.vec_sum);
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

__device__ __forceinline__ float root(float ss, bool smaller, const Args& p) {
  const double sum = smaller ? (double)ss * 0x1p160 : (double)ss;
  return (float)(1.0 / sqrt(sum / (double)p.n + p.eps));
}

// Whole rows in registers: `warps` warps hold one, eight columns per lane and
// chunk, and a thread block holds as many rows as fit.
template <typename T, bool NORM, int CHUNKS>
__global__ void __launch_bounds__(1024) row_kernel(const __grid_constant__ Args p, const int warps) {
  __shared__ float sums[2][32];
  __shared__ uint32_t tops[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mine = warp / warps, first_warp = mine * warps, threads = warps * 32;
  const int t = threadIdx.x - first_warp * 32;
  const int64_t per = (blockDim.x >> 5) / warps;
  int64_t row = blockIdx.x * per + mine;
  const bool live = row < p.rows;
  if (!live) row = p.rows - 1;  // takes part in the barriers
  float y[CHUNKS][8], w[8];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) row_values<T, NORM>(p, row, (int64_t)(c * threads + t) * 8, y[c]);
  // the weight's latency behind the reduction's, where registers allow
  if (NORM && CHUNKS == 1 && p.weight) load_weight(p, (int64_t)t * 8, w);
  if constexpr (NORM) {
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(y[c][j], y[c][j], ss);
    if (p.sum && live)
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) store_sum<T>(p, row, (int64_t)(c * threads + t) * 8, y[c]);
    ss = over_row(ss, sums[0], first_warp, warps, add_f);
    bool smaller = isinf(ss);
    if (__syncthreads_or(smaller)) {
      float s2 = 0.0f;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) s2 = fmaf(y[c][j] * SMALLER, y[c][j] * SMALLER, s2);
      s2 = over_row(s2, sums[1], first_warp, warps, add_f);
      if (smaller) ss = s2;
    }
    const float rstd = root(ss, smaller, p);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (CHUNKS > 1 && p.weight) load_weight(p, (int64_t)(c * threads + t) * 8, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[c][j] = p.weight ? y[c][j] * rstd * w[j] : y[c][j] * rstd;
    }
  }
  uint32_t m = 0;
  if (p.mode == QI8_Q_TOKEN) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) m = max(m, amax_bits(y[c]));
    m = over_row(m, tops, first_warp, warps, max_u);
  }
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int64_t col = (int64_t)(c * threads + t) * 8;
    const uint32_t top = p.mode == QI8_Q_TOKEN ? m : max16(amax_bits(y[c]));
    if (!live || col >= p.n) continue;
    if (p.mode == QI8_Q_TOKEN) emit(p, y[c], top, row, col, c == 0 && t == 0, row);
    else emit(p, y[c], top, row, col, (lane & 15) == 0, row * p.blocks + col / F8_BLOCK);
  }
}

// Rows too long for that are read again for each step (from L2, mostly).
constexpr int LONG_THREADS = 1024;

template <typename T, bool NORM>
__global__ void __launch_bounds__(LONG_THREADS) long_row_kernel(const __grid_constant__ Args p) {
  __shared__ float sums[2][32];
  __shared__ uint32_t tops[32];
  const int64_t row = blockIdx.x, end = (p.n + 127) / 128 * 128;  // whole half warps
  const int64_t col0 = threadIdx.x * 8, step = LONG_THREADS * 8;
  float rstd = 1.0f;
  if constexpr (NORM) {
    bool smaller = false;
    float ss = 0.0f;
    for (int64_t col = col0; col < end; col += step) {
      float y[8];
      row_values<T, NORM>(p, row, col, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(y[j], y[j], ss);
      if (p.sum && col < p.n) store_sum<T>(p, row, col, y);
    }
    ss = over_row(ss, sums[0], 0, LONG_THREADS / 32, add_f);
    if (isinf(ss)) {
      smaller = true;
      ss = 0.0f;
      for (int64_t col = col0; col < end; col += step) {
        float y[8];
        row_values<T, NORM>(p, row, col, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(y[j] * SMALLER, y[j] * SMALLER, ss);
      }
      ss = over_row(ss, sums[1], 0, LONG_THREADS / 32, add_f);
    }
    rstd = root(ss, smaller, p);
  }
  auto final_values = [&](int64_t col, float (&y)[8]) {
    row_values<T, NORM>(p, row, col, y);
    if constexpr (NORM) {
      float w[8];
      if (p.weight) load_weight(p, col, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = p.weight ? y[j] * rstd * w[j] : y[j] * rstd;
    }
  };
  uint32_t m = 0;
  if (p.mode == QI8_Q_TOKEN) {
    for (int64_t col = col0; col < end; col += step) {
      float y[8];
      final_values(col, y);
      m = max(m, amax_bits(y));
    }
    m = over_row(m, tops, 0, LONG_THREADS / 32, max_u);
  }
  for (int64_t first = 0; first < end; first += step) {  // the warp's lanes together
    const int64_t col = first + col0;
    float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (col < p.n) final_values(col, y);
    const uint32_t top = p.mode == QI8_Q_TOKEN ? m : max16(amax_bits(y));
    if (col >= p.n) continue;
    if (p.mode == QI8_Q_TOKEN) emit(p, y, top, row, col, col == 0, row);
    else emit(p, y, top, row, col, (threadIdx.x & 15) == 0, row * p.blocks + col / F8_BLOCK);
  }
}

// No step over whole rows: 16 lanes per block of 128 columns.  A warp takes 2 *
// STEPS neighbouring blocks of one row, all loads before the first use.
constexpr int THREADS = 256;

template <typename T, int STEPS>
__global__ void __launch_bounds__(THREADS) block_kernel(const __grid_constant__ Args p, const unsigned groups) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / groups;
  if (row >= p.rows) return;
  const int64_t col0 = (unit - row * groups) * (STEPS * 256) + lane * 8;
  float y[STEPS][8];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) row_values<T, false>(p, row, col0 + i * 256, y[i]);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int64_t col = col0 + i * 256;
    const uint32_t top = max16(amax_bits(y[i]));
    if (col < p.n) emit(p, y[i], top, row, col, (lane & 15) == 0, row * p.blocks + col / F8_BLOCK);
  }
}

template <typename T, int STEPS>
int launch_blocks(const Args& p, cudaStream_t st) {
  const int64_t groups = (p.blocks + 2 * STEPS - 1) / (2 * STEPS);
  const int64_t grid = (p.rows * groups + THREADS / 32 - 1) / (THREADS / 32);
  QI8_REQUIRE(grid < (1ll << 31), QI8_ESHAPE, "%lld rows of %lld", (long long)p.rows, (long long)p.n);
  block_kernel<T, STEPS><<<(unsigned)grid, THREADS, 0, st>>>(p, (unsigned)groups);
  return check_cuda(cudaGetLastError(), "block_kernel launch");
}

template <typename T, bool NORM, int CHUNKS>
int launch_rows(const Args& p, cudaStream_t st) {
  const int warps = (int)((p.n + 256 * CHUNKS - 1) / (256 * CHUNKS));
  const int per = warps >= 8 ? 1 : 8 / warps;  // rows per thread block
  row_kernel<T, NORM, CHUNKS><<<(unsigned)((p.rows + per - 1) / per), warps * per * 32, 0, st>>>(p, warps);
  return check_cuda(cudaGetLastError(), "row_kernel launch");
}

template <typename T, bool NORM>
int launch_type(const Args& p, cudaStream_t st) {
  if constexpr (!NORM) {
    // few units: one step each spreads them over more SMs
    if (p.mode != QI8_Q_TOKEN)
      return p.blocks < 8 || p.rows * p.blocks < 8 * 8 * 148 ? launch_blocks<T, 1>(p, st) : launch_blocks<T, 4>(p, st);
  }
  if (p.n <= 8192) return launch_rows<T, NORM, 1>(p, st);
  if (p.n <= 16384) return launch_rows<T, NORM, 2>(p, st);
  if (p.n <= 32768) return launch_rows<T, NORM, 4>(p, st);
  long_row_kernel<T, NORM><<<(unsigned)p.rows, LONG_THREADS, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "long_row_kernel launch");
}

template <bool NORM>
int launch(const Args& p, int dtype, cudaStream_t st) {
  if (p.rows == 0 || p.n == 0) return QI8_OK;
  QI8_REQUIRE(p.rows < (1ll << 31), QI8_ESHAPE, "%lld rows", (long long)p.rows);
  switch (dtype) {
    case QI8_BF16: return launch_type<__nv_bfloat16, NORM>(p, st);
    case QI8_F16: return launch_type<__half, NORM>(p, st);
    default: return launch_type<float, NORM>(p, st);
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
  return launch<false>(p, x_dtype, st);
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
  QI8_REQUIRE(eps >= 0.0 && eps < 1e300, QI8_EINVAL, "eps %g", eps);
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
  p.eps = eps;
  p.mode = mode;
  p.vec = rows_aligned(x, ld_x, size, 16) && (!residual || rows_aligned(residual, ld_residual, size, 16));
  p.vec_weight = aligned16(weight);
  p.vec_q = rows_aligned(q_out, ld_q, 1, 8);
  p.vec_sum = sum_out && rows_aligned(sum_out, ld_sum, size, 16);
  return aq::launch<true>(p, x_dtype, static_cast<cudaStream_t>(stream));
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
  p.act = act;
  p.mode = mode;
  p.vec = rows_aligned(gate, ld_gate, size, 16) && rows_aligned(up, ld_up, size, 16);
  p.vec_q = rows_aligned(q_out, ld_q, 1, 8);
  return aq::launch<false>(p, dtype, static_cast<cudaStream_t>(stream));
}
