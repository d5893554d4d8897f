// fp8 quantization with block scales (format: f8.cuh), and back.
//
// Both kernels move each byte once and are bound by HBM: quantizing a weight of 10240 x
// 4096 bf16 takes 25.0 us (5.0 TB/s, 0.77 of the copy rate), 32768 x 4096 72.9 (5.5).
#include <cstdint>

#include "f8.cuh"

namespace qi8 {
namespace {
namespace f8q {

constexpr int THREADS = 512, PASSES = F8_BLOCK * 16 / THREADS;

// One 128 x 128 tile per thread block: 16 lanes by eight columns, 32 rows at a
// time.  The tile stays in registers between its maximum and its codes.  (Blocks that
// stay, with the next tile's loads under way, need 113 registers and took 28.3 us.)
template <typename T>
__global__ void __launch_bounds__(THREADS)
weight_kernel(const T* __restrict__ w, int64_t N, int64_t K, int64_t ld_w, bool vec, uint8_t* __restrict__ q,
              int64_t ld_q, bool vec_q, uint8_t* __restrict__ scale) {
  __shared__ uint32_t warp_max[THREADS / 32];
  const int64_t col = (int64_t)blockIdx.x * F8_BLOCK + (threadIdx.x & 15) * 8;
  const int64_t row = (int64_t)blockIdx.y * F8_BLOCK + (threadIdx.x >> 4);
  wait_for_last_kernel();
  Eight<T> e[PASSES];
  const bool whole = (int64_t)(blockIdx.x + 1) * F8_BLOCK <= K && (int64_t)(blockIdx.y + 1) * F8_BLOCK <= N;
  if (whole && vec) {  // all loads before the first use
#pragma unroll
    for (int i = 0; i < PASSES; ++i) e[i].load(w + (row + THREADS / 16 * i) * ld_w + col);
  } else if (whole && col >= 8 && col + 16 <= K) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) e[i].load_shifted(w + (row + THREADS / 16 * i) * ld_w + col);
  } else {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) e[i].load_some(w + (row + THREADS / 16 * i) * ld_w, col, row + THREADS / 16 * i < N ? K : 0);
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) m = max(m, amax_bits(e[i].get()));
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) m = max(m, warp_max[i]);
  const uint32_t code = f8_scale_code(m);
  const float inv = f8_inverse(code);
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
    if (row + THREADS / 16 * i < N) store_codes(q + (row + THREADS / 16 * i) * ld_q, col, K, f8_codes(e[i].get(), inv), vec_q);
  if (threadIdx.x == 0) scale[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = (uint8_t)code;
}

// Eight columns of a row per thread.
template <typename T>
__global__ void __launch_bounds__(THREADS)
dequant_kernel(const uint8_t* __restrict__ q, int64_t rows, int64_t n, int64_t ld_q, bool vec_q,
               const uint8_t* __restrict__ scale, int tile_shift, T* __restrict__ out, int64_t ld_out, bool vec) {
  wait_for_last_kernel();
  const int64_t per = (n + 7) / 8, blocks = (n + F8_BLOCK - 1) / F8_BLOCK;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < rows * per; i += (int64_t)gridDim.x * THREADS) {
    const int64_t row = i / per, col = (i - row * per) * 8;
    const uint8_t* src = q + row * ld_q;
    uint32_t w[2] = {0, 0};
    if (vec_q && col + 8 <= n) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(src + col));
      w[0] = v.x;
      w[1] = v.y;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < n) w[j >> 2] |= (uint32_t)src[col + j] << (8 * (j & 3));
    }
    const float s = f8_scale(scale[(row >> tile_shift) * blocks + col / F8_BLOCK]);
    F8x f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.v[j] = f8_unpack2((w[j >> 1] >> (16 * (j & 1))) & 0xffffu);
    Eight<T> e;
    e.set(scaled(f, s));
    e.store_some(out + row * ld_out, col, n, vec);
  }
}

template <typename T>
int quant_weight(const void* w, int64_t N, int64_t K, int64_t ld_w, uint8_t* q, int64_t ld_q, uint8_t* scale,
                 cudaStream_t st) {
  const dim3 grid((unsigned)f8_blocks(K), (unsigned)f8_blocks(N));
  return launch_early("weight_kernel launch", weight_kernel<T>, grid, THREADS, 0, 1, st, static_cast<const T*>(w), N, K,
                      ld_w, rows_aligned(w, ld_w, sizeof(T), 16), q, ld_q, rows_aligned(q, ld_q, 1, 8), scale);
}

template <typename T>
int dequant(const uint8_t* q, int64_t rows, int64_t n, int64_t ld_q, const uint8_t* scale, int tile, void* out,
            int64_t ld_out, cudaStream_t st) {
  const int64_t blocks = (rows * ((n + 7) / 8) + THREADS - 1) / THREADS, most = (int64_t)sm_count() * 64;
  return launch_early("dequant_kernel launch", dequant_kernel<T>, dim3((unsigned)(blocks < most ? blocks : most)), THREADS,
                      0, 1, st, q, rows, n, ld_q, rows_aligned(q, ld_q, 1, 8), scale, tile == 1 ? 0 : 7,
                      static_cast<T*>(out), ld_out, rows_aligned(out, ld_out, sizeof(T), 16));
}

}  // namespace f8q
}  // namespace
}  // namespace qi8

using namespace qi8;

extern "C" int qi8_quant_weight_f8(const void* w, int w_dtype, int64_t N, int64_t K, int64_t ld_w, uint8_t* q_out,
                                   int64_t ld_q, uint8_t* scale_out, void* stream) {
  QI8_REQUIRE(device_ok(), QI8_EUNSUPPORTED, "no sm_100 device current");
  QI8_REQUIRE(N >= 0 && K >= 0 && ld_w >= K && ld_q >= K, QI8_ESHAPE, "weight of %lld x %lld, row strides %lld and %lld",
              (long long)N, (long long)K, (long long)ld_w, (long long)ld_q);
  if (N == 0 || K == 0) return QI8_OK;
  QI8_REQUIRE(w && q_out && scale_out, QI8_EINVAL, "null pointer");
  QI8_REQUIRE(f8_blocks(N) <= 65535 && K < (1ll << 31), QI8_ESHAPE, "weight of %lld x %lld: at most 8388480 rows",
              (long long)N, (long long)K);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (w_dtype) {
    case QI8_BF16: return f8q::quant_weight<__nv_bfloat16>(w, N, K, ld_w, q_out, ld_q, scale_out, st);
    case QI8_F16: return f8q::quant_weight<__half>(w, N, K, ld_w, q_out, ld_q, scale_out, st);
    case QI8_F32: return f8q::quant_weight<float>(w, N, K, ld_w, q_out, ld_q, scale_out, st);
  }
  return fail(QI8_EDTYPE, "weight dtype %d: bf16, f16 or f32", w_dtype);
}

extern "C" int qi8_dequant_f8(const uint8_t* q, int64_t rows, int64_t n, int64_t ld_q, const uint8_t* scale, int tile,
                              void* out, int out_dtype, int64_t ld_out, void* stream) {
  QI8_REQUIRE(device_ok(), QI8_EUNSUPPORTED, "no sm_100 device current");
  QI8_REQUIRE(rows >= 0 && n >= 0 && ld_q >= n && ld_out >= n, QI8_ESHAPE,
              "codes of %lld x %lld, row strides %lld and %lld", (long long)rows, (long long)n, (long long)ld_q,
              (long long)ld_out);
  QI8_REQUIRE(tile == 1 || tile == F8_BLOCK, QI8_EINVAL, "tile %d: 1 (activations) or 128 (weights)", tile);
  if (rows == 0 || n == 0) return QI8_OK;
  QI8_REQUIRE(q && scale && out, QI8_EINVAL, "null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (out_dtype) {
    case QI8_BF16: return f8q::dequant<__nv_bfloat16>(q, rows, n, ld_q, scale, tile, out, ld_out, st);
    case QI8_F16: return f8q::dequant<__half>(q, rows, n, ld_q, scale, tile, out, ld_out, st);
    case QI8_F32: return f8q::dequant<float>(q, rows, n, ld_q, scale, tile, out, ld_out, st);
  }
  return fail(QI8_EDTYPE, "output dtype %d: bf16, f16 or f32", out_dtype);
}
