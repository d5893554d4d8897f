// Products of fp8 operands with block scales (format: f8.cuh):
//
//   out[t, n] = sum_kb 2^(ea[t, kb] + eb[n / 128, kb]) sum_{k in kb} a[t, k] b[n, k] + bias[n]
#include <cstdint>

#include "f8.cuh"

namespace qi8 {

int quant_rows_f8(const void* x, int x_dtype, int64_t rows, int64_t n, int64_t ld_x, uint8_t* q, int64_t ld_q,
                  uint8_t* scale, cudaStream_t st);

namespace {
namespace f8g {

// Codes whose rows do not start on 16-byte boundaries -> such rows, zeros behind
// the end.  16 bytes per thread.
__global__ void __launch_bounds__(256)
repitch_kernel(const uint8_t* __restrict__ src, int64_t rows, int64_t K, int64_t ld, uint4* __restrict__ dst) {
  wait_for_last_kernel();
  const int64_t per = (K + 15) / 16;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per, col = (i - row * per) * 16;
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (col + j < K) w[j >> 2] |= (uint32_t)src[row * ld + col + j] << (8 * (j & 3));
    dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

bool is_float(int dtype) { return dtype == QI8_BF16 || dtype == QI8_F16 || dtype == QI8_F32; }

int64_t pitch(int64_t k) { return (k + 15) / 16 * 16; }

// Workspace of one operand: nothing where its rows are aligned already.  A single row
// has no stride.
int64_t copy_bytes(const uint8_t* q, int64_t rows, int64_t K, int64_t ld) {
  return rows_aligned(q, rows == 1 ? 0 : ld, 1, 16) ? 0 : rows * pitch(K);
}

// Brings an operand into the workspace where it has to be.
int align_rows(const uint8_t*& q, int64_t rows, int64_t K, int64_t& ld, uint8_t*& workspace, cudaStream_t st) {
  const int64_t bytes = copy_bytes(q, rows, K, ld);
  if (rows == 1) ld = pitch(K);
  if (bytes == 0) return QI8_OK;
  const int64_t blocks = (bytes / 16 + 255) / 256, most = (int64_t)sm_count() * 32;
  if (int rc = launch_early("repitch_kernel launch", repitch_kernel, dim3((unsigned)(blocks < most ? blocks : most)), 256,
                            0, 1, st, q, rows, K, ld, reinterpret_cast<uint4*>(workspace)))
    return rc;
  q = workspace;
  ld = pitch(K);
  workspace += bytes;
  return QI8_OK;
}

int check_workspace(const void* workspace, int64_t have, int64_t need) {
  QI8_REQUIRE(need == 0 || (workspace && have >= need), QI8_ESHAPE, "workspace of %lld bytes: %lld are needed",
              (long long)have, (long long)need);
  QI8_REQUIRE(need == 0 || aligned16(workspace), QI8_EALIGN, "workspace must be 16-byte aligned");
  return QI8_OK;
}

int check(int64_t M, int64_t K, int64_t N, int64_t ld_b, int64_t ld_out, int out_dtype, const void* bias,
          int bias_dtype) {
  QI8_REQUIRE(device_ok(), QI8_EUNSUPPORTED, "no sm_100 device current");
  constexpr int64_t MOST = (1ll << 31) - 4096;  // rounded up to whole tiles these are 32-bit numbers still
  QI8_REQUIRE(M >= 0 && N >= 0 && K > 0 && M < MOST && N < MOST && K < MOST, QI8_ESHAPE,
              "product of %lld x %lld and %lld x %lld", (long long)M, (long long)K, (long long)N, (long long)K);
  QI8_REQUIRE(ld_b >= K && ld_out >= N, QI8_ESHAPE, "row strides %lld (weight) and %lld (result)", (long long)ld_b,
              (long long)ld_out);
  QI8_REQUIRE(is_float(out_dtype), QI8_EDTYPE, "output dtype %d: bf16, f16 or f32", out_dtype);
  QI8_REQUIRE(!bias || is_float(bias_dtype), QI8_EDTYPE, "bias dtype %d: bf16, f16 or f32", bias_dtype);
  return QI8_OK;
}

}  // namespace f8g
}  // namespace
}  // namespace qi8

using namespace qi8;

extern "C" int64_t qi8_gemm_f8_workspace_bytes(const uint8_t* a, int64_t M, int64_t K, int64_t ld_a, const uint8_t* b,
                                               int64_t N, int64_t ld_b) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return f8g::copy_bytes(a, M, K, ld_a) + f8g::copy_bytes(b, N, K, ld_b);
}

extern "C" int qi8_gemm_f8(const uint8_t* a, const uint8_t* a_scale, int64_t M, int64_t K, int64_t ld_a,
                           const uint8_t* b, const uint8_t* b_scale, int64_t N, int64_t ld_b, const void* bias,
                           int bias_dtype, void* out, int out_dtype, int64_t ld_out, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  if (int rc = f8g::check(M, K, N, ld_b, ld_out, out_dtype, bias, bias_dtype)) return rc;
  QI8_REQUIRE(ld_a >= K, QI8_ESHAPE, "row stride %lld for %lld columns", (long long)ld_a, (long long)K);
  if (M == 0 || N == 0) return QI8_OK;
  QI8_REQUIRE(a && a_scale && b && b_scale && out, QI8_EINVAL, "null pointer");
  if (int rc = f8g::check_workspace(workspace, workspace_bytes, qi8_gemm_f8_workspace_bytes(a, M, K, ld_a, b, N, ld_b)))
    return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (int rc = f8g::align_rows(a, M, K, ld_a, ws, st)) return rc;
  if (int rc = f8g::align_rows(b, N, K, ld_b, ws, st)) return rc;
  const F8Gemm g{a, b, a_scale, b_scale, bias, out, ld_a, ld_b, ld_out, (int)M, (int)N, (int)K, (int)f8_blocks(K),
                 bias_dtype, out_dtype};
  if (gemm_f8_rows_fits((int)M, (int)N, (int)K)) return gemm_f8_rows(g, nullptr, 0, 0, false, st);
  return gemm_f8_tiles(g, st);
}

extern "C" int64_t qi8_linear_f8_workspace_bytes(int64_t M, int64_t K, const uint8_t* b, int64_t N, int64_t ld_b) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return M * f8g::pitch(K) + f8g::pitch(M * f8_blocks(K)) + f8g::copy_bytes(b, N, K, ld_b);
}

extern "C" int qi8_linear_f8(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ld_x, const uint8_t* b,
                             const uint8_t* b_scale, int64_t N, int64_t ld_b, const void* bias, int bias_dtype, void* out,
                             int out_dtype, int64_t ld_out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = f8g::check(M, K, N, ld_b, ld_out, out_dtype, bias, bias_dtype)) return rc;
  QI8_REQUIRE(f8g::is_float(x_dtype), QI8_EDTYPE, "input dtype %d: bf16, f16 or f32", x_dtype);
  QI8_REQUIRE(ld_x >= K, QI8_ESHAPE, "row stride %lld for %lld columns", (long long)ld_x, (long long)K);
  if (M == 0 || N == 0) return QI8_OK;
  QI8_REQUIRE(x && b && b_scale && out, QI8_EINVAL, "null pointer");
  if (int rc = f8g::check_workspace(workspace, workspace_bytes, qi8_linear_f8_workspace_bytes(M, K, b, N, ld_b)))
    return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* q = static_cast<uint8_t*>(workspace);
  uint8_t* s = q + M * f8g::pitch(K);
  uint8_t* ws = s + f8g::pitch(M * f8_blocks(K));
  if (int rc = f8g::align_rows(b, N, K, ld_b, ws, st)) return rc;
  F8Gemm g{q, b, s, b_scale, bias, out, f8g::pitch(K), ld_b, ld_out, (int)M, (int)N, (int)K, (int)f8_blocks(K),
           bias_dtype, out_dtype};
  // Quantized by each block itself, the tokens cost a launch less, but every block the
  // work.  Features x K 4096 x 4096 (weights from HBM): one token 5.5 us so and 6.5 with a
  // kernel for it, two 6.3 and 6.6, three 7.2 and 7.0; 4096 x 2048: four 4.8 and 5.0, six 5.6
  // and 5.4; 4096 x 1024: eight 3.9 and 4.0 (8192 x 1024 5.4 and 5.3); 1024 x 512: 2.3 and 3.3.
  if (gemm_f8_rows_fits((int)M, (int)N, (int)K) && M * K <= 8192)
    return gemm_f8_rows(g, x, x_dtype, ld_x, false, st);
  if (int rc = quant_rows_f8(x, x_dtype, M, K, ld_x, q, f8g::pitch(K), s, st)) return rc;
  if (gemm_f8_rows_fits((int)M, (int)N, (int)K)) return gemm_f8_rows(g, nullptr, 0, 0, true, st);
  return gemm_f8_tiles(g, st);
}
