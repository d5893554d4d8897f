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

using Args = F8Gemm;

// 32 x 32 outputs per thread block, 32 columns of K at a time.
__global__ void __launch_bounds__(256) tile_kernel(const Args p) {
  __shared__ float sa[32][33], sb[32][33];
  const int n0 = blockIdx.x * 32, m0 = blockIdx.y * 32;
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
  float acc[4] = {0, 0, 0, 0};
  for (int k0 = 0; k0 < p.K; k0 += 32) {
    for (int i = r; i < 32; i += 8) {
      const int m = m0 + i, n = n0 + i, k = k0 + c;
      sa[i][c] = m < p.M && k < p.K
                     ? f8_unpack2(p.a[m * p.ld_a + k]).x * f8_scale(p.sa[(int64_t)m * p.KB + k / F8_BLOCK]) : 0.0f;
      sb[i][c] = n < p.N && k < p.K
                     ? f8_unpack2(p.b[n * p.ld_b + k]).x * f8_scale(p.sb[(int64_t)(n / F8_BLOCK) * p.KB + k / F8_BLOCK])
                     : 0.0f;
    }
    __syncthreads();
    for (int k = 0; k < 32; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(sa[r + 8 * i][k], sb[c][k], acc[i]);
    __syncthreads();
  }
  if (n0 + c >= p.N) return;
  const float bias = p.bias ? load_as_f32(p.bias, p.bias_dtype, n0 + c) : 0.0f;
  for (int i = 0; i < 4; ++i)
    if (m0 + r + 8 * i < p.M)
      store_from_f32(p.out, p.out_dtype, (int64_t)(m0 + r + 8 * i) * p.ld_out + n0 + c, acc[i] + bias);
}

bool is_float(int dtype) { return dtype == QI8_BF16 || dtype == QI8_F16 || dtype == QI8_F32; }

int gemm(const Args& p, cudaStream_t st) {
  if (rows_aligned(p.a, p.ld_a, 1, 16) && rows_aligned(p.b, p.ld_b, 1, 16)) return gemm_f8_tiles(p, st);
  const dim3 grid((unsigned)((p.N + 31) / 32), (unsigned)((p.M + 31) / 32));
  tile_kernel<<<grid, 256, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "tile_kernel launch");
}

int64_t pitch(int64_t k) { return (k + 15) / 16 * 16; }

int check(int64_t M, int64_t K, int64_t N, int64_t ld_b, int64_t ld_out, int out_dtype, const void* bias,
          int bias_dtype) {
  QI8_REQUIRE(device_ok(), QI8_EUNSUPPORTED, "no sm_100 device current");
  QI8_REQUIRE(M >= 0 && N >= 0 && K > 0 && M < (1ll << 31) && N < (1ll << 31) && K < (1ll << 31), QI8_ESHAPE,
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
  return 0;
}

extern "C" int qi8_gemm_f8(const uint8_t* a, const uint8_t* a_scale, int64_t M, int64_t K, int64_t ld_a,
                           const uint8_t* b, const uint8_t* b_scale, int64_t N, int64_t ld_b, const void* bias,
                           int bias_dtype, void* out, int out_dtype, int64_t ld_out, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  if (int rc = f8g::check(M, K, N, ld_b, ld_out, out_dtype, bias, bias_dtype)) return rc;
  QI8_REQUIRE(ld_a >= K, QI8_ESHAPE, "row stride %lld for %lld columns", (long long)ld_a, (long long)K);
  if (M == 0 || N == 0) return QI8_OK;
  QI8_REQUIRE(a && a_scale && b && b_scale && out, QI8_EINVAL, "null pointer");
  const F8Gemm p{a, b, a_scale, b_scale, bias, out, ld_a, ld_b, ld_out, (int)M, (int)N, (int)K, (int)f8_blocks(K),
                    bias_dtype, out_dtype};
  return f8g::gemm(p, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t qi8_linear_f8_workspace_bytes(int64_t M, int64_t K, const uint8_t* b, int64_t N, int64_t ld_b) {
  return M * (f8g::pitch(K) + f8_blocks(K));
}

extern "C" int qi8_linear_f8(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ld_x, const uint8_t* b,
                             const uint8_t* b_scale, int64_t N, int64_t ld_b, const void* bias, int bias_dtype, void* out,
                             int out_dtype, int64_t ld_out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = f8g::check(M, K, N, ld_b, ld_out, out_dtype, bias, bias_dtype)) return rc;
  QI8_REQUIRE(f8g::is_float(x_dtype), QI8_EDTYPE, "input dtype %d: bf16, f16 or f32", x_dtype);
  QI8_REQUIRE(ld_x >= K, QI8_ESHAPE, "row stride %lld for %lld columns", (long long)ld_x, (long long)K);
  if (M == 0 || N == 0) return QI8_OK;
  QI8_REQUIRE(x && b && b_scale && out && workspace, QI8_EINVAL, "null pointer");
  QI8_REQUIRE(workspace_bytes >= qi8_linear_f8_workspace_bytes(M, K, b, N, ld_b), QI8_ESHAPE, "workspace of %lld bytes",
              (long long)workspace_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* q = static_cast<uint8_t*>(workspace);
  uint8_t* s = q + M * f8g::pitch(K);
  if (int rc = quant_rows_f8(x, x_dtype, M, K, ld_x, q, f8g::pitch(K), s, st)) return rc;
  const F8Gemm p{q, b, s, b_scale, bias, out, f8g::pitch(K), ld_b, ld_out, (int)M, (int)N, (int)K,
                    (int)f8_blocks(K), bias_dtype, out_dtype};
  return f8g::gemm(p, st);
}
