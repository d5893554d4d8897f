// Weights of 4 bits with group scales (format: int4.cuh): quantization,
// dequantization and the linear layer of a few tokens.
//
//   scale = max(round5(amax(|w| over the group) / 7), 2^-100)
//   code  = rint(w / scale), ties to even, in [-7, 7]
//
// round5 keeps five significant bits (ties to even): a code has three, so
// code * scale is exact in bf16 and every product downstream multiplies the
// weight that dequantization reports.  The scale is at most 1/32 off amax / 7,
// which leaves |w| / scale < 7.25: no code is clipped by more than a quarter
// step.  A group that holds an infinity or a NaN gets scale NaN and code 0, so
// it reads back as NaN as a whole.
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "int4.cuh"

namespace qi8 {
namespace {

// ------------------------------------------------------------ quantization
// A thread handles 16 bytes of codes: words 4 a .. 4 a + 3 of a 128-feature block,
// which are features 32 b + 8 a .. + 7 for b = 0 .. 3.  The quad a = 0 .. 3 covers
// the block, so a group of 32 is the quad's maximum for one b, larger groups
// combine b's in the thread.  Four loads of 16 bytes per thread and step keep HBM
// busy (10240 x 4096 bf16 to codes and back: 62 us with one word per thread and
// step, 40 with four; 20 each).  Threads walk the matrix in the order of the
// codes; the (row, piece) pair advances by a constant step without a division.
constexpr int Q_THREADS = 256;

struct Walk {
  int64_t row;
  int piece;  // of the row, 32 features each
  int64_t step_row;
  int step_piece;
  int pieces;  // per row, a multiple of 4
  __device__ __forceinline__ Walk(int64_t at, int64_t step, int pieces_) : pieces(pieces_) {
    row = at / pieces;
    piece = (int)(at - row * pieces);
    step_row = step / pieces;
    step_piece = (int)(step - step_row * pieces);
  }
  __device__ __forceinline__ void advance() {
    row += step_row;
    piece += step_piece;
    if (piece >= pieces) {
      piece -= pieces;
      ++row;
    }
  }
  // first feature of word b
  __device__ __forceinline__ int feature(int b) const { return (piece >> 2) * 128 + 32 * b + 8 * (piece & 3); }
};

template <bool VEC>
__device__ __forceinline__ void load8(const float* row, int k, int K, float (&v)[8]) {
  if (VEC && k + 8 <= K) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(row + k));
    const float4 b = __ldg(reinterpret_cast<const float4*>(row + k) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k + i < K ? row[k + i] : 0.0f;
}

// Positive finite fp32 to five significant bits, ties to even.
__device__ __forceinline__ float round5(float s) {
  uint32_t b = __float_as_uint(s);
  b = (b + 0x3FFFFu + ((b >> 19) & 1u)) & ~0x7FFFFu;
  return __uint_as_float(b);
}

// rint(w / s) + 8 for |w / s| < 7.5, ties to even, in the low nibble.
// q = w * (1 / s) is off by less than 2^-21.  For 16-bit weights a quotient
// that is no tie is at least 2^-13 away from one (numerator and denominator
// have 11 and 5 bits), so rounding q to multiples of 2^-17 first -- adding 96,
// where that is the spacing of fp32 -- restores exact ties and moves nothing
// across one.  fp32 weights compare the remainder, which fma leaves exact.
template <typename T>
__device__ __forceinline__ uint32_t code_bits(float w, float s, float inv) {
  if constexpr (sizeof(T) == 2) {
    const float t = fmaf(w, inv, 96.0f);
    return __float_as_uint(__fadd_rn(t, 12582912.0f - 96.0f + 8.0f));
  } else {
    float q = rintf(w * inv);
    const float e = fmaf(-q, s, w), h = 0.5f * s, a = fabsf(e);
    if (a > h || (a == h && ((int)q & 1))) q += e > 0.0f ? 1.0f : -1.0f;
    return (uint32_t)((int)q + 8);
  }
}

// Words of 16-bit weights: pairs as they lie in memory, absolute values compared
// as pairs of 16-bit integers, codes joined by multiply-adds (1 instruction per
// weight for each; 10240 x 4096 bf16 take 20 us, 28 as fp32 values, 16 at the copy rate).
template <typename T> struct Piece16 {
  uint4 r[4];
  template <bool VEC>
  __device__ __forceinline__ void load(const T* row, int b, int k, int K) {
    const uint16_t* raw = reinterpret_cast<const uint16_t*>(row);
    if (VEC && k + 8 <= K) r[b] = __ldg(reinterpret_cast<const uint4*>(raw + k));
    else r[b] = ld_act8<false>(raw, k, K);
  }
  __device__ __forceinline__ void clear(int b) { r[b] = make_uint4(0, 0, 0, 0); }
  // largest magnitude of words [b0, b1), as bits of fp32 (NaN above infinity)
  __device__ __forceinline__ uint32_t amax(int b0, int b1) const {
    uint32_t m = 0;
#pragma unroll
    for (int b = b0; b < b1; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = word_of(r[b], i) & 0x7fff7fffu;
        asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(a));
      }
    const uint32_t top = max(m >> 16, m & 0xffffu);
    if constexpr (std::is_same<T, __half>::value)
      return top >= 0x7c00u ? 0x7f800000u : __float_as_uint(__half2float(__ushort_as_half((unsigned short)top)));
    else return top << 16;
  }
  __device__ __forceinline__ uint32_t codes(int b, float, float inv) const {
    // code_bits is 0x4B400000 + code + 8; the constants' sum over the nibbles comes off at the end
    uint32_t c = 0u - (0x4B400000u + 0xB4000000u + 0x40000000u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = word_of(r[b], i);
      float lo, hi;
      if constexpr (std::is_same<T, __half>::value) {
        lo = __half2float(__ushort_as_half((unsigned short)(w & 0xffffu)));
        hi = __half2float(__ushort_as_half((unsigned short)(w >> 16)));
      } else {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xffff0000u);
      }
      c += code_bits<T>(lo, 0.0f, inv) * (1u << (4 * i));
      c += code_bits<T>(hi, 0.0f, inv) * (1u << (4 * i + 16));
    }
    return c;
  }
};
// Words of fp32 weights.
struct Piece32 {
  float v[4][8];
  template <bool VEC>
  __device__ __forceinline__ void load(const float* row, int b, int k, int K) {
    load8<VEC>(row, k, K, v[b]);
  }
  __device__ __forceinline__ void clear(int b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[b][i] = 0.0f;
  }
  __device__ __forceinline__ uint32_t amax(int b0, int b1) const {
    uint32_t m = 0;
#pragma unroll
    for (int b = b0; b < b1; ++b)
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[b][i]) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ uint32_t codes(int b, float s, float inv) const {
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)  // nibble order 0, 2, 4, 6, 1, 3, 5, 7
      c |= (code_bits<float>(v[b][i], s, inv) & 15u) << (4 * ((i >> 1) + 4 * (i & 1)));
    return c;
  }
};

template <typename T, int G, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
quant_i4_kernel(const T* __restrict__ w, int64_t ld, int64_t rows, int K, int Kp, uint32_t* __restrict__ q,
                __nv_bfloat16* __restrict__ scale) {
  constexpr int NS = W4_BLOCK / G, PER = 4 / NS;  // groups per block, words of a group in this thread
  const int pieces = Kp / 32;
  // rows * pieces is a multiple of 4: a quad is all in or all out
  for (Walk at((int64_t)blockIdx.x * Q_THREADS + threadIdx.x, (int64_t)gridDim.x * Q_THREADS, pieces); ;
       at.advance()) {
    const bool in = at.row < rows;
    if (!__any_sync(0xffffffffu, in)) break;
    std::conditional_t<sizeof(T) == 4, Piece32, Piece16<T>> v;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (in) v.template load<VEC>(w + at.row * ld, b, at.feature(b), K);
      else v.clear(b);
    }
    uint32_t word[4], scales[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      uint32_t m = v.amax(j * PER, (j + 1) * PER);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const bool finite = m < 0x7f800000u;
      const float s = fmaxf(round5(__fdiv_rn(__uint_as_float(finite ? m : 0u), 7.0f)), 0x1p-100f);
      const float inv = __frcp_rn(s);
      scales[j] = finite ? __float_as_uint(s) >> 16 : 0x7fffu;  // five significant bits: exact in bf16
#pragma unroll
      for (int b = j * PER; b < (j + 1) * PER; ++b) word[b] = finite ? v.codes(b, s, inv) : 0x88888888u;
    }
    if (!in) continue;
    reinterpret_cast<uint4*>(q)[at.row * pieces + at.piece] = make_uint4(word[0], word[1], word[2], word[3]);
    if ((at.piece & 3) == 0) {
      __nv_bfloat16* s = scale + at.row * (Kp / G) + (at.piece >> 2) * NS;
      if constexpr (NS == 4)
        *reinterpret_cast<uint2*>(s) = make_uint2(scales[0] | scales[1] << 16, scales[2] | scales[3] << 16);
      else if constexpr (NS == 2) *reinterpret_cast<uint32_t*>(s) = scales[0] | scales[1] << 16;
      else *reinterpret_cast<unsigned short*>(s) = (unsigned short)scales[0];
    }
  }
}

// ---------------------------------------------------------- dequantization
template <typename T, int G, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
dequant_i4_kernel(const uint32_t* __restrict__ q, const __nv_bfloat16* __restrict__ scale, int64_t rows, int K, int Kp,
                  T* __restrict__ out, int64_t ld) {
  constexpr int NS = W4_BLOCK / G;
  const int pieces = Kp / 32;
  for (Walk at((int64_t)blockIdx.x * Q_THREADS + threadIdx.x, (int64_t)gridDim.x * Q_THREADS, pieces);
       at.row < rows; at.advance()) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(q) + at.row * pieces + at.piece);
    const __nv_bfloat16* sc = scale + at.row * (Kp / G) + (at.piece >> 2) * NS;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int k = at.feature(b);
      if (k >= K) break;
      const float s = __bfloat162float(sc[b * NS / 4]);
      const uint32_t c = word_of(w, b);
      T* o = out + at.row * ld + k;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t u = (c >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u;
        v[i] = (__uint_as_float(0x4B000000u | u) - 8388616.0f) * s;  // 2^23 + u - (2^23 + 8)
      }
      if (VEC && k + 8 <= K) {
        if constexpr (sizeof(T) == 4) {
          reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
          reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          alignas(16) T h[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = Elem<T>::from_f32(v[i]);
          *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(h);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i < K) o[i] = Elem<T>::from_f32(v[i]);
      }
    }
  }
}

// ------------------------------------------------- linear, a few tokens
// y[t, n] = sum_k W[n, k] x[t, k] + bias[n] for up to 8 NT tokens a block.
// Bound by the weight's bytes (read again, mostly from L2, for every further 8 NT
// tokens): each block takes 16 MT weight rows, its warps
// the 128-feature blocks in turn, and the MMAs (m16n8k16, tokens as the 8
// columns) keep the arithmetic per weight at the unpacking alone.  fp32 sums
// per warp, joined in shared memory in the order of the warps.
// Measured for 1 x 65536 x 8192: 63 us, 4.4 TB/s (0.67 of the copy rate); issue
// slots 66 %, ALU (the unpacking) 55 %, nearly half of the stalls wait for memory.  64
// registers, four blocks per SM: three blocks take 72 us, five with spills 78; two
// and four blocks of codes ahead 76 and 83.  With few blocks per SM a deep
// lookahead helps instead: 1 x 4096 x 4096 6.5 -> 5.4 us.  9 to 16 tokens pair two
// tiles of rows in a warp, which halves the loads of activations: 16 x 32768 x 4096
// 31 us, 37 unpaired with the lookahead; with few blocks it is the other way round,
// 16 x 4096 x 10240 13 us and 18.
constexpr int LIN_WARPS = 8;

template <typename T, int G, int MT, int NT, int AHEAD, bool VEC>
__global__ void __launch_bounds__(LIN_WARPS * 32, NT >= 2 ? 2 : AHEAD == 1 ? 4 : 1)
w4_rows_kernel(const LinArgs p) {
  __shared__ float red[LIN_WARPS][8 * NT][16 * MT + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, a = lane & 3;
  const int n0 = blockIdx.x * 16 * MT;
  const int t0 = blockIdx.y * 8 * NT;

  const uint8_t* q[MT];
  const __nv_bfloat16* sc[MT];
  uint32_t qo[2 * MT], so[2 * MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int64_t n = min(n0 + mt * 16, p.N - 1);
    q[mt] = p.q + n * p.KB * 64;
    sc[mt] = p.scale + n * p.KB * (W4_BLOCK / G);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t r = (uint32_t)(min((int)n + i * 8 + g, p.N - 1) - (int)n);  // rows past the end are read as the last
      qo[2 * mt + i] = r * (uint32_t)p.KB * 64u + a * 16u;
      so[2 * mt + i] = r * (uint32_t)p.KB * (W4_BLOCK / G);
    }
  }
  const uint16_t* x[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int t = t0 + nt * 8 + g;
    x[nt] = p.x + (int64_t)min(t, p.M - 1) * p.ld_x + (VEC ? 8 * a : 0);  // columns past the end repeat the last
  }

  float sum[MT][NT][4] = {};
  w4_blocks<G, MT, AHEAD>(q, sc, qo, so, warp, LIN_WARPS, p.KB, [&](int kb, const W4Frag<G, MT>& f) {
    if (VEC && (kb + 1) * W4_BLOCK <= p.K)
      w4_block<T, G, MT, NT>(f, sum, [&](int nt, int b) {
        return __ldg(reinterpret_cast<const uint4*>(x[nt] + kb * W4_BLOCK + b * 32));
      });
    else
      w4_block<T, G, MT, NT>(f, sum, [&](int nt, int b) {
        return ld_act8<VEC>(x[nt] - (VEC ? 8 * a : 0), kb * W4_BLOCK + b * 32 + a * 8, p.K);
      });
  });

#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[warp][nt * 8 + 2 * a + (i & 1)][mt * 16 + g + 8 * (i >> 1)] = sum[mt][nt][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * MT * 8 * NT; i += LIN_WARPS * 32) {
    const int r = i % (16 * MT), c = i / (16 * MT);
    const int n = n0 + r, t = t0 + c;
    if (n >= p.N || t >= p.M) continue;
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < LIN_WARPS; ++w) y += red[w][c][r];
    y *= w4_unit<T>();
    if (p.bias) y += load_as_f32(p.bias, p.bias_dtype, n);
    store_from_f32(p.out, p.out_dtype, (int64_t)t * p.ld_out + n, y);
  }
}

// Activation rows onto 16-byte boundaries, the last 16 bytes filled with zeros:
// TMA takes no others.
__global__ void align_rows_kernel(const uint16_t* __restrict__ x, int64_t ld_x, int K, uint4* __restrict__ out,
                                  int vecs, int64_t total) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / vecs;
    out[i] = ld_act8<false>(x + t * ld_x, (int)(i - t * vecs) * 8, K);
  }
}

template <typename F>
int with_group(int group, F&& f) {
  switch (group) {
    case 32: return f(std::integral_constant<int, 32>{});
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    default: return fail(QI8_ESHAPE, "group_size must be 32, 64 or 128, got %d", group);
  }
}
template <typename F>
int with_float(int dtype, F&& f) {
  switch (dtype) {
    case QI8_BF16: return f(__nv_bfloat16{});
    case QI8_F16: return f(__half{});
    case QI8_F32: return f(float{});
    default: return fail(QI8_EDTYPE, "bf16, fp16 or fp32 required, got dtype code %d", dtype);
  }
}
template <typename F>
int with_bool(bool b, F&& f) {
  return b ? f(std::true_type{}) : f(std::false_type{});
}

int q_grid(int64_t words) {
  const int64_t need = (words + Q_THREADS - 1) / Q_THREADS;
  const int64_t cap = (int64_t)sm_count() * 8;  // eight blocks of 256 threads fill an SM
  return (int)(need < cap ? need : cap);
}

int check_weight(const void* q, const void* scale, int64_t rows, int64_t K) {
  QI8_REQUIRE(rows >= 0 && rows < (1LL << 40) && K > 0 && K <= (1 << 24), QI8_ESHAPE,
              "4-bit weight of %lld rows, %lld features", (long long)rows, (long long)K);
  QI8_REQUIRE(rows == 0 || (q && scale), QI8_EINVAL, "null pointer");
  QI8_REQUIRE(aligned16(q) && aligned16(scale), QI8_EALIGN, "4-bit codes and scales must be 16-byte aligned");
  return QI8_OK;
}

}  // namespace
}  // namespace qi8

using namespace qi8;

extern "C" int qi8_quant_weight_i4(const void* w, int w_dtype, int64_t rows, int64_t K, int64_t ld_w, int group,
                                   uint8_t* q_out, void* scale_out, void* stream) {
  QI8_REQUIRE(device_ok(), QI8_EUNSUPPORTED, "no sm_100 device current");
  if (int rc = check_weight(q_out, scale_out, rows, K)) return rc;
  QI8_REQUIRE(rows == 0 || w, QI8_EINVAL, "null pointer");
  QI8_REQUIRE(ld_w >= K, QI8_ESHAPE, "row stride %lld below the row's %lld elements", (long long)ld_w, (long long)K);
  const int Kp = (int)w4_padded(K);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_group(group, [&](auto G) {
    return with_float(w_dtype, [&](auto t) {
      using T = decltype(t);
      if (rows == 0) return (int)QI8_OK;
      return with_bool(aligned16(w) && ld_w * sizeof(T) % 16 == 0, [&](auto vec) {
        quant_i4_kernel<T, decltype(G)::value, decltype(vec)::value><<<q_grid(rows * (Kp / 32)), Q_THREADS, 0, st>>>(
            static_cast<const T*>(w), ld_w, rows, (int)K, Kp, reinterpret_cast<uint32_t*>(q_out),
            static_cast<__nv_bfloat16*>(scale_out));
        return check_cuda(cudaGetLastError(), "quant_i4_kernel launch");
      });
    });
  });
}

extern "C" int qi8_dequant_i4(const uint8_t* q, const void* scale, int64_t rows, int64_t K, int group, void* out,
                              int out_dtype, int64_t ld_out, void* stream) {
  QI8_REQUIRE(device_ok(), QI8_EUNSUPPORTED, "no sm_100 device current");
  if (int rc = check_weight(q, scale, rows, K)) return rc;
  QI8_REQUIRE(rows == 0 || out, QI8_EINVAL, "null pointer");
  QI8_REQUIRE(ld_out >= K, QI8_ESHAPE, "row stride %lld below the row's %lld elements", (long long)ld_out,
              (long long)K);
  const int Kp = (int)w4_padded(K);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_group(group, [&](auto G) {
    return with_float(out_dtype, [&](auto t) {
      using T = decltype(t);
      if (rows == 0) return (int)QI8_OK;
      return with_bool(aligned16(out) && ld_out * sizeof(T) % 16 == 0, [&](auto vec) {
        dequant_i4_kernel<T, decltype(G)::value, decltype(vec)::value><<<q_grid(rows * (Kp / 32)), Q_THREADS, 0, st>>>(
            reinterpret_cast<const uint32_t*>(q), static_cast<const __nv_bfloat16*>(scale), rows, (int)K, Kp,
            static_cast<T*>(out), ld_out);
        return check_cuda(cudaGetLastError(), "dequant_i4_kernel launch");
      });
    });
  });
}

namespace {

template <typename T, int G, int MT, int NT, int AHEAD>
int launch_rows(const LinArgs& p, bool vec, cudaStream_t st) {
  const dim3 grid((p.N + 16 * MT - 1) / (16 * MT), (p.M + 8 * NT - 1) / (8 * NT));
  return with_bool(vec, [&](auto v) {
    w4_rows_kernel<T, G, MT, NT, AHEAD, decltype(v)::value><<<grid, LIN_WARPS * 32, 0, st>>>(p);
    return check_cuda(cudaGetLastError(), "w4_rows_kernel launch");
  });
}

}  // namespace

namespace {
// The tcgen05 kernel takes over at 17 tokens, but for small products: it costs
// 8 us before its first result, and the rows kernel with 32 tokens a block reads a
// small weight again from L2 for the next 32.  Rows against tcgen05: 4.3 and 8.7 us
// for 64 x 2048 x 1024, 9.8 and 21 for 128 x 1024 x 4096, 13 and 17 for 256 x 2048 x
// 1024; equal at 2^29 multiply-adds (64 x 4096 x 2048: 10.9 and 11.3), slower beyond
// (64 x 4096 x 4096: 17.7 and 13.9; 32 x 32768 x 4096: 57 and 42) and where K is long
// and the blocks are few (64 x 64 x 16384: 26 and 16, split over clusters).
constexpr int64_t W4_TILES_FROM = 17;
bool few_products(int64_t M, int64_t N, int64_t K) {
  return M <= 4096 && K <= 8192 && M * N * K <= (1LL << 29);
}

bool act_aligned(const void* x, int64_t K, int64_t ld_x) { return aligned16(x) && ld_x % 8 == 0 && K % 8 == 0; }
}  // namespace

extern "C" int64_t qi8_gemm_w4_workspace_bytes(const void* x, int64_t M, int64_t K, int64_t ld_x) {
  if (M < W4_TILES_FROM || act_aligned(x, K, ld_x)) return 0;
  return M * ((K + 7) / 8) * 16;
}

extern "C" int qi8_gemm_w4(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ld_x, const uint8_t* q,
                           const void* scale, int64_t N, int group, const void* bias, int bias_dtype, void* out,
                           int out_dtype, int64_t ld_out, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  QI8_REQUIRE(device_ok(), QI8_EUNSUPPORTED, "no sm_100 device current");
  if (int rc = check_weight(q, scale, N, K)) return rc;
  QI8_REQUIRE(x_dtype == QI8_BF16 || x_dtype == QI8_F16, QI8_EDTYPE, "activations must be bf16 or fp16");
  QI8_REQUIRE(out_dtype == x_dtype || out_dtype == QI8_F32, QI8_EDTYPE,
              "output dtype must be the activations' or fp32");
  QI8_REQUIRE(!bias || bias_dtype == QI8_BF16 || bias_dtype == QI8_F16 || bias_dtype == QI8_F32, QI8_EDTYPE,
              "bias must be bf16, fp16 or fp32");
  QI8_REQUIRE(M >= 0 && M < (1 << 30) && N < (1 << 30), QI8_ESHAPE, "%lld tokens, %lld outputs", (long long)M,
              (long long)N);
  QI8_REQUIRE(ld_x >= K && ld_out >= N, QI8_ESHAPE, "row strides %lld, %lld below the rows' %lld, %lld elements",
              (long long)ld_x, (long long)ld_out, (long long)K, (long long)N);
  QI8_REQUIRE(M == 0 || N == 0 || (x && out), QI8_EINVAL, "null pointer");
  if (int rc = with_group(group, [](auto) { return (int)QI8_OK; })) return rc;
  if (M == 0 || N == 0) return QI8_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool vec = act_aligned(x, K, ld_x);
  LinArgs p{static_cast<const uint16_t*>(x), ld_x, q, static_cast<const __nv_bfloat16*>(scale), bias, bias_dtype,
            out, ld_out, out_dtype, 0, (int)N, (int)K, (int)(w4_padded(K) / W4_BLOCK)};
  p.M = (int)M;
  if (M >= W4_TILES_FROM) {  // aligned from here on, whichever kernel: the bits do not depend on where x lies
    if (const int64_t need = qi8_gemm_w4_workspace_bytes(x, M, K, ld_x)) {
      QI8_REQUIRE(workspace && workspace_bytes >= need, QI8_ESHAPE, "workspace of %lld bytes, %lld needed",
                  (long long)workspace_bytes, (long long)need);
      QI8_REQUIRE(aligned16(workspace), QI8_EALIGN, "workspace must be 16-byte aligned");
      const int vecs = (int)((K + 7) / 8);
      align_rows_kernel<<<q_grid(M * vecs), Q_THREADS, 0, st>>>(p.x, ld_x, p.K, static_cast<uint4*>(workspace), vecs,
                                                                M * vecs);
      if (int rc = check_cuda(cudaGetLastError(), "align_rows_kernel launch")) return rc;
      p.x = static_cast<const uint16_t*>(workspace);
      p.ld_x = vecs * 8;
    }
    if (!few_products(M, N, K)) return gemm_w4_tiles(p, x_dtype, group, st);
  }
  return with_group(group, [&](auto G) {
    constexpr int g = decltype(G)::value;
    return with_bool(x_dtype == QI8_F16, [&](auto half) {
      using T = std::conditional_t<decltype(half)::value, __half, __nv_bfloat16>;
      // few blocks per SM: more of each warp's own in flight, and no rows paired in a warp
      const bool few = p.N <= 32 * sm_count();
      if (p.M >= W4_TILES_FROM) return launch_rows<T, g, 1, 4, 2>(p, true, st);  // rows padded to 16 bytes
      if (p.M > 8) return few ? launch_rows<T, g, 1, 2, 4>(p, vec, st) : launch_rows<T, g, 2, 2, 1>(p, vec, st);
      return few ? launch_rows<T, g, 1, 1, 4>(p, vec, st) : launch_rows<T, g, 1, 1, 1>(p, vec, st);
    });
  });
}
