// The fp8 format with block scales and the pieces that its producers share.
//
//   value = code * 2^e,  code e4m3 (largest value 448),  e >= -100
//
// e is the smallest whole number with amax <= 448 * 2^e.  448 = 1.75 * 2^8, so
// with the fp32 bits of amax, e is the exponent less 8, and one more when the
// mantissa is above 0.75: adding 2^21 - 1 to the bits carries into the exponent
// in just those cases.  A scale is one byte, e + 127, which is the exponent
// field of the fp32 number 2^e; 255 is NaN.  value / 2^e is exact, so a code is
// off by one rounding of e4m3, with a power of two as with any other scale.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace qi8 {

constexpr int F8_BLOCK = 128;  // columns (of a weight: rows too) that share a scale
constexpr int F8_E_MIN = -100;

// A product of fp8 operands: out [M, N] = a [M, K] b [N, K]^T + bias.
struct F8Gemm {
  const uint8_t *a, *b, *sa, *sb;  // codes; scales [M, KB] and [ceil(N / 128), KB]
  const void* bias;
  void* out;
  int64_t ld_a, ld_b, ld_out;
  int M, N, K, KB;  // KB = ceil(K / 128)
  int bias_dtype, out_dtype;
};

// The tcgen05 kernels (gemm_f8_tc.cu): rows of both operands start on 16-byte
// boundaries.
int gemm_f8_tiles(const F8Gemm& g, cudaStream_t st);

// The kernel for single tokens (gemm_f8_rows.cu), where the tokens fit beside its
// ring: rows of codes start on 16-byte boundaries.  x (not null): the tokens as
// numbers of x_dtype, quantized on the way, in place of g.a and g.sa.  after_quant:
// the kernel before on the stream is the tokens' quantizer, so the weight may be read
// before that is done.
bool gemm_f8_rows_fits(int M, int N, int K);
int gemm_f8_rows(const F8Gemm& g, const void* x, int x_dtype, int64_t ld_x, bool after_quant, cudaStream_t st);

inline int64_t f8_blocks(int64_t n) { return (n + F8_BLOCK - 1) / F8_BLOCK; }

namespace {

// The scale byte of a block whose largest |value| has these fp32 bits (an
// infinity or a NaN, which compare above all numbers: 255).
__device__ __forceinline__ uint32_t f8_scale_code(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const int c = (int)((amax_bits + 0x1fffffu) >> 23) - 8;
  return (uint32_t)(c > F8_E_MIN + 127 ? c : F8_E_MIN + 127);
}
// 2^-e and 2^e of a scale byte, NaN for 255.
__device__ __forceinline__ float f8_inverse(uint32_t code) {
  return __uint_as_float(code == 255u ? 0x7fffffffu : (254u - code) << 23);
}
// Bytes of other origin reach down to 2^-127, a subnormal.
__device__ __forceinline__ float f8_scale(uint32_t code) {
  return __uint_as_float(code == 255u ? 0x7fffffffu : code == 0 ? 0x00400000u : code << 23);
}
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ float2 f8_unpack2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Eight consecutive elements of a row as fp32, in pairs: the packed fp32
// instructions take two at a time.
struct F8x {
  float2 v[4];
};

// Bytes `off` (a multiple of the element's size, below 16) to off + 4 WORDS of a row of words.
template <int WORDS>
__device__ __forceinline__ void shift_out(uint32_t (&a)[WORDS + 4], uint32_t off, uint32_t* w) {
#pragma unroll
  for (int i = 0; i < WORDS + 3; ++i) a[i] = off & 4u ? a[i + 1] : a[i];
#pragma unroll
  for (int i = 0; i < WORDS + 1; ++i) a[i] = off & 8u ? a[i + 2] : a[i];
#pragma unroll
  for (int i = 0; i < WORDS; ++i) w[i] = __funnelshift_r(a[i], a[i + 1], 8 * (off & 3u));
}

// The same as they lie in memory.
template <typename T>
struct Eight {
  uint4 v[sizeof(T) / 2];

  // A whole piece on a 16-byte boundary.
  __device__ __forceinline__ void load(const T* at) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
  }
  // A whole piece anywhere: the aligned 16 bytes that it begins and ends in, shifted.
  // These lie in the row when eight columns do before the piece and after it.
  __device__ __forceinline__ void load_shifted(const T* at) {
    constexpr int WORDS = 2 * sizeof(T);
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(at) & 15u);
    const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(at) - off);
    uint32_t a[WORDS + 4];
#pragma unroll
    for (int i = 0; i <= WORDS / 4; ++i) {
      const uint4 c = __ldg(base + i);
      a[4 * i] = c.x;
      a[4 * i + 1] = c.y;
      a[4 * i + 2] = c.z;
      a[4 * i + 3] = c.w;
    }
    shift_out<WORDS>(a, off, reinterpret_cast<uint32_t*>(v));
  }
  // From column `col` on, zero from n on.
  __device__ __forceinline__ void load_some(const T* row, int64_t col, int64_t n) {
    T* e = reinterpret_cast<T*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = col + i < n ? row[col + i] : T(0.0f);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void store(T* at) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(at)[i] = v[i];
  }
  // vec: the row starts on a 16-byte boundary (col is a multiple of 8)
  __device__ __forceinline__ void store_some(T* row, int64_t col, int64_t n, bool vec) const {
    if (vec && col + 8 <= n) {
      store(row + col);
    } else {
      const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < n) row[col + i] = e[i];
    }
  }
  __device__ __forceinline__ F8x get() const {
    F8x f;
    const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = make_float2(Elem<T>::to_f32(e[2 * i]), Elem<T>::to_f32(e[2 * i + 1]));
    return f;
  }
  __device__ __forceinline__ void set(const F8x& f) {
    T* e = reinterpret_cast<T*>(v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        e[2 * i] = f.v[i].x;
        e[2 * i + 1] = f.v[i].y;
      } else if constexpr (std::is_same<T, __half>::value) {
        reinterpret_cast<__half2*>(e)[i] = __float22half2_rn(f.v[i]);
      } else {
        reinterpret_cast<__nv_bfloat162*>(e)[i] = __float22bfloat162_rn(f.v[i]);
      }
    }
  }
};

// Eight elements from column `col` of a row of n >= 1 on, wherever the row starts and
// ends: the aligned 16 bytes that hold them are loaded, all of which hold an element of
// the row, and shifted once they are there.  Columns from n on are zero.
template <typename T>
struct Loose {
  static constexpr int CHUNKS = sizeof(T) / 2 + 1;
  uint4 c[CHUNKS];

  __device__ __forceinline__ void load(const T* row, int64_t col, int64_t n) {
    if (col + 8 <= n) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(row + col);
      const uint4* first = reinterpret_cast<const uint4*>(at & ~(uintptr_t)15);
#pragma unroll
      for (int i = 0; i + 1 < CHUNKS; ++i) c[i] = __ldg(first + i);
      c[CHUNKS - 1] = __ldg(reinterpret_cast<const uint4*>((at + 15) & ~(uintptr_t)15) + (CHUNKS - 2));
    } else {
      const uintptr_t first = reinterpret_cast<uintptr_t>(row + min(col, n - 1)) & ~(uintptr_t)15;
      const uintptr_t last = (reinterpret_cast<uintptr_t>(row + n) - 1) & ~(uintptr_t)15;
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) c[i] = __ldg(reinterpret_cast<const uint4*>(min(first + 16 * i, last)));
    }
  }
  __device__ __forceinline__ Eight<T> get(const T* row, int64_t col, int64_t n) const {
    constexpr int WORDS = 2 * sizeof(T);
    uint32_t a[WORDS + 4];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      a[4 * i] = c[i].x;
      a[4 * i + 1] = c[i].y;
      a[4 * i + 2] = c[i].z;
      a[4 * i + 3] = c[i].w;
    }
    Eight<T> e;
    shift_out<WORDS>(a, (uint32_t)(reinterpret_cast<uintptr_t>(row + col) & 15u), reinterpret_cast<uint32_t*>(e.v));
    if (col + 8 > n) {
      const int left = (int)max(n - col, (int64_t)0);
      T* v = reinterpret_cast<T*>(e.v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= left) v[i] = T(0.0f);
    }
    return e;
  }
};

// The largest |value| as fp32 bits; NaN is above infinity.  One instruction for
// two values.
__device__ __forceinline__ uint32_t amax_bits(const F8x& f) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(f.v[i].x), "f"(f.v[i].y));
  return __float_as_uint(m);
}
// The largest over 16 neighbouring lanes: one block of 128 columns, eight per lane.
__device__ __forceinline__ uint32_t max16(uint32_t m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

__device__ __forceinline__ F8x scaled(const F8x& f, float by) {
  F8x r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = __fmul2_rn(f.v[i], make_float2(by, by));
  return r;
}
__device__ __forceinline__ uint2 f8_codes(const F8x& f, float inv) {
  const F8x s = scaled(f, inv);
  return make_uint2(f8_pack4(s.v[0].x, s.v[0].y, s.v[1].x, s.v[1].y), f8_pack4(s.v[2].x, s.v[2].y, s.v[3].x, s.v[3].y));
}
// int8 scale of a block: amax / 127, at least `least` (an infinity or a NaN stays).
__device__ __forceinline__ float i8_scale(uint32_t amax, float least) {
  const float s = __fdiv_rn(__uint_as_float(amax), 127.0f);
  return s < least ? least : s;
}
// rint(f * inv), |f * inv| < 127.5 or NaN (code 0)
__device__ __forceinline__ uint2 i8_codes(const F8x& f, float inv) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = __float2int_rn(f.v[i].x * inv) & 0xff, b = __float2int_rn(f.v[i].y * inv) & 0xff;
    w[i >> 1] |= (a | (b << 8)) << (16 * (i & 1));
  }
  return make_uint2(w[0], w[1]);
}
// Eight codes of a row.  vec: rows start on 8-byte boundaries; WHOLE: and are whole
// eights long.
template <bool WHOLE = false>
__device__ __forceinline__ void store_codes(uint8_t* row, int64_t col, int64_t n, uint2 c, bool vec) {
  if (WHOLE || (vec && col + 8 <= n)) {
    *reinterpret_cast<uint2*>(row + col) = c;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < n) row[col + i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
  }
}

// Launches a kernel that may start while the one before it on the stream ends: it
// sets itself up, then waits in pdl_wait() before its first access to memory that
// another kernel may write, and lets the next one start after that.  So where the
// kernel before is one of these too, all kernels before that one are done when this
// one starts.  Back to back and without a graph a call takes the GPU 2 us less so.
template <typename... KArgs, typename... Args>
int launch_early(const char* what, void (*kern)(KArgs...), dim3 grid, int block, int smem, int cluster, cudaStream_t st,
                 Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...), what);
}
__device__ __forceinline__ void wait_for_last_kernel() {
  pdl_wait();
  pdl_launch_dependents();
}

// Rows of elements of `size` bytes start on boundaries of `to` bytes.
inline bool rows_aligned(const void* p, int64_t ld, int size, int to) {
  return reinterpret_cast<uintptr_t>(p) % to == 0 && (ld * size) % to == 0;
}

}  // namespace
}  // namespace qi8
