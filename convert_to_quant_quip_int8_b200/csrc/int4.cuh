// The 4-bit weight format and the tensor-core step on it.
//
//   W[n, k] = (u[n, k] - 8) * scale[n, k / group],   group 32, 64 or 128
//
// Rows are padded to Kp, a multiple of 128 features (code 0, u = 8); q holds
// Kp / 2 bytes per row, scale (bf16) Kp / group values per row.
//
// * Eight codes share a 32-bit word, from the lowest nibble in the order of
//   features 0, 2, 4, 6, 1, 3, 5, 7: (word >> 4 i) & 0x000f000f is then the
//   pair of features (2 i, 2 i + 1) in the two halves of a register, where a
//   16-bit MMA operand wants them.  OR-ing a float's exponent above the
//   nibbles gives 128 + u (bf16) or 1024 + u (fp16); one packed subtraction
//   leaves the code itself.  1.4 instructions per weight, nothing rounded.
// * Of the 16 words of a 128-feature block, word 4 a + b holds features
//   32 b + 8 a .. + 7.  A thread of an m16n8k16 quad (a = lane % 4) loads its
//   four words as 16 bytes, and word b of the quad covers exactly the 32
//   features of group block b: no MMA step mixes two groups, so the scales
//   stay out of the operands and multiply the fp32 sums.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace qi8 {

constexpr int W4_BLOCK = 128;  // features per block of 16 words (64 bytes)

inline int64_t w4_padded(int64_t k) { return (k + W4_BLOCK - 1) / W4_BLOCK * W4_BLOCK; }

// One linear layer on a 4-bit weight: y [M, N] = x [M, K] W^T + bias.
struct LinArgs {
  const uint16_t* x;
  int64_t ld_x;
  const uint8_t* q;
  const __nv_bfloat16* scale;
  const void* bias;
  int bias_dtype;
  void* out;
  int64_t ld_out;
  int out_dtype;
  int M, N, K, KB;  // KB = Kp / 128
};

// Lets a kernel have `smem` bytes of shared memory, once per device (Key: a type
// of the kernel's own).
template <typename Key, typename F>
int allow_smem(F* kern, int smem) {
  static bool done[64];
  int dev = 0;
  if (int rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice")) return rc;
  if (dev < 64 && done[dev]) return QI8_OK;
  if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                          "cudaFuncSetAttribute"))
    return rc;
  if (dev < 64) done[dev] = true;
  return QI8_OK;
}

// The tcgen05 kernel (gemm_w4.cu): x rows start on 16-byte boundaries.
int gemm_w4_tiles(const LinArgs& p, int x_dtype, int group, cudaStream_t st);

// (a & b) | c in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// The codes of one word as four packed pairs of T, features in order; bf16 codes
// times 2^-10 if SMALL.
template <typename T, bool SMALL = false>
__device__ __forceinline__ void w4_unpack(uint32_t w, uint32_t (&p)[4]) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
    const uint32_t off = 0x64086408u;  // 1024 + 8
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = and_or(w >> (4 * i), 0x000f000fu, 0x64006400u);
      asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(v), "r"(off));
    }
  } else {
    // 128 + u - (128 + 8), or 2^-10 times that
    const uint32_t base = SMALL ? 0x3e003e00u : 0x43004300u, off = base + 0x00080008u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = and_or(w >> (4 * i), 0x000f000fu, base);
      asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(v), "r"(off));
    }
  }
}

// D[16, 8] += A[16, 16] B[16, 8], 16-bit operands, fp32 sums.
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weights are read once: keep them out of L1, which the activations use.
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int b) {
  return b == 0 ? v.x : b == 1 ? v.y : b == 2 ? v.z : v.w;
}

// Eight consecutive features of an activation row from feature k on, zero from
// K on.  VEC: the row starts on a 16-byte boundary and K is a multiple of 8.
template <bool VEC>
__device__ __forceinline__ uint4 ld_act8(const uint16_t* row, int k, int K) {
  if constexpr (VEC) return k < K ? __ldg(reinterpret_cast<const uint4*>(row + k)) : make_uint4(0, 0, 0, 0);
  else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = k + 2 * i < K ? __ldg(row + k + 2 * i) : 0;
      const uint32_t hi = k + 2 * i + 1 < K ? __ldg(row + k + 2 * i + 1) : 0;
      w[i] = lo | (hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A thread's weights of one 128-feature block for MT tiles of 16 rows: rows
// g and g + 8 of each tile (g = lane / 4), and those rows' scales.
template <int G, int MT>
struct W4Frag {
  uint4 w[2 * MT];
  uint2 s[2 * MT];  // 128 / G bf16 values, the first in the low half

  __device__ __forceinline__ float scale(int r, int j) const {
    const uint32_t v = j < 2 ? s[r].x : s[r].y;
    return __uint_as_float((j & 1) ? (v & 0xffff0000u) : (v << 16));
  }
};

// Calls body(kb, fragment) for the 128-feature blocks first, first + step, ...
// below end.  Row r of the thread (r / 2: tile, r % 2: g or g + 8) has its codes at
// q + qo[r] (from its 16 bytes of a block on) and its scales at sc + so[r]: a base
// that is the same for all threads and 32-bit offsets, which spare registers.
// Codes are loaded AHEAD (1, 2 or 4) blocks ahead.  Scales are loaded four blocks at a time, one
// block by each lane of a quad, and handed round by shuffles: a load that touches
// eight rows takes L1 eight cycles, as many as a row's codes.
template <int G, int MT, int AHEAD, typename Body>
__device__ __forceinline__ void w4_blocks(const uint8_t* const (&q)[MT], const __nv_bfloat16* const (&sc)[MT],
                                          const uint32_t (&qo)[2 * MT], const uint32_t (&so)[2 * MT], int first,
                                          int step, int end, Body&& body) {
  constexpr int NS = W4_BLOCK / G;
  const int a = threadIdx.x & 3;
  W4Frag<G, MT> f;
  uint4 next[AHEAD][2 * MT];
  uint2 s[2 * MT], s_next[2 * MT];
  auto load_scales = [&](int kb, uint2 (&v)[2 * MT]) {
    kb += a * step;
    if (kb >= end) return;
#pragma unroll
    for (int r = 0; r < 2 * MT; ++r) {
      const __nv_bfloat16* at = sc[r >> 1] + (so[r] + (uint32_t)(kb * NS));
      if (NS == 4) v[r] = __ldg(reinterpret_cast<const uint2*>(at));
      else if (NS == 2) v[r].x = __ldg(reinterpret_cast<const uint32_t*>(at));
      else v[r].x = __ldg(reinterpret_cast<const unsigned short*>(at));
    }
  };
  load_scales(first, s_next);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (first + i * step < end)
#pragma unroll
      for (int r = 0; r < 2 * MT; ++r) next[i][r] = ld_stream(q[r >> 1] + (qo[r] + (uint32_t)(first + i * step) * 64u));
  for (int base = first; base < end; base += 4 * step) {
#pragma unroll
    for (int r = 0; r < 2 * MT; ++r) s[r] = s_next[r];
    load_scales(base + 4 * step, s_next);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int kb = base + u * step;
      if (kb >= end) break;
#pragma unroll
      for (int r = 0; r < 2 * MT; ++r) {
        f.w[r] = next[u % AHEAD][r];
        f.s[r].x = __shfl_sync(0xffffffffu, s[r].x, u, 4);
        if (NS == 4) f.s[r].y = __shfl_sync(0xffffffffu, s[r].y, u, 4);
      }
      if (kb + AHEAD * step < end)
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) next[u % AHEAD][r] = ld_stream(q[r >> 1] + (qo[r] + (uint32_t)(kb + AHEAD * step) * 64u));
      body(kb, f);
    }
  }
}

// What the sums of w4_block have to be multiplied by.  bf16 activations reach to
// the end of fp32's range: a group's sum of 128 codes of up to 8 times such a one
// would pass it where the scaled result does not.  So codes enter the MMA times
// 2^-10 (a power of two: nothing rounds), and a group's sum stays finite.
template <typename T>
constexpr float w4_unit() {
  return std::is_same<T, __half>::value ? 1.0f : 1024.0f;
}

// w4_unit * sum[mt][nt] += W X^T over one 128-feature block: lane (g, a) gets rows g
// (elements 0, 1) and g + 8 (2, 3), columns 2 a and 2 a + 1.  act(nt, b)
// returns features 32 b + 8 a .. + 7 of the activation row of column 8 nt + g.
template <typename T, int G, int MT, int NT, typename Act>
__device__ __forceinline__ void w4_block(const W4Frag<G, MT>& f, float (&sum)[MT][NT][4], Act&& act) {
  float d[MT][NT][4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    uint4 x[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) x[nt] = act(nt, b);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t p[4], r[4];
      w4_unpack<T, true>(word_of(f.w[2 * mt], b), p);
      w4_unpack<T, true>(word_of(f.w[2 * mt + 1], b), r);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (b * 32 % G == 0) d[mt][nt][0] = d[mt][nt][1] = d[mt][nt][2] = d[mt][nt][3] = 0.0f;
        mma16816<T>(d[mt][nt], p[0], r[0], p[1], r[1], x[nt].x, x[nt].y);
        mma16816<T>(d[mt][nt], p[2], r[2], p[3], r[3], x[nt].z, x[nt].w);
      }
      if ((b + 1) * 32 % G == 0) {
        const int j = b * 32 / G;
        const float s0 = f.scale(2 * mt, j), s1 = f.scale(2 * mt + 1, j);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sum[mt][nt][0] = fmaf(d[mt][nt][0], s0, sum[mt][nt][0]);
          sum[mt][nt][1] = fmaf(d[mt][nt][1], s0, sum[mt][nt][1]);
          sum[mt][nt][2] = fmaf(d[mt][nt][2], s1, sum[mt][nt][2]);
          sum[mt][nt][3] = fmaf(d[mt][nt][3], s1, sum[mt][nt][3]);
        }
      }
    }
  }
}

}  // namespace qi8
