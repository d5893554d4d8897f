// Linear layer on a 4-bit weight for more than a few tokens, on the tcgen05
// tensor cores (format: int4.cuh):
//
//   y[t, n] = sum_k W[n, k] x[t, k] + bias[n]
//
// The weight rows are the MMA's M (128 TMEM lanes), the tokens its N, so that
// one kernel serves 17 tokens and a long prompt.  Roles of a block:
//   warps 0..3    epilogue: TMEM -> registers -> y (thread = weight row)
//   warps 4..11   unpacking, two groups of four warps that take the
//                 128-feature blocks in turn (thread = weight row): 64 bytes of
//                 codes -> code * scale in 16 bits -> the 128-byte-swizzled A
//                 operand in shared memory
//   warp 12       TMA producer of the activations
//   warp 13       TMEM allocation, MMA issue (one thread)
// A ring of SLOTS slots holds 64 features each (128 x 64 weights, BN x 64
// activations); a slot is full when TMA has written its bytes and the four
// warps of the unpacking group have arrived.
//
// code * scale is exact in bf16 when the scale has five significant bits, as
// qi8_quant_weight_i4 writes it; scales with more are rounded here, half a step
// of the activations' type per product.  fp16 layers shift every row by a power
// of two that brings its largest scale to 2^12, where fp16 holds 32 binades of
// scales exactly, and take it out of the fp32 sums.
//
// Few tiles: a cluster of S blocks splits K and joins its fp32 sums through
// distributed shared memory in the order of the ranks, each block finishing
// 1 / S of the tile's tokens.
//
// Every wait is bounded; on expiry the role sets a status bit, all roles leave
// their loops, copies and MMAs in flight are drained and TMEM is freed.
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "int4.cuh"
#include "tc05.cuh"

namespace qi8 {
namespace {
namespace w4tc {

constexpr int BM = 128;
constexpr int EPI_WARPS = 4, UNPACK_WARP0 = 4, PRODUCER = 12, ISSUER = 13;
constexpr int THREADS = 14 * 32;
constexpr int A_BYTES = BM * 128;  // 64 features in 16 bits

template <int BN> struct Cfg {
  static constexpr int SLOTS = BN == 256 ? 4 : BN == 128 ? 3 : BN == 64 ? 4 : 5;
  static constexpr int OCC = BN == 256 ? 1 : 2;  // blocks per SM
  static constexpr int B_BYTES = BN * 128;
  static constexpr int SLOT_BYTES = A_BYTES + B_BYTES;
  static constexpr int SMEM = 1024 + SLOTS * SLOT_BYTES + 192;
  static constexpr uint32_t TMEM_COLS = 2 * BN;  // two accumulators
  static_assert(OCC * SMEM <= 232448 && BN * 512 <= SLOTS * SLOT_BYTES, "shared memory");
  static_assert((2 * SLOTS + 5) * 8 + 16 <= 192, "barriers");
};

struct Args {
  LinArgs l;
  int n_tiles, t_tiles;  // of 128 weight rows, of BN tokens
  int split;             // blocks per tile (cluster size)
  unsigned int* status;
};

// D fp32, A and B of the same 16-bit type, K-major, M = 128, N = BN
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int bn) {
  constexpr uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}

__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// 32 bytes: a whole sector per thread
__device__ __forceinline__ void ld_codes(uint4& a, uint4& b, const uint8_t* p) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p));
}

// fp16 only: the power of two that brings the row's largest finite scale to
// [2^12, 2^13), as the exponent field of the factor.
__device__ __forceinline__ uint32_t row_shift(const __nv_bfloat16* scale, int count) {
  uint32_t top = 13;
  for (int i = 0; i < count; ++i) {
    const uint32_t e = (__bfloat16_as_ushort(scale[i]) >> 7) & 0xffu;
    if (e < 255) top = max(top, e);
  }
  return 266u - top;
}

// One scale as a packed pair of T.
template <typename T>
__device__ __forceinline__ uint32_t scale_pair(float s, float shift) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __float2half2_rn(s * shift);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const uint32_t u = __float_as_uint(s);
    return __byte_perm(u, u, 0x3232);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t mul_pair(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <typename T, int G, int BN>
__global__ void __launch_bounds__(THREADS, Cfg<BN>::OCC)
gemm_w4_kernel(const __grid_constant__ CUtensorMap tmX, const Args p) {
  using C = Cfg<BN>;
  constexpr int SLOTS = C::SLOTS;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t sA = base, sB = base + SLOTS * A_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw + (base - raw) + SLOTS * C::SLOT_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * SLOTS + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto full_bar = [&](int s) { return smem_u32(bars + s); };
  auto empty_bar = [&](int s) { return smem_u32(bars + SLOTS + s); };
  auto tfull_bar = [&](int b) { return smem_u32(bars + 2 * SLOTS + b); };
  auto tempty_bar = [&](int b) { return smem_u32(bars + 2 * SLOTS + 2 + b); };
  const uint32_t drain_bar = smem_u32(bars + 2 * SLOTS + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const int rank = split > 1 ? (int)cta_rank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(full_bar(s), 1 + 4);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), EPI_WARPS);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == PRODUCER && lane == 0) tma_prefetch_desc(&tmX);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // tiles of this block, 128-feature blocks of each
  const int tiles = p.n_tiles * p.t_tiles;
  const int tile0 = blockIdx.x / split, tile_step = gridDim.x / split;
  const int kb0 = (int)((int64_t)p.l.KB * rank / split), kb1 = (int)((int64_t)p.l.KB * (rank + 1) / split);

  if (warp == PRODUCER) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, issued = 0, issued_ph = 0;
      bool ok = true;
      for (int tile = tile0; ok && tile < tiles; tile += tile_step) {
        const int t0 = (tile / p.n_tiles) * BN;
        for (int kb = 2 * kb0; kb < 2 * kb1; ++kb) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.status, ST_W4_PRODUCER, WAIT_LIMIT_NS)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(full_bar(s), C::B_BYTES);
          tma_load_2d(sB + s * C::B_BYTES, &tmX, kb * 64, t0, full_bar(s));
          issued |= 1u << s;
          issued_ph = (issued_ph & ~(1u << s)) | (ph << s);
          if (++s == SLOTS) s = 0, ph ^= 1u;
        }
      }
      // the last copies land before the block exits, also when nobody reads them any more
      if (!ok)
        for (int t = 0; t < SLOTS; ++t)
          if (issued & (1u << t)) drain_wait(full_bar(t), (issued_ph >> t) & 1u);
    }
  } else if (warp == ISSUER) {
    if (lane == 0) {
      int s = 0, unit = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = tile0; ok && tile < tiles; tile += tile_step, ++unit) {
        const int buf = unit & 1;
        if (!mbar_wait(tempty_bar(buf), ((unit >> 1) & 1) ^ 1u, abort_flag, p.status, ST_W4_MMA, WAIT_LIMIT_NS)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(buf * BN);
        for (int kb = 2 * kb0; kb < 2 * kb1; ++kb) {
          if (!mbar_wait(full_bar(s), ph, abort_flag, p.status, ST_W4_MMA, WAIT_LIMIT_NS)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t da = sw128_desc(sA + s * A_BYTES), db = sw128_desc(sB + s * C::B_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16(d, da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), idesc<T>(BN), kb > 2 * kb0 || k > 0);
          tc_commit(empty_bar(s));
          if (++s == SLOTS) s = 0, ph ^= 1u;
        }
        if (ok) tc_commit(tfull_bar(buf));
      }
      tc_commit(drain_bar);
      drain_wait(drain_bar, 0);
    }
    __syncwarp();
  } else if (warp >= UNPACK_WARP0) {
    const int group = (warp - UNPACK_WARP0) >> 2;
    const int row = ((warp & 3) << 5) + lane;
    const uint32_t a_row = sA + row * 128;
    const uint32_t swz = (uint32_t)(row & 7);
    int s = 2 * group;  // this group's first slot of the ring
    uint32_t ph = 0;
    int block = 0;  // blocks before this tile, over all tiles
    bool ok = true;
    const int kn = kb1 - kb0;
    for (int tile = tile0; ok && tile < tiles; tile += tile_step, block += kn) {
      const int64_t n = min((tile % p.n_tiles) * BM + row, p.l.N - 1);  // rows past the end are read as the last
      const uint8_t* q = p.l.q + (n * p.l.KB + kb0) * 64;
      const __nv_bfloat16* sc = p.l.scale + (n * p.l.KB + kb0) * (W4_BLOCK / G);
      float shift = 1.0f;
      if constexpr (std::is_same<T, __half>::value)
        shift = __uint_as_float(row_shift(sc, kn * (W4_BLOCK / G)) << 23);
      // word 4 a + b of the block in w[a].b
      uint4 w[4], next[4];
      uint2 f, fn;
      auto load = [&](int kb, uint4 (&v)[4], uint2& sv) {
        ld_codes(v[0], v[1], q + kb * 64);
        ld_codes(v[2], v[3], q + kb * 64 + 32);
        const __nv_bfloat16* sp = sc + kb * (W4_BLOCK / G);
        if (G == 32) sv = __ldg(reinterpret_cast<const uint2*>(sp));
        else if (G == 64) sv.x = __ldg(reinterpret_cast<const uint32_t*>(sp));
        else sv.x = __ldg(reinterpret_cast<const unsigned short*>(sp));
      };
      int kb = (block & 1) ^ group;  // blocks alternate between the groups, across tiles too
      if (kb < kn) load(kb, w, f);
      for (; kb < kn; kb += 2) {
        if (kb + 2 < kn) load(kb + 2, next, fn);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.status, ST_W4_UNPACK, WAIT_LIMIT_NS)) {
            ok = false;
            break;
          }
          const uint32_t dst = a_row + s * A_BYTES;
#pragma unroll
          for (int bb = 0; bb < 2; ++bb) {
            const int b = 2 * h + bb, j = b * 32 / G;
            const uint32_t sv = j < 2 ? f.x : f.y;
            const uint32_t sp = scale_pair<T>(__uint_as_float((j & 1) ? (sv & 0xffff0000u) : (sv << 16)), shift);
#pragma unroll
            for (int a = 0; a < 4; ++a) {
              uint32_t v[4];
              w4_unpack<T>(word_of(w[a], b), v);
#pragma unroll
              for (int i = 0; i < 4; ++i) v[i] = mul_pair<T>(v[i], sp);
              st_shared16(dst + (((uint32_t)(bb * 4 + a) ^ swz) << 4), v[0], v[1], v[2], v[3]);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(full_bar(s));
          if (++s == SLOTS) s = 0, ph ^= 1u;
        }
        if (!ok) break;
        s += 2;  // the other group's slots
        if (s >= SLOTS) s -= SLOTS, ph ^= 1u;
#pragma unroll
        for (int a = 0; a < 4; ++a) w[a] = next[a];
        f = fn;
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    int unit = 0;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    for (int tile = tile0; tile < tiles; tile += tile_step, ++unit) {
      const int n = (tile % p.n_tiles) * BM + warp * 32 + lane;
      const int t0 = (tile / p.n_tiles) * BN;
      const int buf = unit & 1;
      float unshift = 1.0f;
      if constexpr (std::is_same<T, __half>::value)
        unshift = __uint_as_float(
            (254u - row_shift(p.l.scale + ((int64_t)min(n, p.l.N - 1) * p.l.KB + kb0) * (W4_BLOCK / G),
                              (kb1 - kb0) * (W4_BLOCK / G))) << 23);
      const float bias = p.l.bias && n < p.l.N ? load_as_f32(p.l.bias, p.l.bias_dtype, n) : 0.0f;
      if (!mbar_wait(tfull_bar(buf), (unit >> 1) & 1, abort_flag, p.status, ST_W4_EPILOGUE, WAIT_LIMIT_NS)) break;
      tc_fence_after();
      if (split == 1) {
        const int t1 = min(BN, p.l.M - t0);
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
          if (c >= t1) break;
          uint32_t r[32];
          tmem_ld32(tmem_base + lanes + (uint32_t)(buf * BN + c), r);
          tmem_wait_ld();
          if (n < p.l.N) {
            const int64_t at = (int64_t)(t0 + c) * p.l.ld_out + n;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (c + j >= t1) break;
              const float y = fmaf(__uint_as_float(r[j]), unshift, bias);
              if (p.l.out_dtype == QI8_F32) static_cast<float*>(p.l.out)[at + j * p.l.ld_out] = y;
              else static_cast<T*>(p.l.out)[at + j * p.l.ld_out] = Elem<T>::from_f32(y);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(buf));
      }
    }
  }

  if (split > 1) {
    // every block's MMAs are done with its ring: the sums go there
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const int tile = tile0;
    const int t0 = (tile / p.n_tiles) * BN, n0 = (tile % p.n_tiles) * BM;
    const int t1 = min(BN, p.l.M - t0);
    if (warp < EPI_WARPS && !*abort_flag) {
      const uint32_t lanes = (uint32_t)(warp * 32) << 16;
      const int row = warp * 32 + lane;
      float unshift = 1.0f;
      if constexpr (std::is_same<T, __half>::value)
        unshift = __uint_as_float(
            (254u - row_shift(p.l.scale + ((int64_t)min(n0 + row, p.l.N - 1) * p.l.KB + kb0) * (W4_BLOCK / G),
                              (kb1 - kb0) * (W4_BLOCK / G))) << 23);
#pragma unroll 1
      for (int c = 0; c < t1; c += 32) {
        uint32_t r[32];
        tmem_ld32(tmem_base + lanes + (uint32_t)c, r);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const int col = c + j;
          // column col belongs to rank col % split, at [source][col / split][row]
          const int dst = col % split, slot = rank * ((BN + split - 1) / split) + col / split;
          if (col < t1)
            st_cluster_f32(mapa(base + (uint32_t)((slot * BM + row) * 4), (uint32_t)dst),
                           __uint_as_float(r[j]) * unshift);
        }
      }
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const float* part = reinterpret_cast<const float*>(smem_raw + (base - raw));
    const int per = (BN + split - 1) / split;
    for (int i = threadIdx.x; i < per * BM; i += THREADS) {
      const int row = i & (BM - 1), c = i / BM;
      const int col = c * split + rank, n = n0 + row;
      if (col >= t1 || n >= p.l.N) continue;
      float y = 0.0f;
      for (int r = 0; r < split; ++r) y += part[(r * per + c) * BM + row];
      if (p.l.bias) y += load_as_f32(p.l.bias, p.l.bias_dtype, n);
      const int64_t at = (int64_t)(t0 + col) * p.l.ld_out + n;
      if (p.l.out_dtype == QI8_F32) static_cast<float*>(p.l.out)[at] = y;
      else static_cast<T*>(p.l.out)[at] = Elem<T>::from_f32(y);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == ISSUER) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM_COLS)
                 : "memory");
  }
}

// Activations [M, K] -> boxes of BN tokens x 64 features, 128-byte swizzle.
int activation_map(CUtensorMap* map, const LinArgs& p, bool half, int bn) {
  EncodeTiledFn fn = encode_fn();
  QI8_REQUIRE(fn, QI8_ECUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)p.K, (cuuint64_t)p.M};
  cuuint64_t strides[1] = {(cuuint64_t)p.ld_x * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)bn}, one[2] = {1, 1};
  const CUresult r = fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                        const_cast<uint16_t*>(p.x), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  QI8_REQUIRE(r == CUDA_SUCCESS, QI8_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return QI8_OK;
}

template <typename T, int G, int BN>
int launch(const LinArgs& l, cudaStream_t st) {
  using C = Cfg<BN>;
  auto kern = gemm_w4_kernel<T, G, BN>;
  int dev = 0;
  if (int rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice")) return rc;
  static bool set[64];
  if (dev >= 64 || !set[dev]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM),
                            "cudaFuncSetAttribute"))
      return rc;
    if (dev < 64) set[dev] = true;
  }
  CUtensorMap map;
  if (int rc = activation_map(&map, l, std::is_same<T, __half>::value, BN)) return rc;
  Args p{l, (l.N + BM - 1) / BM, (l.M + BN - 1) / BN, 1, device_status_ptr()};
  const int64_t tiles = (int64_t)p.n_tiles * p.t_tiles;
  QI8_REQUIRE(tiles < (1 << 30), QI8_ESHAPE, "%lld output tiles", (long long)tiles);
  const int sms = sm_count(), seats = sms * C::OCC;
  // blocks per tile: the split with the least work on the fullest SM, while all
  // blocks are resident at once and each has a few blocks of K
  int64_t best = (tiles + sms - 1) / sms * 64;
  for (int s = 2; s <= 8 && tiles * s <= seats && p.l.KB >= 2 * s; ++s) {
    const int64_t cost = (tiles * s + sms - 1) / sms * 64 / s + 2;  // and a little for joining
    if (cost < best) best = cost, p.split = s;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.split > 1 ? tiles * p.split : tiles < seats ? tiles : seats));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, map, p), "gemm_w4_kernel launch");
}

template <typename T, int G>
int pick(const LinArgs& l, cudaStream_t st) {
  if (l.M <= 32) return launch<T, G, 32>(l, st);
  if (l.M <= 64) return launch<T, G, 64>(l, st);
  if (l.M <= 128) return launch<T, G, 128>(l, st);
  return launch<T, G, 256>(l, st);
}

template <typename T>
int pick_group(const LinArgs& l, int group, cudaStream_t st) {
  return group == 32 ? pick<T, 32>(l, st) : group == 64 ? pick<T, 64>(l, st) : pick<T, 128>(l, st);
}

}  // namespace w4tc
}  // namespace

int gemm_w4_tiles(const LinArgs& l, int x_dtype, int group, cudaStream_t st) {
  return x_dtype == QI8_F16 ? w4tc::pick_group<__half>(l, group, st)
                            : w4tc::pick_group<__nv_bfloat16>(l, group, st);
}

}  // namespace qi8
