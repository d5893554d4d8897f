// Linear layer on a 4-bit weight for more than a few tokens, on the tcgen05
// tensor cores (format: int4.cuh):
//
//   y[t, n] = sum_k W[n, k] x[t, k] + bias[n]
//
// The weight rows are the MMA's M (128 TMEM lanes), the tokens its N, so that
// one kernel serves a batch of single tokens and a long prompt.  Roles of a block:
//   warps 0..3    epilogue: TMEM -> registers -> y (thread = weight row)
//   warps 4..19   unpacking, four groups of four warps (thread = weight row):
//                 half of a 128-feature block, 32 bytes of codes -> code *
//                 scale in 16 bits -> 32 TMEM columns of the A operand
//   warps 20, 22  TMA producers: activations, codes
//   warp 21       TMEM allocation, MMA issue (one thread)
// The A operand lives in TMEM: in shared memory its stores and their fence to the
// async proxy took 800 to 1900 cycles a block (counted with clock64), here 140.
// What bounds the kernel is the MMAs, about 64 cycles for each M = 128, K = 16
// step up to 128 tokens, and as many more cycles a block of the issuing lane's
// waits and commits (slots of 64 features were slower for that); with 256 tokens a
// tile also the epilogues, which the one accumulator does not let overlap.  4096 x
// 10240 x 4096 takes 248 us (1.39 PFLOP/s, 0.84 of measured), fp16 300, with
// groups of 32 363 (row_shift, for every tile), 100 x 10240 x 4096 26 us.
// Rings: codes (stages of two blocks), activations, operand slots of 128
// features.  A group fills about every
// other slot of the sequence and had waited for slot n - 3 - SLOTS or a later one
// to be consumed before it waits for slot n: with SLOTS >= 3 the parity it waits
// for cannot be that of slot n - 2 SLOTS.  Codes are unpacked before the wait.
//
// code * scale is exact in bf16 when the scale has five significant bits, as
// qi8_quant_weight_i4 writes it; scales with more are rounded here, half a step
// of the activations' type per product.  fp16 layers shift every row by a power
// of two that brings its largest scale to 2^12, where fp16 holds 32 binades of
// scales exactly, and take it out of the fp32 sums.
//
// Few tiles: a cluster of S blocks splits K and joins its fp32 sums through
// distributed shared memory in the order of the ranks, each block finishing
// 1 / S of the tile's tokens.  (Tiles of N / SMs rows over all of K instead:
// 17 x 4096 x 4096 took 25 us against 14, 100 x 4096 x 10240 45 against 25.)
// With very few tiles they have 64 rows: 100 x 512 x 4096 11 us, not 14.
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
constexpr int EPI_WARPS = 4, UNPACK_WARP0 = 4, PRODUCER = 20, ISSUER = 21, CODES = 22;
constexpr int UNPACK_WARPS = 16;
constexpr int THREADS = 23 * 32;
constexpr int SLOTS = 4;     // of the weight operand, 128 features each
constexpr int A_COLS = 64;   // TMEM columns of one: two 16-bit features per column
constexpr int SEG = 2;       // 128-feature blocks per stage of the code ring: 128 bytes per row
constexpr int CODE_BARS = 8; // code stages at most

template <int BN> struct Cfg {
  static constexpr int X_SLOTS = BN == 256 ? 3 : BN == 128 ? 5 : BN == 64 ? 8 : 12;
  static constexpr int CODE_BYTES = (BN == 256 ? 32 : BN == 32 ? 96 : 64) * 1024;
  static constexpr int X_BYTES = BN * 256;
  static constexpr int RING = X_SLOTS * X_BYTES + CODE_BYTES;
  static constexpr int BARS = 2 * (SLOTS + X_SLOTS + CODE_BARS) + 5;
  static constexpr int SMEM = 1024 + RING + BARS * 8 + 16;
  static constexpr int ACCS = BN == 256 ? 1 : 2;  // accumulators that fit beside the weight slots
  static_assert(SMEM <= 232448 && (BN + 64) * 512 <= RING, "shared memory; the sums of a split tile");
  static_assert(ACCS * BN + SLOTS * A_COLS <= 512, "tensor memory");
};
constexpr uint32_t TMEM_COLS = 512;

struct Args {
  LinArgs l;
  int rows;              // weight rows per tile, at most 128
  int n_tiles, t_tiles;  // of `rows` weight rows, of BN tokens
  int split;             // blocks per tile (cluster size)
  int code_stages;       // stages of the code ring
  unsigned int* status;
};

// D fp32, A and B of the same 16-bit type, K-major, M = 128, N = BN
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int bn) {
  constexpr uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}

// A in TMEM, B in shared memory
__device__ __forceinline__ void mma_f16(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}
// 32 columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint2 ld_shared8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ void st_cluster_f32x4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d)
               : "memory");
}

// fp16 only: the power of two that brings a row's largest finite scale to
// [2^12, 2^13), as the exponent field of the factor, for row n0 + lane.  The warp
// reads its 32 rows together, a row's scales side by side: a row per lane instead
// touched 32 lines with every load and took 570 us for 4096 x 10240 x 4096 with
// groups of 32, four rows at a time 369.
__device__ __forceinline__ uint32_t row_shift(const __nv_bfloat16* scale, int n0, int n_rows, int pitch, int first,
                                              int count, int lane) {
  uint32_t top[32], mine = 13;
#pragma unroll
  for (int r = 0; r < 32; ++r) top[r] = 13;
  for (int i = lane; i < count; i += 32) {
    uint32_t e[32];  // 32 loads in flight
#pragma unroll
    for (int r = 0; r < 32; ++r)
      e[r] = __bfloat16_as_ushort(scale[(int64_t)min(n0 + r, n_rows - 1) * pitch + first + i]);
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      e[r] = (e[r] >> 7) & 0xffu;
      if (e[r] < 255) top[r] = max(top[r], e[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < 32; ++r) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, top[r]);
    if (r == lane) mine = m;
  }
  return 266u - mine;
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
__global__ void __launch_bounds__(THREADS, 1)
gemm_w4_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmQ,
               const __grid_constant__ Args p) {
  using C = Cfg<BN>;
  constexpr int X_SLOTS = C::X_SLOTS, ACCS = C::ACCS;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t sX = base, sQ = base + X_SLOTS * C::X_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw + (base - raw) + C::RING);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto full_bar = [&](int s) { return smem_u32(bars + s); };
  auto empty_bar = [&](int s) { return smem_u32(bars + SLOTS + s); };
  auto tfull_bar = [&](int b) { return smem_u32(bars + 2 * SLOTS + b); };
  auto tempty_bar = [&](int b) { return smem_u32(bars + 2 * SLOTS + 2 + b); };
  const uint32_t drain_bar = smem_u32(bars + 2 * SLOTS + 4);
  auto qfull_bar = [&](int s) { return smem_u32(bars + 2 * SLOTS + 5 + s); };
  auto qempty_bar = [&](int s) { return smem_u32(bars + 2 * SLOTS + 5 + CODE_BARS + s); };
  auto xfull_bar = [&](int s) { return smem_u32(bars + 2 * (SLOTS + CODE_BARS) + 5 + s); };
  auto xempty_bar = [&](int s) { return smem_u32(bars + 2 * (SLOTS + CODE_BARS) + 5 + X_SLOTS + s); };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const int rank = split > 1 ? (int)cta_rank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(full_bar(s), 8);  // warps of two groups
      mbar_init(empty_bar(s), 1);
    }
    for (int s = 0; s < X_SLOTS; ++s) {
      mbar_init(xfull_bar(s), 1);
      mbar_init(xempty_bar(s), 1);
    }
    for (int s = 0; s < CODE_BARS; ++s) {
      mbar_init(qfull_bar(s), 1);
      mbar_init(qempty_bar(s), UNPACK_WARPS);
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
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == PRODUCER && lane == 0) tma_prefetch_desc(&tmX);
  if (warp == CODES && lane == 0) tma_prefetch_desc(&tmQ);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot, tmem_a = tmem_base + (uint32_t)(ACCS * BN);

  // tiles of this block, 128-feature blocks of each
  const int tiles = p.n_tiles * p.t_tiles;
  const int tile0 = blockIdx.x / split, tile_step = gridDim.x / split;
  const int kb0 = (int)((int64_t)p.l.KB * rank / split), kb1 = (int)((int64_t)p.l.KB * (rank + 1) / split);

  const int kn = kb1 - kb0;

  if (warp == PRODUCER) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, issued = 0, issued_ph = 0;
      bool ok = true;
      for (int tile = tile0; ok && tile < tiles; tile += tile_step) {
        const int t0 = (tile / p.n_tiles) * BN;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(xempty_bar(s), ph ^ 1u, abort_flag, p.status, ST_W4_PRODUCER, WAIT_LIMIT_NS)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(xfull_bar(s), C::X_BYTES);
          tma_load_2d(sX + s * C::X_BYTES, &tmX, kb * 128, t0, xfull_bar(s));
          tma_load_2d(sX + s * C::X_BYTES + C::X_BYTES / 2, &tmX, kb * 128 + 64, t0, xfull_bar(s));
          issued |= 1u << s;
          issued_ph = (issued_ph & ~(1u << s)) | (ph << s);
          if (++s == X_SLOTS) s = 0, ph ^= 1u;
        }
      }
      // the last copies land before the block exits, also when nobody reads them any more
      if (!ok)
        for (int t = 0; t < X_SLOTS; ++t)
          if (issued & (1u << t)) drain_wait(xfull_bar(t), (issued_ph >> t) & 1u);
    }
  } else if (warp == CODES) {
    int s = 0;
    uint32_t ph = 0, issued = 0, issued_ph = 0;
    bool ok = true;
    for (int tile = tile0; ok && tile < tiles; tile += tile_step) {
      const int n0 = (tile % p.n_tiles) * p.rows;
      const int rows = min(p.rows, p.l.N - n0);
      for (int kb = kb0; kb < kb1; kb += SEG) {
        if (!warp_wait(qempty_bar(s), ph ^ 1u, abort_flag, p.status, ST_W4_PRODUCER, WAIT_LIMIT_NS)) {
          ok = false;
          break;
        }
        if (lane == 0) {  // past a split's range too: the box is whole
          mbar_arrive_expect_tx(qfull_bar(s), (uint32_t)(p.rows * SEG) * 64u);
          tma_load_2d(sQ + (uint32_t)(s * p.rows * SEG * 64), &tmQ, kb * 16, n0, qfull_bar(s));
        }
        for (int r = lane; r < rows; r += 32)
          prefetch_l2(p.l.scale + ((int64_t)(n0 + r) * p.l.KB + kb) * (W4_BLOCK / G));
        issued |= 1u << s;
        issued_ph = (issued_ph & ~(1u << s)) | (ph << s);
        if (++s == p.code_stages) s = 0, ph ^= 1u;
      }
    }
    if (!ok)
      for (int t = 0; t < p.code_stages; ++t)
        if (issued & (1u << t)) drain_wait(qfull_bar(t), (issued_ph >> t) & 1u);
  } else if (warp == ISSUER) {
    if (lane == 0) {
      int xs = 0, unit = 0;
      uint32_t xph = 0;
      unsigned seq = 0;  // blocks so far, over all tiles
      bool ok = true;
      for (int tile = tile0; ok && tile < tiles; tile += tile_step, ++unit) {
        const int buf = unit % ACCS;
        if (!mbar_wait(tempty_bar(buf), ((unit / ACCS) & 1) ^ 1u, abort_flag, p.status, ST_W4_MMA, WAIT_LIMIT_NS))
          break;
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(buf * BN);
        for (int kb = 0; kb < kn; ++kb, ++seq) {
          const int s = seq % SLOTS;
          if (!mbar_wait(xfull_bar(xs), xph, abort_flag, p.status, ST_W4_MMA, WAIT_LIMIT_NS) ||
              !mbar_wait(full_bar(s), (seq / SLOTS) & 1u, abort_flag, p.status, ST_W4_MMA, WAIT_LIMIT_NS)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = tmem_a + (uint32_t)(s * A_COLS);
          const uint64_t db = sw128_desc(sX + xs * C::X_BYTES);
#pragma unroll
          for (int k = 0; k < 8; ++k)  // 16 features each: 8 columns of A, 32 bytes of a swizzled half of B
            mma_f16(d, a + 8 * k, db + (uint64_t)((k >> 2) * (C::X_BYTES / 2 / 16) + (k & 3) * 2), idesc<T>(BN),
                    kb > 0 || k > 0);
          tc_commit(empty_bar(s));
          tc_commit(xempty_bar(xs));
          if (++xs == X_SLOTS) xs = 0, xph ^= 1u;
        }
        if (ok) tc_commit(tfull_bar(buf));
      }
      tc_commit(drain_bar);
      drain_wait(drain_bar, 0);
    }
    __syncwarp();
  } else if (warp >= UNPACK_WARP0) {
    // group g of four warps unpacks half g % 2 of block g / 2 of every code stage
    const int g = (warp - UNPACK_WARP0) >> 2, half = g & 1, which = g >> 1;
    const int row = ((warp & 3) << 5) + lane;
    const bool warp_live = ((warp & 3) << 5) < p.rows;  // lanes of the MMA past the tile's rows hold what they hold
    const uint32_t swz = (uint32_t)(row & 7) << 4;      // 128-byte swizzle of the codes
    const uint32_t q_row = sQ + min(row, p.rows - 1) * 128 + half * 8;
    const uint32_t a_row = tmem_a + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(half * 32);
    int qs = 0;
    uint32_t qph = 0;
    unsigned before = 0;  // blocks before this tile, over all tiles
    bool ok = true;
    for (int tile = tile0; ok && tile < tiles; tile += tile_step, before += kn) {
      const int64_t n = min((tile % p.n_tiles) * p.rows + row, p.l.N - 1);  // rows past the end: any scale
      const __nv_bfloat16* sc = p.l.scale + (n * p.l.KB + kb0) * (W4_BLOCK / G);
      float shift = 1.0f;
      if constexpr (std::is_same<T, __half>::value)
        shift = __uint_as_float(row_shift(p.l.scale, (tile % p.n_tiles) * p.rows + ((warp & 3) << 5), p.l.N,
                                          p.l.KB * (W4_BLOCK / G), kb0 * (W4_BLOCK / G), kn * (W4_BLOCK / G), lane)
                                << 23);
      auto load_scales = [&](int kb) -> uint32_t {  // of this half block
        if (kb >= kn) return 0;
        if (G == 32) return __ldg(reinterpret_cast<const uint32_t*>(sc + kb * 4 + half * 2));
        return __ldg(reinterpret_cast<const unsigned short*>(G == 64 ? sc + kb * 2 + half : sc + kb));
      };
      uint32_t f0 = load_scales(which), f1 = load_scales(which + SEG);
      for (int kb = which; kb - which < kn; kb += SEG) {
        const uint32_t f = f0;
        f0 = f1;
        f1 = load_scales(kb + 2 * SEG);
        if (!warp_wait(qfull_bar(qs), qph, abort_flag, p.status, ST_W4_UNPACK, WAIT_LIMIT_NS)) {
          ok = false;
          break;
        }
        // words 4 a + 2 half and the next of the block, unpacked before the slot is there to take them
        uint32_t v[32];
        const bool have = kb < kn;  // the last stage may have one block
        if (have && warp_live) {
          const uint32_t at = q_row + (uint32_t)(qs * p.rows * 128);
          uint2 w[4];
#pragma unroll
          for (int a = 0; a < 4; ++a) w[a] = ld_shared8(at + (((uint32_t)(which * 4 + a) << 4) ^ swz));
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint32_t sp =
                scale_pair<T>(__uint_as_float(G == 32 && b == 1 ? (f & 0xffff0000u) : (f << 16)), shift);
#pragma unroll
            for (int a = 0; a < 4; ++a) {
              uint32_t u[4];
              w4_unpack<T>(b ? w[a].y : w[a].x, u);
#pragma unroll
              for (int e = 0; e < 4; ++e) v[16 * b + 4 * a + e] = mul_pair<T>(u[e], sp);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(qempty_bar(qs));
        if (++qs == p.code_stages) qs = 0, qph ^= 1u;
        if (!have) break;
        const unsigned seq = before + kb;
        const int s = seq % SLOTS;
        if (!warp_wait(empty_bar(s), ((seq / SLOTS) & 1u) ^ 1u, abort_flag, p.status, ST_W4_UNPACK, WAIT_LIMIT_NS)) {
          ok = false;
          break;
        }
        if (warp_live) {
          tc_fence_after();
          tmem_st32(a_row + (uint32_t)(s * A_COLS), v);
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(full_bar(s));
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    int unit = 0;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    for (int tile = tile0; tile < tiles; tile += tile_step, ++unit) {
      const int r0 = warp * 32 + lane, n = (tile % p.n_tiles) * p.rows + r0;
      const int t0 = (tile / p.n_tiles) * BN;
      const int buf = unit % ACCS;
      float unshift = 1.0f;
      if constexpr (std::is_same<T, __half>::value)
        unshift = __uint_as_float((254u - row_shift(p.l.scale, (tile % p.n_tiles) * p.rows + warp * 32, p.l.N,
                                                    p.l.KB * (W4_BLOCK / G), kb0 * (W4_BLOCK / G),
                                                    kn * (W4_BLOCK / G), lane))
                                  << 23);
      const float bias = p.l.bias && n < p.l.N ? load_as_f32(p.l.bias, p.l.bias_dtype, n) : 0.0f;
      if (!warp_wait(tfull_bar(buf), (unit / ACCS) & 1, abort_flag, p.status, ST_W4_EPILOGUE, WAIT_LIMIT_NS)) break;
      tc_fence_after();
      if (split == 1) {
        const int t1 = min(BN, p.l.M - t0);
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
          if (c >= t1) break;
          uint32_t r[32];
          tmem_ld32(tmem_base + lanes + (uint32_t)(buf * BN + c), r);
          tmem_wait_ld();
          if (r0 < p.rows && n < p.l.N) {
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
    const int t0 = (tile / p.n_tiles) * BN, n0 = (tile % p.n_tiles) * p.rows;
    const int t1 = min(BN, p.l.M - t0);
    const int per = ((BN + split - 1) / split + 3) & ~3, pitch = per + 4;  // columns per rank; padded against conflicts
    if (warp < EPI_WARPS && __all_sync(0xffffffffu, !*abort_flag)) {
      const uint32_t lanes = (uint32_t)(warp * 32) << 16;
      const int row = warp * 32 + lane;
      float unshift = 1.0f;
      if constexpr (std::is_same<T, __half>::value)
        unshift = __uint_as_float((254u - row_shift(p.l.scale, n0 + warp * 32, p.l.N, p.l.KB * (W4_BLOCK / G),
                                                    kb0 * (W4_BLOCK / G), kn * (W4_BLOCK / G), lane))
                                  << 23);
      // rank d finishes columns [d per, (d + 1) per); its blocks of sums are [source][row][pitch]
#pragma unroll 1
      for (int c = 0; c < t1; c += 32) {
        uint32_t r[32];
        tmem_ld32(tmem_base + lanes + (uint32_t)c, r);
        tmem_wait_ld();
        if (row < p.rows) {
          int d = c / per, at = c - d * per;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            st_cluster_f32x4(mapa(base + (uint32_t)(((rank * BM + row) * pitch + at) * 4), (uint32_t)d),
                             __uint_as_float(r[j]) * unshift, __uint_as_float(r[j + 1]) * unshift,
                             __uint_as_float(r[j + 2]) * unshift, __uint_as_float(r[j + 3]) * unshift);
            if ((at += 4) >= per) at -= per, ++d;
          }
        }
      }
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const float* part = reinterpret_cast<const float*>(smem_raw + (base - raw));
    for (int i = threadIdx.x; i < per * BM; i += THREADS) {
      const int row = i & (BM - 1), c = i / BM;
      const int col = rank * per + c, n = n0 + row;
      if (col >= t1 || row >= p.rows || n >= p.l.N) continue;
      float y = 0.0f;
      for (int r = 0; r < split; ++r) y += part[(r * BM + row) * pitch + c];
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS)
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

template <typename T, int G, int BN> struct Key {};

template <typename T, int G, int BN>
int launch(const LinArgs& l, cudaStream_t st) {
  using C = Cfg<BN>;
  auto kern = gemm_w4_kernel<T, G, BN>;
  if (int rc = allow_smem<Key<T, G, BN>>(kern, C::SMEM)) return rc;
  const int sms = sm_count();
  Args p{l, BM, (l.N + BM - 1) / BM, (l.M + BN - 1) / BN, 1, 2, device_status_ptr()};
  if ((int64_t)p.n_tiles * p.t_tiles * 16 <= sms) {  // splits of K fill the SMs up to eightfold
    p.rows = BM / 2;
    p.n_tiles = (l.N + p.rows - 1) / p.rows;
  }
  const int64_t tiles = (int64_t)p.n_tiles * p.t_tiles;
  QI8_REQUIRE(tiles < (1 << 30), QI8_ESHAPE, "%lld output tiles", (long long)tiles);
  while (p.split < 8 && tiles * (p.split + 1) <= sms && p.l.KB >= 2 * (p.split + 1)) ++p.split;
  p.code_stages = C::CODE_BYTES / (p.rows * SEG * 64);
  if (p.code_stages > CODE_BARS) p.code_stages = CODE_BARS;
  CUtensorMap map, codes;
  if (int rc = activation_map(&map, l, std::is_same<T, __half>::value, BN)) return rc;
  if (int rc = code_map(&codes, l.q, l.N, l.KB, SEG, p.rows)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.split > 1 ? tiles * p.split : tiles < sms ? tiles : sms));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, map, codes, p), "gemm_w4_kernel launch");
}

// The narrowest MMA that holds all tokens, up to 256: narrower tiles of the same
// tokens would unpack the weight once for each.
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
