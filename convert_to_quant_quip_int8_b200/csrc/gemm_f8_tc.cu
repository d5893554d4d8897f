// Products of fp8 operands with block scales on the tcgen05 tensor cores
// (format: f8.cuh):
//
//   out[t, n] = sum_kb 2^(ea[t, kb] + eb[n / 128, kb]) sum_{k in kb} a[t, k] b[n, k] + bias[n]
//
// Scales that are powers of two are what tcgen05.mma.kind::mxf8f6f4 applies by
// itself: it takes one byte e + 127 per row and 32 columns of K from tensor
// memory, so the four steps of a 128-block read the same byte.  The sums stay in
// the accumulator over all of K.
#include <cmath>
#include <cstdint>

#include "f8.cuh"
#include "tc05.cuh"

namespace qi8 {
namespace {
namespace f8tc {

constexpr int BK = 128;  // columns of K per stage: one swizzled row of codes, one scale
constexpr uint32_t TMEM_COLS = 512;

// e4m3 operands, K-major, fp32 sums, scale bytes (UE8M0); sf: which of the four
// bytes of a scale word this step reads, for both operands
__host__ __device__ constexpr uint32_t idesc(int m, int n, uint32_t sf = 0) {
  return (sf << 4) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24) | (sf << 29);
}

// Four scale bytes, K blocks kb .. kb + 3, of N rows (`row` gives the start of row i).
// words: rows and kb lie on whole words; else a word is shifted out of the two that it
// begins and ends in (8 x 2560 x 2560, where four blocks share 20 K blocks, took 6.7 us
// byte by byte, 6.1 so).  Past the row's end: any.
template <int N, typename F>
__device__ __forceinline__ void scale_words(uint32_t (&w)[N], F&& row, int kb, int KB, bool words) {
  if (words) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(row(i) + kb));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = 0;
#pragma unroll 1  // little code beside that of the other case
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(row(i) + kb), last = reinterpret_cast<uintptr_t>(row(i) + KB - 1);
        const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>((h == 0 ? at : min(at + 3, last)) & ~(uintptr_t)3));
        w[i] = h == 0 ? v : __funnelshift_r(w[i], v, 8 * ((uint32_t)at & 3u));
      }
  }
}

__device__ __forceinline__ void tmem_st4(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// f(the result as what it holds).  Asked for once and not at each store: 100 x 10240 x
// 4096 took 12.7 us else, 12.0 so.
template <typename F>
__device__ __forceinline__ void typed(const F8Gemm& g, F&& f) {
  if (g.out_dtype == QI8_BF16) f(static_cast<__nv_bfloat16*>(g.out));
  else if (g.out_dtype == QI8_F16) f(static_cast<__half*>(g.out));
  else f(static_cast<float*>(g.out));
}

// 32 results `step` elements apart, the first `count` of them.
template <typename T>
__device__ __forceinline__ void store32(T* to, int64_t step, int count, const float (&y)[32]) {
  if (count >= 32) {
#pragma unroll
    for (int j = 0; j < 32; ++j) to[j * step] = Elem<T>::from_f32(y[j]);
  } else {
#pragma unroll
    for (int h = 0; h < 32; h += 8)
      if (h < count)
#pragma unroll
        for (int j = h; j < h + 8; ++j)
          if (j < count) to[j * step] = Elem<T>::from_f32(y[j]);
  }
}

// A warp's 32 rows (m0 on, lane = row) x 32 columns, all of them there, rows of the
// result on 16-byte boundaries.  Stored by rows each instruction touches 32 lines, and
// a tile took 6000 cycles; through shared memory it is 8 (4 with fp32).  Pieces of 16
// bytes are swapped so that eight lanes touch all banks, both ways.
__device__ __forceinline__ void store_tile(const F8Gemm& g, uint4* buf, int m0, int n, const float (&y)[32]) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  if (g.out_dtype == QI8_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      buf[lane * 8 + (i ^ (lane & 7))] = make_uint4(__float_as_uint(y[4 * i]), __float_as_uint(y[4 * i + 1]),
                                                    __float_as_uint(y[4 * i + 2]), __float_as_uint(y[4 * i + 3]));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 3), c = lane & 7;
      if (m0 + r < g.M)
        reinterpret_cast<uint4*>(static_cast<float*>(g.out) + (int64_t)(m0 + r) * g.ld_out + n)[c] = buf[r * 8 + (c ^ (r & 7))];
    }
  } else {
    const bool half = g.out_dtype == QI8_F16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = make_float2(y[8 * i + 2 * j], y[8 * i + 2 * j + 1]);
        if (half) {
          const __half2 h = __float22half2_rn(v);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __nv_bfloat162 h = __float22bfloat162_rn(v);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      buf[lane * 4 + (i ^ ((lane >> 1) & 3))] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 2), c = lane & 3;
      if (m0 + r < g.M)
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(g.out) + (int64_t)(m0 + r) * g.ld_out + n)[c] =
            buf[r * 4 + (c ^ ((r >> 1) & 3))];
    }
  }
}

// ------------------------------------------------- large: pairs of blocks
// A cluster of two blocks computes 256 tokens x 256 features: each block holds
// 128 tokens (TMEM lanes) and loads half of both operands' rows, so that a
// 128-column stage costs 32 KB of L2 reads per block.  Roles of a block:
//   warps 0..7    epilogue (warp w: lanes 32 (w % 4), every other half)
//   warps 8..11   scales: global memory -> tensor memory, four K blocks at a time
//   warp 12       TMA producer
//   warp 13       TMEM allocation; MMA issue (the even block's)
// Two accumulators of 256 columns and the scales do not fit 512 columns, so the
// accumulators share 64: the epilogue reads those first, and the next tile's
// MMAs wait for just that.  Tiles may have fewer features, where that fills the last
// wave of blocks better.
// The issuing warp sets the pace: an MMA takes it 72 cycles, a wait 110, a commit
// 60 to 100 (clock64), and the tensor cores, which queue about 14 MMAs, 128 cycles
// for each.  A stage of one K block cost it 700 cycles per block, two blocks a stage
// keep it below the 512 of the MMAs.  4096 x 10240 x 4096 with its quantization takes
// 142 us alone (2420 TFLOP/s, 0.72 of twice the measured bf16 rate) and 154 us back to
// back for seconds, where the board's 1 kW sets the clock: zeros take 107 us.
namespace pair {

constexpr int EPI_WARPS = 8, SCALE_WARP0 = 8, SCALE_WARPS = 4, PRODUCER = 12, ISSUER = 13;
constexpr int THREADS = 14 * 32;
constexpr int STAGES = 3, OPERAND = 128 * BK, STAGE = 4 * OPERAND;  // two K blocks of both operands
constexpr int ACC1 = 192;                           // columns of accumulator 1; 64 are both accumulators'
constexpr int SCALES = 448, SLOT = 16, SLOTS = 4;   // 8 columns of b, 4 of a
constexpr int BARS = 2 * STAGES + 4 + 2 * SLOTS + 2;
constexpr int EPI_BYTES = 32 * 32 * 4 + 32 * 4;  // of an epilogue warp: a tile on its way out, the bias
constexpr int SMEM = 1024 + STAGES * STAGE + EPI_WARPS * EPI_BYTES + BARS * 8 + 16;
static_assert(SMEM <= 232448 && SCALES + SLOTS * SLOT <= (int)TMEM_COLS && ACC1 + 256 <= SCALES, "memories");

struct Args {
  F8Gemm g;
  int m_tiles, n_tiles;
  int bn;  // features of a tile, a multiple of 32 up to 256
  bool words_a, words_b, vec_out;
  unsigned int* status;
};

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma(int one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                    uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.ne.b32 q, %7, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accum), "r"(one)
      : "memory");
}
// arrives on the barrier at this offset in both blocks once all earlier MMAs are done
__device__ __forceinline__ void commit(int one, uint32_t bar, uint16_t mask) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
      "h"(mask), "r"(one)
      : "memory");
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
gemm_f8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ Args p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const uint32_t sA = base, sB = base + STAGES * 2 * OPERAND;
  uint8_t* epi = sm + STAGES * STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi + EPI_WARPS * EPI_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto full_bar = [&](int s) { return smem_u32(bars + s); };
  auto empty_bar = [&](int s) { return smem_u32(bars + STAGES + s); };
  auto tfull_bar = [&](int b) { return smem_u32(bars + 2 * STAGES + b); };
  auto tempty_bar = [&](int b) { return smem_u32(bars + 2 * STAGES + 2 + b); };
  auto sfull_bar = [&](int b) { return smem_u32(bars + 2 * STAGES + 4 + b); };
  auto sempty_bar = [&](int b) { return smem_u32(bars + 2 * STAGES + 4 + SLOTS + b); };
  const uint32_t tshared_bar = smem_u32(bars + BARS - 2), drain_bar = smem_u32(bars + BARS - 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  const bool leader = rank == 0;
  const int pair0 = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {  // warps of both blocks
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 2 * EPI_WARPS);
    }
    for (int b = 0; b < SLOTS; ++b) {
      mbar_init(sfull_bar(b), 2 * SCALE_WARPS);
      mbar_init(sempty_bar(b), 1);
    }
    mbar_init(tshared_bar, 2 * EPI_WARPS);
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == PRODUCER && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  wait_for_last_kernel();
  const uint32_t tmem = *tmem_slot;
  const int KB = p.g.KB, tiles = p.m_tiles * p.n_tiles;

  if (warp == PRODUCER) {
    if (lane == 0) {
      const uint32_t full0 = mapa(full_bar(0), 0);
      int s = 0;
      uint32_t ph = 0, issued = 0, issued_ph = 0;
      bool ok = true;
      for (int tile = pair0; ok && tile < tiles; tile += pairs) {
        const int m0 = (tile % p.m_tiles) * 256 + (int)rank * 128, n0 = (tile / p.m_tiles) * p.bn + (int)rank * (p.bn / 2);
        for (int kb = 0; kb < KB; kb += 2) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.status, ST_F8_PRODUCER, WAIT_LIMIT_NS)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(full_bar(s), 2 * 2 * (OPERAND + (uint32_t)p.bn / 2 * BK));
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // past the last K block: zeros
            tma_load(sA + (2 * s + i) * OPERAND, &tmA, (kb + i) * BK, m0, full0 + 8 * s);
            tma_load(sB + (2 * s + i) * OPERAND, &tmB, (kb + i) * BK, n0, full0 + 8 * s);
          }
          issued |= 1u << s;
          issued_ph = (issued_ph & ~(1u << s)) | (ph << s);
          if (++s == STAGES) s = 0, ph ^= 1u;
        }
      }
      // copies that no MMA waits for any more land before the blocks exit
      if (!ok && leader)
        for (int t = 0; t < STAGES; ++t)
          if (issued & (1u << t)) drain_wait(full_bar(t), (issued_ph >> t) & 1u);
    }
  } else if (warp == ISSUER) {
    // the whole warp, so that addresses and descriptors stay in uniform registers; one lane issues
    if (leader) {
      const int one = lane == 0;
      int s = 0, unit = 0;
      uint32_t ph = 0;
      unsigned slot = 0;  // scale slots used so far
      bool ok = true;
      for (int tile = pair0; ok && tile < tiles; tile += pairs, ++unit) {
        const int buf = unit & 1;
        if (!warp_wait(tempty_bar(buf), ((unit >> 1) & 1) ^ 1u, abort_flag, p.status, ST_F8_MMA, WAIT_LIMIT_NS)) break;
        if (unit > 0 && p.bn > ACC1 &&
            !warp_wait(tshared_bar, (unit - 1) & 1, abort_flag, p.status, ST_F8_MMA, WAIT_LIMIT_NS)) break;
        tc_fence_after();
        const uint32_t d = tmem + (buf ? ACC1 : 0);
        for (int kb = 0; ok && kb < KB; kb += 4, ++slot) {  // one slot of scales
          const uint32_t sb = tmem + SCALES + (slot % SLOTS) * SLOT;
          if (!warp_wait(sfull_bar(slot % SLOTS), (slot / SLOTS) & 1, abort_flag, p.status, ST_F8_MMA, WAIT_LIMIT_NS)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int h = 0; h < 4; h += 2) {  // one stage
            if (kb + h >= KB) break;
            if (!warp_wait(full_bar(s), ph, abort_flag, p.status, ST_F8_MMA, WAIT_LIMIT_NS)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t da = sw128_desc(sA + 2 * s * OPERAND), db = sw128_desc(sB + 2 * s * OPERAND);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (kb + h + i >= KB) break;
#pragma unroll
              for (int k = 0; k < BK / 32; ++k)
                mma(one, d, da + (i * OPERAND / 16 + 2 * k), db + (i * OPERAND / 16 + 2 * k), idesc(256, p.bn, h + i),
                    sb + 8, sb, h + i + k > 0 || kb > 0);
            }
            commit(one, empty_bar(s), 3);
            if (++s == STAGES) s = 0, ph ^= 1u;
          }
          if (ok) commit(one, sempty_bar(slot % SLOTS), 3);
        }
        if (ok) commit(one, tfull_bar(buf), 3);
      }
      commit(one, drain_bar, 1);
      if (one) drain_wait(drain_bar, 0);
    }
  } else if (warp >= SCALE_WARP0) {
    // ---------------------------------------------------------- scales
    // word i: token (feature) 32 i + lane, in the same lane of all four quarters of
    // tensor memory
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + SCALES;
    const uint32_t sfull0 = mapa(sfull_bar(0), 0);
    auto load = [&](int tile, int kb, uint32_t (&a)[4], uint32_t (&b)[8]) {
      const int m0 = (tile % p.m_tiles) * 256 + (int)rank * 128, n0 = (tile / p.m_tiles) * p.bn;
      const int last = (p.g.N - 1) / F8_BLOCK;
      scale_words(a, [&](int i) { return p.g.sa + (int64_t)min(m0 + 32 * i + lane, p.g.M - 1) * KB; }, kb, KB, p.words_a);
      scale_words(b, [&](int i) { return p.g.sb + (int64_t)min((n0 + 32 * i + lane) / F8_BLOCK, last) * KB; }, kb, KB,
                  p.words_b);
    };
    unsigned slot = 0;
    bool ok = true;
    uint32_t a[4], b[8];
    if (pair0 < tiles) load(pair0, 0, a, b);
    for (int tile = pair0; ok && tile < tiles; tile += pairs) {
      for (int kb = 0; kb < KB; kb += 4, ++slot) {
        uint32_t a_next[4] = {0, 0, 0, 0}, b_next[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (kb + 4 < KB) load(tile, kb + 4, a_next, b_next);
        else if (tile + pairs < tiles) load(tile + pairs, 0, a_next, b_next);
        if (!warp_wait(sempty_bar(slot % SLOTS), ((slot / SLOTS) & 1) ^ 1u, abort_flag, p.status, ST_F8_SCALES,
                       WAIT_LIMIT_NS)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t at = lanes + (slot % SLOTS) * SLOT;
        const uint32_t lo[4] = {b[0], b[1], b[2], b[3]}, hi[4] = {b[4], b[5], b[6], b[7]};
        tmem_st4(at, lo);
        tmem_st4(at + 4, hi);
        tmem_st4(at + 8, a);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(sfull0 + 8 * (slot % SLOTS));
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = a_next[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = b_next[i];
      }
    }
  } else {
    // -------------------------------------------------------- epilogue
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t tempty0 = mapa(tempty_bar(0), 0), tshared0 = mapa(tshared_bar, 0);
    uint4* my_tile = reinterpret_cast<uint4*>(epi + warp * 32 * 32 * 4);
    float* my_bias = reinterpret_cast<float*>(epi + EPI_WARPS * 32 * 32 * 4) + warp * 32;
    int unit = 0;
    for (int tile = pair0; tile < tiles; tile += pairs, ++unit) {
      const int buf = unit & 1;
      const int m0 = (tile % p.m_tiles) * 256 + (int)rank * 128 + quarter * 32;
      const int n0 = (tile / p.m_tiles) * p.bn, end = min(n0 + p.bn, p.g.N);
      // every other 32 columns, those first that the accumulators share: the lowest
      // 64 of accumulator 1, the highest 64 of accumulator 0
      auto chunk = [&](int i) { return (buf ? 2 * i : 6 - 2 * i) + half; };
      if (!warp_wait(tfull_bar(buf), (unit >> 1) & 1, abort_flag, p.status, ST_F8_EPILOGUE, WAIT_LIMIT_NS)) break;
      tc_fence_after();
      const uint32_t acc = lanes + (buf ? ACC1 : 0);
      uint32_t r[2][32];
      if (32 * chunk(0) < p.bn) tmem_ld32(acc + 32 * chunk(0), r[0]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        tmem_wait_ld();
        if (i < 3 && 32 * chunk(i + 1) < p.bn) tmem_ld32(acc + 32 * chunk(i + 1), r[(i + 1) & 1]);
        if (i == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_cluster(tshared0);
        }
        if (i == 3) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_cluster(tempty0 + 8 * buf);
        }
        if (32 * chunk(i) >= p.bn) continue;
        const int n = n0 + 32 * chunk(i);
        float y[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j] = __uint_as_float(r[i & 1][j]);
        if (p.g.bias) {
          __syncwarp();
          my_bias[lane] = n + lane < p.g.N ? load_as_f32(p.g.bias, p.g.bias_dtype, n + lane) : 0.0f;
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; ++j) y[j] += my_bias[j];
        }
        if (p.vec_out && n + 32 <= end) store_tile(p.g, my_tile, m0, n, y);
        else if (m0 + lane < p.g.M && n < end)
          typed(p.g, [&](auto* out) { store32(out + (int64_t)(m0 + lane) * p.g.ld_out + n, 1, end - n, y); });
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == ISSUER) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

}  // namespace pair

// ------------------------------------------ few tokens: weights on the lanes
// The weight rows are the MMA's M (128 TMEM lanes, of which a tile may use
// fewer), the tokens its N.  A tile has `rows` weight rows, so that the tiles of a
// weight that is read once fill the SMs; a cluster of `split` blocks may share a
// tile's K and joins its fp32 sums through distributed shared memory in the order of
// the ranks.  Roles of a block:
//   warps 0..3   epilogue: TMEM -> registers -> out (thread = weight row)
//   warps 4..7   scales: global memory -> tensor memory, four K blocks at a time
//   warp 8       TMA producer: weight rows and tokens, one or two K blocks per stage
//   warps 9, 10  MMA issue, every other stage each; warp 9 TMEM allocation
// Two issuers, because one takes 430 cycles for a K block's waits, MMAs and commits
// however few the tokens.  16 x 10240 x 4096 takes 9.8 us (weights from HBM; 4.3 TB/s,
// and 5.9 from one K block to the next: HBM), 100 x 10240 x 4096 11.9, where a block
// reads 14 KB of tokens from L2 beside each 10 KB of weights and L2 sets the pace (0.27
// us a K block against 0.22).  The rest is launch, first loads and the way out.
namespace few {

constexpr int BM = 128;
constexpr int EPI_WARPS = 4, SCALE_WARP0 = 4, SCALE_WARPS = 4, PRODUCER = 8, ISSUER0 = 9;
constexpr int THREADS = 11 * 32;
constexpr int RING = 216 * 1024, MAX_STAGES = 8;
constexpr int ISSUERS = 2;                         // each with an accumulator of its own
constexpr int SCALES = 448, SLOT = 16, SLOTS = 4;  // 8 columns of the tokens, 4 of the weight rows
constexpr int BARS = 2 * MAX_STAGES + 4 + 2 * SLOTS + 1;
constexpr int SMEM = 1024 + RING + BARS * 8 + 16;  // the ring, behind it a split tile's sums

struct Args {
  F8Gemm g;
  int rows, n_tiles, t_tiles, split, stages;
  int bn;    // tokens of a tile, a multiple of 16
  int join;  // where the sums of a split tile's blocks meet, from the ring's start
  bool words_a, words_b;
  unsigned int* status;
};

// K blocks per stage of the ring
__host__ __device__ constexpr int kps(int bn) { return bn == 128 ? 1 : 2; }
// The issuer of a tile's first stage: they take turns over all stages.
template <int KPS>
__device__ __forceinline__ int first_issuer(int unit, int kn) { return (unit * ((kn + KPS - 1) / KPS)) & 1; }
// tokens that each block of a split tile finishes
__host__ __device__ constexpr int join_per(int bn, int split) { return ((bn + split - 1) / split + 3) & ~3; }

__device__ __forceinline__ void mma(int one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                    uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.ne.b32 q, %7, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accum), "r"(one)
      : "memory");
}
__device__ __forceinline__ void commit(int one, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(one)
      : "memory");
}
__device__ __forceinline__ void tmem_st1(uint32_t addr, uint32_t r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(addr), "r"(r) : "memory");
}
__device__ __forceinline__ void st_cluster_f32x4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d)
               : "memory");
}
// 32 columns of an accumulator, or of the two issuers' accumulators
template <int BN>
__device__ __forceinline__ void sums(uint32_t at, bool two, float (&y)[32]) {
  uint32_t v[32], u[32];
  tmem_ld32(at, v);
  if (two) tmem_ld32(at + BN, u);
  tmem_wait_ld();
#pragma unroll
  for (int j = 0; j < 32; ++j) y[j] = __uint_as_float(v[j]) + (two ? __uint_as_float(u[j]) : 0.0f);
}

template <int BN, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
gemm_f8_few_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ Args p) {
  constexpr int KPS = kps(BN);             // K blocks per stage
  constexpr int ACCS = BN == 128 ? 1 : 2;  // tiles that may be under way
  static_assert(ACCS * ISSUERS * BN <= SCALES && SCALES + SLOTS * SLOT <= (int)TMEM_COLS && SMEM <= 232448, "memories");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const int w_bytes = p.rows * BK, x_bytes = p.bn * BK, stage_bytes = KPS * (w_bytes + x_bytes);
  // an MMA reads 128 rows from a stage's weights on, past a smaller tile's into what follows
  const uint32_t sW = base, sX = base + p.stages * KPS * w_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + RING);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto full_bar = [&](int s) { return smem_u32(bars + s); };
  auto empty_bar = [&](int s) { return smem_u32(bars + MAX_STAGES + s); };
  auto tfull_bar = [&](int b) { return smem_u32(bars + 2 * MAX_STAGES + b); };
  auto tempty_bar = [&](int b) { return smem_u32(bars + 2 * MAX_STAGES + 2 + b); };
  auto sfull_bar = [&](int b) { return smem_u32(bars + 2 * MAX_STAGES + 4 + b); };
  auto sempty_bar = [&](int b) { return smem_u32(bars + 2 * MAX_STAGES + 4 + SLOTS + b); };
  const uint32_t drain_bar = smem_u32(bars + BARS - 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = SPLIT ? p.split : 1, rank = SPLIT ? (int)cta_rank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), ISSUERS);
      mbar_init(tempty_bar(b), EPI_WARPS);
    }
    for (int b = 0; b < SLOTS; ++b) {
      mbar_init(sfull_bar(b), SCALE_WARPS);
      mbar_init(sempty_bar(b), ISSUERS);
    }
    mbar_init(drain_bar, ISSUERS);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == ISSUER0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == PRODUCER && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // waited for where blocks first reach into one another's memory
  if (SPLIT) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  wait_for_last_kernel();
  const uint32_t tmem = *tmem_slot;
  const int tiles = p.n_tiles * p.t_tiles;
  const int tile0 = blockIdx.x / split, tile_step = gridDim.x / split;
  const int KB = p.g.KB;
  const int kb0 = (int)((int64_t)KB * rank / split), kb1 = (int)((int64_t)KB * (rank + 1) / split), kn = kb1 - kb0;

  if (warp == PRODUCER) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, issued = 0, issued_ph = 0;
      bool ok = true;
      for (int tile = tile0; ok && tile < tiles; tile += tile_step) {
        const int n0 = (tile % p.n_tiles) * p.rows, t0 = (tile / p.n_tiles) * p.bn;
        for (int kb = kb0; kb < kb1; kb += KPS) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.status, ST_F8_PRODUCER, WAIT_LIMIT_NS)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(full_bar(s), (uint32_t)stage_bytes);
#pragma unroll
          for (int i = 0; i < KPS; ++i) {  // past the split's last K block too: the stage is whole
            tma_load_2d(sW + (s * KPS + i) * w_bytes, &tmB, (kb + i) * BK, n0, full_bar(s));
            tma_load_2d(sX + (s * KPS + i) * x_bytes, &tmA, (kb + i) * BK, t0, full_bar(s));
          }
          issued |= 1u << s;
          issued_ph = (issued_ph & ~(1u << s)) | (ph << s);
          if (++s == p.stages) s = 0, ph ^= 1u;
        }
      }
      // copies that no MMA waits for any more land before the block exits
      if (!ok)
        for (int t = 0; t < p.stages; ++t)
          if (issued & (1u << t)) drain_wait(full_bar(t), (issued_ph >> t) & 1u);
    }
  } else if (warp >= ISSUER0) {
    // The whole warp, so that addresses and descriptors stay in uniform registers; one
    // lane issues.  Each issuer has every other stage of the ring, and so sees every
    // phase of its stages' barriers.
    const int which = warp - ISSUER0;
    const int one = lane == 0;
    int s = which, unit = 0;
    uint32_t ph = 0;
    unsigned slot = 0;
    bool ok = true;
    for (int tile = tile0; ok && tile < tiles; tile += tile_step, ++unit) {
      const int buf = unit % ACCS;
      if (!warp_wait(tempty_bar(buf), ((unit / ACCS) & 1) ^ 1u, abort_flag, p.status, ST_F8_MMA, WAIT_LIMIT_NS)) break;
      tc_fence_after();
      const uint32_t d = tmem + (buf * ISSUERS + which) * BN;
      const int first = (which ^ first_issuer<KPS>(unit, kn)) * KPS;  // K block of this issuer's first stage
      uint32_t sums_there = 0;
      for (int kb = 0; ok && kb < kn; kb += 4, ++slot) {  // one slot of scales
        const uint32_t sb = tmem + SCALES + (slot % SLOTS) * SLOT;
        if (!warp_wait(sfull_bar(slot % SLOTS), (slot / SLOTS) & 1, abort_flag, p.status, ST_F8_MMA, WAIT_LIMIT_NS)) {
          ok = false;
          break;
        }
#pragma unroll
        for (int h0 = 0; h0 < 4; h0 += KPS * ISSUERS) {  // one stage
          const int h = h0 + first;
          if (kb + h >= kn) break;
          if (!warp_wait(full_bar(s), ph, abort_flag, p.status, ST_F8_MMA, WAIT_LIMIT_NS)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t dw = sw128_desc(sW + s * KPS * w_bytes), dx = sw128_desc(sX + s * KPS * x_bytes);
#pragma unroll
          for (int i = 0; i < KPS; ++i) {
            if (kb + h + i >= kn) break;
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              mma(one, d, dw + (uint64_t)(i * (w_bytes >> 4) + 2 * k), dx + (uint64_t)(i * (x_bytes >> 4) + 2 * k),
                  idesc(BM, p.bn, h + i), sb + 8, sb, i + k > 0 ? 1u : sums_there);
          }
          sums_there = 1;
          commit(one, empty_bar(s));
          if ((s += ISSUERS) >= p.stages) s = which, ph ^= 1u;
        }
        if (ok) commit(one, sempty_bar(slot % SLOTS));
      }
      if (ok) commit(one, tfull_bar(buf));
    }
    commit(one, drain_bar);
    if (one) drain_wait(drain_bar, 0);
  } else if (warp >= SCALE_WARP0) {
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + SCALES;
    const int last = (p.g.N - 1) / F8_BLOCK;
    auto load = [&](int tile, int kb, uint32_t (&w)[4], uint32_t (&x)[BN / 32]) {
      const int n0 = (tile % p.n_tiles) * p.rows, t0 = (tile / p.n_tiles) * p.bn;
      const bool whole = (kb & 3) == 0;
      scale_words(w, [&](int i) { return p.g.sb + (int64_t)min((n0 + 32 * i + lane) / F8_BLOCK, last) * KB; }, kb, KB,
                  p.words_b && whole);
      scale_words(x, [&](int i) { return p.g.sa + (int64_t)min(t0 + 32 * i + lane, p.g.M - 1) * KB; }, kb, KB,
                  p.words_a && whole);
    };
    unsigned slot = 0;
    bool ok = true;
    uint32_t w[4], x[BN / 32];
    load(tile0, kb0, w, x);
    for (int tile = tile0; ok && tile < tiles; tile += tile_step) {
      for (int kb = kb0; kb < kb1; kb += 4, ++slot) {
        uint32_t w_next[4], x_next[BN / 32];
        const bool more = kb + 4 < kb1;
        load(more || tile + tile_step >= tiles ? tile : tile + tile_step, more ? kb + 4 : kb0, w_next, x_next);
        if (!warp_wait(sempty_bar(slot % SLOTS), ((slot / SLOTS) & 1) ^ 1u, abort_flag, p.status, ST_F8_SCALES,
                       WAIT_LIMIT_NS)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t at = lanes + (slot % SLOTS) * SLOT;
        tmem_st4(at + 8, w);
#pragma unroll
        for (int i = 0; i < BN / 32; ++i) tmem_st1(at + i, x[i]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sfull_bar(slot % SLOTS));
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = w_next[i];
#pragma unroll
        for (int i = 0; i < BN / 32; ++i) x[i] = x_next[i];
      }
    }
  } else {
    int unit = 0;
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const int r = warp * 32 + lane;
    for (int tile = tile0; tile < tiles; tile += tile_step, ++unit) {
      const int n = (tile % p.n_tiles) * p.rows + r, t0 = (tile / p.n_tiles) * p.bn;
      const int buf = unit % ACCS;
      const float bias = p.g.bias && n < p.g.N ? load_as_f32(p.g.bias, p.g.bias_dtype, n) : 0.0f;
      if (!warp_wait(tfull_bar(buf), (unit / ACCS) & 1, abort_flag, p.status, ST_F8_EPILOGUE, WAIT_LIMIT_NS)) break;
      tc_fence_after();
      if constexpr (!SPLIT) {
        const int t1 = min(p.bn, p.g.M - t0);
        // of a tile of one stage one accumulator has sums
        const int acc0 = (buf * ISSUERS + (kn > KPS ? 0 : first_issuer<KPS>(unit, kn))) * BN;
        if (warp * 32 < p.rows)
#pragma unroll 1
          for (int c = 0; c < t1; c += 32) {
            float v[32];
            sums<BN>(lanes + (uint32_t)(acc0 + c), kn > KPS, v);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += bias;
            if (r < p.rows && n < p.g.N)
              typed(p.g, [&](auto* out) { store32(out + (int64_t)(t0 + c) * p.g.ld_out + n, p.g.ld_out, t1 - c, v); });
          }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(buf));
      }
    }
  }

  if constexpr (SPLIT) {
    // one tile per cluster
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    tc_fence_after();
    const int n0 = (tile0 % p.n_tiles) * p.rows, t0 = (tile0 / p.n_tiles) * p.bn, t1 = min(p.bn, p.g.M - t0);
    const int per = join_per(p.bn, split);
    if (warp < EPI_WARPS && __all_sync(0xffffffffu, !*abort_flag)) {
      const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
      const int r = warp * 32 + lane;
      // rank d finishes tokens [d per, (d + 1) per): sums as [source][four tokens][row]
#pragma unroll 1
      for (int c = 0; c < t1; c += 32) {
        float v[32];
        sums<BN>(lanes + (uint32_t)c, kn > KPS, v);
        if (r < p.rows) {
          int d = c / per, at = c - d * per;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            if (c + j >= p.bn) break;  // past the last rank's
            st_cluster_f32x4(mapa(base + (uint32_t)(p.join + ((rank * per + at) * BM + 4 * r) * 4), (uint32_t)d), v[j],
                             v[j + 1], v[j + 2], v[j + 3]);
            if ((at += 4) >= per) at -= per, ++d;
          }
        }
      }
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const float* part = reinterpret_cast<const float*>(sm + p.join);
    typed(p.g, [&](auto* out) {
      using T = std::remove_pointer_t<decltype(out)>;
      for (int i = threadIdx.x; i < per / 4 * BM; i += THREADS) {  // four tokens of a row
        const int r = i & (BM - 1), c = i / BM * 4;
        const int t = rank * per + c, n = n0 + r;
        if (t >= t1 || r >= p.rows || n >= p.g.N) continue;
        float y[4] = {0, 0, 0, 0};
        for (int s = 0; s < split; ++s) {
          const float4 v = *reinterpret_cast<const float4*>(part + (s * per + c) * BM + 4 * r);
          y[0] += v.x;
          y[1] += v.y;
          y[2] += v.z;
          y[3] += v.w;
        }
        const float bias = p.g.bias ? load_as_f32(p.g.bias, p.g.bias_dtype, n) : 0.0f;
        T* to = out + (int64_t)(t0 + t) * p.g.ld_out + n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (t + j < t1) to[j * p.g.ld_out] = Elem<T>::from_f32(y[j] + bias);
      }
    });
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == ISSUER0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

}  // namespace few

// Codes [rows, K] -> boxes of `box` rows x 128 columns, 128-byte swizzle, zeros outside.
int code_map8(CUtensorMap* map, const uint8_t* q, int64_t rows, int64_t K, int64_t ld, int box) {
  EncodeTiledFn fn = encode_fn();
  QI8_REQUIRE(fn, QI8_ECUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t boxes[2] = {(cuuint32_t)BK, (cuuint32_t)box}, one[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(q), dims, strides, boxes, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  QI8_REQUIRE(r == CUDA_SUCCESS, QI8_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return QI8_OK;
}

// Scale rows that can be read a word at a time.
bool word_rows(const uint8_t* s, int KB) { return KB % 4 == 0 && reinterpret_cast<uintptr_t>(s) % 4 == 0; }

int launch_pair(const F8Gemm& g, cudaStream_t st) {
  static bool done[64];
  int dev = 0;
  QI8_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !done[dev]) {
    QI8_CUDA(cudaFuncSetAttribute(pair::gemm_f8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, pair::SMEM));
    if (dev < 64) done[dev] = true;
  }
  // Features per tile, by the last wave: a K block takes 2 cycles per feature, or what
  // issuing its MMAs takes, a tile about 1500 more.  512 x 10240 x 4096 takes 25.4 us in
  // tiles of 160, 27.7 in tiles of 256; 1024 x 4096 x 4096 17.2 with 256, 24 with 224 (a
  // second wave).  Halves of a tile that are no whole 16s are slower than these.
  int bn = 256;
  double best = 1e300;
  for (int n = 256; n >= 128; n -= 32) {
    const int64_t tiles = (int64_t)((g.M + 255) / 256) * ((g.N + n - 1) / n);
    const int64_t waves = (2 * tiles + sm_count() - 1) / sm_count();
    const double cycles = (double)waves * ((n < 160 ? 320 : 2 * n) * (double)g.KB + 1500.0);
    if (cycles < best) best = cycles, bn = n;
  }
  CUtensorMap ma, mb;
  if (int rc = code_map8(&ma, g.a, g.M, g.K, g.ld_a, 128)) return rc;
  if (int rc = code_map8(&mb, g.b, g.N, g.K, g.ld_b, bn / 2)) return rc;
  pair::Args p{g, (g.M + 255) / 256, (g.N + bn - 1) / bn, bn, word_rows(g.sa, g.KB), word_rows(g.sb, g.KB),
               rows_aligned(g.out, g.ld_out, elem_size(g.out_dtype), 16), device_status_ptr()};
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  QI8_REQUIRE(tiles < (1 << 30), QI8_ESHAPE, "%lld output tiles", (long long)tiles);
  const int64_t pairs = tiles < sm_count() / 2 ? tiles : sm_count() / 2;
  return launch_early("gemm_f8_pair_kernel launch", pair::gemm_f8_pair_kernel, dim3((unsigned)(2 * pairs)), pair::THREADS,
                      pair::SMEM, 1, st, ma, mb, p);  // its clusters are in its attributes
}

template <int BN, bool SPLIT>
int launch_few(const F8Gemm& g, int rows, int split, cudaStream_t st) {
  static bool done[64];
  int dev = 0;
  QI8_CUDA(cudaGetDevice(&dev));
  auto kern = few::gemm_f8_few_kernel<BN, SPLIT>;
  if (dev >= 64 || !done[dev]) {
    QI8_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, few::SMEM));
    if (dev < 64) done[dev] = true;
  }
  const int t_tiles = (g.M + BN - 1) / BN, bn = ((g.M + t_tiles - 1) / t_tiles + 15) & ~15;
  CUtensorMap ma, mb;
  if (int rc = code_map8(&ma, g.a, g.M, g.K, g.ld_a, bn)) return rc;
  if (int rc = code_map8(&mb, g.b, g.N, g.K, g.ld_b, rows)) return rc;
  const int join = SPLIT ? split * few::BM * few::join_per(bn, split) * 4 : 0;
  int stages = (few::RING - join) / (few::kps(BN) * (rows + bn) * BK) / few::ISSUERS * few::ISSUERS;
  if (stages > few::MAX_STAGES) stages = few::MAX_STAGES;
  QI8_REQUIRE(stages >= few::ISSUERS, QI8_ESHAPE, "no room for two stages");
  few::Args p{g, rows, (g.N + rows - 1) / rows, t_tiles, split, stages, bn, few::RING - join, word_rows(g.sa, g.KB),
              word_rows(g.sb, g.KB), device_status_ptr()};
  const int64_t tiles = (int64_t)p.n_tiles * p.t_tiles;
  QI8_REQUIRE(tiles < (1 << 30), QI8_ESHAPE, "%lld output tiles", (long long)tiles);
  const int64_t blocks = SPLIT ? tiles * split : tiles < sm_count() ? tiles : sm_count();
  return launch_early("gemm_f8_few_kernel launch", kern, dim3((unsigned)blocks), few::THREADS, few::SMEM, split, st, ma, mb,
                      p);
}

}  // namespace f8tc
}  // namespace

int gemm_f8_tiles(const F8Gemm& g, cudaStream_t st) {
  using namespace f8tc;
  const int sms = sm_count();
  // Tiles of 128 weight rows and up to 128 tokens, as far as one wave of blocks goes:
  // 512 x 4096 x 4096 takes 14.5 us so and 16.2 in tiles of 256 x 256, 512 x 10240 x
  // 4096 (320 tiles) 37 and 30.  Up to 128 tokens half of a 256-token tile would be
  // empty: 100 x 32768 x 4096 takes 30.1 us so and 32.5 in those.
  const int64_t t_tiles = ((int64_t)g.M + 127) / 128, n_tiles = ((int64_t)g.N + 127) / 128;
  if (g.M > 128 && n_tiles * t_tiles > sms) return launch_pair(g, st);
  // Blocks that share a tile's K: a K block takes 0.21 us up to 64 tokens and 0.27 with
  // 128, or what the weight takes from HBM, the join 1.4 us and 0.003 for each token and
  // block.  Fitted to 21 shapes of 9 to 256 tokens, of which it misses the best choice in
  // two, by 5 % at most (64 x 4224 x 8192 and x 10240, beside them, by 6): 16 x 4096 x 4096
  // takes 8.7 us with whole tiles, 7.4 with two blocks each and 7.0 with four, 100 x 4096 x
  // 10240 21.7, 15.9 and 14.5, 100 x 8192 x 4096 12.2 and, with two, 13.4; 16 x 4224 x 4096
  // 7.4 with two and 7.1 with four.  Of clusters of two 74 run at once on 148 SMs, of four
  // 33, of eight 15; three blocks were never faster than two or four.
  const int bn = (int)((g.M + t_tiles - 1) / t_tiles + 15) & ~15;
  const double block_us = bn <= 64 ? 0.21 : 0.21 + 0.06 / 64 * (bn - 64), read_us = (double)g.N * g.K / 5.5e6;
  int split = 1, room = sms;
  double best = fmax(g.KB * block_us, read_us);
  for (int s : {2, 4, 8}) {
    const int there = s == 2 ? sms : s == 8 ? sms * 30 / 37 : sms * 33 / 37;
    const double us = fmax((g.KB + s - 1) / s * block_us, read_us) + 1.4 + 0.003 * bn * s;
    if (s <= g.KB && n_tiles * t_tiles * s <= there && us < best) best = us, split = s, room = there;
  }
  // as few rows per tile as spread them over the SMs in as many waves
  const int64_t waves = (n_tiles * t_tiles * split + room - 1) / room, most = waves * room / (t_tiles * split);
  const int least = split > 1 ? 64 : 32;
  int rows = (int)(((int64_t)g.N + most - 1) / most + 15) & ~15;
  rows = rows < least ? least : rows > 128 ? 128 : rows;
  const auto launch = split > 1 ? bn <= 32 ? launch_few<32, true> : bn <= 64 ? launch_few<64, true> : launch_few<128, true>
                      : bn <= 32 ? launch_few<32, false> : bn <= 64 ? launch_few<64, false> : launch_few<128, false>;
  return launch(g, rows, split, st);
}

}  // namespace qi8
