// Products of fp8 operands with block scales for single tokens (format: f8.cuh),
// on m16n8k32 steps fed from shared memory.
//
// A thread block computes 16 features.  One warp copies the weight rows, 1024
// columns at a time, into a ring that holds a row of 4096 columns as a whole; eight
// warps take one block of 128 columns of each such piece and add up in the order of
// the warps.  The tokens' codes lie in shared memory as a whole, copied or, for few
// of them, quantized here while the weight is on its way.  Rows are 16 bytes longer
// than whole 128s, so that eight of them read as one ldmatrix row block touch all
// banks once.
//
// Against the tcgen05 kernel this one starts sooner (no tensor memory, maps or
// scales to set up), but every block reads the tokens, up to eight, beside its 16
// weight rows, and none shares its K with others.  1 x 4096 x 4096 with its quantization
// takes 5.9 us with the weight from HBM: launch, one latency of HBM and the join of
// eight warps stand beside 2.6 us of reading.
#include <cstdint>

#include "f8.cuh"
#include "tc05.cuh"

namespace qi8 {
namespace {
namespace f8r {

constexpr int ROWS = 16, MOST_TOKENS = 8, WARPS = 8, COPIER = WARPS, THREADS = (WARPS + 1) * 32;
constexpr int PIECE = WARPS * F8_BLOCK;           // columns of K per stage
constexpr int PIECE_PITCH = PIECE + 16, STAGE = ROWS * PIECE_PITCH;
constexpr int MAX_STAGES = 4;
constexpr int SM_SMEM = 228 * 1024;
constexpr int STATIC_SMEM = 6000;  // of a block beside its ring and tokens, rounded up
// Largest K, up to four tokens and beyond (gemm_f8_rows_fits).
constexpr int FEW_TOKENS = 4, FEW_K = 5120, MOST_K = 2560;

// Bytes between tokens in shared memory, and of all of them with their scales.
constexpr int pitch_for(int KB) { return KB * F8_BLOCK + 16; }
constexpr int tokens_for(int M, int KB) { return M * (pitch_for(KB) + KB); }
// Two blocks of any size share an SM.
static_assert(MAX_STAGES * STAGE + tokens_for(FEW_TOKENS, FEW_K / F8_BLOCK) <= SM_SMEM / 2 - STATIC_SMEM &&
                  MAX_STAGES * STAGE + tokens_for(MOST_TOKENS, MOST_K / F8_BLOCK) <= SM_SMEM / 2 - STATIC_SMEM,
              "shared memory");

struct Args {
  F8Gemm g;
  const void* x;  // tokens to quantize, in place of codes
  int64_t ld_x;
  bool vec_x;
  int stages, x_pitch;
  bool after_quant;
  unsigned int* status;
};

// D[16, 8] += A[16, 32] B[32, 8], e4m3, fp32 sums
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four blocks of eight rows x 16 bytes; lane l gives the address of row l % 8 of block l / 8.
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Contiguous bytes, whole 16s, global to shared memory.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// Of the four codes in a word, those at columns below K.
__device__ __forceinline__ uint32_t below(uint32_t w, int k, int K) {
  const int left = K - k;
  return left >= 4 ? w : left <= 0 ? 0u : w & ((1u << (8 * left)) - 1u);
}

// 2^(ea + eb) for two scale bytes as two factors of about half the exponent each:
// multiplied one after the other they overflow, or vanish, only where the result does.
__device__ __forceinline__ float2 both_scales(uint32_t a, uint32_t b) {
  if (a == 255u || b == 255u) return make_float2(__uint_as_float(0x7fffffffu), 1.0f);
  const int e = (int)(a + b) - 254, h = e >> 1;
  return make_float2(__uint_as_float((uint32_t)(h + 127) << 23), __uint_as_float((uint32_t)(e - h + 127) << 23));
}

template <typename X>  // uint8_t: codes
__global__ void __launch_bounds__(THREADS) gemm_f8_rows_kernel(const __grid_constant__ Args p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float part[WARPS][ROWS][MOST_TOKENS + 1];
  __shared__ __align__(16) uint8_t zeros[F8_BLOCK];
  __shared__ uint64_t bars[2 * MAX_STAGES];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * ROWS, M = p.g.M, K = p.g.K, KB = p.g.KB;
  const int pieces = (K + PIECE - 1) / PIECE;
  const uint32_t ring = smem_u32(smem);
  uint8_t* codes = smem + p.stages * STAGE;
  uint8_t* scales = codes + M * p.x_pitch;  // [KB][M]
  auto full_bar = [&](int s) { return smem_u32(bars + s); };
  auto empty_bar = [&](int s) { return smem_u32(bars + MAX_STAGES + s); };
  if (threadIdx.x == COPIER * 32) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), WARPS);
    }
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < F8_BLOCK / 4) reinterpret_cast<uint32_t*>(zeros)[threadIdx.x] = 0;
  __syncthreads();

  // one piece of the block's rows into a stage; lane = row
  const uint8_t* my_row = p.g.b + (int64_t)min(n0 + lane, p.g.N - 1) * p.g.ld_b;
  auto copy_piece = [&](int i, int s) {
    const int k = i * PIECE, bytes = min(PIECE, (K - k + 15) & ~15);
    if (lane == 0) mbar_arrive_expect_tx(full_bar(s), ROWS * bytes);
    __syncwarp();
    if (lane < ROWS) bulk_copy(ring + s * STAGE + lane * PIECE_PITCH, my_row + k, bytes, full_bar(s));
  };
  if (warp == COPIER) {
    if (!p.after_quant) pdl_wait();
    for (int i = 0; i < pieces && i < p.stages; ++i) copy_piece(i, i);
  }

  // the tokens, by all warps but that one
  if (warp < WARPS) {
    wait_for_last_kernel();
    if constexpr (std::is_same<X, uint8_t>::value) {
      const int per = KB * (F8_BLOCK / 16);
      for (int i = threadIdx.x; i < M * per; i += WARPS * 32) {
        const int t = i / per, k = (i - t * per) * 16;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k < K) v = __ldg(reinterpret_cast<const uint4*>(p.g.a + t * p.g.ld_a + k));
        if (k + 16 > K) v = make_uint4(below(v.x, k, K), below(v.y, k + 4, K), below(v.z, k + 8, K), below(v.w, k + 12, K));
        *reinterpret_cast<uint4*>(codes + t * p.x_pitch + k) = v;
      }
      for (int i = threadIdx.x; i < M * KB; i += WARPS * 32) {
        const int t = i / KB, kb = i - t * KB;
        scales[kb * M + t] = __ldg(p.g.sa + i);
      }
    } else {
      // eight columns per lane, 16 lanes per block of 128
      const int per = KB * 16;
      for (int i0 = 0; i0 < M * per; i0 += WARPS * 32) {
        const int i = i0 + threadIdx.x, t = i / per, k = (i - t * per) * 8;
        const bool live = t < M;
        Eight<X> e;
        const X* row = static_cast<const X*>(p.x) + (live ? t : 0) * p.ld_x;
        if (live && p.vec_x && k + 8 <= K) e.load(row + k);
        else e.load_some(row, k, live ? K : 0);
        const F8x f = e.get();
        const uint32_t code = f8_scale_code(max16(amax_bits(f)));
        if (!live) continue;
        *reinterpret_cast<uint2*>(codes + t * p.x_pitch + k) = f8_codes(f, f8_inverse(code));
        if ((lane & 15) == 0) scales[k / F8_BLOCK * M + t] = (uint8_t)code;
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
  }

  if (warp == COPIER) {
    int s = 0, sent = p.stages;
    uint32_t ph = 0;
    for (; sent < pieces; ++sent) {
      if (!warp_wait(empty_bar(s), ph, abort_flag, p.status, ST_F8_PRODUCER, WAIT_LIMIT_NS)) break;
      copy_piece(sent, s);
      if (++s == p.stages) s = 0, ph ^= 1u;
    }
    // nobody may be waiting any more, but what is on its way lands before the block exits
    for (int j = sent - p.stages; j < sent; ++j) drain_wait(full_bar(j % p.stages), (j / p.stages) & 1u);
  } else {
    float acc[4] = {};
    // rows and 16-byte halves of an A block: (0..7, 0), (8..15, 0), (0..7, 1), (8..15, 1)
    const uint32_t a_at = (uint32_t)((lane & 15) * PIECE_PITCH + warp * F8_BLOCK + (lane >> 4) * 16);
    const uint8_t* sw = p.g.sb + (int64_t)(n0 / F8_BLOCK) * KB;
    int s = 0;
    uint32_t ph = 0;
    for (int i = 0; i < pieces; ++i) {
      const int kb = i * WARPS + warp;
      const bool mine = kb < KB;
      const uint32_t w_scale = mine ? __ldg(sw + kb) : 127u;
      if (!warp_wait(full_bar(s), ph, abort_flag, p.status, ST_F8_MMA, WAIT_LIMIT_NS)) break;
      if (mine) {
        uint32_t a[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) ldmatrix4(a[j], ring + s * STAGE + a_at + 32 * j);
        if ((kb + 1) * F8_BLOCK > K) {  // nothing was copied past K's 16 bytes, and those may hold anything
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int h = 0; h < 4; ++h)
              a[j][h] = below(a[j][h], kb * F8_BLOCK + 32 * j + 16 * (h >> 1) + 4 * (lane & 3), K);
        }
        // lane l: token l % 8, 16 bytes l / 8 of 64
        const int tok = lane & 7;
        const uint32_t b_at = (tok < M ? smem_u32(codes + tok * p.x_pitch + kb * F8_BLOCK) : smem_u32(zeros)) + (lane >> 3) * 16;
        uint32_t b[2][4];
        ldmatrix4(b[0], b_at);
        ldmatrix4(b[1], b_at + 64);
        float d[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) mma(d, a[j], b[j >> 1][2 * (j & 1)], b[j >> 1][2 * (j & 1) + 1]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int t = 2 * (lane & 3) + u;
          const float2 f = both_scales(t < M ? scales[kb * M + t] : 127u, w_scale);
          acc[u] = fmaf(d[u] * f.y, f.x, acc[u]);
          acc[u + 2] = fmaf(d[u + 2] * f.y, f.x, acc[u + 2]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty_bar(s));
      if (++s == p.stages) s = 0, ph ^= 1u;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) part[warp][(lane >> 2) + 8 * (j >> 1)][2 * (lane & 3) + (j & 1)] = acc[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * M; i += THREADS) {
    const int t = i / ROWS, r = i % ROWS, n = n0 + r;
    if (n >= p.g.N) continue;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) y += part[k][r][t];
    if (p.g.bias) y += load_as_f32(p.g.bias, p.g.bias_dtype, n);
    store_from_f32(p.g.out, p.g.out_dtype, t * p.g.ld_out + n, y);
  }
}

// Stages of the ring: as many as there are pieces of K, up to four.
int stages_for(int K) {
  const int pieces = (K + PIECE - 1) / PIECE;
  return pieces < MAX_STAGES ? pieces : MAX_STAGES;
}
int smem_for(int M, int K) { return stages_for(K) * STAGE + tokens_for(M, (int)f8_blocks(K)); }

template <typename X>
int launch(const Args& p, int smem, cudaStream_t st) {
  static bool done[64];
  int dev = 0;
  QI8_CUDA(cudaGetDevice(&dev));
  auto kern = gemm_f8_rows_kernel<X>;
  if (dev >= 64 || !done[dev]) {
    QI8_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SM_SMEM / 2));
    if (dev < 64) done[dev] = true;
  }
  // Where most SMs take as many blocks as any, so much shared memory that no more fit:
  // else some SMs get one more and others one less.  1 x 4096 x 4096 (256 blocks, of
  // which three fit an SM) took 6.9 us so and takes 5.9; 2560 x 2560 (160 blocks) is 2 %
  // faster without.
  const int sms = sm_count(), blocks = (p.g.N + ROWS - 1) / ROWS, each = (blocks + sms - 1) / sms;
  const int more = SM_SMEM / (each + 1);
  if (smem < more && each * sms - blocks < sms / 2) smem = more;
  return launch_early("gemm_f8_rows_kernel launch", kern, dim3((unsigned)blocks), THREADS, smem, 1, st, p);
}

}  // namespace f8r
}  // namespace

// Where this kernel is the faster one (cold weights, tcgen05 second): 1 x 4096 x 4096
// 5.7 us and 6.7, 1 x 4096 x 5120 6.5 and 7.6, 2 x 4096 x 4096 5.8 and 6.8, 4 x 4096 x
// 4096 6.7 and 6.9, 8 x 4096 x 4096 7.9 and 6.9, 8 x 2560 x 2560 5.6 and 6.1, 1 x 10240 x
// 2048 8.3 and 6.9, 4 x 2048 x 6144 7.2 and 6.4.  Tokens beyond four cost it steps, many
// blocks their start, and it does not split K.  All blocks have to run at once: 1 x 6144
// x 4096 (three per SM) takes 7.6 us and 8.2, two tokens (two per SM) 10.1 and 8.2.
bool gemm_f8_rows_fits(int M, int N, int K) {
  using namespace f8r;
  if (M > MOST_TOKENS || N > 8192 || K > FEW_K || (M > FEW_TOKENS && (K > MOST_K || (int64_t)N * K > 10500000)))
    return false;
  const int per_sm = SM_SMEM / (smem_for(M, K) + STATIC_SMEM);
  return (N + ROWS - 1) / ROWS <= (per_sm < 7 ? per_sm : 7) * sm_count();
}

int gemm_f8_rows(const F8Gemm& g, const void* x, int x_dtype, int64_t ld_x, bool after_quant, cudaStream_t st) {
  f8r::Args p{g, x, ld_x, x && rows_aligned(x, ld_x, elem_size(x_dtype), 16), f8r::stages_for(g.K),
              f8r::pitch_for(g.KB), after_quant, device_status_ptr()};
  const int smem = f8r::smem_for(g.M, g.K);
  if (!x) return f8r::launch<uint8_t>(p, smem, st);
  switch (x_dtype) {
    case QI8_BF16: return f8r::launch<__nv_bfloat16>(p, smem, st);
    case QI8_F16: return f8r::launch<__half>(p, smem, st);
    default: return f8r::launch<float>(p, smem, st);
  }
}

}  // namespace qi8
