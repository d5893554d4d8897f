// The streaming engine of the products with few tokens: 4-bit weights are read
// once, at the rate of HBM, and everything else hides behind that.
//
// One block per SM works through a list of tasks.  A task is MT tiles of up to
// 16 weight rows, all of K, against up to 8 NT activation rows.
//   producer warp   one TMA box per tile and segment of 16 blocks of 128 features
//                   (1 KB a row) into a ring of STAGES: pieces of 1 KB keep DRAM
//                   pages open (64 bytes per row and step, the size of one block,
//                   reached 0.9 TB/s, one bulk copy per row 2.6)
//   W warps         one block each of a segment: 16 bytes per row and thread from
//                   the ring, unpacked in registers, mma.sync m16n8k16 with the
//                   rows as M and the tokens as N; fp32 sums of the whole task
//                   stay in registers, then go to a buffer in shared memory
//   finishing warps add the W sums in order and do what the task is for
// Nothing waits for the whole block: ring and buffers have full and empty
// barriers.  Blocks of K rotate over the warps from task to task, so that a K of
// 17 blocks does not cost two rounds of 16.
//
// Scales are read straight from global memory one step ahead; the producer has
// prefetched their sectors into L2 when it issued the segment's copies.
#pragma once

#include "common.cuh"
#include "int4.cuh"
#include "tc05.cuh"

namespace qi8 {
namespace {
namespace stream {

constexpr int SEG = 16;                      // blocks of 128 features per segment
constexpr int FINISH_WARPS = 2;
constexpr int COL_PITCH = 20;                // floats per column of a tile's sums (16 rows), conflict-free

template <int MT, int NT, int W> struct Cfg {
  static constexpr int STAGE_BYTES = 16 * MT * SEG * 64;
  static constexpr int STAGES = MT == 1 ? 8 : 4;
  static constexpr int TILE = 8 * NT * COL_PITCH;                // floats of one warp's sums of one tile
  static constexpr int SUM_BYTES = W * MT * TILE * 4;
  static constexpr int BARS = 2 * STAGES + 4;
  static constexpr int SMEM = 128 + STAGES * STAGE_BYTES + 2 * SUM_BYTES + BARS * 8 + 16;
  static constexpr int THREADS = (W + 1 + FINISH_WARPS) * 32;
};

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr)
               : "memory");
  return v;
}
// the finishing warps among themselves
__device__ __forceinline__ void finish_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(FINISH_WARPS * 32) : "memory");
}

// true when it is for all of them: after a wait has expired they leave together
__device__ __forceinline__ bool finish_vote(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)ok), "n"(FINISH_WARPS * 32)
      : "memory");
  return all != 0;
}

// Height of the tiles of `rows` rows, as equal as they can be, at most 16.
__host__ __device__ inline int tile_height(int rows, int mt) {
  const int tasks = (rows + 16 * mt - 1) / (16 * mt);
  return tasks ? (rows + tasks * mt - 1) / (tasks * mt) : 0;
}

// J: struct of static constants MT, NT, W, G, VEC, type T and
//   J(args)                        in every thread, after the kernel has started
//   int tasks(), int KB(), int K(), int height()   weight rows per tile
//   const __nv_bfloat16* scales()
//   int rows()                                     of the whole weight
//   int row(int j, int mt)                         first weight row of tile mt; a tile may pass
//                                                  the weight's end (zeros), not its start
//   const uint16_t* activation(int j, int col)     any row where there is no token
//   void finish(int j, const float* sums, int tid)   by 32 FINISH_WARPS threads
//   void finish_all(int tid)                         after the last task
template <typename J>
__device__ __forceinline__ void run(J& job, const CUtensorMap* codes, uint8_t* smem_raw, unsigned int* status) {
  constexpr int MT = J::MT, NT = J::NT, W = J::W, G = J::G;
  using C = Cfg<MT, NT, W>;
  using T = typename J::T;
  constexpr int NS = W4_BLOCK / G;
  uint8_t* smem = smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u);
  float* sums = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE_BYTES + 2 * C::SUM_BYTES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + C::BARS);
  const uint32_t ring = smem_u32(smem);
  auto full = [&](int s) { return smem_u32(bars + s); };
  auto empty = [&](int s) { return smem_u32(bars + C::STAGES + s); };
  auto sfull = [&](int b) { return smem_u32(bars + 2 * C::STAGES + b); };
  auto sempty = [&](int b) { return smem_u32(bars + 2 * C::STAGES + 2 + b); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), W);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(sfull(b), W);
      mbar_init(sempty(b), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const int tasks = job.tasks(), KB = job.KB(), height = job.height();
  const uint32_t pitch = (uint32_t)min(SEG, KB) * 64u;
  // every block starts at another segment, or all would ask the same L2 slices for
  // the same activations at the same time
  const int segs = (KB + SEG - 1) / SEG;
  auto segment = [&](int i) { return (int)((blockIdx.x + (unsigned)i) % (unsigned)segs) * SEG; };

  if (warp == W) {
    // ------------------------------------------------------------ producer
    int s = 0;
    uint32_t ph = 0, issued = 0, issued_ph = 0;
    bool ok = true;
    for (int j = 0; ok && j < tasks; ++j) {
      for (int i = 0; i < segs; ++i) {
        const int kb = segment(i);
        if (!warp_wait(empty(s), ph ^ 1u, abort_flag, status, ST_W4_PRODUCER, WAIT_LIMIT_NS)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(full(s), pitch * (uint32_t)(height * MT));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            tma_load_2d(ring + s * C::STAGE_BYTES + (uint32_t)(mt * 16) * pitch, codes, kb * 16, job.row(j, mt),
                        full(s));
        }
        // the segment's scales into L2
        for (int i = lane; i < 16 * MT; i += 32)
          if ((i & 15) < height) {
            const __nv_bfloat16* sc =
                job.scales() + ((int64_t)min(job.row(j, i >> 4) + (i & 15), job.rows() - 1) * KB + kb) * NS;
            prefetch_l2(sc);
            if (G < 128) prefetch_l2(sc + min(SEG, KB - kb) * NS - 1);
          }
        issued |= 1u << s;
        issued_ph = (issued_ph & ~(1u << s)) | (ph << s);
        if (++s == C::STAGES) s = 0, ph ^= 1u;
      }
    }
    if (!ok)
      for (int t = 0; t < C::STAGES; ++t)
        if (issued & (1u << t)) drain_wait(full(t), (issued_ph >> t) & 1u);
  } else if (warp < W) {
    // ------------------------------------------------------------ products
    const int g = lane >> 2, a = lane & 3;
    uint32_t at_row[2 * MT];  // of the thread's rows in a stage
#pragma unroll
    for (int r = 0; r < 2 * MT; ++r)
      at_row[r] = (uint32_t)((r >> 1) * 16 + min((r & 1) * 8 + g, height - 1)) * pitch + a * 16;
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int j = 0; ok && j < tasks; ++j) {
      const uint16_t* x[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) x[nt] = job.activation(j, nt * 8 + g) + 8 * a;
      const __nv_bfloat16* sc[2 * MT];
#pragma unroll
      for (int r = 0; r < 2 * MT; ++r)
        sc[r] = job.scales() +
                (int64_t)min(job.row(j, r >> 1) + min((r & 1) * 8 + g, height - 1), job.rows() - 1) * KB * NS;
      // this warp's block of a segment: the one with (block + j KB) % W == warp
      const int mine = (int)(((unsigned)warp - (unsigned)j * (unsigned)KB) % W);
      float sum[MT][NT][4] = {};
      W4Frag<G, MT> f;
      auto load_scales = [&](int kb) {
        if (kb < KB)
#pragma unroll
          for (int r = 0; r < 2 * MT; ++r) f.load_scale(r, sc[r] + kb * NS);
      };
      load_scales(segment(0) + mine);
      for (int i = 0; i < segs; ++i) {
        const int kb0 = segment(i), next0 = i + 1 < segs ? segment(i + 1) : KB;
        if (!warp_wait(full(s), ph, abort_flag, status, ST_W4_UNPACK, WAIT_LIMIT_NS)) {
          ok = false;
          break;
        }
        // SEG / W blocks of the segment, W apart
#pragma unroll
        for (int part = 0; part < SEG / W; ++part) {
          const int kb = kb0 + mine + part * W;
          const bool have = kb < KB;
          if (have) {
            const uint32_t at = ring + s * C::STAGE_BYTES + (mine + part * W) * 64;
#pragma unroll
            for (int r = 0; r < 2 * MT; ++r) f.w[r] = ld_shared16(at + at_row[r]);
          }
          if (part == SEG / W - 1) {
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(s));
          }
          const W4Frag<G, MT> now = f;
          load_scales(part + 1 < SEG / W ? kb + W : next0 + mine);
          if (!have) continue;
          // columns without a token repeat the last one; nobody reads them
          if (J::VEC && (kb + 1) * W4_BLOCK <= job.K())
            w4_block<T, G, MT, NT>(now, sum, [&](int nt, int b) {
              return __ldg(reinterpret_cast<const uint4*>(x[nt] + kb * W4_BLOCK + b * 32));
            });
          else
            w4_block<T, G, MT, NT>(now, sum, [&](int nt, int b) {
              return ld_act8<J::VEC>(x[nt] - 8 * a, kb * W4_BLOCK + b * 32 + a * 8, job.K());
            });
        }
        if (++s == C::STAGES) s = 0, ph ^= 1u;
      }
      if (!ok) break;
      const int buf = j & 1;
      if (!warp_wait(sempty(buf), ((j >> 1) & 1) ^ 1u, abort_flag, status, ST_W4_UNPACK, WAIT_LIMIT_NS)) break;
      float* out = sums + (buf * W + warp) * MT * C::TILE;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            out[mt * C::TILE + (nt * 8 + 2 * a + (i & 1)) * COL_PITCH + g + 8 * (i >> 1)] = sum[mt][nt][i];
      __syncwarp();
      if (lane == 0) mbar_arrive(sfull(buf));
    }
  } else {
    // ----------------------------------------------------------- finishing
    const int tid = threadIdx.x - (W + 1) * 32;
    bool ok = true;
    for (int j = 0; j < tasks; ++j) {
      const int buf = j & 1;
      ok = finish_vote(tid != 0 || mbar_wait(sfull(buf), (j >> 1) & 1, abort_flag, status, ST_W4_EPILOGUE, WAIT_LIMIT_NS));
      if (ok) job.finish(j, sums + buf * W * MT * C::TILE, tid);
      finish_sync();
      if (tid == 0) mbar_arrive(sempty(buf));
    }
    if (ok) job.finish_all(tid);
  }
}

}  // namespace stream
}  // namespace
}  // namespace qi8
