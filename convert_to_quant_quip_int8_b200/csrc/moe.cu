// A mixture-of-experts layer for a few tokens, experts in 4-bit weights
// (format: int4.cuh):
//
//   l = x R^T                        router logits, 64-bit sums
//   S = the top_k largest of l       equal ones: lowest expert first
//   p = softmax(l) on S, divided by its sum if renormalize
//   y = sum_{e in S} p_e D_e (act(G_e x) * (U_e x))
//
// act is SiLU or GELU (erf).  w13 [E, 2 I, H] holds G_e above U_e, w2 [E, H, I]
// is D_e.  Up to 64 tokens run together, so that an expert's weights are read
// once for all of its tokens; longer inputs take several turns.
//
// Five launches, bound by the bytes of the experts in use; each starts while the
// one before it drains (programmatic dependent launch):
//   moe_logits_kernel   a block per expert and eight tokens
//   moe_route_kernel    one block: the choice, its weights, tokens by expert
//   moe_expert_kernel   gate and up: 16 rows of G and of U per warp, h = act(g) * u
//   moe_expert_kernel   down: 32 rows of D per warp, fp32 rows per (token, choice)
//   moe_combine_kernel  y = sum of a token's rows with its weights, in the order of
//                       the choices: no atomics, the same bits every time
// An expert's tokens come in chunks of up to `cap` pairs (token, choice): as many
// as the MMA columns of a task hold.  The warps of a block share a chunk; they
// split K where blocks would be few, the rows otherwise (the activations then come
// from L2 once per block, not once per warp).
//
// h is held as two bf16 numbers (value and remainder, 16 significant bits
// together): rounding it to one would cost as much accuracy as the output's
// own rounding, and the second column of the MMA costs no bytes.  bf16 for fp16
// layers too: h can pass fp16's range, and codes are exact in both types.
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "int4.cuh"

namespace qi8 {
namespace {

constexpr int MOE_TOKENS = 64;  // one bit each in an expert's mask
constexpr int MOE_WARPS = 8;
constexpr int MOE_MAX_EXPERTS = 1024;

// What the route kernel leaves for the others, in the workspace.
struct Route {
  int* n_chunks;  // of all experts with tokens, in the experts' order
  int* expert;    // [chunk]
  int* first;     // [chunk] its first pair
  int* count;     // [chunk] its pairs
  int* token;     // [pair]
  int* pair;      // [token][choice]
  float* weight;  // [token][choice]
};

struct MoeArgs {
  const uint16_t* x;
  int64_t ld_x;
  const void* router;
  int router_dtype;
  const uint8_t* q13;
  const __nv_bfloat16* s13;
  const uint8_t* q2;
  const __nv_bfloat16* s2;
  void* out;
  int64_t ld_out;
  int dtype;
  int T, H, E, I, top_k;
  int renorm, act;
  int cap;         // pairs per chunk
  double* logits;  // [T, E]
  __nv_bfloat16* h;  // [pair][2][Ip]
  float* part;       // [pair][Hp], Hp = H to a multiple of 4
  Route r;
};

// ------------------------------------------------------------------ router
// The choice of experts has to be that of the exact logits, so the sums are
// fp64 (products of 16- or 24-bit factors are exact in it).
constexpr int LOGIT_TOKENS = 8;

// Eight values from k on as fp64, zeros from n on.
template <typename T>
__device__ __forceinline__ void load8_f64(const T* row, bool vec, int k, int n, double (&v)[8]) {
  if (vec && k + 8 <= n) {
    alignas(16) T b[8];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      reinterpret_cast<uint4*>(b)[i] = __ldg(reinterpret_cast<const uint4*>(row + k) + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (double)Elem<T>::to_f32(b[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < n ? (double)Elem<T>::to_f32(row[k + i]) : 0.0;
  }
}

template <typename T, typename R>
__global__ void __launch_bounds__(MOE_WARPS * 32)
moe_logits_kernel(const MoeArgs p) {
  __shared__ double part[LOGIT_TOKENS][MOE_WARPS];
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = blockIdx.x, t0 = blockIdx.y * LOGIT_TOKENS;
  const int tokens = min(LOGIT_TOKENS, p.T - t0);
  const R* w = static_cast<const R*>(p.router) + (int64_t)e * p.H;
  const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)t0 * p.ld_x;
  const bool wvec = aligned16(p.router) && (int64_t)p.H * sizeof(R) % 16 == 0;
  const bool xvec = aligned16(p.x) && p.ld_x % 8 == 0;
  double acc[LOGIT_TOKENS] = {};
  for (int k = threadIdx.x * 8; k < p.H; k += MOE_WARPS * 256) {
    double r[8];
    load8_f64(w, wvec, k, p.H, r);
#pragma unroll
    for (int t = 0; t < LOGIT_TOKENS; ++t) {
      if (t >= tokens) break;
      double v[8];
      load8_f64(x + t * p.ld_x, xvec, k, p.H, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[t] = fma(v[i], r[i], acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < LOGIT_TOKENS; ++t) {
    if (t >= tokens) break;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);
    if (lane == 0) part[t][warp] = acc[t];
  }
  __syncthreads();
  if (threadIdx.x < tokens) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < MOE_WARPS; ++i) sum += part[threadIdx.x][i];
    p.logits[(int64_t)(t0 + threadIdx.x) * p.E + e] = sum;
  }
}

// Order of the logits as unsigned numbers: -0 equals 0, NaN above all.
__device__ __forceinline__ unsigned long long order_key(double v) {
  if (v != v) return ~0ull;
  const long long b = __double_as_longlong(v + 0.0);
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

__device__ __forceinline__ double order_value(unsigned long long key) {
  return __longlong_as_double((long long)(key >> 63 ? key & 0x7fffffffffffffffull : ~key));
}

// One warp chooses for token t; lane l holds the keys of experts l, l + 32, ...
template <int PER_LANE>
__device__ __forceinline__ void choose(const MoeArgs& p, int t, int lane, unsigned long long* mask, int* ids,
                                       float* wts) {
  const double* l = p.logits + (int64_t)t * p.E;
  unsigned long long key[PER_LANE];
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) key[i] = i * 32 + lane < p.E ? order_key(l[i * 32 + lane]) : 0;
  double top = 0.0;
  float total = 0.0f, mine = 0.0f, mine2 = 0.0f;  // of choices lane and lane + 32
  for (int j = 0; j < p.top_k; ++j) {
    unsigned long long best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i)
      if (key[i] > best) best = key[i], at = i;  // the lowest expert of the lane among equal ones
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(best >> 32));
    const bool in_hi = (unsigned)(best >> 32) == hi;
    const unsigned lo = __reduce_max_sync(0xffffffffu, in_hi ? (unsigned)best : 0u);
    const bool in = in_hi && (unsigned)best == lo;
    const int e = (int)__reduce_min_sync(0xffffffffu, in ? (unsigned)(at * 32 + lane) : 0xffffffffu);
    const unsigned long long won = (unsigned long long)hi << 32 | lo;
    const double v = won == ~0ull ? __longlong_as_double(0x7ff8000000000000ll) : order_value(won);
    if (j == 0) top = v;
    if (in && at * 32 + lane == e) {
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i)
        if (i == at) key[i] = 0;
      atomicOr(&mask[e], 1ull << t);
      ids[t * p.top_k + j] = e;
    }
    const float w = expf((float)(v - top));
    total += w;
    if ((j & 31) == lane) (j < 32 ? mine : mine2) = w;
  }
  if (!p.renorm) {
    total = 0.0f;
    for (int e = lane; e < p.E; e += 32) total += expf((float)(l[e] - top));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane < p.top_k) wts[t * p.top_k + lane] = mine / total;
  if (lane + 32 < p.top_k) wts[t * p.top_k + lane + 32] = mine2 / total;
}

__global__ void __launch_bounds__(512)
moe_route_kernel(const MoeArgs p) {
  __shared__ unsigned long long mask[MOE_MAX_EXPERTS];
  __shared__ int first[MOE_MAX_EXPERTS];
  extern __shared__ int ids[];  // [token][choice]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) mask[e] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  for (int t = warp; t < p.T; t += warps) {
    if (p.E <= 64) choose<2>(p, t, lane, mask, ids, p.r.weight);
    else if (p.E <= 256) choose<8>(p, t, lane, mask, ids, p.r.weight);
    else choose<32>(p, t, lane, mask, ids, p.r.weight);
  }
  __syncthreads();

  // experts with tokens, in order: warp 0 runs over all of them
  if (warp == 0) {
    int chunks = 0, pairs = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      const int n = e < p.E ? __popcll(mask[e]) : 0, nc = (n + p.cap - 1) / p.cap;
      int pair_end = n, chunk_end = nc;  // inclusive sums over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, pair_end, o), b = __shfl_up_sync(0xffffffffu, chunk_end, o);
        if (lane >= o) pair_end += a, chunk_end += b;
      }
      if (n) {
        first[e] = pairs + pair_end - n;
        for (int c = 0; c < nc; ++c) {
          const int at = chunks + chunk_end - nc + c;
          p.r.expert[at] = e;
          p.r.first[at] = first[e] + c * p.cap;
          p.r.count[at] = min(p.cap, n - c * p.cap);
        }
      }
      chunks += __shfl_sync(0xffffffffu, chunk_end, 31);
      pairs += __shfl_sync(0xffffffffu, pair_end, 31);
    }
    if (lane == 0) *p.r.n_chunks = chunks;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.T * p.top_k; i += blockDim.x) {
    const int t = i / p.top_k, e = ids[i];
    const int at = first[e] + __popcll(mask[e] & ((1ull << t) - 1));
    p.r.token[at] = t;
    p.r.pair[i] = at;
  }
}

// ----------------------------------------------------------- gate and up
__device__ __forceinline__ float gate_act(float g, int act) {
  if (act == QI8_ACT_GELU) return gelu_erf(g);
  return g / (1.0f + expf(-g));
}

// h of column `col` and row i0 + r of a chunk, as value and remainder.
__device__ __forceinline__ void store_h(const MoeArgs& p, __nv_bfloat16* h, int Ip, int col, int i, float g, float u) {
  const float v = i < p.I ? gate_act(g, p.act) * u : 0.0f;  // zeros to the padded end
  // next to fp32's largest numbers, where rounding would give an infinity, cut
  const __nv_bfloat16 hi = fabsf(v) < 0x1.ffp127f ? __float2bfloat16_rn(v) : __float2bfloat16_rz(v);
  const float rest = v - __bfloat162float(hi);
  h[(int64_t)col * 2 * Ip + i] = hi;
  h[((int64_t)col * 2 + 1) * Ip + i] = __float2bfloat16_rn(isfinite(rest) ? rest : 0.0f);  // infinities, NaN: hi alone
}

// One chunk of tokens against the rows of one expert.
// UP:   tile 0 of a warp is 16 rows of G, tile 1 the same of U; columns are pairs.
// down: two tiles of 16 rows of D; columns 2 j, 2 j + 1 are value and remainder of
//       pair j, so that a thread holds both.
// RW warps side by side over the rows, KW over the 128-feature blocks of K.
template <typename T, int G, int NT, int RW, bool VEC, bool UP>
__global__ void __launch_bounds__(MOE_WARPS * 32, NT == 4 ? 1 : 2)
moe_expert_kernel(const MoeArgs p) {
  constexpr int KW = MOE_WARPS / RW, NS = W4_BLOCK / G;
  constexpr float unit = w4_unit<T>();
  __shared__ float red[KW > 1 ? KW : 1][KW > 1 ? 2 : 1][KW > 1 ? 8 * NT : 1][KW > 1 ? 17 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, a = lane & 3;
  const int rw = warp % RW, kw = warp / RW;
  pdl_wait();
  pdl_launch_dependents();
  const int c = blockIdx.y;
  if (c >= *p.r.n_chunks) return;
  const int e = p.r.expert[c], first = p.r.first[c], count = p.r.count[c];
  const int K = UP ? p.H : p.I, KB = (K + W4_BLOCK - 1) / W4_BLOCK;
  const int Ip = (p.I + W4_BLOCK - 1) / W4_BLOCK * W4_BLOCK;
  const int n0 = (blockIdx.x * RW + rw) * (UP ? 16 : 32);
  const int rows = UP ? p.I : p.H;
  if (KW == 1 && n0 >= (UP ? Ip : p.H)) return;

  const uint8_t* q[2];
  const __nv_bfloat16* sc[2];
  uint32_t qo[4], so[4];
  const int b0 = min(blockIdx.x * RW * (UP ? 16 : 32), rows - 1);  // the block's first row
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) {
    const int64_t row = UP ? ((int64_t)e * 2 + mt) * p.I + b0 : (int64_t)e * p.H + b0;
    q[mt] = (UP ? p.q13 : p.q2) + row * KB * 64;
    sc[mt] = (UP ? p.s13 : p.s2) + row * KB * NS;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t r = (uint32_t)(min(n0 + (UP ? 0 : mt * 16) + i * 8 + g, rows - 1) - b0);  // past the end: the last
      qo[2 * mt + i] = r * (uint32_t)KB * 64u + a * 16u;
      so[2 * mt + i] = r * (uint32_t)KB * NS;
    }
  }
  const uint16_t* x[NT];  // columns past the end repeat the last
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = nt * 8 + g;
    if (UP) x[nt] = p.x + (int64_t)p.r.token[first + min(col, count - 1)] * p.ld_x + (VEC ? 8 * a : 0);
    else x[nt] = reinterpret_cast<const uint16_t*>(p.h) + ((int64_t)first * 2 + min(col, 2 * count - 1)) * Ip + 8 * a;
  }
  float sum[2][NT][4] = {};
  w4_blocks<G, 2, 1>(q, sc, qo, so, kw, KW, KB, [&](int kb, const W4Frag<G, 2>& f) {
    if (!UP || (VEC && (kb + 1) * W4_BLOCK <= K))
      w4_block<T, G, 2, NT>(f, sum, [&](int nt, int b) {
        return *reinterpret_cast<const uint4*>(x[nt] + kb * W4_BLOCK + b * 32);
      });
    else
      w4_block<T, G, 2, NT>(f, sum, [&](int nt, int b) {
        return ld_act8<VEC>(x[nt] - (VEC ? 8 * a : 0), kb * W4_BLOCK + b * 32 + a * 8, K);
      });
  });

  const int64_t Hp = (p.H + 3) & ~3;
  __nv_bfloat16* h = p.h + (int64_t)first * 2 * Ip;
  float* part = p.part + (int64_t)first * Hp;
  if constexpr (KW == 1) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = g + 8 * (i >> 1);
        if constexpr (UP) {
          const int col = nt * 8 + 2 * a + (i & 1);
          if (col < count) store_h(p, h, Ip, col, n0 + r, sum[0][nt][i] * unit, sum[1][nt][i] * unit);
        } else if ((i & 1) == 0) {
          const int pair = nt * 4 + a;
          if (pair < count) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
              if (n0 + mt * 16 + r < p.H) part[pair * Hp + n0 + mt * 16 + r] = (sum[mt][nt][i] + sum[mt][nt][i + 1]) * unit;
          }
        }
      }
  } else {
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[kw][mt][nt * 8 + 2 * a + (i & 1)][g + 8 * (i >> 1)] = sum[mt][nt][i];
    __syncthreads();
    for (int i = threadIdx.x; i < (UP ? 16 : 32) * count; i += MOE_WARPS * 32) {
      if constexpr (UP) {
        const int r = i & 15, col = i >> 4;
        float gv = 0.0f, uv = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; ++w) gv += red[w][0][col][r], uv += red[w][1][col][r];
        if (n0 + r < Ip) store_h(p, h, Ip, col, n0 + r, gv * unit, uv * unit);
      } else {
        const int r = i & 15, mt = (i >> 4) & 1, pair = i >> 5, n = n0 + mt * 16 + r;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; ++w) v += red[w][mt][2 * pair][r] + red[w][mt][2 * pair + 1][r];
        if (n < p.H) part[pair * Hp + n] = v * unit;
      }
    }
  }
}

// ---------------------------------------------------------------- combine
// Four features of y per thread.
__global__ void __launch_bounds__(128)
moe_combine_kernel(const MoeArgs p) {
  pdl_wait();
  const int64_t Hp = (p.H + 3) & ~3;
  const int n = (blockIdx.x * 128 + threadIdx.x) * 4, t = blockIdx.y;
  if (n >= p.H) return;
  float y[4] = {};
  for (int j = 0; j < p.top_k; ++j) {
    const float w = p.r.weight[t * p.top_k + j];
    const float4 v = *reinterpret_cast<const float4*>(p.part + p.r.pair[t * p.top_k + j] * Hp + n);
    y[0] = fmaf(w, v.x, y[0]);
    y[1] = fmaf(w, v.y, y[1]);
    y[2] = fmaf(w, v.z, y[2]);
    y[3] = fmaf(w, v.w, y[3]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < p.H) store_from_f32(p.out, p.dtype, (int64_t)t * p.ld_out + n + i, y[i]);
}

// --------------------------------------------------------------- workspace
struct Layout {
  int64_t logits, h, part, n_chunks, expert, first, count, token, pair, weight, bytes;
};
Layout layout(int64_t T, int64_t H, int64_t E, int64_t I, int64_t k) {
  const int64_t pairs = T * k;  // and never more chunks
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  Layout l;
  l.logits = take(T * E * 8);
  l.h = take(pairs * 2 * w4_padded(I) * 2);
  l.part = take(pairs * ((H + 3) & ~3) * 4);
  l.n_chunks = take(4);
  l.expert = take(pairs * 4);
  l.first = take(pairs * 4);
  l.count = take(pairs * 4);
  l.token = take(pairs * 4);
  l.pair = take(pairs * 4);
  l.weight = take(pairs * 4);
  l.bytes = at;
  return l;
}

// In stream order, but scheduled while the kernel before it drains: each waits in
// pdl_wait for that one's results.
template <typename... KArgs, typename... Args>
int launch_after(void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st, const char* what,
                 const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, args...), what);
}

template <typename T, int G, int NT, bool VEC, bool UP>
int launch_expert(const MoeArgs& p, cudaStream_t st) {
  const int64_t pairs = (int64_t)p.T * p.top_k;
  const unsigned chunks = (unsigned)(pairs < p.E + pairs / p.cap ? pairs : p.E + pairs / p.cap);
  const int rows = UP ? (int)w4_padded(p.I) : p.H, tile = UP ? 16 : 32;
  const unsigned tiles = (unsigned)((rows + tile - 1) / tile);
  // eight warps over the rows when that makes two blocks per SM
  const int64_t used = pairs < p.E ? pairs : p.E;
  if (used * (tiles / MOE_WARPS) >= 2 * sm_count())
    return launch_after(moe_expert_kernel<T, G, NT, MOE_WARPS, VEC, UP>,
                        dim3((tiles + MOE_WARPS - 1) / MOE_WARPS, chunks), MOE_WARPS * 32, 0, st,
                        "moe_expert_kernel launch", p);
  return launch_after(moe_expert_kernel<T, G, NT, 1, VEC, UP>, dim3(tiles, chunks), MOE_WARPS * 32, 0, st,
                      "moe_expert_kernel launch", p);
}

// NTU, NTD: columns of eight for gate and up (one per pair), for down (two per pair)
template <typename T, int G, int NTU, int NTD>
int run_up_down(const MoeArgs& p, cudaStream_t st) {
  const bool vec = aligned16(p.x) && p.ld_x % 8 == 0 && p.H % 8 == 0;
  if (int rc = vec ? launch_expert<T, G, NTU, true, true>(p, st) : launch_expert<T, G, NTU, false, true>(p, st))
    return rc;
  return launch_expert<__nv_bfloat16, G, NTD, true, false>(p, st);
}

template <typename T, int G>
int run_experts(const MoeArgs& p, cudaStream_t st) {
  const int rc = p.cap == 4   ? run_up_down<T, G, 1, 1>(p, st)
                 : p.cap == 8 ? run_up_down<T, G, 1, 2>(p, st)
                              : run_up_down<T, G, 2, 4>(p, st);
  if (rc) return rc;
  return launch_after(moe_combine_kernel, dim3((p.H + 511) / 512, p.T), 128, 0, st, "moe_combine_kernel launch", p);
}

template <typename T>
int run_chunk(MoeArgs p, int group, cudaStream_t st) {
  // An expert has at most T pairs, T top_k / E on average.  Columns cost registers
  // and so occupancy, a second chunk reads the expert again, mostly from L2: 8 pairs
  // on average take 107 us in chunks of 8 and 117 in chunks of 16 (64 tokens, 64
  // experts of 1024), 12 on average 295 and 278 (48 tokens, 8 experts of 10240), 2
  // the same time in chunks of 4 and 8.
  const int pairs = p.T * p.top_k;
  p.cap = p.T <= 4 || pairs <= 3 * p.E ? 4 : p.T <= 8 || pairs <= 10 * p.E ? 8 : 16;
  const dim3 grid(p.E, (p.T + LOGIT_TOKENS - 1) / LOGIT_TOKENS);
  if (p.router_dtype == QI8_F32) moe_logits_kernel<T, float><<<grid, MOE_WARPS * 32, 0, st>>>(p);
  else moe_logits_kernel<T, T><<<grid, MOE_WARPS * 32, 0, st>>>(p);
  if (int rc = check_cuda(cudaGetLastError(), "moe_logits_kernel launch")) return rc;
  if (int rc = launch_after(moe_route_kernel, dim3(1), 512, p.T * p.top_k * 4, st, "moe_route_kernel launch", p))
    return rc;
  if (group == 32) return run_experts<T, 32>(p, st);
  if (group == 64) return run_experts<T, 64>(p, st);
  return run_experts<T, 128>(p, st);
}

constexpr int MOE_MAX_TOP = 64;  // choices of 64 tokens fit the route kernel's shared memory

int check_sizes(int64_t T, int64_t H, int64_t E, int64_t I, int top_k) {
  QI8_REQUIRE(T >= 0 && T < (1 << 30) && H > 0 && H <= (1 << 20) && I > 0 && I <= (1 << 20), QI8_ESHAPE,
              "%lld tokens of %lld features, experts of %lld", (long long)T, (long long)H, (long long)I);
  QI8_REQUIRE(E > 0 && E <= MOE_MAX_EXPERTS, QI8_ESHAPE, "%lld experts: 1 to %d are supported", (long long)E,
              MOE_MAX_EXPERTS);
  QI8_REQUIRE(top_k > 0 && top_k <= E && top_k <= MOE_MAX_TOP, QI8_ESHAPE,
              "top_k %d: 1 to %d and at most the %lld experts", top_k, MOE_MAX_TOP, (long long)E);
  return QI8_OK;
}

}  // namespace
}  // namespace qi8

using namespace qi8;

extern "C" int64_t qi8_moe_w4_workspace_bytes(int64_t T, int64_t H, int64_t E, int64_t I, int top_k) {
  if (check_sizes(T, H, E, I, top_k)) return 0;
  return layout(T < MOE_TOKENS ? T : MOE_TOKENS, H, E, I, top_k).bytes;
}

extern "C" int qi8_moe_w4(const void* x, int x_dtype, int64_t T, int64_t H, int64_t ld_x, const void* router,
                          int router_dtype, int64_t E, const uint8_t* q13, const void* s13, int64_t I,
                          const uint8_t* q2, const void* s2, int group, int top_k, int renormalize, int act, void* out,
                          int64_t ld_out, void* workspace, int64_t workspace_bytes, void* stream) {
  QI8_REQUIRE(device_ok(), QI8_EUNSUPPORTED, "no sm_100 device current");
  if (int rc = check_sizes(T, H, E, I, top_k)) return rc;
  QI8_REQUIRE(x_dtype == QI8_BF16 || x_dtype == QI8_F16, QI8_EDTYPE, "activations must be bf16 or fp16");
  QI8_REQUIRE(router_dtype == x_dtype || router_dtype == QI8_F32, QI8_EDTYPE,
              "router weights must be the activations' dtype or fp32");
  QI8_REQUIRE(group == 32 || group == 64 || group == 128, QI8_ESHAPE, "group_size must be 32, 64 or 128, got %d",
              group);
  QI8_REQUIRE(act == QI8_ACT_SILU || act == QI8_ACT_GELU, QI8_EINVAL, "activation must be SiLU or GELU");
  QI8_REQUIRE(ld_x >= H && ld_out >= H, QI8_ESHAPE, "row strides %lld, %lld below %lld features", (long long)ld_x,
              (long long)ld_out, (long long)H);
  if (T == 0) return QI8_OK;
  QI8_REQUIRE(x && router && q13 && s13 && q2 && s2 && out && workspace, QI8_EINVAL, "null pointer");
  QI8_REQUIRE(aligned16(q13) && aligned16(s13) && aligned16(q2) && aligned16(s2) && aligned16(workspace), QI8_EALIGN,
              "4-bit codes, scales and the workspace must be 16-byte aligned");
  const Layout l = layout(T < MOE_TOKENS ? T : MOE_TOKENS, H, E, I, top_k);
  QI8_REQUIRE(workspace_bytes >= l.bytes, QI8_ESHAPE, "workspace of %lld bytes, %lld needed",
              (long long)workspace_bytes, (long long)l.bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  MoeArgs p{static_cast<const uint16_t*>(x), ld_x, router, router_dtype, q13,
            static_cast<const __nv_bfloat16*>(s13), q2, static_cast<const __nv_bfloat16*>(s2), out, ld_out, x_dtype,
            0, (int)H, (int)E, (int)I, top_k, renormalize != 0, act, 0,
            reinterpret_cast<double*>(ws + l.logits), reinterpret_cast<__nv_bfloat16*>(ws + l.h),
            reinterpret_cast<float*>(ws + l.part),
            {reinterpret_cast<int*>(ws + l.n_chunks), reinterpret_cast<int*>(ws + l.expert),
             reinterpret_cast<int*>(ws + l.first), reinterpret_cast<int*>(ws + l.count),
             reinterpret_cast<int*>(ws + l.token), reinterpret_cast<int*>(ws + l.pair),
             reinterpret_cast<float*>(ws + l.weight)}};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int64_t t = 0; t < T; t += MOE_TOKENS) {
    p.T = (int)(T - t < MOE_TOKENS ? T - t : MOE_TOKENS);
    const int rc = x_dtype == QI8_F16 ? run_chunk<__half>(p, group, st) : run_chunk<__nv_bfloat16>(p, group, st);
    if (rc) return rc;
    p.x += p.T * ld_x;
    p.out = static_cast<uint8_t*>(p.out) + p.T * ld_out * 2;
  }
  return QI8_OK;
}
