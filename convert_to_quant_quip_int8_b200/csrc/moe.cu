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
// Four launches, bound by the bytes of the experts in use:
//   moe_logits_kernel  one warp per (expert, token quad)
//   moe_route_kernel   one block: the choice, its weights, tokens by expert
//   moe_up_kernel      one block per (expert, 16 rows of G and of U); h = act(g) * u
//   moe_down_kernel    one block per 16 rows of y: every expert in use, all
//                      tokens; its sums never leave the block, so nothing is
//                      added atomically and the result does not depend on order
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
  int* n_used;                    // experts with tokens
  int* expert;                    // [used] which
  int* first;                     // [used] its first pair
  unsigned long long* mask;       // [used] its tokens
  int* token;                     // [pair]
  float* weight;                  // [pair]
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
  double* logits;  // [T, E]
  __nv_bfloat16* h;  // [pair][2][Ip]
  Route r;
};

// ------------------------------------------------------------------ router
// The choice of experts has to be that of the exact logits, so the sums are
// fp64 (products of 16- or 24-bit factors are exact in it).
constexpr int LOGIT_TOKENS = 4;

template <typename T>
__device__ __forceinline__ double elem64(const T* p, int64_t i) {
  return (double)Elem<T>::to_f32(p[i]);
}

template <typename T, typename R>
__global__ void __launch_bounds__(MOE_WARPS * 32)
moe_logits_kernel(const MoeArgs p) {
  const int lane = threadIdx.x & 31;
  const int e = blockIdx.x * MOE_WARPS + (threadIdx.x >> 5);
  if (e >= p.E) return;
  const int t0 = blockIdx.y * LOGIT_TOKENS;
  const R* w = static_cast<const R*>(p.router) + (int64_t)e * p.H;
  const T* x = reinterpret_cast<const T*>(p.x);
  double acc[LOGIT_TOKENS] = {};
  for (int k = lane; k < p.H; k += 32) {
    const double r = elem64(w, k);
#pragma unroll
    for (int j = 0; j < LOGIT_TOKENS; ++j) {
      const int t = min(t0 + j, p.T - 1);
      acc[j] = fma(elem64(x, (int64_t)t * p.ld_x + k), r, acc[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < LOGIT_TOKENS; ++j) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
    if (lane == 0 && t0 + j < p.T) p.logits[(int64_t)(t0 + j) * p.E + e] = acc[j];
  }
}

// Order of the logits as unsigned numbers: -0 equals 0, NaN above all.
__device__ __forceinline__ unsigned long long order_key(double v) {
  if (v != v) return ~0ull;
  const long long b = __double_as_longlong(v + 0.0);
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

__global__ void __launch_bounds__(512)
moe_route_kernel(const MoeArgs p) {
  __shared__ unsigned long long mask[MOE_MAX_EXPERTS];
  __shared__ int first[MOE_MAX_EXPERTS];
  extern __shared__ unsigned char dyn[];  // per (token, choice): expert, weight
  int* ids = reinterpret_cast<int*>(dyn);
  float* wts = reinterpret_cast<float*>(ids + p.T * p.top_k);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) mask[e] = 0;
  __syncthreads();

  for (int t = warp; t < p.T; t += warps) {
    const double* l = p.logits + (int64_t)t * p.E;
    // each choice is the greatest (logit, lower expert first) below the last one
    unsigned long long last_key = ~0ull;
    int last_e = -1;
    double top = 0.0;
    for (int j = 0; j < p.top_k; ++j) {
      unsigned long long best = 0;
      int best_e = 0x7fffffff;
      for (int e = lane; e < p.E; e += 32) {
        const unsigned long long key = order_key(l[e]);
        const bool below = key < last_key || (key == last_key && e > last_e);
        if (below && (key > best || (key == best && e < best_e))) best = key, best_e = e;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long ok = __shfl_xor_sync(0xffffffffu, best, o);
        const int oe = __shfl_xor_sync(0xffffffffu, best_e, o);
        if (ok > best || (ok == best && oe < best_e)) best = ok, best_e = oe;
      }
      last_key = best;
      last_e = best_e;
      if (j == 0) top = l[best_e];
      if (lane == 0) {
        ids[t * p.top_k + j] = best_e;
        atomicOr(&mask[best_e], 1ull << t);
      }
    }
    __syncwarp();
    float total = 0.0f;
    if (p.renorm)
      for (int j = lane; j < p.top_k; j += 32) total += expf((float)(l[ids[t * p.top_k + j]] - top));
    else
      for (int e = lane; e < p.E; e += 32) total += expf((float)(l[e] - top));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    for (int j = lane; j < p.top_k; j += 32)
      wts[t * p.top_k + j] = expf((float)(l[ids[t * p.top_k + j]] - top)) / total;
  }
  __syncthreads();

  // experts with tokens, in order: warp 0 runs over all of them
  if (warp == 0) {
    int used = 0, pairs = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      const unsigned long long m = e < p.E ? mask[e] : 0;
      const int n = __popcll(m);
      int before = n;  // inclusive sum over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      const unsigned some = __ballot_sync(0xffffffffu, m != 0);
      if (m) {
        const int at = used + __popc(some & ((1u << lane) - 1));
        first[e] = pairs + before - n;
        p.r.expert[at] = e;
        p.r.first[at] = first[e];
        p.r.mask[at] = m;
      }
      used += __popc(some);
      pairs += __shfl_sync(0xffffffffu, before, 31);
    }
    if (lane == 0) *p.r.n_used = used;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.T * p.top_k; i += blockDim.x) {
    const int t = i / p.top_k, e = ids[i];
    const int at = first[e] + __popcll(mask[e] & ((1ull << t) - 1));
    p.r.token[at] = t;
    p.r.weight[at] = wts[i];
  }
}

// ----------------------------------------------------------- gate and up
__device__ __forceinline__ float gate_act(float g, int act) {
  if (act == QI8_ACT_GELU) return gelu_erf(g);
  return g / (1.0f + expf(-g));
}

// Tokens c0 .. of the block's expert, eight times NT of them.
template <typename T, int G, int NT, bool VEC>
__device__ __forceinline__ void up_tokens(const MoeArgs& p, int e, int row0, int pair0, int count,
                                          float (*red)[2][8 * NT][17]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, a = lane & 3;
  const int KB = (p.H + W4_BLOCK - 1) / W4_BLOCK;
  const uint8_t* q[4];
  const __nv_bfloat16* sc[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = min(row0 + (r & 1) * 8 + g, p.I - 1);
    const int64_t n = ((int64_t)e * 2 + (r >> 1)) * p.I + i;  // gate rows, then up rows
    q[r] = p.q13 + n * KB * 64 + a * 16;
    sc[r] = p.s13 + n * KB * (W4_BLOCK / G);
  }
  const uint16_t* x[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int c = nt * 8 + g;
    x[nt] = c < count ? p.x + (int64_t)p.r.token[pair0 + c] * p.ld_x : nullptr;
  }
  float sum[2][NT][4] = {};
  W4Frag<G, 2> cur, next;
  int kb = warp;
  if (kb < KB)
#pragma unroll
    for (int r = 0; r < 4; ++r) cur.load(r, q[r] + (int64_t)kb * 64, sc[r] + kb * (W4_BLOCK / G));
  for (; kb < KB; kb += MOE_WARPS) {
    const int nx = kb + MOE_WARPS;
    if (nx < KB)
#pragma unroll
      for (int r = 0; r < 4; ++r) next.load(r, q[r] + (int64_t)nx * 64, sc[r] + nx * (W4_BLOCK / G));
    w4_block<T, G, 2, NT>(cur, sum, [&](int nt, int b) {
      return x[nt] ? ld_act8<VEC>(x[nt], kb * W4_BLOCK + b * 32 + a * 8, p.H) : make_uint4(0, 0, 0, 0);
    });
    cur = next;
  }
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[warp][mt][nt * 8 + 2 * a + (i & 1)][g + 8 * (i >> 1)] = sum[mt][nt][i];
  __syncthreads();
  const int Ip = (p.I + W4_BLOCK - 1) / W4_BLOCK * W4_BLOCK;
  for (int i = threadIdx.x; i < 16 * 8 * NT; i += MOE_WARPS * 32) {
    const int r = i & 15, c = i >> 4;
    if (c >= count) continue;
    float gv = 0.0f, uv = 0.0f;
#pragma unroll
    for (int w = 0; w < MOE_WARPS; ++w) gv += red[w][0][c][r], uv += red[w][1][c][r];
    const float v = row0 + r < p.I ? gate_act(gv, p.act) * uv : 0.0f;
    const __nv_bfloat16 hi = __float2bfloat16_rn(v);
    const float rest = v - __bfloat162float(hi);
    __nv_bfloat16* h = p.h + (int64_t)(pair0 + c) * 2 * Ip + row0 + r;
    h[0] = hi;
    h[Ip] = __float2bfloat16_rn(isfinite(rest) ? rest : 0.0f);  // an infinite or NaN value is in hi alone
  }
  __syncthreads();
}

template <typename T, int G, bool VEC>
__global__ void __launch_bounds__(MOE_WARPS * 32)
moe_up_kernel(const MoeArgs p) {
  __shared__ __align__(16) unsigned char red[MOE_WARPS * 2 * 16 * 17 * sizeof(float)];
  if ((int)blockIdx.y >= *p.r.n_used) return;
  const int e = p.r.expert[blockIdx.y], pair0 = p.r.first[blockIdx.y];
  const int count = __popcll(p.r.mask[blockIdx.y]);
  const int row0 = blockIdx.x * 16;
  for (int c = 0; c < count; c += 16) {
    if (count - c <= 8)
      up_tokens<T, G, 1, VEC>(p, e, row0, pair0 + c, count - c, reinterpret_cast<float(*)[2][8][17]>(red));
    else
      up_tokens<T, G, 2, VEC>(p, e, row0, pair0 + c, min(count - c, 16), reinterpret_cast<float(*)[2][16][17]>(red));
  }
}

// ------------------------------------------------------------------- down
// Columns 2 j and 2 j + 1 of the MMA are value and remainder of pair j.
template <int G, int NT>
__device__ __forceinline__ void down_pairs(const MoeArgs& p, const uint8_t* const (&q)[2],
                                           const __nv_bfloat16* const (&sc)[2], int kb0, int kb1, int pair0, int count,
                                           float (*ysum)[17]) {
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, a = lane & 3;
  const int Ip = (p.I + W4_BLOCK - 1) / W4_BLOCK * W4_BLOCK;
  const uint16_t* x[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int c = nt * 8 + g;
    x[nt] = c < 2 * count ? reinterpret_cast<const uint16_t*>(p.h) + ((int64_t)pair0 * 2 + c) * Ip : nullptr;
  }
  float sum[1][NT][4] = {};
  W4Frag<G, 1> cur, next;
#pragma unroll
  for (int r = 0; r < 2; ++r) cur.load(r, q[r] + (int64_t)kb0 * 64, sc[r] + kb0 * (W4_BLOCK / G));
  for (int kb = kb0; kb < kb1; ++kb) {
    if (kb + 1 < kb1)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        next.load(r, q[r] + (int64_t)(kb + 1) * 64, sc[r] + (kb + 1) * (W4_BLOCK / G));
    w4_block<__nv_bfloat16, G, 1, NT>(cur, sum, [&](int nt, int b) {
      return x[nt] ? *reinterpret_cast<const uint4*>(x[nt] + kb * W4_BLOCK + b * 32 + a * 8) : make_uint4(0, 0, 0, 0);
    });
    cur = next;
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int j = nt * 4 + a;
    if (j < count) {
      float* y = ysum[p.r.token[pair0 + j]];
      const float w = p.r.weight[pair0 + j];
      y[g] = fmaf(w, sum[0][nt][0] + sum[0][nt][1], y[g]);
      y[g + 8] = fmaf(w, sum[0][nt][2] + sum[0][nt][3], y[g + 8]);
    }
  }
  __syncwarp();
}

template <int G>
__global__ void __launch_bounds__(MOE_WARPS * 32)
moe_down_kernel(const MoeArgs p) {
  extern __shared__ unsigned char dyn[];
  float(*ysum)[17] = reinterpret_cast<float(*)[17]>(dyn);  // [warp][token][16]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 16;
  for (int i = threadIdx.x; i < MOE_WARPS * p.T * 17; i += MOE_WARPS * 32) ysum[0][i] = 0.0f;
  __syncthreads();

  const int KB = (p.I + W4_BLOCK - 1) / W4_BLOCK;
  const int64_t items = (int64_t)*p.r.n_used * KB;  // (expert, block of I), split evenly over the warps
  int64_t at = items * warp / MOE_WARPS;
  const int64_t end = items * (warp + 1) / MOE_WARPS;
  while (at < end) {
    const int u = (int)(at / KB), kb0 = (int)(at - (int64_t)u * KB);
    const int kb1 = (int)min((int64_t)KB, kb0 + (end - at));
    const int e = p.r.expert[u], pair0 = p.r.first[u], count = __popcll(p.r.mask[u]);
    const uint8_t* q[2];
    const __nv_bfloat16* sc[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t n = (int64_t)e * p.H + min(n0 + r * 8 + (lane >> 2), p.H - 1);
      q[r] = p.q2 + n * KB * 64 + (lane & 3) * 16;
      sc[r] = p.s2 + n * KB * (W4_BLOCK / G);
    }
    float(*mine)[17] = ysum + warp * p.T;
    for (int c = 0; c < count; c += 16) {
      const int left = count - c;
      if (left <= 4) down_pairs<G, 1>(p, q, sc, kb0, kb1, pair0 + c, left, mine);
      else if (left <= 8) down_pairs<G, 2>(p, q, sc, kb0, kb1, pair0 + c, left, mine);
      else down_pairs<G, 4>(p, q, sc, kb0, kb1, pair0 + c, min(left, 16), mine);
    }
    at += kb1 - kb0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.T * 16; i += MOE_WARPS * 32) {
    const int t = i >> 4, r = i & 15;
    if (n0 + r >= p.H) continue;
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < MOE_WARPS; ++w) y += ysum[w * p.T + t][r];
    store_from_f32(p.out, p.dtype, (int64_t)t * p.ld_out + n0 + r, y);
  }
}

// --------------------------------------------------------------- workspace
struct Layout {
  int64_t logits, h, n_used, expert, first, mask, token, weight, bytes;
};
Layout layout(int64_t T, int64_t E, int64_t I, int64_t k) {
  const int64_t pairs = T * k, used = pairs < E ? pairs : E;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  Layout l;
  l.logits = take(T * E * 8);
  l.h = take(pairs * 2 * w4_padded(I) * 2);
  l.mask = take(used * 8);
  l.n_used = take(4);
  l.expert = take(used * 4);
  l.first = take(used * 4);
  l.token = take(pairs * 4);
  l.weight = take(pairs * 4);
  l.bytes = at;
  return l;
}

template <typename T, int G>
int run_experts(const MoeArgs& p, cudaStream_t st) {
  const int64_t pairs = (int64_t)p.T * p.top_k;
  const unsigned used = (unsigned)(pairs < p.E ? pairs : p.E);
  const unsigned Ip = (unsigned)w4_padded(p.I);
  const dim3 grid(Ip / 16, used);
  if (aligned16(p.x) && p.ld_x % 8 == 0 && p.H % 8 == 0) moe_up_kernel<T, G, true><<<grid, MOE_WARPS * 32, 0, st>>>(p);
  else moe_up_kernel<T, G, false><<<grid, MOE_WARPS * 32, 0, st>>>(p);
  if (int rc = check_cuda(cudaGetLastError(), "moe_up_kernel launch")) return rc;
  moe_down_kernel<G><<<(p.H + 15) / 16, MOE_WARPS * 32, MOE_WARPS * p.T * 17 * sizeof(float), st>>>(p);
  return check_cuda(cudaGetLastError(), "moe_down_kernel launch");
}

template <typename T>
int run_chunk(const MoeArgs& p, int group, cudaStream_t st) {
  const dim3 grid((p.E + MOE_WARPS - 1) / MOE_WARPS, (p.T + LOGIT_TOKENS - 1) / LOGIT_TOKENS);
  if (p.router_dtype == QI8_F32) moe_logits_kernel<T, float><<<grid, MOE_WARPS * 32, 0, st>>>(p);
  else moe_logits_kernel<T, T><<<grid, MOE_WARPS * 32, 0, st>>>(p);
  if (int rc = check_cuda(cudaGetLastError(), "moe_logits_kernel launch")) return rc;
  moe_route_kernel<<<1, 512, p.T * p.top_k * 8, st>>>(p);
  if (int rc = check_cuda(cudaGetLastError(), "moe_route_kernel launch")) return rc;
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
  return layout(T < MOE_TOKENS ? T : MOE_TOKENS, E, I, top_k).bytes;
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
  const Layout l = layout(T < MOE_TOKENS ? T : MOE_TOKENS, E, I, top_k);
  QI8_REQUIRE(workspace_bytes >= l.bytes, QI8_ESHAPE, "workspace of %lld bytes, %lld needed",
              (long long)workspace_bytes, (long long)l.bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  MoeArgs p{static_cast<const uint16_t*>(x), ld_x, router, router_dtype, q13,
            static_cast<const __nv_bfloat16*>(s13), q2, static_cast<const __nv_bfloat16*>(s2), out, ld_out, x_dtype,
            0, (int)H, (int)E, (int)I, top_k, renormalize != 0, act,
            reinterpret_cast<double*>(ws + l.logits), reinterpret_cast<__nv_bfloat16*>(ws + l.h),
            {reinterpret_cast<int*>(ws + l.n_used), reinterpret_cast<int*>(ws + l.expert),
             reinterpret_cast<int*>(ws + l.first), reinterpret_cast<unsigned long long*>(ws + l.mask),
             reinterpret_cast<int*>(ws + l.token), reinterpret_cast<float*>(ws + l.weight)}};
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
