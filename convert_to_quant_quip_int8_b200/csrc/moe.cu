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
//   moe_up_kernel      streaming engine (w4_stream.cuh): tasks are 16 rows of G
//                      and of U of one expert, h = act(g) * u
//   moe_down_kernel    streaming engine: a block takes a share of y's rows and
//                      goes through every expert in use; its sums never leave the
//                      block, so nothing is added atomically and the result does
//                      not depend on order
// An expert's tokens come in chunks of up to `cap` pairs (token, choice): as many
// as the MMA columns of a task hold.
//
// h is held as two bf16 numbers (value and remainder, 16 significant bits
// together): rounding it to one would cost as much accuracy as the output's
// own rounding, and the second column of the MMA costs no bytes.  bf16 for fp16
// layers too: h can pass fp16's range, and codes are exact in both types.
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "int4.cuh"
#include "w4_stream.cuh"

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
  float* weight;  // [pair]
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
  int height;      // rows of y per tile of the down product
  unsigned int* status;
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
    p.r.weight[at] = wts[i];
  }
}

// ----------------------------------------------------------- gate and up
__device__ __forceinline__ float gate_act(float g, int act) {
  if (act == QI8_ACT_GELU) return gelu_erf(g);
  return g / (1.0f + expf(-g));
}

// Tasks: (chunk, 16 rows of I), chunk-major, an equal share for every block.
template <typename T_, int G_, int NT_, bool VEC_>
struct UpJob {
  using T = T_;
  static constexpr int G = G_, MT = 2, NT = NT_, W = 16;
  static constexpr bool VEC = VEC_;
  const MoeArgs& p;
  int tiles;
  int lo, hi;
  __device__ __forceinline__ explicit UpJob(const MoeArgs& p_) : p(p_) {
    tiles = (p.I + 15) / 16;
    const int64_t all = (int64_t)*p.r.n_chunks * tiles;  // below 2^28
    lo = (int)(all * blockIdx.x / gridDim.x);
    hi = (int)(all * (blockIdx.x + 1) / gridDim.x);
  }
  __device__ __forceinline__ int tasks() const { return hi - lo; }
  __device__ __forceinline__ int KB() const { return (p.H + W4_BLOCK - 1) / W4_BLOCK; }
  __device__ __forceinline__ int K() const { return p.H; }
  __device__ __forceinline__ int height() const { return 16; }
  __device__ __forceinline__ int rows() const { return 2 * p.E * p.I; }
  __device__ __forceinline__ const __nv_bfloat16* scales() const { return p.s13; }
  __device__ __forceinline__ int chunk(int j) const { return (lo + j) / tiles; }
  __device__ __forceinline__ int first_row(int j) const { return (lo + j) % tiles * 16; }
  // gate rows, then up rows; a tile that passes the end of one reads what follows, for nothing
  __device__ __forceinline__ int row(int j, int mt) const {
    return (2 * p.r.expert[chunk(j)] + mt) * p.I + first_row(j);
  }
  __device__ __forceinline__ const uint16_t* activation(int j, int col) const {
    const int c = chunk(j);
    return p.x + (int64_t)p.r.token[p.r.first[c] + min(col, p.r.count[c] - 1)] * p.ld_x;
  }
  __device__ __forceinline__ void finish(int j, const float* sums, int tid) const {
    constexpr int TILE = stream::Cfg<MT, NT, W>::TILE;
    const int c = chunk(j), i0 = first_row(j), count = p.r.count[c];
    const int Ip = (p.I + W4_BLOCK - 1) / W4_BLOCK * W4_BLOCK;
    __nv_bfloat16* h = p.h + (int64_t)p.r.first[c] * 2 * Ip + i0;
    for (int i = tid; i < 16 * count; i += stream::FINISH_WARPS * 32) {
      const int r = i & 15, col = i >> 4;
      float gv = 0.0f, uv = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        gv += sums[w * MT * TILE + col * stream::COL_PITCH + r];
        uv += sums[(w * MT + 1) * TILE + col * stream::COL_PITCH + r];
      }
      const float v = i0 + r < p.I ? gate_act(gv, p.act) * uv : 0.0f;
      const __nv_bfloat16 hi = __float2bfloat16_rn(v);
      const float rest = v - __bfloat162float(hi);
      h[(int64_t)col * 2 * Ip + r] = hi;
      // an infinite or NaN value is in hi alone
      h[(int64_t)col * 2 * Ip + Ip + r] = __float2bfloat16_rn(isfinite(rest) ? rest : 0.0f);
    }
    // zeros from the last rows to the padded end of h
    if (i0 + 16 >= p.I)
      for (int i = tid; i < (Ip - i0 - 16) * count * 2; i += stream::FINISH_WARPS * 32)
        h[(int64_t)(i % (2 * count)) * Ip + 16 + i / (2 * count)] = __float2bfloat16_rn(0.0f);
  }
  __device__ __forceinline__ void finish_all(int) const {}
};

template <typename T, int G, int NT, bool VEC>
__global__ void __launch_bounds__(stream::Cfg<2, NT, 16>::THREADS, 1)
moe_up_kernel(const __grid_constant__ CUtensorMap codes, const __grid_constant__ MoeArgs p) {
  extern __shared__ __align__(128) uint8_t smem[];
  UpJob<T, G, NT, VEC> job(p);
  stream::run(job, &codes, smem, p.status);
}

// ------------------------------------------------------------------- down
// Tasks: (tile of the block's rows, chunk).  Columns 2 j and 2 j + 1 of the MMA
// are value and remainder of pair j.
template <int G_, int NT_>
struct DownJob {
  using T = __nv_bfloat16;
  static constexpr int G = G_, MT = 1, NT = NT_, W = 16;
  static constexpr bool VEC = true;
  const MoeArgs& p;
  float (*y)[17];  // [token][row]
  int chunks, r0, r1, tiles;
  __device__ __forceinline__ DownJob(const MoeArgs& p_, float (*y_)[17]) : p(p_), y(y_) {
    chunks = *p.r.n_chunks;
    r0 = (int)((int64_t)p.H * blockIdx.x / gridDim.x);
    r1 = (int)((int64_t)p.H * (blockIdx.x + 1) / gridDim.x);
    tiles = (r1 - r0 + p.height - 1) / p.height;
  }
  __device__ __forceinline__ int tasks() const { return tiles * chunks; }
  __device__ __forceinline__ int KB() const { return (p.I + W4_BLOCK - 1) / W4_BLOCK; }
  __device__ __forceinline__ int K() const { return KB() * W4_BLOCK; }
  __device__ __forceinline__ int height() const { return p.height; }
  __device__ __forceinline__ int rows() const { return p.E * p.H; }
  __device__ __forceinline__ const __nv_bfloat16* scales() const { return p.s2; }
  // the last tile of a block may overlap the one before, or pass the block's first row
  __device__ __forceinline__ int first_row(int j) const { return max(min(r0 + j / chunks * p.height, r1 - p.height), 0); }
  __device__ __forceinline__ int row(int j, int) const { return p.r.expert[j % chunks] * p.H + first_row(j); }
  __device__ __forceinline__ const uint16_t* activation(int j, int col) const {
    const int c = j % chunks;
    return reinterpret_cast<const uint16_t*>(p.h) +
           ((int64_t)p.r.first[c] * 2 + min(col, 2 * p.r.count[c] - 1)) * K();
  }
  __device__ __forceinline__ void finish(int j, const float* sums, int tid) const {
    constexpr int TILE = stream::Cfg<MT, NT, W>::TILE;
    const int c = j % chunks, first = p.r.first[c];
    for (int i = tid; i < 16 * p.r.count[c]; i += stream::FINISH_WARPS * 32) {
      const int r = i & 15, pair = i >> 4;  // pairs of a chunk are of different tokens
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float* s = sums + w * TILE + 2 * pair * stream::COL_PITCH + r;
        v += s[0] + s[stream::COL_PITCH];
      }
      float* at = &y[p.r.token[first + pair]][r];
      *at = fmaf(p.r.weight[first + pair], v, *at);
    }
    if (c < chunks - 1) return;
    stream::finish_sync();
    for (int i = tid; i < 16 * p.T; i += stream::FINISH_WARPS * 32) {
      const int r = i & 15, t = i >> 4, n = first_row(j) + r;
      if (r < p.height && n >= r0 && n < r1) store_from_f32(p.out, p.dtype, (int64_t)t * p.ld_out + n, y[t][r]);
      y[t][r] = 0.0f;
    }
  }
  __device__ __forceinline__ void finish_all(int) const {}
};

template <int G, int NT>
__global__ void __launch_bounds__(stream::Cfg<1, NT, 16>::THREADS, 1)
moe_down_kernel(const __grid_constant__ CUtensorMap codes, const __grid_constant__ MoeArgs p) {
  extern __shared__ __align__(128) uint8_t smem[];
  float(*y)[17] = reinterpret_cast<float(*)[17]>(smem + stream::Cfg<1, NT, 16>::SMEM);  // behind the engine's
  for (int i = threadIdx.x; i < p.T * 17; i += blockDim.x) y[0][i] = 0.0f;  // seen after the engine's first barrier
  DownJob<G, NT> job(p, y);
  stream::run(job, &codes, smem, p.status);
}

// --------------------------------------------------------------- workspace
struct Layout {
  int64_t logits, h, n_chunks, expert, first, count, token, weight, bytes;
};
Layout layout(int64_t T, int64_t E, int64_t I, int64_t k) {
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
  l.n_chunks = take(4);
  l.expert = take(pairs * 4);
  l.first = take(pairs * 4);
  l.count = take(pairs * 4);
  l.token = take(pairs * 4);
  l.weight = take(pairs * 4);
  l.bytes = at;
  return l;
}

template <typename Tag, typename K>
int launch_stream(K kern, int threads, int smem, int grid, const CUtensorMap& codes, const MoeArgs& p,
                  cudaStream_t st, const char* what) {
  if (int rc = allow_smem<Tag>(kern, smem)) return rc;
  kern<<<grid, threads, smem, st>>>(codes, p);
  return check_cuda(cudaGetLastError(), what);
}

// NTU, NTD: columns of eight for gate and up (one per pair), for down (two per pair)
template <typename T, int G, int NTU, int NTD, bool VEC>
int run_up_down(MoeArgs p, cudaStream_t st) {
  using CU = stream::Cfg<2, NTU, 16>;
  using CD = stream::Cfg<1, NTD, 16>;
  constexpr int y_bytes = MOE_TOKENS * 17 * 4;
  static_assert(CU::SMEM <= 232448 && CD::SMEM + y_bytes <= 232448, "shared memory");
  const int KU = (int)(w4_padded(p.H) / W4_BLOCK), KD = (int)(w4_padded(p.I) / W4_BLOCK);
  CUtensorMap up, down;
  if (int rc = code_map(&up, p.q13, (int64_t)2 * p.E * p.I, KU, KU < stream::SEG ? KU : stream::SEG, 16)) return rc;
  if (int rc = launch_stream<UpJob<T, G, NTU, VEC>>(moe_up_kernel<T, G, NTU, VEC>, CU::THREADS, CU::SMEM, sm_count(),
                                                    up, p, st, "moe_up_kernel launch"))
    return rc;
  const int need = (p.H + 3) / 4;  // at least four rows a block
  const int grid = need < sm_count() ? need : sm_count();
  p.height = stream::tile_height((p.H + grid - 1) / grid, 1);
  if (int rc = code_map(&down, p.q2, (int64_t)p.E * p.H, KD, KD < stream::SEG ? KD : stream::SEG, p.height)) return rc;
  return launch_stream<DownJob<G, NTD>>(moe_down_kernel<G, NTD>, CD::THREADS, CD::SMEM + y_bytes, grid, down, p, st,
                                        "moe_down_kernel launch");
}

template <typename T, int G>
int run_experts(const MoeArgs& p, cudaStream_t st) {
  const bool vec = aligned16(p.x) && p.ld_x % 8 == 0 && p.H % 8 == 0;
  if (p.cap == 4) return vec ? run_up_down<T, G, 1, 1, true>(p, st) : run_up_down<T, G, 1, 1, false>(p, st);
  if (p.cap == 8) return vec ? run_up_down<T, G, 1, 2, true>(p, st) : run_up_down<T, G, 1, 2, false>(p, st);
  return vec ? run_up_down<T, G, 2, 4, true>(p, st) : run_up_down<T, G, 2, 4, false>(p, st);
}

template <typename T>
int run_chunk(MoeArgs p, int group, cudaStream_t st) {
  // an expert has at most T pairs, T top_k / E on average
  p.cap = p.T <= 4 ? 4 : p.T <= 8 || p.T * p.top_k <= 6 * p.E ? 8 : 16;
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
  QI8_REQUIRE(2 * E * I < (1LL << 31) && E * H < (1LL << 31), QI8_ESHAPE, "%lld experts of %lld x %lld: too many rows",
              (long long)E, (long long)I, (long long)H);
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
            0, (int)H, (int)E, (int)I, top_k, renormalize != 0, act, 0, 0, device_status_ptr(),
            reinterpret_cast<double*>(ws + l.logits), reinterpret_cast<__nv_bfloat16*>(ws + l.h),
            {reinterpret_cast<int*>(ws + l.n_chunks), reinterpret_cast<int*>(ws + l.expert),
             reinterpret_cast<int*>(ws + l.first), reinterpret_cast<int*>(ws + l.count),
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
