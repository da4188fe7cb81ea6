// Load-balance loss of a top-k router, the per-expert counts, and the gradient
// of the logits.
//
// For the live tokens t (mask[t] set, or no mask; a row whose logits are all
// -inf has no expert to weigh and is not live), n of them:
//   p_t = softmax(logits_t) in fp32,  P_e = sum_t p_te / n,
//   counts_e = live (t, j) with topi[t, j] = e,  f_e = counts_e / (k n),
//   loss = E sum_e f_e P_e                      (1 when the load is even)
//   dlogits_tj = dloss (E / n) p_tj (f_j - sum_e f_e p_te)
// f is a count and carries no gradient.  n = 0 gives loss 0 and gradient 0.
//
// Bound: one read of the logits forward; one read and one write backward (the
// softmax is recomputed: storing p would cost a write and a read more).  A row
// is split over G lanes of 8 consecutive experts each (one 16-byte load for
// 16-bit logits), G the smallest power of two with 8 G >= E, so a warp holds
// 32 / G rows and the softmax needs log2 G shuffles.  Each lane sums p of its
// own 8 experts over its rows in registers; blocks leave their sums as partials
// that one block adds in block order: no floating-point atomics, the same bits
// every time.  Counts are integers, where order does not matter.  Batches of
// at most SINGLE_ELEMS logits take one block and one launch.
// Measured, forward and backward: 512 tokens, 8 experts 8.5 us; 131072 tokens, 64
// experts, fp32 (34 MB) 31 us, under a host call of 90 (one by one and cold the
// partial sums 18.8, bound by their instructions at 2 a cycle and SM, the one block
// that joins them 6.9 and the gradient 16.3).
#include <algorithm>

#include "common.cuh"

namespace b200q {
namespace balance {

constexpr int THREADS = 1024, GRAD_THREADS = 256;
constexpr int MAX_EXPERTS = 256, MAX_K = 8;
// Logits up to which one block and one launch take the batch.  us with one block /
// with as many as there are rows for, bf16: 8 experts 16384 7.4 / 7.7, 32768 9.7 /
// 7.7; 64 experts 8192 6.1 / 6.0, 16384 6.5 / 6.9, 32768 9.1 / 7.0; 256 experts,
// top 8, 16384 6.6 / 6.8, 32768 9.3 / 7.0.
constexpr int64_t SINGLE_ELEMS = 16384;
constexpr int MAX_BLOCKS = 148;  // one per SM: few partials to add
constexpr int UNROLL = 2;        // rows per lane requested before the first is used

template <class T>
__device__ __forceinline__ float tf(T v);
template <>
__device__ __forceinline__ float tf<float>(float v) { return v; }
template <>
__device__ __forceinline__ float tf<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float tf<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T ft(float v);
template <>
__device__ __forceinline__ float ft<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half ft<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 ft<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight consecutive logits of a row, -inf past E.  VEC: E % 8 == 0, 16-byte aligned rows.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int e0, int E, float* v) {
  if (VEC) {
    if (e0 < E) {
      constexpr int W = sizeof(T) * 8 / 16;
      uint4 u[W];
#pragma unroll
      for (int i = 0; i < W; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(row + e0) + i);
      const T* h = reinterpret_cast<const T*>(u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = tf<T>(h[i]);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = !VEC && e0 + i < E ? tf<T>(row[e0 + i]) : -INFINITY;
}

// The same of row t, -inf where the row is past the batch or masked.
template <class T, bool VEC>
__device__ __forceinline__ void load_row(const T* logits, const uint8_t* mask, int64_t t, int64_t T_, int e0, int E,
                                         float* v) {
  // both loads at once: what a masked row holds is dropped after it has come
  const bool in = t < T_, keep = in && (!mask || mask[t]);
  if (in) load8<T, VEC>(logits + t * E, e0, E, v);
  if (!keep)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = -INFINITY;
}

// Softmax of a row over its G lanes, in place (zeros past E); returns whether
// the row has a logit above -inf.  A NaN anywhere makes the row NaN.
template <int G>
__device__ __forceinline__ bool softmax8(float* v) {
  float m = -INFINITY;
  bool any = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m = fmaxf(m, v[i]);
    any |= !(v[i] == -INFINITY);
  }
  int has = any;
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    has |= __shfl_xor_sync(0xffffffffu, has, o);
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = expf(v[i] - m);
    sum += v[i];
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = 1.f / sum;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= inv;
  return has;
}

// Adds nb blocks' partials in block order and writes loss, counts and coef
// (coef[e] = E f_e / n, the per-expert factor of the gradient).
template <int NT>
__device__ void finish(const float* p_part, const int* c_part, const int* n_part, int nb, int E, int k, float* loss,
                       int32_t* counts, float* coef) {
  __shared__ float s_p[NT], s_loss[NT / 32];
  __shared__ int s_c[NT], s_n[NT / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int n = 0;
  for (int b = tid; b < nb; b += NT) n += n_part[b];
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) s_n[warp] = n;
  // thread (slice, expert): SL slices of the blocks per expert
  const int EP = E <= 8 ? 8 : E <= 16 ? 16 : E <= 32 ? 32 : E <= 64 ? 64 : E <= 128 ? 128 : 256;
  const int SL = NT / EP, e = tid % EP, sl = tid / EP;
  float p = 0.f;
  int c = 0;
  if (e < E) {
#pragma unroll 8
    for (int b = sl * nb / SL; b < (sl + 1) * nb / SL; ++b) {
      p += p_part[(size_t)b * E + e];
      c += c_part[(size_t)b * E + e];
    }
  }
  s_p[tid] = p;
  s_c[tid] = c;
  __syncthreads();
  n = 0;
  for (int w = 0; w < NT / 32; ++w) n += s_n[w];
  float term = 0.f;
  if (tid < E) {
    for (int s = 1; s < SL; ++s) {
      p += s_p[s * EP + tid];
      c += s_c[s * EP + tid];
    }
    counts[tid] = c;
    const float inv = n > 0 ? 1.f / (float)n : 0.f;
    const float ef = (float)E * ((float)c * inv / (float)k);  // E f_e
    coef[tid] = ef * inv;
    term = n > 0 ? ef * (p * inv) : 0.f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) term += __shfl_xor_sync(0xffffffffu, term, o);
  if (lane == 0) s_loss[warp] = term;
  __syncthreads();
  if (tid == 0) {
    float t = 0.f;
    for (int w = 0; w < NT / 32; ++w) t += s_loss[w];
    *loss = t;
  }
}

// One block's share of the rows -> sums of p, counts and live tokens.  A
// block that is alone finishes the loss itself.
template <class T, int G, bool VEC>
__global__ void __launch_bounds__(THREADS) partial_kernel(const T* __restrict__ logits, const int32_t* __restrict__ topi,
                                                          const uint8_t* __restrict__ mask, int64_t T_, int E, int k,
                                                          float* p_part, int* c_part, int* n_part, float* loss,
                                                          int32_t* counts, float* coef, int* status) {
  constexpr int RPW = 32 / G;  // rows per warp and step
  __shared__ float s_p[THREADS / 32][MAX_EXPERTS];
  __shared__ int s_c[MAX_EXPERTS], s_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gl = lane % G, gr = lane / G, e0 = gl * 8;
  for (int e = tid; e < MAX_EXPERTS; e += THREADS) s_c[e] = 0;
  if (tid == 0) s_n = 0;
  __syncthreads();
  float acc[8] = {};
  int n = 0;
  bool bad = false;
  const int64_t step = (int64_t)gridDim.x * (THREADS / 32) * RPW;
  // every lane of a warp makes the same number of steps (shuffles inside)
  for (int64_t t0 = ((int64_t)blockIdx.x * (THREADS / 32) + warp) * RPW; t0 < T_; t0 += UNROLL * step) {
    float v[UNROLL][8];
    int choice[UNROLL];  // this lane's first choice of each row
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t t = t0 + u * step + gr;
      load_row<T, VEC>(logits, mask, t, T_, e0, E, v[u]);
      choice[u] = t < T_ && gl < k ? topi[t * k + gl] : -1;
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (!softmax8<G>(v[u])) continue;  // not live; the row's G lanes agree and the shuffles are behind
      const int64_t t = t0 + u * step + gr;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e0 + i < E) acc[i] += v[u][i];
      n += gl == 0;
      for (int j = gl; j < k; j += G) {
        const int e = j == gl ? choice[u] : topi[t * k + j];
        if (e >= 0 && e < E)
          atomicAdd(&s_c[e], 1);
        else if (e != -1)
          bad = true;
      }
    }
    __syncwarp();
  }
  if (bad && status) atomicOr(status, B200Q_DEV_ERR_BOUNDS);
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0 && n) atomicAdd(&s_n, n);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int o = G; o < 32; o <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    if (gr == 0) s_p[warp][e0 + i] = acc[i];
  }
  __syncthreads();
  for (int e = tid; e < E; e += THREADS) {
    float p = 0.f;
    for (int w = 0; w < THREADS / 32; ++w) p += s_p[w][e];
    p_part[(size_t)blockIdx.x * E + e] = p;
    c_part[(size_t)blockIdx.x * E + e] = s_c[e];
  }
  if (tid == 0) n_part[blockIdx.x] = s_n;
  pdl_launch_next();
  if (gridDim.x == 1) {
    __syncthreads();  // the block's own global writes are visible to all its threads
    finish<THREADS>(p_part, c_part, n_part, 1, E, k, loss, counts, coef);
  }
}

__global__ void __launch_bounds__(THREADS) finish_kernel(const float* p_part, const int* c_part, const int* n_part,
                                                         int nb, int E, int k, float* loss, int32_t* counts,
                                                         float* coef) {
  pdl_wait_previous();
  finish<THREADS>(p_part, c_part, n_part, nb, E, k, loss, counts, coef);
}

template <class T, int G, bool VEC>
__global__ void __launch_bounds__(GRAD_THREADS) grad_kernel(const T* __restrict__ logits, const uint8_t* __restrict__ mask,
                                                       const float* __restrict__ coef,
                                                       const float* __restrict__ dloss, int64_t T_, int E,
                                                       T* __restrict__ dlogits) {
  constexpr int RPW = 32 / G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane % G, gr = lane / G, e0 = gl * 8;
  const float g = *dloss;
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = e0 + i < E ? coef[e0 + i] : 0.f;
  const int64_t step = (int64_t)gridDim.x * (GRAD_THREADS / 32) * RPW;
  float next[8];  // the row after this one is requested before this one is used
  int64_t t0 = ((int64_t)blockIdx.x * (GRAD_THREADS / 32) + warp) * RPW;
  load_row<T, VEC>(logits, mask, t0 + gr, T_, e0, E, next);
  for (; t0 < T_; t0 += step) {
    const int64_t t = t0 + gr;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = next[i];
    load_row<T, VEC>(logits, mask, t + step, T_, e0, E, next);
    const bool live = softmax8<G>(v);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) dot = fmaf(v[i], f[i], dot);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (t >= T_) continue;
    T out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = ft<T>(live ? g * v[i] * (f[i] - dot) : 0.f);
    T* row = dlogits + t * E;
    if (VEC) {
      if (e0 < E) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) * 8 / 16); ++i)
          reinterpret_cast<uint4*>(row + e0)[i] = reinterpret_cast<const uint4*>(out)[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e0 + i < E) row[e0 + i] = out[i];
    }
  }
}

int lanes_per_row(int64_t E) {
  int g = 1;
  while (8 * g < E) g *= 2;
  return g;
}

int blocks_for(int64_t T, int64_t E) {
  if (T * E <= SINGLE_ELEMS) return 1;
  const int64_t rows = (THREADS / 32) * (32 / lanes_per_row(E));  // per block and step
  return (int)std::min<int64_t>((T + rows - 1) / rows, MAX_BLOCKS);
}

// Calls f with the logits type, G and VEC as compile-time values.
template <class T, class F>
void by_width(int g, bool vec, F f) {
  auto w = [&](auto gc) {
    if (vec)
      f(gc, std::true_type{});
    else
      f(gc, std::false_type{});
  };
  switch (g) {
    case 1: return w(std::integral_constant<int, 1>{});
    case 2: return w(std::integral_constant<int, 2>{});
    case 4: return w(std::integral_constant<int, 4>{});
    case 8: return w(std::integral_constant<int, 8>{});
    case 16: return w(std::integral_constant<int, 16>{});
    default: return w(std::integral_constant<int, 32>{});
  }
}

static int check_shape(int64_t T, int64_t E, int dtype) {
  if (dtype != B200Q_DTYPE_FP16 && dtype != B200Q_DTYPE_BF16 && dtype != B200Q_DTYPE_FP32)
    return fail(B200Q_ERR_UNSUPPORTED, "moe_balance: dtype must be fp16, bf16 or fp32");
  if (E < 2 || E > MAX_EXPERTS) return fail(B200Q_ERR_SHAPE, "moe_balance: need 2 <= E <= 256");
  if (T < 0 || T > (1ll << 27)) return fail(B200Q_ERR_SHAPE, "moe_balance: need 0 <= T <= 2^27");
  return B200Q_OK;
}

template <class T>
void launch_forward(const void* logits, const int32_t* topi, const uint8_t* mask, int64_t T_, int E, int k,
                    float* loss, int32_t* counts, float* coef, void* scratch, int* status, cudaStream_t st) {
  const int nb = blocks_for(T_, E);
  float* pp = reinterpret_cast<float*>(scratch);
  int* cp = reinterpret_cast<int*>(pp + (size_t)nb * E);
  int* np = cp + (size_t)nb * E;
  const bool vec = E % 8 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
  by_width<T>(lanes_per_row(E), vec, [&](auto gc, auto vc) {
    partial_kernel<T, decltype(gc)::value, decltype(vc)::value>
        <<<nb, THREADS, 0, st>>>(reinterpret_cast<const T*>(logits), topi, mask, T_, E, k, pp, cp, np, loss, counts,
                                 coef, status);
  });
  if (nb > 1) {  // its start overlaps the partial kernel's end
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, finish_kernel, (const float*)pp, (const int*)cp, (const int*)np, nb, E, k, loss, counts, coef);
  }
}

template <class T>
void launch_grad(const void* logits, const uint8_t* mask, const float* coef, const float* dloss, int64_t T_, int E,
                 void* dlogits, cudaStream_t st) {
  const int g = lanes_per_row(E);
  const int64_t rows = (GRAD_THREADS / 32) * (32 / g);
  const unsigned nb = (unsigned)std::min<int64_t>((T_ + rows - 1) / rows, 8 * 148);
  const bool vec = E % 8 == 0 && ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(dlogits)) & 15) == 0;
  by_width<T>(g, vec, [&](auto gc, auto vc) {
    grad_kernel<T, decltype(gc)::value, decltype(vc)::value><<<nb, GRAD_THREADS, 0, st>>>(
        reinterpret_cast<const T*>(logits), mask, coef, dloss, T_, E, reinterpret_cast<T*>(dlogits));
  });
}

}  // namespace balance
}  // namespace b200q

extern "C" {

size_t b200q_moe_balance_scratch_bytes(int64_t T, int64_t E) {
  if (T < 0 || E < 2 || E > b200q::balance::MAX_EXPERTS) return 256;
  const size_t nb = (size_t)b200q::balance::blocks_for(T, E);
  return nb * (2 * (size_t)E + 1) * 4;
}

int b200q_moe_balance(const void* logits, const int32_t* topi, const uint8_t* mask, int64_t T, int64_t E, int64_t k,
                      int dtype, float* loss, int32_t* counts, float* coef, void* scratch, size_t scratch_bytes,
                      void* workspace, void* stream) {
  using namespace b200q;
  using namespace b200q::balance;
  int rc = check_shape(T, E, dtype);
  if (rc) return rc;
  if (k < 1 || k > MAX_K || k > E) return fail(B200Q_ERR_SHAPE, "moe_balance: need 1 <= k <= min(8, E)");
  if (!loss || !counts || !coef || (T > 0 && (!logits || !topi)))
    return fail(B200Q_ERR_SHAPE, "moe_balance: null pointer argument");
  if (!scratch || scratch_bytes < b200q_moe_balance_scratch_bytes(T, E))
    return fail(B200Q_ERR_WORKSPACE, "moe_balance: scratch of " +
                                         std::to_string(b200q_moe_balance_scratch_bytes(T, E)) + " bytes required");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int* status = reinterpret_cast<int*>(workspace);
  if (dtype == B200Q_DTYPE_FP16)
    launch_forward<__half>(logits, topi, mask, T, (int)E, (int)k, loss, counts, coef, scratch, status, st);
  else if (dtype == B200Q_DTYPE_BF16)
    launch_forward<__nv_bfloat16>(logits, topi, mask, T, (int)E, (int)k, loss, counts, coef, scratch, status, st);
  else
    launch_forward<float>(logits, topi, mask, T, (int)E, (int)k, loss, counts, coef, scratch, status, st);
  return check_cuda(cudaGetLastError(), "moe_balance launch");
}

int b200q_moe_balance_grad(const void* logits, const uint8_t* mask, const float* coef, const float* dloss, int64_t T,
                           int64_t E, int dtype, void* dlogits, void* stream) {
  using namespace b200q;
  using namespace b200q::balance;
  int rc = check_shape(T, E, dtype);
  if (rc) return rc;
  if (T == 0) return B200Q_OK;
  if (!logits || !coef || !dloss || !dlogits) return fail(B200Q_ERR_SHAPE, "moe_balance_grad: null pointer argument");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == B200Q_DTYPE_FP16)
    launch_grad<__half>(logits, mask, coef, dloss, T, (int)E, dlogits, st);
  else if (dtype == B200Q_DTYPE_BF16)
    launch_grad<__nv_bfloat16>(logits, mask, coef, dloss, T, (int)E, dlogits, st);
  else
    launch_grad<float>(logits, mask, coef, dloss, T, (int)E, dlogits, st);
  return check_cuda(cudaGetLastError(), "moe_balance_grad launch");
}

}  // extern "C"
