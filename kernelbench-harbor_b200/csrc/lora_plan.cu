// The batch's plan (tokens grouped by adapter, tiles) and the C entry points
// of the multi-adapter operators.
//
// One block: 32 warps take 32 consecutive ranges of the tokens, count their
// ids into a table of their own (a match within the warp gives a token's rank
// among its equals), a scan over segments and warps turns the counts into
// first positions, and a second walk writes the tokens: a stable counting sort
// without atomics, so a plan is the same every time.  A batch needs it once for
// all projections of a model.  Bound: latency, ~T / 1024 dependent steps twice:
// 4.6 us for 64 tokens, 8.2 for 8192, 44 for 65536 (one block is enough for a
// batch of a serving or training step; more would gain from several).
#include <type_traits>

#include "lora_seg.cuh"

namespace b200q {
namespace lora {

constexpr int PLAN_THREADS = 1024, PLAN_WARPS = 32;

__device__ __forceinline__ int segment_of(int64_t id, int L) { return id >= 0 && id < L ? (int)id : L; }

__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const int64_t* __restrict__ ids, int T, int L,
                                                            int32_t* __restrict__ plan, PlanLayout lay, int* status) {
  extern __shared__ int sm[];
  int* cnt = sm;                               // [32][L + 1]
  int* off = sm + PLAN_WARPS * (L + 1);        // [L + 2] first position of a segment
  int* ts = off + (L + 2);                     // [L + 2] first small tile
  int* tl = ts + (L + 2);                      // [L + 2] first large tile
  __shared__ int s_sum[3][PLAN_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < PLAN_WARPS * (L + 1); i += PLAN_THREADS) cnt[i] = 0;
  __syncthreads();
  const int t0 = (int)((int64_t)warp * T / PLAN_WARPS), t1 = (int)((int64_t)(warp + 1) * T / PLAN_WARPS);
  int* mine = cnt + warp * (L + 1);
  bool bad = false;
  for (int b = t0; b < t1; b += 32) {
    const int t = b + lane;
    const int64_t id = t < t1 ? ids[t] : -1;
    bad |= id < -1 || id >= L;
    const int seg = t < t1 ? segment_of(id, L) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, seg);
    if (seg >= 0 && lane == __ffs(same) - 1) mine[seg] += __popc(same);
    __syncwarp();
  }
  if (bad && status) atomicOr(status, B200Q_DEV_ERR_BOUNDS);
  __syncthreads();
  // segment `tid`: its length, then an exclusive scan of lengths and tile counts
  int v[3] = {0, 0, 0}, x[3];
  if (tid <= L) {
    for (int w = 0; w < PLAN_WARPS; ++w) v[0] += cnt[w * (L + 1) + tid];
    v[1] = (v[0] + ROWS_S - 1) / ROWS_S;
    v[2] = (v[0] + ROWS_L - 1) / ROWS_L;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    x[j] = v[j];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x[j], o);
      if (lane >= o) x[j] += u;
    }
    if (lane == 31) s_sum[j][warp] = x[j];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    int before = 0;
    for (int w = 0; w < warp; ++w) before += s_sum[j][w];
    x[j] += before;
  }
  if (tid <= L) {
    off[tid] = x[0] - v[0];
    ts[tid] = x[1] - v[1];
    tl[tid] = x[2] - v[2];
    plan[lay.seg + tid] = x[0] - v[0];
    int at = x[0] - v[0];
    for (int w = 0; w < PLAN_WARPS; ++w) {
      const int c = cnt[w * (L + 1) + tid];
      cnt[w * (L + 1) + tid] = at;
      at += c;
    }
    if (tid == L) {
      off[L + 1] = x[0];
      ts[L + 1] = x[1];
      tl[L + 1] = x[2];
      plan[lay.seg + L + 1] = x[0];
      plan[0] = x[1];
      plan[1] = x[2];
    }
  }
  __syncthreads();
  for (int b = t0; b < t1; b += 32) {
    const int t = b + lane;
    const int seg = t < t1 ? segment_of(ids[t], L) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, seg);
    int at = 0;
    if (seg >= 0) at = mine[seg] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (seg >= 0) {
      plan[lay.order + at] = t;
      if (lane == __ffs(same) - 1) mine[seg] += __popc(same);
    }
    __syncwarp();
  }
  // tile tables: the segment of tile i by bisection of the first-tile array
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    const int* first = kind ? tl : ts;
    const int rows = kind ? ROWS_L : ROWS_S;
    int4* out = reinterpret_cast<int4*>(plan + (kind ? lay.large : lay.small));
    for (int i = tid; i < first[L + 1]; i += PLAN_THREADS) {
      int lo = 0, hi = L + 1;  // first[lo] <= i < first[hi]
      while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (first[m] <= i)
          lo = m;
        else
          hi = m;
      }
      const int a = off[lo] + (i - first[lo]) * rows;
      out[i] = make_int4(lo < L ? lo : -1, a, min(rows, off[lo + 1] - a), 0);
    }
  }
}

int launch_grads(const void* x, const void* dy, const float* lo, const float* dlo, const int32_t* plan,
                 const PlanLayout& lay, int64_t T, int64_t D, int64_t N, int64_t r, int64_t L, int dtype, float* part,
                 void* dA, void* dB, cudaStream_t st);
size_t grads_part_bytes(int64_t T, int64_t D, int64_t N, int64_t r, int64_t L, int dtype);

// Up to this many tokens the one-launch cluster kernel runs, above it the
// tiled pair (which needs room for the row between).  Measured, bf16, us with
// one launch / the pair, one adapter:
//   4096 x 4096:   r 16, 64 tokens 5.5 / 8.9, 256 6.7 / 10.0, 512 7.4 / 11.0; r 32 7.5 / 10.0, 9.6 / 11.2, 11.3 / 12.7
//   14336 -> 4096: r 16, 256 tokens 9.3 / 16.8; 4096 -> 14336: 10.6 / 12.2
// At ranks 33 to 64 a CTA takes 160 KB of shared memory, so one fits an SM, and
// above 128 tokens the tiles soon take a second round of clusters:
//   4096 x 4096:   r 64, 64 tokens 13.2 / 11.4, 128 13.2 / 12.9, 256 25.3 / 14.0; of 8 adapters 12.9 / 12.6, 13.2 / 13.2, 25.2 / 13.6
//   4096 -> 14336: 128 tokens 18.3 / 14.1, of 8 adapters 18.4 / 23.8, 256 35.0 / 15.6 and 35.0 / 23.3
// The transposed form (dx) differs from these by less than 1.5 us.
constexpr int64_t SMALL_MAX_T = 256, SMALL_MAX_T_HIGH = 128;

static int launch(const Args& a, int dtype, bool tr, cudaStream_t st) {
  const bool small = a.T <= (a.r > 32 && a.mid ? SMALL_MAX_T_HIGH : SMALL_MAX_T);
  return small ? launch_small(a, dtype, tr, st) : launch_tiles(a, dtype, tr, st);
}

static int check_sizes(const char* what, int64_t T, int64_t D, int64_t N, int64_t r, int64_t L, int dtype) {
  const std::string w(what);
  if (dtype != B200Q_DTYPE_FP16 && dtype != B200Q_DTYPE_BF16)
    return fail(B200Q_ERR_UNSUPPORTED, w + ": dtype must be fp16 or bf16");
  if (T < 0 || T > MAX_TOKENS) return fail(B200Q_ERR_SHAPE, w + ": need 0 <= T <= 2^24");
  if (L < 1 || L > MAX_ADAPTERS) return fail(B200Q_ERR_SHAPE, w + ": need 1 <= L <= 1023");
  if (r < 1 || r > MAX_RANK) return fail(B200Q_ERR_SHAPE, w + ": need 1 <= r <= 64");
  if (D < 1 || N < 1 || D > (1 << 22) || N > (1 << 22)) return fail(B200Q_ERR_SHAPE, w + ": need 1 <= D, N <= 2^22");
  return B200Q_OK;
}

static bool misaligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 15) return true;
  return false;
}

}  // namespace lora
}  // namespace b200q

extern "C" {

size_t b200q_lora_plan_bytes(int64_t T, int64_t L) {
  if (T < 0 || T > b200q::lora::MAX_TOKENS || L < 1 || L > b200q::lora::MAX_ADAPTERS) return 0;
  return (size_t)b200q::lora::plan_layout(T, L).words * 4;
}

int b200q_lora_plan(const int64_t* lora_ids, int64_t T, int64_t L, int32_t* plan, size_t plan_bytes, void* workspace,
                    void* stream) {
  using namespace b200q;
  using namespace b200q::lora;
  if (T < 0 || T > MAX_TOKENS) return fail(B200Q_ERR_SHAPE, "lora_plan: need 0 <= T <= 2^24");
  if (L < 1 || L > MAX_ADAPTERS) return fail(B200Q_ERR_SHAPE, "lora_plan: need 1 <= L <= 1023");
  if (!plan || (T > 0 && !lora_ids)) return fail(B200Q_ERR_SHAPE, "lora_plan: null pointer argument");
  if (plan_bytes < b200q_lora_plan_bytes(T, L))
    return fail(B200Q_ERR_WORKSPACE, "lora_plan: a plan of " + std::to_string(b200q_lora_plan_bytes(T, L)) + " bytes required");
  if (misaligned({plan})) return fail(B200Q_ERR_ALIGN, "lora_plan: plan must be 16-byte aligned");
  const int smem = (int)((PLAN_WARPS * (L + 1) + 3 * (L + 2)) * 4);
  if (smem > 48 * 1024) {
    const int rc = allow_smem((const void*)plan_kernel, smem, "cudaFuncSetAttribute(lora plan)");
    if (rc) return rc;
  }
  plan_kernel<<<1, PLAN_THREADS, smem, reinterpret_cast<cudaStream_t>(stream)>>>(
      lora_ids, (int)T, (int)L, plan, plan_layout(T, L), reinterpret_cast<int*>(workspace));
  return check_cuda(cudaGetLastError(), "lora_plan launch");
}

size_t b200q_lora_mid_bytes(int64_t T, int64_t r) {
  if (T < 0 || r < 1 || r > b200q::lora::MAX_RANK) return 0;
  return (size_t)T * b200q::lora::mid_pitch(r) * 4;
}

int b200q_lora_apply(const void* x, const void* base, const void* A, const void* B, const float* scaling,
                     const int32_t* plan, int64_t T, int64_t D, int64_t N, int64_t r, int64_t L, int dtype, void* y,
                     float* lo, void* workspace, void* stream) {
  using namespace b200q;
  using namespace b200q::lora;
  int rc = check_sizes("lora_apply", T, D, N, r, L, dtype);
  if (rc) return rc;
  if (T == 0) return B200Q_OK;
  if (!x || !A || !B || !plan || !y || (!lo && T > SMALL_MAX_T))
    return fail(B200Q_ERR_SHAPE, "lora_apply: null pointer argument");
  if (misaligned({x, base, A, B, plan, y, lo})) return fail(B200Q_ERR_ALIGN, "lora_apply: pointers must be 16-byte aligned");
  const Args a = {x, base, A, B, scaling, plan, plan_layout(T, L), (int)D, (int)N, (int)r, mid_pitch(r), y, lo, T, L,
                  reinterpret_cast<int*>(workspace)};
  return launch(a, dtype, false, reinterpret_cast<cudaStream_t>(stream));
}

size_t b200q_lora_backward_scratch_bytes(int64_t T, int64_t D, int64_t N, int64_t r, int64_t L, int dtype) {
  using namespace b200q::lora;
  if (check_sizes("lora_backward", T, D, N, r, L, dtype) || T == 0) return 0;
  return b200q_lora_mid_bytes(T, r) + grads_part_bytes(T, D, N, r, L, dtype);
}

int b200q_lora_backward(const void* x, const void* dy, const void* base, const void* A, const void* B,
                        const float* scaling, const int32_t* plan, const float* lo, int64_t T, int64_t D, int64_t N,
                        int64_t r, int64_t L, int dtype, void* scratch, size_t scratch_bytes, void* dx, void* dA,
                        void* dB, void* workspace, void* stream) {
  using namespace b200q;
  using namespace b200q::lora;
  int rc = check_sizes("lora_backward", T, D, N, r, L, dtype);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool need_dlo = dx || dA;
  if (!dx && !dA && !dB) return B200Q_OK;
  if (T > 0 && (!plan || !dy || (need_dlo && (!A || !B)) || (dA && !x) || (dB && !lo)))
    return fail(B200Q_ERR_SHAPE, "lora_backward: null pointer argument");
  if (misaligned({x, dy, base, A, B, plan, lo, scratch, dx, dA, dB}))
    return fail(B200Q_ERR_ALIGN, "lora_backward: pointers must be 16-byte aligned");
  if (T > 0 && (!scratch || scratch_bytes < b200q_lora_backward_scratch_bytes(T, D, N, r, L, dtype)))
    return fail(B200Q_ERR_WORKSPACE, "lora_backward: scratch of " +
                                         std::to_string(b200q_lora_backward_scratch_bytes(T, D, N, r, L, dtype)) +
                                         " bytes required");
  float* dlo = reinterpret_cast<float*>(scratch);
  float* part = dlo + b200q_lora_mid_bytes(T, r) / 4;
  if (T > 0 && need_dlo) {
    const Args a = {dy, base, B, A, scaling, plan, plan_layout(T, L), (int)N, (int)D, (int)r, mid_pitch(r), dx, dlo, T, L,
                    reinterpret_cast<int*>(workspace)};
    if ((rc = launch(a, dtype, true, st))) return rc;
  }
  return dA || dB ? launch_grads(x, dy, lo, dlo, plan, plan_layout(T, L), T, D, N, r, L, dtype, part, dA, dB, st) : B200Q_OK;
}

}  // extern "C"
