// Input gradient of the frozen W4A16 projection for few rows (M <= 16):
//   dx[m, k] = sum_n dy[m, n] ((nib(k, n) - z[k/g, n]) s[k/g, n]).
//
// With one 16-row operand the dequantising tensor-core tile (w4a16_tc.cu's
// MODE_DX, 128 rows of dy) spends its time on rows that are not there.  Here
// mma.sync m16n8k16 takes dy as the 16 rows, and the weight, dequantised as the
// forward does, straight from a lane's packed words as the other fragment.  Of
// the contraction any order serves that both operands share: a lane's 32 columns
// of a weight row are its parts of 8 k16 steps, in the order in which a word
// unpacks, so no dequantised value passes through shared memory.
// A CTA takes 128 weight rows: 8 column parts x 2 halves of 64 rows, one warp
// each; the two warps at the same columns share a two-stage TMA ring of dy, words,
// scales and zero points.  The S CTAs of a cluster share the columns too; sums are
// joined in a fixed order.
// Bound: HBM (the packed weight once: 32 MB at N=4096, K=14336, 4.9 us at the
// measured copy rate) but for the instructions: 15 per packed word, 8 of them on
// the half-rate fp16 pipe.  Measured there: 15.0 us, 9 us of it in the products (by
// clock stamps), 2 in start and 1.5 in joining.  Before: the same tile fed by
// 16-byte copies of the lanes 23 us (they held up the load unit), 64-row tiles with
// the scale on dy's side 21 us, the 128-row tensor-core tile 29 us.
#include <algorithm>

#include "w4a16_dq.cuh"

namespace b200q {
namespace dx16 {

constexpr int TILE = 128, ROWS = 64, RB = ROWS / 8;  // weight rows of a CTA, of a warp; a warp's 8-row blocks
constexpr int WC = 8, WARPS = WC * TILE / ROWS, THREADS = WARPS * 32;  // warps across the columns; all
constexpr int CHUNK = 128;  // columns of a step of the two warps that share them
constexpr int MAX_S = 8, STAGES = 2;
// A stage: dy as two boxes of 64 columns (128-byte swizzle), the packed words, the groups' scales and zero points
constexpr int DY_BYTES = 16 * CHUNK * 2, W_BYTES = TILE * CHUNK / 2, SZ_BYTES = CHUNK * 2;
constexpr int OFF_W = DY_BYTES, OFF_S = OFF_W + W_BYTES;
constexpr int RPITCH = TILE + 4, RED = (WC + 1) * 16 * RPITCH * 4;
template <int GROUPS>
constexpr int STAGE_BYTES = (OFF_S + 2 * GROUPS * SZ_BYTES + 1023) / 1024 * 1024;
template <int GROUPS>
constexpr int SMEM = 1024 + WC * STAGES * STAGE_BYTES<GROUPS> + 256;
static_assert(SMEM<4> <= 227 * 1024 && RED <= WC * STAGES * STAGE_BYTES<1>, "shared memory budget");

// 8 consecutive values -> the pairs (0,4) (1,5) (2,6) (3,7)
__device__ __forceinline__ void pairs(const uint4 v, uint32_t* p) {
  p[0] = prmt(v.x, v.z, 0x5410);
  p[1] = prmt(v.x, v.z, 0x7632);
  p[2] = prmt(v.y, v.w, 0x5410);
  p[3] = prmt(v.y, v.w, 0x7632);
}

__device__ __forceinline__ uint4 lds(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

template <bool BF16>
__device__ __forceinline__ void mma(float* d, const uint32_t (*a)[4], int j, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0][j]), "r"(a[1][j]), "r"(a[0][j + 1]), "r"(a[1][j + 1]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0][j]), "r"(a[1][j]), "r"(a[0][j + 1]), "r"(a[1][j + 1]), "r"(b0), "r"(b1));
}

template <bool BF16>
__device__ __forceinline__ uint16_t rounded(float v) {
  if (BF16) {
    const __nv_bfloat16 b = __float2bfloat16_rn(v);
    return *reinterpret_cast<const uint16_t*>(&b);
  }
  const __half h = __float2half_rn(v);
  return *reinterpret_cast<const uint16_t*>(&h);
}

// GROUPS: weight groups of a tile (1: the group size is 128 or 256).
template <bool BF16, int GROUPS>
__global__ void __launch_bounds__(THREADS, 1)
    dgrad_small_kernel(const __grid_constant__ CUtensorMap tm_dy, const __grid_constant__ CUtensorMap tm_w,
                       const __grid_constant__ CUtensorMap tm_s, const __grid_constant__ CUtensorMap tm_z,
                       uint16_t* __restrict__ dx, int M, int N, int K, int group, int S, int* status) {
  extern __shared__ uint8_t sm_raw[];
  uint8_t* const sm = align_smem_1024(sm_raw);
  constexpr int STAGE = STAGE_BYTES<GROUPS>, SUBS = GROUPS == 4 ? 2 : 1;  // groups of a warp's rows
  uint64_t* const full = reinterpret_cast<uint64_t*>(sm + WC * STAGES * STAGE);  // [wc][stage]
  const int tile = (int)blockIdx.x / S, rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wc = warp % WC, half = warp / WC;  // columns and rows of the tile
  uint8_t* const ring = sm + wc * STAGES * STAGE;
  uint64_t* const bar = full + wc * STAGES;
  const bool asks = half == 0 && lane == 0;
  auto request = [&](int n, int slot) {  // one thread; beyond the tensors' ends the copies write zeros
    uint8_t* const st = ring + slot * STAGE;
    mbar_arrive_expect_tx(bar + slot, DY_BYTES + W_BYTES + 2 * GROUPS * SZ_BYTES);
    tma_load_2d(st + OFF_W, &tm_w, n / 8, tile * TILE, bar + slot);
    tma_load_2d(st, &tm_dy, n, 0, bar + slot);
    tma_load_2d(st + DY_BYTES / 2, &tm_dy, n + CHUNK / 2, 0, bar + slot);
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      const int row = (tile * TILE + i * (TILE / GROUPS)) / group;
      tma_load_2d(st + OFF_S + i * SZ_BYTES, &tm_s, n, row, bar + slot);
      tma_load_2d(st + OFF_S + (GROUPS + i) * SZ_BYTES, &tm_z, n, row, bar + slot);
    }
  };
  // Steps of this warp pair: every (S WC)-th chunk
  const int chunks = (N + CHUNK - 1) / CHUNK, stride = S * WC, first = rank * WC + wc;
  const int steps = first < chunks ? (chunks - first + stride - 1) / stride : 0;
  auto column = [&](int step) { return (first + step * stride) * CHUNK; };
  if (asks) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i) mbar_init(bar + i, 1);
    fence_barrier_init();
    for (int i = 0; i < STAGES && i < steps; ++i) request(column(i), i);
  }
  __syncthreads();  // the barriers are there
  float tot[RB][4] = {};
  bool ok = true;
  for (int step = 0; step < steps; ++step) {
    const int slot = step % STAGES;
    const uint8_t* const st = ring + slot * STAGE;
    ok = ok && mbar_wait(bar + slot, (step / STAGES) & 1, status);
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub) {
      constexpr int NB = RB / SUBS;
      uint4 wb[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) wb[b] = lds(st + OFF_W + (half * ROWS + (sub * NB + b) * 8 + g) * (CHUNK / 2) + t * 16);
      const uint8_t* const srow = st + OFF_S + (GROUPS == 1 ? 0 : half * SUBS + sub) * SZ_BYTES;
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // 8 of the lane's 32 columns: its part of two k16 steps
        const tc::ColQ q = tc::load_colq<BF16>(srow, srow + GROUPS * SZ_BYTES, 4 * t + i);
        uint32_t a[2][4];  // dy of rows g, g + 8
#pragma unroll
        for (int h = 0; h < 2; ++h)
          pairs(lds(st + (t >> 1) * (DY_BYTES / 2) + (g + 8 * h) * 128 + (((t & 1) * 4 + i) ^ g) * 16), a[h]);
#pragma unroll
        for (int b = 0; b < NB; b += 2) {  // two row blocks in turn: their products do not wait for one another
          const uint4 v0 = tc::dequant_word<BF16>(reinterpret_cast<const uint32_t*>(&wb[b])[i], q);
          const uint4 v1 = tc::dequant_word<BF16>(reinterpret_cast<const uint32_t*>(&wb[b + 1])[i], q);
          float *c0 = tot[sub * NB + b], *c1 = tot[sub * NB + b + 1];
          mma<BF16>(c0, a, 0, v0.x, v0.y);
          mma<BF16>(c1, a, 0, v1.x, v1.y);
          mma<BF16>(c0, a, 2, v0.z, v0.w);
          mma<BF16>(c1, a, 2, v1.z, v1.w);
        }
      }
    }
    asm volatile("bar.sync %0, 64;" ::"r"(1 + wc) : "memory");  // both warps have read the stage
    if (asks && ok && step + STAGES < steps) request(column(step + STAGES), slot);
  }
  if (asks && !ok)  // given up: what was asked for may still arrive
    for (int i = 0; i < STAGES && i < steps; ++i) {
      const int last = steps - 1 - (steps - 1 - i) % STAGES;
      mbar_wait(bar + i, (last / STAGES) & 1, nullptr);
    }
  __syncthreads();
  // the warps' sums, then the cluster's, in order
  float* red = reinterpret_cast<float*>(sm);  // [wc][16][RPITCH], then this CTA's sums
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    float* r = red + (wc * 16 + g) * RPITCH + half * ROWS + 8 * b + 2 * t;
    *reinterpret_cast<float2*>(r) = make_float2(tot[b][0], tot[b][1]);
    *reinterpret_cast<float2*>(r + 8 * RPITCH) = make_float2(tot[b][2], tot[b][3]);
  }
  __syncthreads();
  float* const part = red + WC * 16 * RPITCH;
#pragma unroll
  for (int i = tid; i < 16 * TILE / 2; i += THREADS) {
    const int m = i / (TILE / 2), c = i % (TILE / 2) * 2;
    float2 v = make_float2(0.f, 0.f);
#pragma unroll
    for (int q = 0; q < WC; ++q) {
      const float2 u = *reinterpret_cast<const float2*>(red + (q * 16 + m) * RPITCH + c);
      v.x += u.x, v.y += u.y;
    }
    if (S > 1)
      *reinterpret_cast<float2*>(part + m * RPITCH + c) = v;
    else if (m < M && tile * TILE + c < K)  // K is even
      *reinterpret_cast<uint32_t*>(dx + (size_t)m * K + tile * TILE + c) =
          (uint32_t)rounded<BF16>(v.x) | (uint32_t)rounded<BF16>(v.y) << 16;
  }
  if (S == 1) return;
  cluster_sync();
  const int nq = TILE / S, q0 = rank * nq;  // this rank's columns of the tile
  for (int i = tid; i < 16 * nq / 2; i += THREADS) {
    const int m = i / (nq / 2), c = q0 + i % (nq / 2) * 2;
    if (m >= M || tile * TILE + c >= K) continue;
    float2 v = make_float2(0.f, 0.f);
    const uint32_t addr = smem_u32(part + m * RPITCH + c);
    for (int q = 0; q < S; ++q) {
      float2 u;
      asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(u.x), "=f"(u.y) : "r"(map_shared_rank(addr, q)) : "memory");
      v.x += u.x, v.y += u.y;
    }
    *reinterpret_cast<uint32_t*>(dx + (size_t)m * K + tile * TILE + c) =
        (uint32_t)rounded<BF16>(v.x) | (uint32_t)rounded<BF16>(v.y) << 16;
  }
  cluster_sync();  // the others have read this CTA's sums
}

}  // namespace dx16

int w4a16_dgrad_small(const void* dy, const int32_t* qweight, const void* scales, const void* zeros, void* dx, int64_t M,
                      int64_t N, int64_t K, int64_t group, int dtype, void* workspace, cudaStream_t stream) {
  using namespace dx16;
  const bool bf = dtype == B200Q_DTYPE_BF16;
  const int groups = group == 32 ? 4 : group == 64 ? 2 : 1;
  auto kern = groups == 4   ? (bf ? dgrad_small_kernel<true, 4> : dgrad_small_kernel<false, 4>)
              : groups == 2 ? (bf ? dgrad_small_kernel<true, 2> : dgrad_small_kernel<false, 2>)
                            : (bf ? dgrad_small_kernel<true, 1> : dgrad_small_kernel<false, 1>);
  const int smem = groups == 4 ? SMEM<4> : groups == 2 ? SMEM<2> : SMEM<1>;
  int rc = allow_smem((const void*)kern, smem, "cudaFuncSetAttribute(w4a16 dgrad small)");
  if (rc) return rc;
  const CUtensorMapDataType dt = bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tm_dy, tm_w, tm_s, tm_z;
  rc = encode_2d(&tm_dy, dt, dy, (uint64_t)N, (uint64_t)M, (uint64_t)N * 2, CHUNK / 2, 16, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc)
    rc = encode_2d(&tm_w, CU_TENSOR_MAP_DATA_TYPE_INT32, qweight, (uint64_t)N / 8, (uint64_t)K, (uint64_t)N / 2, CHUNK / 8,
                   TILE, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (!rc)
    rc = encode_2d(&tm_s, dt, scales, (uint64_t)N, (uint64_t)(K / group), (uint64_t)N * 2, CHUNK, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (!rc)
    rc = encode_2d(&tm_z, dt, zeros, (uint64_t)N, (uint64_t)(K / group), (uint64_t)N * 2, CHUNK, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc) return rc;
  // the split of the columns with the shortest estimate: rounds of co-resident
  // clusters x (a pair's steps + 2 for start and joining)
  const int64_t tiles = (K + TILE - 1) / TILE, chunks = (N + CHUNK - 1) / CHUNK;
  int S = 1;
  int64_t best = INT64_MAX;
  const int* fit = resident_clusters((const void*)kern, THREADS, smem);
  for (int s = 1; s <= MAX_S && (s == 1 || s * WC < chunks + WC); s *= 2) {
    const int64_t cost = ((tiles + fit[s] - 1) / fit[s]) * ((chunks + s * WC - 1) / (s * WC) + 2);
    if (cost < best) best = cost, S = s;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * S));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, tm_dy, tm_w, tm_s, tm_z, reinterpret_cast<uint16_t*>(dx), (int)M, (int)N,
                                       (int)K, (int)group, S, reinterpret_cast<int*>(workspace)),
                    "w4a16 dgrad small launch");
}

}  // namespace b200q
