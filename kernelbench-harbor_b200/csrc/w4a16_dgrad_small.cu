// Input gradient of the frozen W4A16 projection for few rows (M <= 16):
//   dx[m, k] = sum_n (dy[m, n] s[k/g, n]) (nib(k, n) - z[k/g, n]).
//
// With one 16-row operand the dequantising tensor-core tile (w4a16_tc.cu's
// MODE_DX, 128 rows) spends its time forming weights for rows that are not
// there.  Here the scale goes to the other side of the product: A = dy . s, 16
// rows x 128 columns per warp, once per weight group, and B = nib - z, an exact
// small integer, straight from a lane's 16 packed bytes into the fragment of
// mma.sync m16n8k16.  Of the contraction any order serves that both operands
// share: a lane's 32 columns of a weight row are its parts of 8 k16 steps, so
// nothing passes through shared memory.  A = dy . s is rounded once to the
// activation type (where the other path rounds nib - z times s); fp16 scales a
// row by a power of two first, since s takes it towards the subnormals.
// A CTA takes 64 weight rows; its 8 warps and the S CTAs of its cluster share
// the columns, and their sums are added in a fixed order.
// Bound: HBM (the packed weight once: 32 MB at N=4096, K=14336, 4.9 us at the
// measured copy rate) but for the instructions: 9 integer and half-precision
// operations per packed word, and forming A for each 64 weight rows, half as
// many again.  Measured there: 21 us, against 29 us for the 128-row tile.
#include <algorithm>

#include "w4a16_dq.cuh"

namespace b200q {
namespace dx16 {

using tc::as_u32;
using tc::fma_f16x2;
using tc::mul_bf16x2;
using tc::mul_f16x2;
using tc::sub_bf16x2;
using tc::sub_f16x2;

constexpr int TILE = 64, RB = TILE / 8;  // weight rows of a CTA; 8-row blocks
constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int CHUNK = 128;  // columns of a warp's step
constexpr int MAX_S = 8;
constexpr int RPITCH = TILE + 4;
constexpr int STAGES = 3, STAGE = TILE * CHUNK / 2;  // a warp's ring of packed weights: a lane's 16 bytes of 8 row blocks
constexpr int RED = (WARPS + 1) * 16 * RPITCH * 4;
constexpr int SMEM = WARPS * STAGES * STAGE > RED ? WARPS * STAGES * STAGE : RED;

// 8 consecutive values -> the pairs (0,4) (1,5) (2,6) (3,7)
__device__ __forceinline__ void pairs(const uint4 v, uint32_t* p) {
  p[0] = prmt(v.x, v.z, 0x5410);
  p[1] = prmt(v.x, v.z, 0x7632);
  p[2] = prmt(v.y, v.w, 0x5410);
  p[3] = prmt(v.y, v.w, 0x7632);
}

// larger magnitude of each half (its sign bit means nothing)
__device__ __forceinline__ uint32_t max_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Exponent e of the largest magnitude among the 4 lanes' 32 fp16 values each
// (0 where all are 0, the type's largest where one is infinite) and 2^-e twice.
__device__ __forceinline__ uint32_t scale_of(const uint32_t (*v)[4], int& e) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max_f16x2(m, v[i][j]);
  m = max_f16x2(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max_f16x2(m, __shfl_xor_sync(0xffffffffu, m, 2));
  m &= 0x7FFF7FFFu;
  const uint32_t top = max(m & 0xffffu, m >> 16) >> 10;  // biased exponent; 0: zero or subnormal, 31: infinite
  // 2^-e has to be a normal fp16: e in -15 .. 14 (2^15 <= v: one step short of [1, 2), still far from the range's end)
  e = top == 0 ? -14 : min((int)top, 29) - 15;
  if (m == 0) e = 0;
  const uint32_t inv = (uint32_t)(15 - e) << 10;
  return inv | (inv << 16);
}

// A load that stays where it is written (the compiler would gather all of them at the top and spill)
__device__ __forceinline__ uint4 ldg_ordered(const uint32_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <bool BF16>
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// GT: weight rows of the tile that share a group (the group size, at most TILE).
template <bool BF16, int GT>
__global__ void __launch_bounds__(THREADS, 2)
    dgrad_small_kernel(const uint16_t* __restrict__ dy, const uint32_t* __restrict__ qw,
                       const uint16_t* __restrict__ scales, const uint16_t* __restrict__ zeros,
                       uint16_t* __restrict__ dx, int M, int N, int K, int group, int S) {
  extern __shared__ __align__(16) uint8_t sm[];
  const int k0 = (int)(blockIdx.x / S) * TILE, rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int words = N / 8;
  float tot[RB][4] = {};
  uint8_t* ring = sm + warp * STAGES * STAGE + lane * 16;
  auto request = [&](int n0, int slot) {  // the packed words that this lane multiplies in the step at n0
    const int n = n0 + 32 * t;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const bool here = n < N && k0 + 8 * b < K;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(ring + slot * STAGE + b * 512)),
                   "l"(here ? qw + (size_t)(k0 + 8 * b + g) * words + n / 8 : qw), "r"(here ? 16 : 0)
                   : "memory");
    }
  };
  const int nstep = S * WARPS * CHUNK, nfirst = (rank * WARPS + warp) * CHUNK;
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    request(nfirst + i * nstep, i);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  int slot = 0;
  for (int n0 = nfirst; n0 < N; n0 += nstep) {
    request(n0 + (STAGES - 1) * nstep, slot == 0 ? STAGES - 1 : slot - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const int n = n0 + 32 * t;  // this lane's 32 columns: all inside the row or none (N % 32 == 0)
    const bool in = n < N;
#pragma unroll
    for (int sub = 0; sub < TILE / GT; ++sub) {
      const int ks = k0 + sub * GT;
      if (ks >= K) break;  // K is a multiple of the group
      const uint16_t* srow = scales + (size_t)(ks / group) * N + n;
      const uint16_t* zrow = zeros + (size_t)(ks / group) * N + n;
      // pairs of columns (0,4) (1,5) (2,6) (3,7) of each word, as the unpacked nibbles come: the zero points as the
      // subtraction wants them, and dy . s of rows g, g + 8
      uint32_t zp[4][4], sp[4][4], a[2][4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 zv = in ? ldg_ordered(reinterpret_cast<const uint32_t*>(zrow) + 4 * i) : make_uint4(0, 0, 0, 0);
        pairs(zv, zp[i]);
        if (!BF16) {  // 1024 + z, and -(64 + z) for the nibbles that stay 16 times too large
          zp[i][0] = fma_f16x2(zp[i][0], 0x3C003C00u, 0x64006400u);
          zp[i][1] = fma_f16x2(zp[i][1], 0xBC00BC00u, 0xD400D400u);
          zp[i][2] = fma_f16x2(zp[i][2], 0x3C003C00u, 0x64006400u);
          zp[i][3] = fma_f16x2(zp[i][3], 0xBC00BC00u, 0xD400D400u);
        } else {  // 128 + z
#pragma unroll
          for (int j = 0; j < 4; ++j) zp[i][j] = as_u32(__hadd2(tc::as_b2(zp[i][j]), __float2bfloat162_rn(128.f)));
        }
        pairs(in ? ldg_ordered(reinterpret_cast<const uint32_t*>(srow) + 4 * i) : make_uint4(0, 0, 0, 0), sp[i]);
      }
      float fac[2] = {1.f, 1.f};
      uint32_t sinv = 0;
      int es = 0;
      if (!BF16) {
        sinv = scale_of(sp, es);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sp[i][j] = mul_f16x2(sp[i][j], sinv);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pairs(in && g + 8 * h < M ? ldg_ordered(reinterpret_cast<const uint32_t*>(dy + (size_t)(g + 8 * h) * N + n) + 4 * i)
                                    : make_uint4(0, 0, 0, 0),
                a[h][i]);
        if (!BF16) {  // row and scales brought to [1, 2) at their largest, exactly; their product is the one rounding
          int ed;
          const uint32_t dinv = scale_of(a[h], ed);
          fac[h] = __uint_as_float((uint32_t)(127 + es + ed) << 23);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) a[h][i][j] = mul_f16x2(mul_f16x2(a[h][i][j], dinv), sp[i][j]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) a[h][i][j] = mul_bf16x2(a[h][i][j], sp[i][j]);
        }
      }
      if (sub == 0) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");  // this lane's own copies
#pragma unroll
      for (int b = 0; b < GT / 8; ++b) {
        float c[4] = {};
        const uint4 wb = *reinterpret_cast<const uint4*>(ring + slot * STAGE + (sub * (GT / 8) + b) * 512);
        const uint32_t ww[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t v[4];
          if (!BF16) {
            const uint32_t r16 = 0x2C002C00u, w8 = ww[i] >> 8;  // 1/16
            v[0] = sub_f16x2(and_or(ww[i], 0x000F000Fu, 0x64006400u), zp[i][0]);
            v[1] = fma_f16x2(and_or(ww[i], 0x00F000F0u, 0x64006400u), r16, zp[i][1]);
            v[2] = sub_f16x2(and_or(w8, 0x000F000Fu, 0x64006400u), zp[i][2]);
            v[3] = fma_f16x2(and_or(w8, 0x00F000F0u, 0x64006400u), r16, zp[i][3]);
          } else {
            v[0] = sub_bf16x2(and_or(ww[i], 0x000F000Fu, 0x43004300u), zp[i][0]);
            v[1] = sub_bf16x2(and_or(ww[i] >> 4, 0x000F000Fu, 0x43004300u), zp[i][1]);
            v[2] = sub_bf16x2(and_or(ww[i] >> 8, 0x000F000Fu, 0x43004300u), zp[i][2]);
            v[3] = sub_bf16x2(and_or(ww[i] >> 12, 0x000F000Fu, 0x43004300u), zp[i][3]);
          }
          mma<BF16>(c, a[0][i][0], a[1][i][0], a[0][i][1], a[1][i][1], v[0], v[1]);
          mma<BF16>(c, a[0][i][2], a[1][i][2], a[0][i][3], a[1][i][3], v[2], v[3]);
        }
        float* o = tot[sub * (GT / 8) + b];
        o[0] = fmaf(c[0], fac[0], o[0]);
        o[1] = fmaf(c[1], fac[0], o[1]);
        o[2] = fmaf(c[2], fac[1], o[2]);
        o[3] = fmaf(c[3], fac[1], o[3]);
      }
    }
    slot = slot + 1 == STAGES ? 0 : slot + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* red = reinterpret_cast<float*>(sm);  // [warp][16][RPITCH], then this CTA's sums
  // the warps' sums, then the cluster's
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    *reinterpret_cast<float2*>(red + (warp * 16 + g) * RPITCH + 8 * b + 2 * t) = make_float2(tot[b][0], tot[b][1]);
    *reinterpret_cast<float2*>(red + (warp * 16 + g + 8) * RPITCH + 8 * b + 2 * t) = make_float2(tot[b][2], tot[b][3]);
  }
  __syncthreads();
  float* part = red + WARPS * 16 * RPITCH;
  for (int i = tid; i < 16 * TILE; i += THREADS) {
    const int m = i / TILE, c = i % TILE;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < WARPS; ++q) v += red[(q * 16 + m) * RPITCH + c];
    part[m * RPITCH + c] = v;
  }
  if (S > 1)
    cluster_sync();
  else
    __syncthreads();
  // this rank's columns of the tile
  const int q0 = rank * TILE / S, q1 = (rank + 1) * TILE / S, nq = q1 - q0;
  for (int i = tid; i < M * nq; i += THREADS) {
    const int m = i / nq, c = q0 + i % nq;
    if (k0 + c >= K) continue;
    float v = 0.f;
    if (S > 1) {
      const uint32_t addr = smem_u32(part + m * RPITCH + c);
      for (int q = 0; q < S; ++q) {
        float u;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u) : "r"(map_shared_rank(addr, q)) : "memory");
        v += u;
      }
    } else {
      v = part[m * RPITCH + c];
    }
    uint16_t r;
    if (BF16) {
      const __nv_bfloat16 b = __float2bfloat16_rn(v);
      r = *reinterpret_cast<const uint16_t*>(&b);
    } else {
      const __half h = __float2half_rn(v);
      r = *reinterpret_cast<const uint16_t*>(&h);
    }
    dx[(size_t)m * K + k0 + c] = r;
  }
  if (S > 1) cluster_sync();  // the others have read this CTA's sums
}

}  // namespace dx16

int w4a16_dgrad_small(const void* dy, const int32_t* qweight, const void* scales, const void* zeros, void* dx, int64_t M,
                      int64_t N, int64_t K, int64_t group, int dtype, cudaStream_t stream) {
  using namespace dx16;
  const uintptr_t any = reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(qweight) |
                        reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(zeros);
  if (any & 15) return fail(B200Q_ERR_ALIGN, "w4a16 dgrad: pointers must be 16-byte aligned");
  const bool bf = dtype == B200Q_DTYPE_BF16;
  auto kern = group == 32 ? (bf ? dgrad_small_kernel<true, 32> : dgrad_small_kernel<false, 32>)
                          : (bf ? dgrad_small_kernel<true, 64> : dgrad_small_kernel<false, 64>);
  int rc = allow_smem((const void*)kern, SMEM, "cudaFuncSetAttribute(w4a16 dgrad small)");
  if (rc) return rc;
  // the split of the columns with the shortest estimate: rounds of co-resident
  // clusters x (a warp's steps + 2 for start and joining)
  const int64_t tiles = (K + TILE - 1) / TILE, chunks = (N + CHUNK - 1) / CHUNK;
  int S = 1;
  int64_t best = INT64_MAX;
  const int* fit = resident_clusters((const void*)kern, THREADS, SMEM);
  for (int s = 1; s <= MAX_S && (s == 1 || s * WARPS < chunks + WARPS); s *= 2) {
    const int64_t cost = ((tiles + fit[s] - 1) / fit[s]) * ((chunks + s * WARPS - 1) / (s * WARPS) + 2);
    if (cost < best) best = cost, S = s;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * S));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, reinterpret_cast<const uint16_t*>(dy),
                                       reinterpret_cast<const uint32_t*>(qweight),
                                       reinterpret_cast<const uint16_t*>(scales),
                                       reinterpret_cast<const uint16_t*>(zeros), reinterpret_cast<uint16_t*>(dx), (int)M,
                                       (int)N, (int)K, (int)group, S),
                    "w4a16 dgrad small launch");
}

}  // namespace b200q
