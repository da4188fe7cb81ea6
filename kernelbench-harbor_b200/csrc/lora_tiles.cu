// Many tokens (prefill, training): shrink and expand as two launches over tiles
// of up to 128 rows of one adapter.
//
// shrink: 8 warps of 16 rows; rows go from HBM straight into the multiply's
// fragments (two 64-wide stages ahead, in registers), P comes through a
// 4-stage ring in shared memory that all warps read.  The contraction of a tile
// is split over a cluster of S CTAs, so that short batches fill the GPU; the
// partial sums meet through distributed shared memory in rank order.
// expand: a CTA takes a tile's 128 output columns: mid split into two halves of
// the type in registers, Q staged once, base requested before anything else.
// Bound: HBM -- x once, base once, y once; mid (4 r bytes a token) stays in L2.
#include <type_traits>

#include "lora_seg.cuh"

namespace b200q {
namespace lora {

constexpr int SK = 64;   // contraction depth of a stage
constexpr int SSTG = 4;  // stages of P in shared memory
constexpr int MAX_SPLIT = 8;
constexpr int NC = 128;  // output columns of an expand CTA

template <int RP, bool TR>
struct ShrinkCfg {
  static constexpr int PITCH = RP * 2 + 16;                              // !TR: bytes per contraction row
  static constexpr int STAGE = TR ? RP * SK * 2 : SK * PITCH;            // TR: rank rows of 64 values
  static constexpr int PART = ROWS_L * (RP + 4) * 4;                     // partial sums, over the ring
  static constexpr int SMEM = SSTG * STAGE > PART ? SSTG * STAGE : PART;
};

template <class T, int RP, bool TR, bool VEC>
__global__ void __launch_bounds__(THREADS, VEC ? 2 : 1) lora_shrink_tile_kernel(const Args a, int S) {
  using C = ShrinkCfg<RP, TR>;
  extern __shared__ __align__(16) uint8_t sm[];
  const int tile = blockIdx.x / S, rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int32_t* plan = a.plan;
  if (tile >= plan[1]) return;
  const int4 tl = reinterpret_cast<const int4*>(plan + a.lay.large)[tile];
  if (tl.x < 0) return;  // a whole cluster at a time
  const int32_t* rows = plan + a.lay.order + tl.y;
  const int count = tl.z, D = a.D, r = a.r;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int m = warp * 16 + g;
  const int64_t ra = m < count ? rows[m] : -1, rb = m + 8 < count ? rows[m + 8] : -1;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* P = reinterpret_cast<const T*>(a.P) + (size_t)tl.x * D * r;
  const int nst = (D + SK - 1) / SK;
  const int s0 = (int)((int64_t)rank * nst / S), s1 = (int)((int64_t)(rank + 1) * nst / S);

  auto stage_p = [&](int st) {
    uint8_t* buf = sm + (st - s0) % SSTG * C::STAGE;
    constexpr int PIECES = SK * RP / 8;
#pragma unroll
    for (int i = 0; i < (PIECES + THREADS - 1) / THREADS; ++i) {
      const int idx = tid + i * THREADS;
      if (PIECES % THREADS && idx >= PIECES) break;
      if (!TR) {
        const int k = idx / (RP / 8), pc = idx % (RP / 8), kk = st * SK + k;
        stage8<T, VEC>(buf + row32(k) * C::PITCH + pc * 16, P + (size_t)kk * r, pc * 8, r, kk < D, P);
      } else {
        const int n = idx / (SK / 8), pc = idx % (SK / 8);  // odd rows have their 64-byte halves swapped: no bank conflicts
        stage8<T, VEC>(buf + n * (SK * 2) + ((pc ^ ((n & 1) << 2)) << 4), P + (size_t)n * D, st * SK + pc * 8, D, n < r, P);
      }
    }
  };
  auto load_x = [&](int st, uint4* v) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = st * SK + 32 * h + 8 * t;
      v[2 * h] = ra >= 0 ? ld8<T, VEC>(x + ra * D, k, D) : make_uint4(0, 0, 0, 0);
      v[2 * h + 1] = rb >= 0 ? ld8<T, VEC>(x + rb * D, k, D) : make_uint4(0, 0, 0, 0);
    }
  };
  float acc[RP / 8][4] = {};
  auto multiply = [&](int st, const uint4* v) {
    const uint8_t* buf = sm + (st - s0) % SSTG * C::STAGE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 xa = v[2 * h], xb = v[2 * h + 1];
      const uint32_t row = smem_u32(buf + (32 * h + lane) * C::PITCH);
#pragma unroll
      for (int j = 0; j < RP / 8; ++j) {
        uint32_t b[4];
        if (!TR) {
          ldmatrix_x4_trans(b, row + j * 16);
        } else {
          const int n = 8 * j + g;
          const uint4 w = *reinterpret_cast<const uint4*>(buf + n * (SK * 2) + (((4 * h + t) ^ ((n & 1) << 2)) << 4));
          b[0] = w.x, b[1] = w.y, b[2] = w.z, b[3] = w.w;
        }
        mma16816<T>(acc[j], xa.x, xb.x, xa.y, xb.y, b[0], b[1]);
        mma16816<T>(acc[j], xa.z, xb.z, xa.w, xb.w, b[2], b[3]);
      }
    }
  };
  uint4 xr[3][4] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (s0 + i < s1) load_x(s0 + i, xr[i]);
#pragma unroll
  for (int i = 0; i < SSTG - 1; ++i) {
    if (s0 + i < s1) stage_p(s0 + i);
    cp_async_commit();
  }
  for (int st = s0; st < s1; st += 3) {
#pragma unroll
    for (int u = 0; u < 3; ++u) {
      const int c = st + u;
      if (c < s1) {
        if (c + 2 < s1) load_x(c + 2, xr[(u + 2) % 3]);
        cp_async_wait<SSTG - 2>();
        __syncthreads();  // stage c has landed for every thread; the slot filled next was read before
        if (c + SSTG - 1 < s1) stage_p(c + SSTG - 1);
        cp_async_commit();
        multiply(c, xr[u]);
      }
    }
  }
  const float scale = a.scaling ? a.scaling[tl.x] : 1.f;
  if (S == 1) {
#pragma unroll
    for (int j = 0; j < RP / 8; ++j) {
      const int col = 8 * j + 2 * t;
      if (!VEC && col >= a.mp) break;
      const bool in0 = col < r, in1 = col + 1 < r;  // past the rank: an exact 0, whatever x holds
      if (ra >= 0)
        *reinterpret_cast<float2*>(a.mid + ra * a.mp + col) =
            make_float2(in0 ? acc[j][0] * scale : 0.f, in1 ? acc[j][1] * scale : 0.f);
      if (rb >= 0)
        *reinterpret_cast<float2*>(a.mid + rb * a.mp + col) =
            make_float2(in0 ? acc[j][2] * scale : 0.f, in1 ? acc[j][3] * scale : 0.f);
    }
    return;
  }
  cp_async_wait<0>();
  __syncthreads();
  float* part = reinterpret_cast<float*>(sm);
  constexpr int PP = RP + 4;
#pragma unroll
  for (int j = 0; j < RP / 8; ++j) {
    *reinterpret_cast<float2*>(part + m * PP + 8 * j + 2 * t) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(part + (m + 8) * PP + 8 * j + 2 * t) = make_float2(acc[j][2], acc[j][3]);
  }
  cluster_sync();
  const int q0 = rank * ROWS_L / S, q1 = min((rank + 1) * ROWS_L / S, count);
  for (int i = tid; i < (q1 - q0) * (RP / 4); i += THREADS) {
    const int row = q0 + i / (RP / 4), col = i % (RP / 4) * 4;
    const uint32_t addr = smem_u32(part + row * PP + col);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < S; ++c) {
      float4 u;
      asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                   : "=f"(u.x), "=f"(u.y), "=f"(u.z), "=f"(u.w)
                   : "r"(map_shared_rank(addr, c))
                   : "memory");
      s.x += u.x, s.y += u.y, s.z += u.z, s.w += u.w;
    }
    if (VEC || col < a.mp)
      *reinterpret_cast<float4*>(a.mid + (size_t)rows[row] * a.mp + col) =
          make_float4(col < r ? s.x * scale : 0.f, col + 1 < r ? s.y * scale : 0.f, col + 2 < r ? s.z * scale : 0.f,
                      col + 3 < r ? s.w * scale : 0.f);
  }
  cluster_sync();  // the others have read this CTA's part
}

template <int RP, bool TR>
struct ExpandCfg {
  static constexpr int QWORDS = NC / 2 + 4;                                   // !TR: words per rank row
  static constexpr int APITCH = RP == 16 ? 32 : RP == 32 ? 96 : 160;          // TR: bytes per column row, 8 words mod 32 (no conflicts)
  static constexpr int SMEM = TR ? NC * APITCH : RP * QWORDS * 4;
};

template <class T, int RP, bool TR, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) lora_expand_tile_kernel(const Args a) {
  using C = ExpandCfg<RP, TR>;
  extern __shared__ __align__(16) uint8_t sm[];
  const int32_t* plan = a.plan;
  const int nb = (a.N + NC - 1) / NC, tile = blockIdx.x / nb;  // a tile's column blocks run side by side
  if (tile >= plan[1]) return;
  const int4 tl = reinterpret_cast<const int4*>(plan + a.lay.large)[tile];
  const int32_t* rows = plan + a.lay.order + tl.y;
  const int count = tl.z, N = a.N, r = a.r, n0 = blockIdx.x % nb * NC;
  const T* base = reinterpret_cast<const T*>(a.base);
  T* y = reinterpret_cast<T*>(a.y);
  if (tl.x < 0) {
    copy_rows<T, VEC>(base, y, rows, count, N, n0, min(n0 + NC, N));
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int m = warp * 16 + g;
  const int64_t ra = m < count ? rows[m] : -1, rb = m + 8 < count ? rows[m + 8] : -1;
  uint4 bv[NC / 32][2];
#pragma unroll
  for (int q = 0; q < NC / 32; ++q) {
    const int n = n0 + q * 32 + 8 * t;
    bv[q][0] = base && ra >= 0 ? ld8<T, VEC>(base + ra * N, n, N) : make_uint4(0, 0, 0, 0);
    bv[q][1] = base && rb >= 0 ? ld8<T, VEC>(base + rb * N, n, N) : make_uint4(0, 0, 0, 0);
  }
  const T* Q = reinterpret_cast<const T*>(a.Q) + (size_t)tl.x * r * N;
  if (!TR) {
    uint32_t* qb = reinterpret_cast<uint32_t*>(sm);
#pragma unroll
    for (int i = 0; i < RP * (NC / 8) / THREADS; ++i) {
      // 8 rank rows in fragment order x 4 lanes of 8 columns, warps over the column groups
      const int idx = i * WARPS + warp, q = idx % (NC / 32), row = idx / (NC / 32) * 8 + g, k = k_of_row16(row);
      const uint4 v = k < r ? ld8<T, VEC>(Q + (size_t)k * N, n0 + q * 32 + 8 * t, N) : make_uint4(0, 0, 0, 0);
      uint32_t* dst = qb + row * C::QWORDS + q * 16 + t;
      dst[0] = v.x;
      dst[4] = v.y;
      dst[8] = v.z;
      dst[12] = v.w;
    }
  } else {
    constexpr int PIECES = NC * RP / 8;
#pragma unroll
    for (int i = 0; i < PIECES / THREADS; ++i) {
      const int idx = tid + i * THREADS, c = idx / (RP / 8), pc = idx % (RP / 8), col = n0 + c;
      // column 32 q + 8 a + 2 p + b is row 32 q + 8 p + 2 a + b: a fragment's columns together
      const int row = (c & ~31) | (((c >> 1) & 3) << 3) | (((c >> 3) & 3) << 1) | (c & 1);
      stage8<T, VEC>(sm + row * C::APITCH + pc * 16, Q + (size_t)col * r, pc * 8, r, col < N, Q);
    }
    cp_async_commit();
  }
  // mid: rows m, m + 8; values 4t .. 4t + 3 of each 16 ranks, split into hi + lo
  float fac[2];
  uint2 ha[RP / 16][2], la[RP / 16][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t row = h ? rb : ra;
    float4 v[RP / 16];
    float mx = 0.f;
#pragma unroll
    for (int k = 0; k < RP / 16; ++k) {
      v[k] = row >= 0 && (VEC || 16 * k + 4 * t < a.mp)
                 ? *reinterpret_cast<const float4*>(a.mid + row * a.mp + 16 * k + 4 * t)
                 : make_float4(0.f, 0.f, 0.f, 0.f);
      const float f[4] = {fabsf(v[k].x), fabsf(v[k].y), fabsf(v[k].z), fabsf(v[k].w)};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (f[e] < INFINITY) mx = fmaxf(mx, f[e]);
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    float inv;
    pow2_of(mx, fac[h], inv);
#pragma unroll
    for (int k = 0; k < RP / 16; ++k) {
      T hi[4], lo[4];
      split(v[k].x * inv, hi[0], lo[0]);
      split(v[k].y * inv, hi[1], lo[1]);
      split(v[k].z * inv, hi[2], lo[2]);
      split(v[k].w * inv, hi[3], lo[3]);
      ha[k][h] = make_uint2(pack2(hi[0], hi[1]), pack2(hi[2], hi[3]));
      la[k][h] = make_uint2(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]));
    }
  }
  if (TR) cp_async_wait<0>();
  __syncthreads();
#pragma unroll
  for (int q = 0; q < NC / 32; ++q) {
    float c[4][4] = {};
#pragma unroll
    for (int k = 0; k < RP / 16; ++k) {
      uint32_t b[8];
      if (!TR) {
        const uint32_t addr = smem_u32(reinterpret_cast<uint32_t*>(sm) +
                                       (16 * k + 8 * ((lane >> 3) & 1) + (lane & 7)) * C::QWORDS + q * 16 + (lane >> 4) * 4);
        ldmatrix_x4_trans(b, addr);
        ldmatrix_x4_trans(b + 4, addr + 32);
      } else {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const uint2 w = *reinterpret_cast<const uint2*>(sm + (32 * q + 8 * p + g) * C::APITCH + (16 * k + 4 * t) * 2);
          b[2 * p] = w.x;
          b[2 * p + 1] = w.y;
        }
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        mma16816<T>(c[p], ha[k][0].x, ha[k][1].x, ha[k][0].y, ha[k][1].y, b[2 * p], b[2 * p + 1]);
        mma16816<T>(c[p], la[k][0].x, la[k][1].x, la[k][0].y, la[k][1].y, b[2 * p], b[2 * p + 1]);
      }
    }
    const int n = n0 + q * 32 + 8 * t;
    if (ra >= 0) st8<T, VEC>(y + ra * N, n, N, add8<T>(bv[q][0], c, 0, fac[0]));
    if (rb >= 0) st8<T, VEC>(y + rb * N, n, N, add8<T>(bv[q][1], c, 2, fac[1]));
  }
}

int launch_tiles(const Args& a, int dtype, bool tr, cudaStream_t st) {
  const bool vec = a.D % 8 == 0 && a.N % 8 == 0 && a.r % 8 == 0;
  return by_type(dtype, a.r, vec, [&](auto tc, auto rc, auto vc) -> int {
    using T = decltype(tc);
    constexpr int RP = decltype(rc)::value;
    constexpr bool VEC = decltype(vc)::value;
    auto shrink = tr ? lora_shrink_tile_kernel<T, RP, true, VEC> : lora_shrink_tile_kernel<T, RP, false, VEC>;
    auto expand = tr ? lora_expand_tile_kernel<T, RP, true, VEC> : lora_expand_tile_kernel<T, RP, false, VEC>;
    const int smem_s = tr ? ShrinkCfg<RP, true>::SMEM : ShrinkCfg<RP, false>::SMEM;
    const int smem_e = tr ? ExpandCfg<RP, true>::SMEM : ExpandCfg<RP, false>::SMEM;
    const int64_t blocks = a.lay.max_large * ((a.N + NC - 1) / NC);
    if (blocks > (1ll << 31) - 1) return fail(B200Q_ERR_SHAPE, "lora_apply: size too large");
    cudaError_t e = cudaFuncSetAttribute(shrink, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_s);
    if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(lora shrink)");
    // the contraction is split until the tiles' clusters fill the SMs twice
    // over, as long as a part keeps two stages
    const int64_t tiles = (a.T + ROWS_L - 1) / ROWS_L, nst = (a.D + SK - 1) / SK;
    int S = 1;
    while (S < MAX_SPLIT && tiles * S < 2 * num_sms(-1) && nst >= 4 * S) S *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.lay.max_large * S));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem_s;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)S;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, shrink, a, S);
    if (e != cudaSuccess) return check_cuda(e, "lora shrink launch");
    if (!a.y) return B200Q_OK;  // mid alone was asked for
    expand<<<(unsigned)blocks, THREADS, smem_e, st>>>(a);
    return check_cuda(cudaGetLastError(), "lora expand launch");
  });
}

}  // namespace lora
}  // namespace b200q
