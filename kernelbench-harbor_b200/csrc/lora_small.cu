// Few tokens (decode): shrink and expand in one launch.
//
// A cluster of CL CTAs takes one tile of up to 16 rows of one adapter.  Each
// CTA contracts 1/CL of the row's width with its part of P (its 8 warps take
// 32-wide chunks in turn), the 16 x r partial sums meet in every CTA through
// distributed shared memory, added in rank order, and each CTA expands 1/CL of
// the output columns.  The row between, mid, is written once for a backward
// pass.  Bound: latency -- 0.3 to 4 MB of adapters and rows at decode, against
// one launch, two dependent rounds of loads and one cluster barrier; the first
// group's Q, and base, are requested before the shrink starts.  Measured: 4.9 us
// for one token, 5.5 us for 64 tokens of 8 adapters, at 4096 x 4096, r = 16.
#include <type_traits>

#include "lora_seg.cuh"

namespace b200q {
namespace lora {

constexpr int CL = 8;       // CTAs per tile (the portable cluster size)
constexpr int STAGES = 3;   // chunks of P a warp keeps in shared memory
constexpr int QROW = 20;    // words per rank row of a warp's 32-column group of Q: 16 + 4 against bank conflicts

template <int RP>
struct SmallCfg {
  static constexpr int PITCH = RP * 2 + 16;          // bytes per contraction row of a staged chunk of P
  static constexpr int RING = WARPS * STAGES * 32 * PITCH;
  static constexpr int RED = WARPS * ROWS_S * RP * 4;  // per-warp partial sums, over the ring
  static constexpr int QBUF = WARPS * RP * QROW * 4;
  static constexpr int OFF_Q = RING > RED ? RING : RED;
  static constexpr int OFF_PART = OFF_Q + QBUF;
  static constexpr int HPITCH = RP + 8;  // elements per row of the split mid
  static constexpr int OFF_HI = OFF_PART + ROWS_S * RP * 4;
  static constexpr int OFF_LO = OFF_HI + ROWS_S * HPITCH * 2;
  static constexpr int OFF_FAC = OFF_LO + ROWS_S * HPITCH * 2;
  static constexpr int SMEM = OFF_FAC + ROWS_S * 4;
};

template <class T, int RP, bool TR, bool VEC>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(THREADS) lora_small_kernel(const Args a) {
  using C = SmallCfg<RP>;
  extern __shared__ __align__(16) uint8_t sm[];
  const int32_t* plan = a.plan;
  const int tile = blockIdx.x / CL, rank = (int)cluster_ctarank();
  if (tile >= plan[0]) return;  // a whole cluster at a time
  const int4 tl = reinterpret_cast<const int4*>(plan + a.lay.small)[tile];
  const int32_t* rows = plan + a.lay.order + tl.y;
  const int count = tl.z, D = a.D, N = a.N, r = a.r;
  const T* base = reinterpret_cast<const T*>(a.base);
  T* y = reinterpret_cast<T*>(a.y);
  const int ng = (N + 31) / 32;  // 32-column groups; this CTA's are [g0, g1)
  const int g0 = rank * ng / CL, g1 = (rank + 1) * ng / CL;
  if (tl.x < 0) {
    if (y) copy_rows<T, VEC>(base, y, rows, count, N, g0 * 32, min(g1 * 32, N), base + a.T * N);
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int64_t ra = g < count ? rows[g] : -1, rb = g + 8 < count ? rows[g + 8] : -1;
  const T* P = reinterpret_cast<const T*>(a.P) + (size_t)tl.x * D * r;
  const T* Q = reinterpret_cast<const T*>(a.Q) + (size_t)tl.x * r * N;
  const T* const p_end = reinterpret_cast<const T*>(a.P) + a.L * D * r;
  const T* const q_end = reinterpret_cast<const T*>(a.Q) + a.L * N * r;

  // ---------------------------------------------------------------- first expand group: loads in flight early
  uint4 bv[2], qv[TR ? 1 : RP / 8];
  uint2 qt[TR ? RP / 16 : 1][4];
  auto load_group = [&](int q) {
    const int n = q * 32 + 8 * t;
    bv[0] = base && ra >= 0 ? ld8<T, VEC, false>(base + ra * N, n, N, base + a.T * N) : make_uint4(0, 0, 0, 0);
    bv[1] = base && rb >= 0 ? ld8<T, VEC, false>(base + rb * N, n, N, base + a.T * N) : make_uint4(0, 0, 0, 0);
    if constexpr (!TR) {
#pragma unroll
      for (int i = 0; i < RP / 8; ++i) {  // rank rows in fragment order, 4 lanes per row
        const int k = k_of_row16(i * 8 + g);
        qv[i] = k < r ? ld8<T, VEC>(Q + (size_t)k * N, n, N, q_end) : make_uint4(0, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int col = q * 32 + 8 * (g >> 1) + 2 * p + (g & 1);
#pragma unroll
        for (int s = 0; s < RP / 16; ++s)
          qt[s][p] = col < N ? ld4<T, VEC>(Q + (size_t)col * r, 16 * s + 4 * t, r) : make_uint2(0, 0);
      }
    }
  };
  if (y && g0 + warp < g1) load_group(g0 + warp);

  // ---------------------------------------------------------------- shrink: this CTA's chunks of 32
  float acc[RP / 8][4] = {};
  const int nch = (D + 31) / 32;
  const int c1 = (rank + 1) * nch / CL;
  const T* x = reinterpret_cast<const T*>(a.x);
  uint8_t* ring = sm + warp * STAGES * 32 * C::PITCH;
  uint4 xv[2], pv[TR ? RP / 8 : 1];
  auto load_x = [&](int c) {
    const int k = 32 * c + 8 * t;
    xv[0] = ra >= 0 ? ld8<T, VEC>(x + ra * D, k, D, x + a.T * D) : make_uint4(0, 0, 0, 0);
    xv[1] = rb >= 0 ? ld8<T, VEC>(x + rb * D, k, D, x + a.T * D) : make_uint4(0, 0, 0, 0);
    if (TR) {
#pragma unroll
      for (int j = 0; j < RP / 8; ++j)
        pv[j] = 8 * j + g < r ? ld8<T, VEC>(P + (size_t)(8 * j + g) * D, k, D, p_end) : make_uint4(0, 0, 0, 0);
    }
  };
  // 32 contraction rows of P: to the ring by asynchronous copies (VEC), else to registers and from there
  uint4 pq[TR || VEC ? 1 : RP / 8];
  auto stage_p = [&](int c, int s) {
    if constexpr (!TR) {
#pragma unroll
      for (int i = 0; i < RP / 8; ++i) {
        const int idx = lane + 32 * i, k = idx / (RP / 8), pc = idx % (RP / 8), kk = 32 * c + k;
        const T* piece = P + (size_t)kk * r + pc * 8;
        if constexpr (VEC)
          copy16<false, 0>(smem_u32(ring + s * 32 * C::PITCH + row32(k) * C::PITCH + pc * 16), piece, r - pc * 8, kk < D, P,
                           r % 8 != 0);
        else
          pq[i] = kk < D ? ld8_any<T>(piece, r - pc * 8, p_end) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  auto put_p = [&](int s) {
    if constexpr (!TR && !VEC) {
#pragma unroll
      for (int i = 0; i < RP / 8; ++i) {
        const int idx = lane + 32 * i, k = idx / (RP / 8), pc = idx % (RP / 8);
        sts16(smem_u32(ring + s * 32 * C::PITCH + row32(k) * C::PITCH + pc * 16), pq[i]);
      }
    }
  };
  const int c0 = rank * nch / CL + warp;
  constexpr int AHEAD = VEC ? STAGES - 1 : 1;  // chunks of P requested before they are used
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) {
    if (c0 + s * WARPS < c1) stage_p(c0 + s * WARPS, s);
    cp_async_commit();
  }
  if (c0 < c1) load_x(c0);
  int s = 0;
  for (int c = c0; c < c1; c += WARPS) {
    const uint4 xa = xv[0], xb = xv[1];
    uint4 pc_[TR ? RP / 8 : 1];
    if (TR) {
#pragma unroll
      for (int j = 0; j < RP / 8; ++j) pc_[j] = pv[j];
    }
    if (!TR) {
      if (VEC)
        cp_async_wait<STAGES - 2>();
      else
        put_p(s);
      __syncwarp();
    }
    if (c + WARPS < c1) {
      load_x(c + WARPS);
      if (!VEC) stage_p(c + WARPS, 0);
    }
    const uint32_t row = smem_u32(ring + s * 32 * C::PITCH + lane * C::PITCH);
#pragma unroll
    for (int j = 0; j < RP / 8; ++j) {
      uint32_t b[4];
      if (TR) {
        b[0] = pc_[j].x, b[1] = pc_[j].y, b[2] = pc_[j].z, b[3] = pc_[j].w;
      } else {
        ldmatrix_x4_trans(b, row + j * 16);
      }
      mma16816<T>(acc[j], xa.x, xb.x, xa.y, xb.y, b[0], b[1]);
      mma16816<T>(acc[j], xa.z, xb.z, xa.w, xb.w, b[2], b[3]);
    }
    if (!TR) {
      __syncwarp();  // every lane has read the slot that is filled next
      if (VEC) {
        const int cn = c + (STAGES - 1) * WARPS;
        if (cn < c1) stage_p(cn, s == 0 ? STAGES - 1 : s - 1);
        cp_async_commit();
      }
      s = s + 1 == STAGES ? 0 : s + 1;
    }
  }

  // ---------------------------------------------------------------- sums over the warps, then over the cluster
  cp_async_wait<0>();
  __syncthreads();
  float* red = reinterpret_cast<float*>(sm);
#pragma unroll
  for (int j = 0; j < RP / 8; ++j) {
    *reinterpret_cast<float2*>(red + (warp * ROWS_S + g) * RP + 8 * j + 2 * t) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(red + (warp * ROWS_S + g + 8) * RP + 8 * j + 2 * t) = make_float2(acc[j][2], acc[j][3]);
  }
  __syncthreads();
  constexpr int EPT = RP / 16;  // values per thread: 16 threads per row
  const int mrow = tid >> 4, mcol = (tid & 15) * EPT;
  float v[EPT];
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    v[e] = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v[e] += red[(w * ROWS_S + mrow) * RP + mcol + e];
  }
  float* part = reinterpret_cast<float*>(sm + C::OFF_PART);
#pragma unroll
  for (int e = 0; e < EPT; ++e) part[mrow * RP + mcol + e] = v[e];
  cluster_sync();
  const float scale = a.scaling ? a.scaling[tl.x] : 1.f;
  float mx = 0.f;
  const uint32_t paddr = smem_u32(part + mrow * RP + mcol);
#pragma unroll
  for (int e = 0; e < EPT; ++e) v[e] = 0.f;
#pragma unroll
  for (int c = 0; c < CL; ++c) {
    const uint32_t from = map_shared_rank(paddr, c);
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      float u;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u) : "r"(from + 4 * e) : "memory");
      v[e] += u;
    }
  }
  // the others may read this CTA's part until they arrive, too
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    v[e] = mcol + e < r ? v[e] * scale : 0.f;  // past the rank: an exact 0, whatever x holds
    if (fabsf(v[e]) < INFINITY) mx = fmaxf(mx, fabsf(v[e]));
  }
  if (a.mid && rank == 0 && mrow < count) {
    float* mid = a.mid + (size_t)rows[mrow] * a.mp;
#pragma unroll
    for (int e = 0; e < EPT; ++e) mid[mcol + e] = v[e];
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float fac, inv;
  scale_of<T>(mx, fac, inv);
  T* hi = reinterpret_cast<T*>(sm + C::OFF_HI);
  T* lo = reinterpret_cast<T*>(sm + C::OFF_LO);
  float* facs = reinterpret_cast<float*>(sm + C::OFF_FAC);
#pragma unroll
  for (int e = 0; e < EPT; ++e) split(v[e] * inv, hi[mrow * C::HPITCH + mcol + e], lo[mrow * C::HPITCH + mcol + e]);
  if ((tid & 15) == 0) facs[mrow] = fac;
  __syncthreads();
  if (!y) {  // mid alone was asked for
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    return;
  }

  // ---------------------------------------------------------------- expand: this CTA's columns
  uint2 ha[RP / 16][2], la[RP / 16][2];  // rows g, g + 8; values 4t .. 4t + 3 of each 16 ranks
#pragma unroll
  for (int k = 0; k < RP / 16; ++k) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      ha[k][h] = *reinterpret_cast<const uint2*>(hi + (g + 8 * h) * C::HPITCH + 16 * k + 4 * t);
      la[k][h] = *reinterpret_cast<const uint2*>(lo + (g + 8 * h) * C::HPITCH + 16 * k + 4 * t);
    }
  }
  const float fa = facs[g], fb = facs[g + 8];
  uint32_t* qb = reinterpret_cast<uint32_t*>(sm + C::OFF_Q) + warp * RP * QROW;
  for (int q = g0 + warp; q < g1; q += WARPS) {
    float c[4][4] = {};
    const uint4 b0 = bv[0], b1 = bv[1];
    if (!TR) {
      // words to the column order of the output fragment: word p of lane t's 8 columns to tile p, place t
#pragma unroll
      for (int i = 0; i < RP / 8; ++i) {
        uint32_t* row = qb + (i * 8 + g) * QROW + t;
        row[0] = qv[i].x;
        row[4] = qv[i].y;
        row[8] = qv[i].z;
        row[12] = qv[i].w;
      }
      __syncwarp();
      if (q + WARPS < g1) load_group(q + WARPS);
      const uint32_t addr = smem_u32(qb + (8 * ((lane >> 3) & 1) + (lane & 7)) * QROW + (lane >> 4) * 4);
#pragma unroll
      for (int k = 0; k < RP / 16; ++k) {
#pragma unroll
        for (int p = 0; p < 4; p += 2) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, addr + (k * 16 * QROW + p * 4) * 4);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            mma16816<T>(c[p + i], ha[k][0].x, ha[k][1].x, ha[k][0].y, ha[k][1].y, b[2 * i], b[2 * i + 1]);
            mma16816<T>(c[p + i], la[k][0].x, la[k][1].x, la[k][0].y, la[k][1].y, b[2 * i], b[2 * i + 1]);
          }
        }
      }
      __syncwarp();  // the buffer is rewritten by the next group
    } else {
      uint2 qc[RP / 16][4];
#pragma unroll
      for (int k = 0; k < RP / 16; ++k)
#pragma unroll
        for (int p = 0; p < 4; ++p) qc[k][p] = qt[k][p];
      if (q + WARPS < g1) load_group(q + WARPS);
#pragma unroll
      for (int k = 0; k < RP / 16; ++k)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          mma16816<T>(c[p], ha[k][0].x, ha[k][1].x, ha[k][0].y, ha[k][1].y, qc[k][p].x, qc[k][p].y);
          mma16816<T>(c[p], la[k][0].x, la[k][1].x, la[k][0].y, la[k][1].y, qc[k][p].x, qc[k][p].y);
        }
    }
    const int n = q * 32 + 8 * t;
    if (ra >= 0) st8<T, VEC>(y + ra * N + n, N - n, add8<T>(b0, c, 0, fa));
    if (rb >= 0) st8<T, VEC>(y + rb * N + n, N - n, add8<T>(b1, c, 2, fb));
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

int launch_small(const Args& a, int dtype, bool tr, cudaStream_t st) {
  const bool vec = aligned_widths(a.D, a.N, a.r);
  return by_type(dtype, a.r, vec, [&](auto tc, auto rc, auto vc) -> int {
    using T = decltype(tc);
    constexpr int RP = decltype(rc)::value;
    constexpr bool VEC = decltype(vc)::value;
    auto kern = tr ? lora_small_kernel<T, RP, true, VEC> : lora_small_kernel<T, RP, false, VEC>;
    constexpr int smem = SmallCfg<RP>::SMEM;
    const int rc2 = allow_smem((const void*)kern, smem, "cudaFuncSetAttribute(lora small)");
    if (rc2) return rc2;
    kern<<<(unsigned)(a.lay.max_small * CL), THREADS, smem, st>>>(a);
    return check_cuda(cudaGetLastError(), "lora_apply launch");
  });
}

}  // namespace lora
}  // namespace b200q
