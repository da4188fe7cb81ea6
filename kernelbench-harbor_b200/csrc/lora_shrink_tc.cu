// Many tokens, aligned rows, ranks 33 to 64: the shrink product
//   mid[rows, r] = s X[rows, K] . P[K, r]
// with its accumulator (a 128-row tile of one adapter, fp32) in tensor memory.
//
// 8 warps only copy: 16-byte asynchronous copies of the tile's (gathered) rows
// and of P's stage into 64-column ring slots, in the 128-byte-swizzled layouts
// that the multiply reads: X K-major; P as stored, MN-major forward (rank
// contiguous), K-major backward.  A ninth warp issues, from one thread, 4
// tcgen05.mma (M128 K16) per stage.  The contraction of a tile is split
// over a cluster of S CTAs, whose sums meet through distributed shared memory
// in rank order.
// Bound: HBM, the rows once, and L2, P once per tile (half as much again): 29 us
// for 117 MB of rows at D=14336, r=64, 4096 tokens (18 us at the measured copy
// rate).  The form with register fragments (lora_tiles.cu) takes 45 us there: at
// rank 64 most of its instructions load fragments.  At ranks up to 32 it is as
// fast, without tensor memory.
#include "lora_seg.cuh"

namespace b200q {
namespace lora {

constexpr int TC_STG = 4, TC_LAG = 2;  // ring slots; stages between a copy's request and its hand-over
constexpr int TC_X = 128 * 128, TC_P = 64 * 128, TC_STAGE = TC_X + TC_P;
constexpr int RP = 64;  // rank, and tensor-memory columns
static_assert(SHRINK_TC_SMEM == TC_STG * TC_STAGE + 1024, "lora_seg.cuh has the launch's size");

template <class T, bool TR>
__global__ void __launch_bounds__(SHRINK_TC_THREADS, 2) lora_shrink_tc_kernel(const Args a, int S) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[TC_STG], empty[TC_STG], done;
  __shared__ uint32_t s_tmem;
  __shared__ int s_err;
  const int tile = blockIdx.x / S, rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int32_t* plan = a.plan;
  if (tile >= plan[1]) return;
  const int4 tl = reinterpret_cast<const int4*>(plan + a.lay.large)[tile];
  if (tl.x < 0) return;  // a whole cluster at a time
  uint8_t* sm = align_smem_1024(raw);
  const uint32_t smem = smem_u32(sm);
  const int32_t* rows = plan + a.lay.order + tl.y;
  const int count = tl.z, D = a.D, r = a.r;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nst = (D + 63) / 64;
  const int s0 = (int)((int64_t)rank * nst / S), n = (int)((int64_t)(rank + 1) * nst / S) - s0;
  if (tid == 0) {
    for (int s = 0; s < TC_STG; ++s) {
      mbar_init(&full[s], THREADS);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    fence_barrier_init();
    s_err = 0;
  }
  if (warp == WARPS) tmem_alloc(&s_tmem, RP);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  if (warp < WARPS) {
    // ---------------------------------------------------------------- copies
    const T* x = reinterpret_cast<const T*>(a.x);
    const T* P = reinterpret_cast<const T*>(a.P) + (size_t)tl.x * D * r;
    const int pc = tid & 7, prow = tid >> 3;
    const T* src[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      src[i] = x + (size_t)rows[prow + 32 * i < count ? prow + 32 * i : 0] * D + s0 * 64 + pc * 8;
    constexpr int NP = 2, PSTEP = 32;  // pieces of P per thread, rows between them
    const int q = tid & 7, prk = tid >> 3;
    const T* psrc[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i)
      psrc[i] = TR ? P + (size_t)(prk + i * PSTEP) * D + s0 * 64 + q * 8 : P + (size_t)(s0 * 64 + prk + i * PSTEP) * r + q * 8;
    const bool halves = r % 8 != 0;  // A's rows are 8-byte aligned only
    const uint32_t wdst = smem + prow * 128 + ((pc ^ (prow & 7)) << 4);
    const uint32_t pdst = smem + TC_X + prk * 128 + ((q ^ (prk & 7)) << 4);
    int kst = s0 * 64, slot = 0;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      if (i >= TC_STG && !mbar_wait(&empty[slot], ((i / TC_STG) - 1) & 1, a.status)) {
        ok = false;
        break;
      }
      const uint32_t w = wdst + slot * TC_STAGE, p = pdst + slot * TC_STAGE;
      if (kst + 64 <= D && (TR || !halves)) {  // a whole stage: no column to check
        static_for<4>([&](auto j) { cp_async16_ahead<32 * j * 128>(w, src[j], prow + 32 * j < count ? 16 : 0); });
        static_for<NP>([&](auto j) {
          cp_async16<j * PSTEP * 128>(p, psrc[j], (TR ? prk + j * PSTEP < r : q * 8 < r) ? 16 : 0);
        });
      } else {
        static_for<4>([&](auto j) { copy16<true, 32 * j * 128>(w, src[j], D - kst - pc * 8, prow + 32 * j < count, x); });
        static_for<NP>([&](auto j) {
            if constexpr (!TR)
              copy16<false, j * PSTEP * 128>(p, psrc[j], r - q * 8, kst + prk + j * PSTEP < D, P, halves);
            else
              copy16<false, j * PSTEP * 128>(p, psrc[j], D - kst - q * 8, prk + j * PSTEP < r, P);
          });
      }
      cp_async_commit();
#pragma unroll
      for (int j = 0; j < 4; ++j) src[j] += 64;
#pragma unroll
      for (int j = 0; j < NP; ++j) psrc[j] += TR ? 64 : 64 * r;
      kst += 64;
      slot = (slot + 1) % TC_STG;
      if (i >= TC_LAG) {
        cp_async_wait<TC_LAG>();
        fence_proxy_async_smem();  // this thread's copies, before the multiply's reads
        mbar_arrive(&full[(i - TC_LAG) % TC_STG]);
      }
    }
    cp_async_wait<0>();
    fence_proxy_async_smem();
    if (ok)
      for (int i = max(0, n - TC_LAG); i < n; ++i) mbar_arrive(&full[i % TC_STG]);
    else
      s_err = 1;
  } else if (lane == 0) {
    // ---------------------------------------------------------------- products
    constexpr uint32_t idesc = idesc_f16(128, RP, std::is_same<T, __nv_bfloat16>::value ? 1 : 0, 0, TR ? 0 : 1);
    for (int i = 0; i < n; ++i) {
      const int s = i % TC_STG;
      if (!mbar_wait(&full[s], (i / TC_STG) & 1, a.status)) {
        s_err = 1;
        break;
      }
      tc_fence_after();
      const uint32_t xa = smem + s * TC_STAGE, pa = xa + TC_X;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // X (and P backward) K-major: 8-row groups 1024 B apart, a k16 step 32 B;
        // P forward MN-major: one atom of 64 columns, 8-row k groups 1024 B apart, a k16 step two of them
        const uint64_t ad = smem_desc(xa + k * 32, 16, 1024, 2);
        const uint64_t bd = TR ? smem_desc(pa + k * 32, 16, 1024, 2) : smem_desc(pa + k * 2048, 1024, 1024, 2);
        tc_mma_f16_ss(tmem, ad, bd, idesc, (i | k) != 0);
      }
      tc_commit(&empty[s]);
    }
    tc_commit(&done);
  }
  __syncwarp();
  pdl_launch_next();
  // ---------------------------------------------------------------- sums: tensor memory -> shared memory -> the cluster
  constexpr int PP = RP + 4;
  float* part = reinterpret_cast<float*>(sm);
  if (!mbar_wait(&done, 0, a.status)) s_err = 1;
  __syncwarp();
  tc_fence_after();
  if (warp < WARPS) {
    // lane quadrant warp % 4, half of the columns
    const int c0 = (warp >> 2) * 32;
    uint32_t v[32];
    tmem_ld32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0, v);
    tmem_ld_wait();
    float* row = part + ((warp & 3) * 32 + lane) * PP + c0;
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      *reinterpret_cast<float4*>(row + i) = make_float4(__uint_as_float(v[i]), __uint_as_float(v[i + 1]),
                                                        __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
  }
  tc_fence_before();
  __syncthreads();
  if (S > 1) cluster_sync();
  if (warp == WARPS) {
    tc_fence_after();
    tmem_dealloc(tmem, RP);
  }
  const float scale = a.scaling ? a.scaling[tl.x] : 1.f;
  const int q0 = rank * ROWS_L / S, q1 = min((rank + 1) * ROWS_L / S, count);
  if (!s_err) {
    for (int i = tid; i < (q1 - q0) * (RP / 4); i += SHRINK_TC_THREADS) {
      const int row = q0 + i / (RP / 4), col = i % (RP / 4) * 4;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      if (S == 1) {
        s = *reinterpret_cast<const float4*>(part + row * PP + col);
      } else {
        const uint32_t addr = smem_u32(part + row * PP + col);
        for (int c = 0; c < S; ++c) {
          float4 u;
          asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                       : "=f"(u.x), "=f"(u.y), "=f"(u.z), "=f"(u.w)
                       : "r"(map_shared_rank(addr, c))
                       : "memory");
          s.x += u.x, s.y += u.y, s.z += u.z, s.w += u.w;
        }
      }
      // past the rank: an exact 0, whatever x holds
      *reinterpret_cast<float4*>(a.mid + (size_t)rows[row] * a.mp + col) =
          make_float4(col < r ? s.x * scale : 0.f, col + 1 < r ? s.y * scale : 0.f, col + 2 < r ? s.z * scale : 0.f,
                      col + 3 < r ? s.w * scale : 0.f);
    }
  }
  if (S > 1) cluster_sync();  // the others have read this CTA's part
}

const void* shrink_tc_kernel(int dtype, bool tr) {
  if (dtype == B200Q_DTYPE_FP16)
    return tr ? (const void*)lora_shrink_tc_kernel<__half, true> : (const void*)lora_shrink_tc_kernel<__half, false>;
  return tr ? (const void*)lora_shrink_tc_kernel<__nv_bfloat16, true> : (const void*)lora_shrink_tc_kernel<__nv_bfloat16, false>;
}

}  // namespace lora
}  // namespace b200q
