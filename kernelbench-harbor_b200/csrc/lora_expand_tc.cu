// Many tokens an adapter, aligned rows, ranks 33 to 64: the expand product
//   y[rows, N] = base + mid[rows, r] . Q[r, N]
// on 128-row tiles of one adapter, 64 columns at a time, the sums in tensor memory.
//
// The tile's mid rows are split into two halves of the type once (scaled by a
// power of two per row, scale_of) and stay in shared memory as two
// K-major operands; a ring of 3 stages holds base's 64 columns and the stage of
// Q (as stored: MN-major forward, K-major backward), both by 16-byte
// asynchronous copies in the 128-byte swizzle.  One thread issues a stage's 8
// tcgen05.mma (M128 N64 K16; 4 k steps, both halves) into one of two
// accumulators while the stage before is stored: the warps read a row per lane
// from tensor memory, add base in place in shared memory, and leave as whole
// 128-byte lines.
// Bound: HBM, base and y once; the steps run near the measured copy rate, start
// (plan, rows, mid, halves: 3 us) beside them.  After the shrink at N=14336, D=4096,
// r=64, 8192 tokens of two adapters 129 us for both (142 with register fragments);
// 4096 tokens, N=4096, D=14336: 52.4 and 54.1.
#include "lora_seg.cuh"

namespace b200q {
namespace lora {

constexpr int ETC_STG = 3, ETC_W = 128 * 128, ETC_Q = 64 * 128, ETC_STAGE = ETC_W + ETC_Q;
constexpr int ETC_MID = 128 * 128;  // bytes of one half of mid
constexpr int ERP = 64, ECOLS = 64;  // ranks; columns of a stage and of an accumulator
static_assert(EXPAND_TC_SMEM == 2 * ETC_MID + ETC_STG * ETC_STAGE + 1024, "lora_seg.cuh has the launch's size");

template <class T, bool TR>
__global__ void __launch_bounds__(THREADS, 2) lora_expand_tc_kernel(const Args a, int parts, int steps) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t done[2];
  __shared__ uint32_t s_tmem;
  __shared__ float s_fac[ROWS_L];
  const int32_t* plan = a.plan;
  const int tile = blockIdx.x / parts;  // a tile's parts run side by side
  if (tile >= plan[1]) {
    pdl_wait_previous();
    return;
  }
  const int4 tl = reinterpret_cast<const int4*>(plan + a.lay.large)[tile];
  const int32_t* rows = plan + a.lay.order + tl.y;
  const int count = tl.z, N = a.N, r = a.r, n0 = blockIdx.x % parts * steps * ECOLS;
  const int nst = min(steps, (N - n0 + ECOLS - 1) / ECOLS);
  const T* base = reinterpret_cast<const T*>(a.base);
  T* y = reinterpret_cast<T*>(a.y);
  if (tl.x < 0) {
    copy_rows<T, true>(base, y, rows, count, N, n0, min(n0 + steps * ECOLS, N), base + a.T * N);
    pdl_wait_previous();
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* const sm = align_smem_1024(raw);
  const uint32_t smem = smem_u32(sm), ring = smem + 2 * ETC_MID;
  if (tid == 0) {
    mbar_init(&done[0], 1);
    mbar_init(&done[1], 1);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&s_tmem, 2 * ECOLS);
  // this thread's pieces: 16 bytes of rows tid / 8 + 32 i of base and y, and of Q's rows
  const int pc = tid & 7, prow = tid >> 3;
  const uint32_t wdst = prow * 128 + ((pc ^ (prow & 7)) << 4);  // the same piece of 32 rows further on is 4096 bytes on
  size_t off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) off[i] = (size_t)rows[prow + 32 * i < count ? prow + 32 * i : 0] * N + n0 + pc * 8;
  const T* const Q = reinterpret_cast<const T*>(a.Q) + (size_t)tl.x * r * N;
  const T* qsrc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    qsrc[i] = TR ? Q + (size_t)(n0 + prow + 32 * i) * r + pc * 8 : Q + (size_t)min(prow + 32 * i, r - 1) * N + n0 + pc * 8;
  const bool halves = r % 8 != 0;  // TR: A's rows are 8-byte aligned only
  auto request = [&](int st) {
    const uint32_t to = ring + st % ETC_STG * ETC_STAGE;
    const int c = n0 + st * ECOLS;
    if (base)
      static_for<4>([&](auto i) {
        copy16<true, 32 * i * 128>(to + wdst, base + off[i] + st * ECOLS, N - c - pc * 8, prow + 32 * i < count, base);
      });
    static_for<2>([&](auto i) {
      if constexpr (TR)
        copy16<false, 32 * i * 128>(to + ETC_W + wdst, qsrc[i] + (size_t)st * ECOLS * r, r - pc * 8, c + prow + 32 * i < N, Q,
                                    halves);
      else
        copy16<false, 32 * i * 128>(to + ETC_W + wdst, qsrc[i] + st * ECOLS, N - c - pc * 8, prow + 32 * i < r, Q);
    });
  };
#pragma unroll
  for (int i = 0; i < ETC_STG; ++i) {
    if (i < nst) request(i);
    cp_async_commit();
  }
  {
    // mid as two halves of the type: a warp's 16 rows, two at a time, four values per lane
    const float* src[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = warp * 16 + 2 * i + (lane >> 4);
      src[i] = m < count ? a.mid + (size_t)rows[m] * a.mp + 4 * (lane & 15) : nullptr;
    }
    pdl_wait_previous();  // mid comes from the kernel before; all else was there when that one began
    float4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = src[i] ? *reinterpret_cast<const float4*>(src[i]) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = warp * 16 + 2 * i + (lane >> 4);
      const float f[4] = {fabsf(v[i].x), fabsf(v[i].y), fabsf(v[i].z), fabsf(v[i].w)};
      float mx = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (f[e] < INFINITY) mx = fmaxf(mx, f[e]);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      float fac, inv;
      scale_of<T>(mx, fac, inv);
      if ((lane & 15) == 0) s_fac[m] = fac;
      T hi[4], lo[4];
      split(v[i].x * inv, hi[0], lo[0]);
      split(v[i].y * inv, hi[1], lo[1]);
      split(v[i].z * inv, hi[2], lo[2]);
      split(v[i].w * inv, hi[3], lo[3]);
      const uint32_t to = m * 128 + ((((lane & 15) >> 1) ^ (m & 7)) << 4) + (lane & 1) * 8;
      *reinterpret_cast<uint2*>(sm + to) = make_uint2(pack2(hi[0], hi[1]), pack2(hi[2], hi[3]));
      *reinterpret_cast<uint2*>(sm + ETC_MID + to) = make_uint2(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]));
    }
  }
  cp_async_wait<ETC_STG - 1>();
  fence_proxy_async_smem();  // this thread's copies and halves, before the multiply's reads
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  auto multiply = [&](int st) {  // one thread
    constexpr uint32_t idesc = idesc_f16(128, ECOLS, std::is_same<T, __nv_bfloat16>::value ? 1 : 0, 0, TR ? 0 : 1);
    const uint32_t qa = ring + st % ETC_STG * ETC_STAGE + ETC_W;
#pragma unroll
    for (int k = 0; k < ERP / 16; ++k) {
      const uint64_t bd = TR ? smem_desc(qa + k * 32, 16, 1024, 2) : smem_desc(qa + k * 2048, 1024, 1024, 2);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        tc_mma_f16_ss(tmem + (st & 1) * ECOLS, smem_desc(smem + h * ETC_MID + k * 32, 16, 1024, 2), bd, idesc, (k | h) != 0);
    }
    tc_commit(&done[st & 1]);
  };
  if (tid == 0) multiply(0);
  // the row and the 32 columns that this lane takes from tensor memory
  const int row = (warp & 3) * 32 + lane, half = warp >> 2;
  const float fac = s_fac[row];
  bool ok = true;
  int last = 0;
  for (int st = 0; st < nst; ++st) {
    uint8_t* const wide = sm + 2 * ETC_MID + st % ETC_STG * ETC_STAGE;
    if (ok && !mbar_wait(&done[st & 1], (st >> 1) & 1, a.status)) {
      ok = false;
      last = st;
    }
    __syncwarp();
    tc_fence_after();
    uint32_t acc[32];
    tmem_ld32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (st & 1) * ECOLS + half * 32, acc);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4* const at = reinterpret_cast<uint4*>(wide + row * 128 + (((half * 4 + i) ^ (row & 7)) << 4));
      const uint4 u = base ? *at : make_uint4(0, 0, 0, 0);
      const T* b = reinterpret_cast<const T*>(&u);
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = pack2(ft<T>(fmaf(__uint_as_float(acc[8 * i + 2 * e]), fac, tf<T>(b[2 * e]))),
                     ft<T>(fmaf(__uint_as_float(acc[8 * i + 2 * e + 1]), fac, tf<T>(b[2 * e + 1]))));
      *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
    cp_async_wait<1>();  // the next stage's
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && ok && st + 1 < nst) {
      tc_fence_after();
      multiply(st + 1);
    }
    if (n0 + st * ECOLS + pc * 8 < N && ok) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (prow + 32 * i < count)
          *reinterpret_cast<uint4*>(y + off[i] + st * ECOLS) = *reinterpret_cast<const uint4*>(wide + wdst + 32 * i * 128);
    }
    __syncthreads();  // the stage is read, by all
    if (st + ETC_STG < nst) request(st + ETC_STG);
    cp_async_commit();
  }
  cp_async_wait<0>();
  if (tid == 0 && !ok) mbar_wait(&done[last & 1], (last >> 1) & 1, nullptr);  // given up: no product is left running
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * ECOLS);
  }
}

const void* expand_tc_kernel(int dtype, bool tr) {
  if (dtype == B200Q_DTYPE_FP16)
    return tr ? (const void*)lora_expand_tc_kernel<__half, true> : (const void*)lora_expand_tc_kernel<__half, false>;
  return tr ? (const void*)lora_expand_tc_kernel<__nv_bfloat16, true> : (const void*)lora_expand_tc_kernel<__nv_bfloat16, false>;
}

}  // namespace lora
}  // namespace b200q
