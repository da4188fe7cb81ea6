// Gradients of the adapters: for each adapter a over its tokens,
//   dA[a] [D, r] = sum_t x[t]^T dlo[t],   dB[a] [r, N] = sum_t lo[t]^T dy[t],
// lo and dlo in fp32 with the scaling included (lora_seg.cuh's mid).  An
// adapter without tokens gets zeros.
//
// Both are one product, thin^T . wide over the tokens, so one launch does both:
// a CTA owns CT columns of x or of dy, one adapter and 1/S of its tokens, and
// steps through them TK at a time: the wide rows by asynchronous copies into a
// ring of GSTG stages, the thin rows through registers, split into two halves
// of the type one stage ahead (fp16: scaled by a power of two that follows the
// largest value seen, the sums with it).  A warp takes 32 columns and one half
// of the stage's tokens.  The two halves, and the S parts of a token range, which
// a second launch joins, are added in a fixed order: deterministic.  (As a
// cluster the parts would need no second launch, but clusters of 3 fill only
// 142 x 3 of the SMs' 444 places: 144 column blocks took two rounds.)
// Bound: HBM, x and dy once; at r = 64 the legacy tensor rate is as near (two
// halves: 4 T r (D + N) flop).  Measured, one adapter, 8192 tokens, 4096 + 14336
// columns (302 MB), r = 16: 63 us, 4.8 TB/s; the copies alone take 52.
#include <type_traits>

#include "lora_seg.cuh"

namespace b200q {
namespace lora {

constexpr int CT = 128;  // columns of a CTA
constexpr int TK = 64;   // tokens of a stage
constexpr int WPITCH = CT * 2 + 16;
constexpr int OPITCH = CT + 1;
constexpr int TOKS = 8;  // stages of token indices kept (more than GSTG + 2)

template <int RP>
struct GradCfg {
  // stages of the wide rows and CTAs per SM: as many bytes in flight either way, more warps where they fit
  static constexpr int GSTG = RP == 64 ? 4 : 3, CTAS = RP == 64 ? 2 : 3;
  static constexpr int TPITCH = RP * 2 + 16;
  static constexpr int WIDE = GSTG * TK * WPITCH;
  static constexpr int THIN = TK * TPITCH;  // one half of one stage; two stages are kept
  static constexpr int OUT = RP * OPITCH * 4;
  static constexpr int SMEM = WIDE + 4 * THIN > OUT ? WIDE + 4 * THIN : OUT;
  static constexpr int VPT = TK * RP / 4 / THREADS;  // float4 of the thin rows per thread
};

struct GradArgs {
  const void *x, *dy;
  const float *lo, *dlo;
  const int32_t* plan;
  PlanLayout lay;
  int D, N, r, mp, nbd;
  int64_t T;
  void *dA, *dB;
  float* part;  // S > 1: [S][L][blocks][RP][CT] sums
};

// Rounds a block's sums [rank][column] into dA [column][rank] or dB [rank][column].
template <class T>
__device__ __forceinline__ void write_block(const GradArgs& a, const float* out, int block, int seg) {
  const bool da = block < a.nbd;
  const int W = da ? a.D : a.N, r = a.r, w0 = (da ? block : block - a.nbd) * CT, nc = min(CT, W - w0);
  T* dst = reinterpret_cast<T*>(da ? a.dA : a.dB) + (size_t)seg * W * r;
  if (da) {
    for (int i = threadIdx.x; i < nc * r; i += THREADS)  // nc * r consecutive values of dA
      dst[(size_t)w0 * r + i] = ft<T>(out[i % r * OPITCH + i / r]);
  } else {
    for (int i = threadIdx.x; i < CT * r; i += THREADS) {
      const int j = i / CT, c = i % CT;
      if (c < nc) dst[(size_t)j * W + w0 + c] = ft<T>(out[j * OPITCH + c]);
    }
  }
}

template <class T, int RP, bool VEC>
__global__ void __launch_bounds__(THREADS, VEC ? GradCfg<RP>::CTAS : 2) lora_grads_kernel(const GradArgs a, int S) {
  using C = GradCfg<RP>;
  constexpr int GSTG = C::GSTG;
  constexpr bool F16 = std::is_same<T, __half>::value;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int s_tok[TOKS][TK];
  __shared__ unsigned s_max[4];
  const bool da = (int)blockIdx.x < a.nbd;  // columns of x (dA) or of dy (dB)
  const T* wide = reinterpret_cast<const T*>(da ? a.x : a.dy);
  const float* thin = da ? a.dlo : a.lo;
  const int W = da ? a.D : a.N;
  const int w0 = (da ? blockIdx.x : blockIdx.x - a.nbd) * CT;
  const int seg = blockIdx.y, rank = blockIdx.z;
  const int b0 = a.plan[a.lay.seg + seg], b1 = a.plan[a.lay.seg + seg + 1];
  const int nst_all = (b1 - b0 + TK - 1) / TK;
  // whole stages per part
  const int f0 = b0 + (int)((int64_t)rank * nst_all / S) * TK;
  const int f1 = min(b1, b0 + (int)((int64_t)(rank + 1) * nst_all / S) * TK);
  const int nst = (f1 - f0 + TK - 1) / TK;
  const int32_t* order = a.plan + a.lay.order;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int cg = warp & 3, half = warp >> 2;

  auto load_tokens = [&](int st) {  // threads 0 .. TK - 1
    const int i = f0 + st * TK + tid;
    s_tok[st % TOKS][tid] = i < f1 ? order[i] : -1;
  };
  const T* wcol = wide + w0 + (tid & 15) * 8;
  const int wleft = W - w0 - (tid & 15) * 8;
  uint4 wv[VEC ? 1 : TK / 16];  // rows of any alignment: to registers a stage ahead, then to the ring
  auto stage_wide = [&](int st) {
    // this thread's 16 bytes of rows tid / 16 + 16 i
    const uint32_t dst = smem_u32(sm) + st % GSTG * (TK * WPITCH) + (tid >> 4) * WPITCH + (tid & 15) * 16;
    const int* toks = &s_tok[st % TOKS][tid >> 4];
    static_for<TK / 16>([&](auto i) {
      const int tok = toks[16 * i];
      if constexpr (VEC)
        copy16<true, 16 * i * WPITCH>(dst, wcol + (size_t)max(tok, 0) * W, wleft, tok >= 0, wide);
      else
        wv[i] = tok >= 0 ? ld8_any<T>(wcol + (size_t)tok * W, wleft, wide + a.T * W) : make_uint4(0, 0, 0, 0);
    });
  };
  auto put_wide = [&](int st) {
    if constexpr (!VEC) {
      const uint32_t dst = smem_u32(sm) + st % GSTG * (TK * WPITCH) + (tid >> 4) * WPITCH + (tid & 15) * 16;
      static_for<TK / 16>([&](auto i) { sts16<16 * i * WPITCH>(dst, wv[i]); });
    }
  };
  float4 tv[C::VPT];
  auto load_thin = [&](int st) {
#pragma unroll
    for (int i = 0; i < C::VPT; ++i) {
      const int idx = tid + i * THREADS, row = idx / (RP / 4), col = idx % (RP / 4) * 4;
      const int tok = s_tok[st % TOKS][row];
      tv[i] = tok >= 0 ? *reinterpret_cast<const float4*>(thin + (size_t)tok * a.mp + col)
                       : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  auto note_max = [&](int st) {  // fp16: the largest exponent of the finite values in tv
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < C::VPT; ++i) {
      const float f[4] = {tv[i].x, tv[i].y, tv[i].z, tv[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned x = (__float_as_uint(f[e]) >> 23) & 0xffu;
        if (x != 255) m = max(m, x);
      }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) atomicMax(&s_max[st & 3], m);
  };
  float acc[RP / 16][4][4] = {};
  float fac = 1.f, inv = 1.f;  // fp16: sums and thin rows carry inv = 1 / fac
  unsigned emax = 0;
  // splits tv into stage st's buffer; returns what the sums have to be multiplied by before they take that stage
  auto put_thin = [&](int st) {
    float scale = 1.f;
    if (F16) {
      const unsigned m = s_max[st & 3];
      if (m > emax) {
        float nf, ni;
        scale_of<T>(__uint_as_float(m << 23), nf, ni);
        scale = fac * ni;  // both powers of two
        fac = nf;
        inv = ni;
        emax = m;
      }
    }
    uint8_t* hi_ = sm + C::WIDE + (st & 1) * 2 * C::THIN;
    uint8_t* lo_ = hi_ + C::THIN;
#pragma unroll
    for (int i = 0; i < C::VPT; ++i) {
      const int idx = tid + i * THREADS, row = idx / (RP / 4), col = idx % (RP / 4) * 4;
      T hi[4], lo[4];
      split(tv[i].x * inv, hi[0], lo[0]);
      split(tv[i].y * inv, hi[1], lo[1]);
      split(tv[i].z * inv, hi[2], lo[2]);
      split(tv[i].w * inv, hi[3], lo[3]);
      *reinterpret_cast<uint2*>(hi_ + row * C::TPITCH + col * 2) = make_uint2(pack2(hi[0], hi[1]), pack2(hi[2], hi[3]));
      *reinterpret_cast<uint2*>(lo_ + row * C::TPITCH + col * 2) = make_uint2(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]));
    }
    return scale;
  };

  if (tid < 4) s_max[tid] = 0;
  if (tid < TK) {
    for (int i = 0; i < GSTG + 1; ++i) load_tokens(i);
  }
  __syncthreads();
  float rescale = 1.f;
  if (nst > 0) {
    load_thin(0);
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < GSTG - 1; ++i) {
        if (i < nst) stage_wide(i);
        cp_async_commit();
      }
    } else {
      stage_wide(0);
      put_wide(0);
      if (nst > 1) stage_wide(1);
    }
    if (F16) {
      note_max(0);
      __syncthreads();
    }
    put_thin(0);
    load_thin(1);
    if (F16) note_max(1);
  }
  for (int st = 0; st < nst; ++st) {
    cp_async_wait<GSTG - 2>();
    __syncthreads();  // stage st's wide and thin rows are in place; everyone is done with stage st - 1
    rescale = 1.f;
    if (st + 1 < nst) rescale = put_thin(st + 1);
    if (F16 && tid == 0) s_max[(st + 3) & 3] = 0;  // next used by note_max(st + 3), a barrier from here
    if constexpr (VEC) {
      if (st + GSTG - 1 < nst) stage_wide(st + GSTG - 1);
      cp_async_commit();
    } else {
      if (st + 1 < nst) put_wide(st + 1);
      if (st + 2 < nst) stage_wide(st + 2);
    }
    if (st + 2 < nst) load_thin(st + 2);
    if (tid < TK) load_tokens(st + GSTG + 1);
    // A: thin^T (rank rows), B: wide (this warp's 32 columns), k: this warp's half of the tokens
    const uint32_t wb = smem_u32(sm + st % GSTG * TK * WPITCH) + (32 * half + 8 * ((lane >> 3) & 1) + (lane & 7)) * WPITCH +
                        (cg * 32 + 8 * (lane >> 4)) * 2;
    const uint32_t th = smem_u32(sm + C::WIDE + (st & 1) * 2 * C::THIN) +
                        (32 * half + 8 * (lane >> 4) + (lane & 7)) * C::TPITCH + 16 * ((lane >> 3) & 1);
    static_for<2>([&](auto k) {
      uint32_t b[8];
      ldmatrix_x4_trans<k * 16 * WPITCH>(b, wb);
      ldmatrix_x4_trans<k * 16 * WPITCH + 32>(b + 4, wb);
      static_for<RP / 16>([&](auto i) {
        uint32_t h[4], l[4];
        ldmatrix_x4_trans<k * 16 * C::TPITCH + i * 32>(h, th);
        ldmatrix_x4_trans<C::THIN + k * 16 * C::TPITCH + i * 32>(l, th);
#pragma unroll
        for (int p = 0; p < 4; ++p) mma16816<T>(acc[i][p], h[0], h[1], h[2], h[3], b[2 * p], b[2 * p + 1]);
#pragma unroll
        for (int p = 0; p < 4; ++p) mma16816<T>(acc[i][p], l[0], l[1], l[2], l[3], b[2 * p], b[2 * p + 1]);
      });
    });
    if (F16) {
      if (rescale != 1.f) {
#pragma unroll
        for (int i = 0; i < RP / 16; ++i)
#pragma unroll
          for (int p = 0; p < 4; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][p][e] *= rescale;
      }
      if (st + 2 < nst) note_max(st + 2);
    }
  }
  cp_async_wait<0>();
  __syncthreads();
  float* out = reinterpret_cast<float*>(sm);
#pragma unroll
  for (int h = 1; h >= 0; --h) {
    if (half == h) {
#pragma unroll
      for (int i = 0; i < RP / 16; ++i)
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float* o = out + (16 * i + g + 8 * (e >> 1)) * OPITCH + cg * 32 + 8 * p + 2 * t + (e & 1);
            *o = acc[i][p][e] * fac + (h == 0 ? *o : 0.f);
          }
    }
    if (h) __syncthreads();
  }
  pdl_launch_next();
  __syncthreads();
  if (S > 1) {
    float* dst = a.part + (((size_t)rank * gridDim.y + seg) * gridDim.x + blockIdx.x) * (RP * CT);
    for (int i = tid; i < RP * CT; i += THREADS) dst[i] = out[i / CT * OPITCH + i % CT];
    return;
  }
  write_block<T>(a, out, blockIdx.x, seg);
}

// The sums of the S parts of a block, in order.
template <class T, int RP>
__global__ void __launch_bounds__(THREADS) lora_grads_join_kernel(const GradArgs a, int S) {
  __shared__ float out[RP * OPITCH];
  pdl_wait_previous();
  constexpr int N4 = RP * CT / 4 / THREADS;  // 16 bytes at a time, a part's all in flight together
  static_assert(N4 * 4 * THREADS == RP * CT, "whole rounds");
  const size_t step = (size_t)gridDim.y * gridDim.x * (RP * CT / 4);
  const float4* src = reinterpret_cast<const float4*>(a.part) +
                      ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * (RP * CT / 4) + threadIdx.x;
  float4 v[N4] = {};
#pragma unroll 2
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int k = 0; k < N4; ++k) {
      const float4 u = src[s * step + k * THREADS];
      v[k].x += u.x, v[k].y += u.y, v[k].z += u.z, v[k].w += u.w;
    }
#pragma unroll
  for (int k = 0; k < N4; ++k) {
    const int i = (threadIdx.x + k * THREADS) * 4;
    float* o = out + i / CT * OPITCH + i % CT;
    o[0] = v[k].x, o[1] = v[k].y, o[2] = v[k].z, o[3] = v[k].w;
  }
  __syncthreads();
  write_block<T>(a, out, blockIdx.x, blockIdx.y);
}

constexpr int MAX_PARTS = 8;

// Parts of the tokens: the shortest estimate, for adapters of equal shares:
// rounds of co-resident CTAs x (stages of a part + 5).  More than one part only
// where the column blocks leave places free, so the parts' sums stay small.
template <class T, int RP, bool VEC>
int parts_of(int64_t T_, int64_t blocks, int64_t L) {
  const int64_t fit = resident_clusters((const void*)lora_grads_kernel<T, RP, VEC>, THREADS, GradCfg<RP>::SMEM)[1];
  const int64_t nst = (T_ + TK * L - 1) / (TK * L);
  int S = 1;
  int64_t best = INT64_MAX;
  for (int s = 1; s <= MAX_PARTS && (s == 1 || (T_ >= 4 * TK * s && blocks * s <= 2 * fit)); ++s) {
    const int64_t cost = (blocks * s + fit - 1) / fit * ((nst + s - 1) / s + 5);
    if (cost < best) best = cost, S = s;
  }
  return S;
}

static int64_t column_blocks(int64_t W) { return (W + CT - 1) / CT; }

size_t grads_part_bytes(int64_t T_, int64_t D, int64_t N, int64_t r, int64_t L, int dtype) {
  size_t bytes = 0;
  by_type(dtype, r, aligned_widths(D, N, r), [&](auto tc, auto rc, auto vc) -> int {
    using T = decltype(tc);
    constexpr int RP = decltype(rc)::value;
    const int64_t blocks = (column_blocks(D) + column_blocks(N)) * L;
    const int S = parts_of<T, RP, decltype(vc)::value>(T_, blocks, L);
    bytes = S > 1 ? (size_t)S * blocks * (RP * CT) * 4 : 0;
    return 0;
  });
  return bytes;
}

int launch_grads(const void* x, const void* dy, const float* lo, const float* dlo, const int32_t* plan,
                 const PlanLayout& lay, int64_t T_, int64_t D, int64_t N, int64_t r, int64_t L, int dtype, float* part,
                 void* dA, void* dB, cudaStream_t st) {
  if (T_ == 0) {
    cudaError_t e = cudaSuccess;
    if (dA) e = cudaMemsetAsync(dA, 0, (size_t)L * D * r * 2, st);
    if (dB && e == cudaSuccess) e = cudaMemsetAsync(dB, 0, (size_t)L * N * r * 2, st);
    return check_cuda(e, "lora_grads memset");
  }
  const int nbd = dA ? (int)column_blocks(D) : 0, nbn = dB ? (int)column_blocks(N) : 0;
  const GradArgs a = {x, dy, lo, dlo, plan, lay, (int)D, (int)N, (int)r, mid_pitch(r), nbd, T_, dA, dB, part};
  return by_type(dtype, r, aligned_widths(D, N, r), [&](auto tc, auto rc, auto vc) -> int {
    using T = decltype(tc);
    constexpr int RP = decltype(rc)::value;
    constexpr bool VEC = decltype(vc)::value;
    auto kern = lora_grads_kernel<T, RP, VEC>;
    constexpr int smem = GradCfg<RP>::SMEM;
    const int rc2 = allow_smem((const void*)kern, smem, "cudaFuncSetAttribute(lora grads)");
    if (rc2) return rc2;
    // as in grads_part_bytes, whichever gradients are wanted
    const int S = parts_of<T, RP, VEC>(T_, (column_blocks(D) + column_blocks(N)) * L, L);
    kern<<<dim3((unsigned)(nbd + nbn), (unsigned)L, (unsigned)S), THREADS, smem, st>>>(a, S);
    if (S > 1) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(nbd + nbn), (unsigned)L);
      cfg.blockDim = dim3(THREADS);
      cfg.stream = st;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      cudaLaunchKernelEx(&cfg, lora_grads_join_kernel<T, RP>, a, S);
    }
    return check_cuda(cudaGetLastError(), "lora_grads launch");
  });
}

}  // namespace lora
}  // namespace b200q
