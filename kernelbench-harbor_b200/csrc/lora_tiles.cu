// Many tokens (prefill, training): shrink and expand as two launches over tiles
// of up to 128 rows of one adapter, both streaming wide rows through a ring of
// 3 or 4 stages of 128 rows x 64 columns in shared memory (asynchronous 16-byte
// copies, 8 lanes to a row's 128 bytes), so that the CTAs of an SM keep ~96 KB
// of HBM reads in flight.
//
// shrink: a warp takes 32 rows and one 32-wide half of every stage (a piece of
// P then serves two row blocks; at rank 64, where their sums would fill the
// registers, 16 rows and both halves); the halves and, with the contraction of
// a tile split over a cluster of S CTAs, the CTAs' sums are added in a fixed
// order.
// expand: the stage is base's, beside the 64 columns of Q, whose words are put
// in the order in which a thread ends with 8 consecutive columns, so that base
// and y pass as 16-byte pieces.  A warp takes 16 rows; mid is split into two
// halves of the type once, in registers, and serves all the CTA's columns.
// Bound: HBM -- x once, base once, y once; mid (4 r bytes a token) stays in L2.
// Measured, 8192 tokens, r = 16: shrink of 14336 columns (235 MB) 42.6 us, 5.5
// TB/s; expand to 14336 columns (470 MB) 79 us, 5.9 TB/s.
#include <algorithm>
#include <type_traits>

#include "lora_seg.cuh"

namespace b200q {
namespace lora {

constexpr int SK = 64;  // columns of a stage
constexpr int ROWB = SK * 2;               // bytes of a stage's wide row; 16-byte pieces are XOR-swizzled by the row
constexpr int WIDE = ROWS_L * ROWB;        // bytes of a stage's wide rows
constexpr int MAX_SPLIT = 8;

// Stages of the ring and CTAs per SM: 4 and 2, or 3 and 3 -- as many bytes in
// flight, and half as many warps again to hide each other's latencies, but 85
// registers a thread.  Up to rank 16 these are enough; at rank 64 they never are.
// At rank 32 the shrink spills with them, and the expand, with a few words, gains
// where an adapter has few tokens: 8192 tokens in 16s, 4096 x 4096, bf16 209 us
// with three and 230 with two, in 512s 54.6 and 50.8 (with the shrink, r = 32).
// What two cost the shrink: splits of 8 fit one round for fewer tiles, and 4000
// tokens of 8 adapters there take 37.5 us instead of 34.6.
__host__ __device__ constexpr int stages_of(int ctas) { return ctas == 2 ? 4 : 3; }
__host__ __device__ constexpr int shrink_ctas(int rp, bool vec) { return !vec || rp >= 32 ? 2 : 3; }
__host__ __device__ constexpr int expand_ctas(int rp, bool vec, bool few) { return !vec || rp == 64 || (rp == 32 && !few) ? 2 : 3; }
// tokens per adapter up to which the expand kernel takes three CTAs
constexpr int FEW_TOKENS = 32;
// Tokens per adapter, and values of y, from which rank 64 expands through tensor
// memory (lora_expand_tc.cu): below, its tiles' start costs more than the
// fragments that it saves.  4096 tokens, D=4096, N=14336, bf16, shrink and expand:
// 82.2 us with fragments and 74.8 without in 128s, 113.5 and 124.8 in 64s; N=1408,
// D=2048: 14.3 and 13.0 us at 1024 tokens, 11.8 and 13.0 at 512.
constexpr int TC_TOKENS = 96;
constexpr int64_t TC_VALUES = 1 << 20;

// Swizzle of a row's 16-byte pieces: 8 rows x 1 piece (a fragment's words) and
// 2 rows x 4 pieces (a quarter warp's 16-byte loads) both meet all banks once.
__device__ __forceinline__ int swz(int row) { return ((row & 1) << 2) | ((row >> 1) & 3); }

// The 64 contraction rows of P / the rank rows of Q lie RP or 64 values wide.
template <int RP, bool TR, bool VEC>
struct ShrinkCfg {
  static constexpr int STG = stages_of(shrink_ctas(RP, VEC));
  static constexpr int PITCH = RP * 2 + 16;                    // !TR: bytes per contraction row
  static constexpr int THIN = TR ? RP * ROWB : SK * PITCH;     // TR: rank rows of 64 values
  static constexpr int STAGE = WIDE + THIN;
  static constexpr int PP = RP + 4;                            // floats per row of the partial sums, over the ring
  static constexpr int PART = ROWS_L * PP * 4;
  static constexpr int SMEM = STG * STAGE > PART ? STG * STAGE : PART;
};

template <class T, int RP, bool TR, bool VEC>
__global__ void __launch_bounds__(THREADS, shrink_ctas(RP, VEC)) lora_shrink_tile_kernel(const Args a, int S) {
  using C = ShrinkCfg<RP, TR, VEC>;
  constexpr int STG = C::STG;
  extern __shared__ __align__(128) uint8_t sm[];
  const int tile = blockIdx.x / S, rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int32_t* plan = a.plan;
  if (tile >= plan[1]) return;
  const int4 tl = reinterpret_cast<const int4*>(plan + a.lay.large)[tile];
  if (tl.x < 0) return;  // a whole cluster at a time
  const int32_t* rows = plan + a.lay.order + tl.y;
  const int count = tl.z, D = a.D, r = a.r;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  // a warp's rows are 16 NM mg .., its 32-wide parts of a stage half .. half + NH - 1
  constexpr int NM = RP == 64 ? 1 : 2, NH = RP == 64 ? 2 : 1;
  const int mg = NM == 1 ? warp : warp & 3, half = NM == 1 ? 0 : warp >> 2;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* P = reinterpret_cast<const T*>(a.P) + (size_t)tl.x * D * r;
  const int nst = (D + SK - 1) / SK;
  const int s0 = (int)((int64_t)rank * nst / S), s1 = (int)((int64_t)(rank + 1) * nst / S);

  // this thread's pieces of a stage: 16 bytes of rows tid / 8 + 32 i, and of P; pointers advance by a stage
  const int pc = tid & 7, prow = tid >> 3;
  const T* src[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    src[i] = x + (size_t)rows[prow + 32 * i < count ? prow + 32 * i : 0] * D + s0 * SK + pc * 8;
  constexpr int PIECES = SK * RP / 8, NP = (PIECES + THREADS - 1) / THREADS;
  constexpr int PSTEP = TR ? THREADS / 8 : THREADS / (RP / 8);  // rows of P between a thread's pieces
  static_assert(PSTEP % 32 == 0, "row32(row + PSTEP) = row32(row) + PSTEP, and swz(row + PSTEP) = swz(row)");
  const int q = TR ? tid & 7 : tid % (RP / 8), prk = TR ? tid >> 3 : tid / (RP / 8);
  const bool has_p = PIECES % THREADS == 0 || tid < PIECES;
  const T* psrc[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i)
    psrc[i] = TR ? P + (size_t)(prk + i * PSTEP) * D + s0 * SK + q * 8 : P + (size_t)(s0 * SK + prk + i * PSTEP) * r + q * 8;
  const uint32_t smem = smem_u32(sm), wdst = prow * ROWB + ((pc ^ swz(prow)) << 4);
  const bool halves = r % 8 != 0;  // A's rows are 8-byte aligned only
  const uint32_t pdst = WIDE + (TR ? prk * ROWB + ((q ^ swz(prk)) << 4) : row32(prk) * C::PITCH + q * 16);
  int kst = s0 * SK;     // first column of the stage that is requested next
  uint32_t in = smem;    // and its ring slot
  auto advance = [&]() {
#pragma unroll
    for (int i = 0; i < 4; ++i) src[i] += SK;
#pragma unroll
    for (int i = 0; i < NP; ++i) psrc[i] += TR ? SK : SK * r;
    kst += SK;
  };
  auto next = [&](uint32_t slot) { return slot == smem + (STG - 1) * C::STAGE ? smem : slot + C::STAGE; };
  auto stage = [&]() {  // VEC: asynchronous copies
    if (kst + SK <= D && (TR || !halves)) {  // a whole stage: no column to check
      static_for<4>([&](auto i) {
        cp_async16_ahead<32 * i * ROWB>(in + wdst, src[i], prow + 32 * i < count ? 16 : 0);
      });
      if (has_p)
        static_for<NP>([&](auto i) {
          cp_async16<i * PSTEP*(TR ? ROWB : C::PITCH)>(in + pdst, psrc[i], (TR ? prk + i * PSTEP < r : q * 8 < r) ? 16 : 0);
        });
    } else {
      static_for<4>([&](auto i) {
        copy16<true, 32 * i * ROWB>(in + wdst, src[i], D - kst - pc * 8, prow + 32 * i < count, x);
      });
      if (has_p)
        static_for<NP>([&](auto i) {
          if constexpr (!TR)
            copy16<false, i * PSTEP * C::PITCH>(in + pdst, psrc[i], r - q * 8, kst + prk + i * PSTEP < D, P, halves);
          else
            copy16<false, i * PSTEP * ROWB>(in + pdst, psrc[i], D - kst - q * 8, prk + i * PSTEP < r, P);
        });
    }
    advance();
    in = next(in);
  };
  // otherwise: to registers a stage ahead, then to the ring
  uint4 wv[VEC ? 1 : 4], pv[VEC ? 1 : NP];
  auto request = [&]() {
    if constexpr (!VEC) {
      const T* const x_end = x + a.T * D;
      const T* const p_end = reinterpret_cast<const T*>(a.P) + a.L * D * r;
      static_for<4>([&](auto i) {
        wv[i] = prow + 32 * i < count ? ld8_any<T>(src[i], D - kst - pc * 8, x_end) : make_uint4(0, 0, 0, 0);
      });
      static_for<NP>([&](auto i) {
        const bool here = has_p && (TR ? prk + i * PSTEP < r : kst + prk + i * PSTEP < D);
        pv[i] = here ? ld8_any<T>(psrc[i], TR ? D - kst - q * 8 : r - q * 8, p_end) : make_uint4(0, 0, 0, 0);
      });
      advance();
    }
  };
  auto deposit = [&]() {
    if constexpr (!VEC) {
      static_for<4>([&](auto i) { sts16<32 * i * ROWB>(in + wdst, wv[i]); });
      if (has_p) static_for<NP>([&](auto i) { sts16<i * PSTEP*(TR ? ROWB : C::PITCH)>(in + pdst, pv[i]); });
      in = next(in);
    }
  };
  float acc[NM][RP / 8][4] = {};
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < STG - 1; ++i) {
      if (s0 + i < s1) stage();
      cp_async_commit();
    }
  } else if (s0 < s1) {
    request();
    deposit();
    if (s0 + 1 < s1) request();
  }
  // where this lane reads a stage: its rows' pieces of either half, and P's
  const uint32_t xrow = (16 * NM * mg + g) * ROWB;
  uint32_t xoff[NH], poff[NH];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    const uint32_t piece = ((4 * (half + h) + t) ^ swz(g)) << 4;
    xoff[h] = xrow + piece;
    poff[h] = WIDE + (TR ? g * ROWB + piece : (32 * (half + h) + lane) * C::PITCH);
  }
  uint32_t slot = smem;
  for (int st = s0; st < s1; ++st) {
    cp_async_wait<STG - 2>();
    __syncthreads();  // stage st has landed for every thread; the slot filled next was read before
    if constexpr (VEC) {
      if (st + STG - 1 < s1) stage();
      cp_async_commit();
    } else {
      if (st + 1 < s1) deposit();
      if (st + 2 < s1) request();
    }
    if (16 * NM * mg < count) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        uint4 xv[NM][2];
        static_for<NM>([&](auto m) {
          xv[m][0] = lds16<16 * m * ROWB>(slot + xoff[h]);
          xv[m][1] = lds16<(16 * m + 8) * ROWB>(slot + xoff[h]);
        });
        // fragments of 4 column tiles at a time, then their products: none waits for the one before
        constexpr int JB = RP / 8 < 4 ? RP / 8 : 4;
        static_for<RP / 8 / JB>([&](auto j0) {
          uint32_t b[JB][4];
          static_for<JB>([&](auto j) {
            if constexpr (!TR) {
              ldmatrix_x4_trans<(j0 * JB + j) * 16>(b[j], slot + poff[h]);
            } else {
              const uint4 w = lds16<(j0 * JB + j) * 8 * ROWB>(slot + poff[h]);
              b[j][0] = w.x, b[j][1] = w.y, b[j][2] = w.z, b[j][3] = w.w;
            }
          });
#pragma unroll
          for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int j = 0; j < JB; ++j)
              mma16816<T>(acc[m][j0 * JB + j], xv[m][0].x, xv[m][1].x, xv[m][0].y, xv[m][1].y, b[j][0], b[j][1]);
#pragma unroll
          for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int j = 0; j < JB; ++j)
              mma16816<T>(acc[m][j0 * JB + j], xv[m][0].z, xv[m][1].z, xv[m][0].w, xv[m][1].w, b[j][2], b[j][3]);
        });
      }
    }
    slot = next(slot);
  }
  pdl_launch_next();
  cp_async_wait<0>();
  __syncthreads();
  // the two halves of the stages, then the CTAs of the cluster
  float* part = reinterpret_cast<float*>(sm);
#pragma unroll
  for (int h = NM - 1; h >= 0; --h) {
    if (half == h) {
#pragma unroll
      for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int j = 0; j < RP / 8; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float2* p = reinterpret_cast<float2*>(part + (16 * (NM * mg + m) + 8 * e + g) * C::PP + 8 * j + 2 * t);
            float2 v = make_float2(acc[m][j][2 * e], acc[m][j][2 * e + 1]);
            if (NM == 2 && h == 0) v.x += p->x, v.y += p->y;
            *p = v;
          }
    }
    if (h) __syncthreads();
  }
  if (S > 1)
    cluster_sync();
  else
    __syncthreads();
  const float scale = a.scaling ? a.scaling[tl.x] : 1.f;
  const int q0 = rank * ROWS_L / S, q1 = min((rank + 1) * ROWS_L / S, count);
  for (int i = tid; i < (q1 - q0) * (RP / 4); i += THREADS) {
    const int row = q0 + i / (RP / 4), col = i % (RP / 4) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (S == 1) {
      s = *reinterpret_cast<const float4*>(part + row * C::PP + col);
    } else {
      const uint32_t addr = smem_u32(part + row * C::PP + col);
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
  if (S > 1) cluster_sync();  // the others have read this CTA's part
}

template <int RP, bool TR, int CTAS>
struct ExpandCfg {
  static constexpr int STG = stages_of(CTAS);
  // !TR: bytes per rank row of 64 columns; TR: per column row of RP ranks, 8 words mod 32 (no bank conflicts)
  static constexpr int PITCH = !TR ? ROWB + 16 : RP == 16 ? 32 : RP == 32 ? 96 : 160;
  static constexpr int THIN = (TR ? SK : RP) * PITCH;
  static constexpr int STAGE = WIDE + THIN;
  static constexpr int SMEM = STG * STAGE;
};

// CTA = (tile, part): `steps` 64-column steps from step part * steps on.
template <class T, int RP, bool TR, bool VEC, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) lora_expand_tile_kernel(const Args a, int parts, int steps) {
  using C = ExpandCfg<RP, TR, CTAS>;
  constexpr int STG = C::STG;
  extern __shared__ __align__(128) uint8_t sm[];
  const int32_t* plan = a.plan;
  const int tile = blockIdx.x / parts;  // a tile's parts run side by side
  if (tile >= plan[1]) {
    pdl_wait_previous();
    return;
  }
  const int4 tl = reinterpret_cast<const int4*>(plan + a.lay.large)[tile];
  const int32_t* rows = plan + a.lay.order + tl.y;
  const int count = tl.z, N = a.N, r = a.r, n0 = blockIdx.x % parts * steps * SK;
  const int nst = min(steps, (N - n0 + SK - 1) / SK);
  const T* base = reinterpret_cast<const T*>(a.base);
  T* y = reinterpret_cast<T*>(a.y);
  if (tl.x < 0) {
    copy_rows<T, VEC>(base, y, rows, count, N, n0, min(n0 + steps * SK, N), base + a.T * N);
    pdl_wait_previous();
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const T* Q = reinterpret_cast<const T*>(a.Q) + (size_t)tl.x * r * N;
  const int pc = tid & 7, prow = tid >> 3;
  const T* src[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    src[i] = base ? base + (size_t)rows[prow + 32 * i < count ? prow + 32 * i : 0] * N + n0 + pc * 8 : nullptr;
  constexpr int PIECES = SK * RP / 8, NP = (PIECES + THREADS - 1) / THREADS;
  constexpr int PSTEP = TR ? THREADS / (RP / 8) : THREADS / 8;  // rows of Q between a thread's pieces
  static_assert(PSTEP % 32 == 0, "the row orders repeat every 32");
  const int q = TR ? tid % (RP / 8) : tid & 7, qrow = TR ? tid / (RP / 8) : tid >> 3;
  const bool has_q = PIECES % THREADS == 0 || tid < PIECES;
  const T* qsrc[NP];
  int qin[NP];  // TR: bytes of the piece inside the rank; !TR: whether the rank row exists
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = qrow + i * PSTEP, k = k_of_row16(row);  // !TR: rank rows in fragment order
    qsrc[i] = TR ? Q + (size_t)(n0 + row) * r + q * 8 : Q + (size_t)(k < r ? k : 0) * N + n0 + q * 8;
    qin[i] = TR ? (q * 8 < r ? 16 : 0) : k < r;
  }
  // TR: column 32 w + 8 a + 2 p + b is row 32 w + 8 p + 2 a + b: a fragment's columns together
  const uint32_t smem = smem_u32(sm), wdst = prow * ROWB + ((pc ^ swz(prow)) << 4);
  const uint32_t qdst = WIDE + (TR ? ((qrow & ~31) | (((qrow >> 1) & 3) << 3) | (((qrow >> 3) & 3) << 1) | (qrow & 1)) * C::PITCH + q * 16
                                   : qrow * C::PITCH + (q >> 2) * 64 + (q & 3) * 4);
  int cst = n0;
  uint32_t in = smem;
  auto advance = [&]() {
#pragma unroll
    for (int i = 0; i < 4; ++i) src[i] += SK;
    if (TR) {
#pragma unroll
      for (int i = 0; i < NP; ++i) qsrc[i] += SK * r;
    }
    cst += SK;
  };
  auto next = [&](uint32_t slot) { return slot == smem + (STG - 1) * C::STAGE ? smem : slot + C::STAGE; };
  const bool halves = r % 8 != 0;  // TR: A's rows are 8-byte aligned only
  // VEC: base (and, TR, A's rows) by asynchronous copies
  auto stage = [&]() {
    if (cst + SK <= N && !(TR && halves)) {
      if (base)
        static_for<4>([&](auto i) {
          cp_async16_ahead<32 * i * ROWB>(in + wdst, src[i], prow + 32 * i < count ? 16 : 0);
        });
      if (TR && has_q) static_for<NP>([&](auto i) { cp_async16<i * PSTEP * C::PITCH>(in + qdst, qsrc[i], qin[i]); });
    } else {
      if (base)
        static_for<4>([&](auto i) {
          copy16<true, 32 * i * ROWB>(in + wdst, src[i], N - cst - pc * 8, prow + 32 * i < count, base);
        });
      if (TR && has_q)
        static_for<NP>([&](auto i) {
          copy16<false, i * PSTEP * C::PITCH>(in + qdst, qsrc[i], r - q * 8, cst + qrow + i * PSTEP < N, Q, halves);
        });
    }
    advance();
    in = next(in);
  };
  // otherwise: to registers a stage ahead, then to the ring
  const T* const q_end = reinterpret_cast<const T*>(a.Q) + a.L * N * r;
  uint4 wv[VEC ? 1 : 4], av[VEC || !TR ? 1 : NP];
  auto request = [&]() {
    if constexpr (!VEC) {
      static_for<4>([&](auto i) {
        wv[i] = base && prow + 32 * i < count ? ld8_any<T, false>(src[i], N - cst - pc * 8, base + a.T * N) : make_uint4(0, 0, 0, 0);
      });
      if constexpr (TR)
        static_for<NP>([&](auto i) {
          av[i] = has_q && cst + qrow + i * PSTEP < N ? ld8_any<T>(qsrc[i], r - q * 8, q_end) : make_uint4(0, 0, 0, 0);
        });
      advance();
    }
  };
  auto deposit = [&]() {
    if constexpr (!VEC) {
      if (base) static_for<4>([&](auto i) { sts16<32 * i * ROWB>(in + wdst, wv[i]); });
      if constexpr (TR)
        if (has_q) static_for<NP>([&](auto i) { sts16<i * PSTEP * C::PITCH>(in + qdst, av[i]); });
      in = next(in);
    }
  };
  // !TR: Q through registers, since its words change places: word p of the 8
  // columns of lane t goes to tile p, place t
  uint4 qv[TR ? 1 : NP];
  auto load_q = [&](int st) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      qv[i] = has_q && qin[i] ? ld8<T, VEC>(qsrc[i], 0, N - n0 - st * SK - q * 8, q_end) : make_uint4(0, 0, 0, 0);
      qsrc[i] += SK;
    }
  };
  auto put_q = [&](uint32_t to) {
    if (has_q)
      static_for<NP>([&](auto i) {
        asm volatile("st.shared.u32 [%0+%5], %1;\n\tst.shared.u32 [%0+%5+16], %2;\n\tst.shared.u32 [%0+%5+32], %3;\n\t"
                     "st.shared.u32 [%0+%5+48], %4;" ::"r"(to + qdst), "r"(qv[i].x), "r"(qv[i].y), "r"(qv[i].z), "r"(qv[i].w),
                     "n"(i * PSTEP * C::PITCH)
                     : "memory");
      });
  };
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < STG - 1; ++i) {
      if (i < nst) stage();
      cp_async_commit();
    }
  } else {
    request();
    deposit();
    if (nst > 1) request();
  }
  if constexpr (!TR) load_q(0);
  // mid: rows m, m + 8; values 4t .. 4t + 3 of each 16 ranks, split into hi + lo
  const int m = warp * 16 + g;
  const int64_t ra = m < count ? rows[m] : -1, rb = m + 8 < count ? rows[m + 8] : -1;
  pdl_wait_previous();  // mid comes from the kernel before; all else was there when that one began
  float fac[2];
  uint2 ha[RP / 16][2], la[RP / 16][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t row = h ? rb : ra;
    float4 v[RP / 16];
    float mx = 0.f;
#pragma unroll
    for (int k = 0; k < RP / 16; ++k) {
      v[k] = row >= 0 ? *reinterpret_cast<const float4*>(a.mid + row * a.mp + 16 * k + 4 * t)
                      : make_float4(0.f, 0.f, 0.f, 0.f);
      const float f[4] = {fabsf(v[k].x), fabsf(v[k].y), fabsf(v[k].z), fabsf(v[k].w)};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (f[e] < INFINITY) mx = fmaxf(mx, f[e]);
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    float inv;
    scale_of<T>(mx, fac[h], inv);
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
  T* ya = y + (ra >= 0 ? ra : 0) * N + n0 + 8 * t;
  T* yb = y + (rb >= 0 ? rb : 0) * N + n0 + 8 * t;
  int left = N - n0 - 8 * t;  // columns of the row from this lane's on
  // where this lane reads a stage: base's pieces of either 32 columns, and Q's fragments
  const uint32_t boff[2] = {(uint32_t)(m * ROWB + ((t ^ swz(g)) << 4)), (uint32_t)(m * ROWB + (((4 + t) ^ swz(g)) << 4))};
  const uint32_t foff = WIDE + (TR ? g * C::PITCH + 8 * t
                                   : (8 * ((lane >> 3) & 1) + (lane & 7)) * C::PITCH + (lane >> 4) * 16);
  uint32_t slot = smem;
  for (int st = 0; st < nst; ++st) {
    if constexpr (!TR) put_q(slot);  // this slot's last readers are two barriers back
    cp_async_wait<STG - 2>();
    __syncthreads();
    if constexpr (VEC) {
      if (st + STG - 1 < nst) stage();
      cp_async_commit();
    } else {
      if (st + 1 < nst) deposit();
      if (st + 2 < nst) request();
    }
    if constexpr (!TR) {
      if (st + 1 < nst) load_q(st + 1);
    }
    if (16 * warp < count) {
      static_for<2>([&](auto w) {  // 32 columns each
        float c[4][4] = {};
        static_for<RP / 16>([&](auto k) {
          uint32_t b[8];
          if constexpr (!TR) {
            ldmatrix_x4_trans<16 * k * C::PITCH + w * 64>(b, slot + foff);
            ldmatrix_x4_trans<16 * k * C::PITCH + w * 64 + 32>(b + 4, slot + foff);
          } else {
            static_for<4>([&](auto p) {
              const uint2 u = lds8<(32 * w + 8 * p) * C::PITCH + 32 * k>(slot + foff);
              b[2 * p] = u.x;
              b[2 * p + 1] = u.y;
            });
          }
#pragma unroll
          for (int p = 0; p < 4; ++p)
            mma16816<T>(c[p], ha[k][0].x, ha[k][1].x, ha[k][0].y, ha[k][1].y, b[2 * p], b[2 * p + 1]);
#pragma unroll
          for (int p = 0; p < 4; ++p)
            mma16816<T>(c[p], la[k][0].x, la[k][1].x, la[k][0].y, la[k][1].y, b[2 * p], b[2 * p + 1]);
        });
        uint4 ua = make_uint4(0, 0, 0, 0), ub = ua;
        if (base) {
          ua = lds16<0>(slot + boff[w]);
          ub = lds16<8 * ROWB>(slot + boff[w]);
        }
        if (ra >= 0) st8<T, VEC>(ya + 32 * w, left - 32 * w, add8<T>(ua, c, 0, fac[0]));
        if (rb >= 0) st8<T, VEC>(yb + 32 * w, left - 32 * w, add8<T>(ub, c, 2, fac[1]));
      });
    }
    ya += SK;
    yb += SK;
    left -= SK;
    slot = next(slot);
  }
}

// Launches a shrink kernel (kern<<<tiles x S>>>(args, S)) with the split of the
// contraction that has the shortest estimate: rounds of co-resident clusters x
// (stages of a part + 5 for start, joining and ending), for about half a tile
// more than T / 128 with each adapter that ends inside one.
// `fit`: resident_clusters of the kernel, `per`: times as many really fit.
template <class Kern>
int launch_split(Kern kern, int threads, int smem, const Args& a, cudaStream_t st, const int* fit, int per) {
  const int64_t whole = (a.T + ROWS_L - 1) / ROWS_L, tiles = whole + std::min(a.L, whole) / 2, nst = (a.D + SK - 1) / SK;
  int S = 1;
  int64_t best = INT64_MAX;
  for (int s = 1; s <= MAX_SPLIT && (s == 1 || nst >= 4 * s); ++s) {
    const int64_t at_once = (int64_t)per * fit[s], cost = ((tiles + at_once - 1) / at_once) * ((nst + s - 1) / s + 5);
    if (cost < best) best = cost, S = s;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.lay.max_large * S));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a, S), "lora shrink launch");
}

int launch_tiles(const Args& a, int dtype, bool tr, cudaStream_t st) {
  const bool vec = aligned_widths(a.D, a.N, a.r);
  return by_type(dtype, a.r, vec, [&](auto tc, auto rc, auto vc) -> int {
    using T = decltype(tc);
    constexpr int RP = decltype(rc)::value;
    constexpr bool VEC = decltype(vc)::value;
    constexpr int FEW = expand_ctas(RP, VEC, true), MANY = expand_ctas(RP, VEC, false);
    const bool few = a.T <= FEW_TOKENS * a.L;
    ExpandFn expand =
        tr ? (few ? lora_expand_tile_kernel<T, RP, true, VEC, FEW> : lora_expand_tile_kernel<T, RP, true, VEC, MANY>)
           : (few ? lora_expand_tile_kernel<T, RP, false, VEC, FEW> : lora_expand_tile_kernel<T, RP, false, VEC, MANY>);
    int smem_e = tr ? (few ? ExpandCfg<RP, true, FEW>::SMEM : ExpandCfg<RP, true, MANY>::SMEM)
                    : (few ? ExpandCfg<RP, false, FEW>::SMEM : ExpandCfg<RP, false, MANY>::SMEM);
    int per_e = 1;
    if (VEC && RP == 64 && a.T > TC_TOKENS * a.L && a.T * a.N >= TC_VALUES) {
      expand = reinterpret_cast<ExpandFn>(const_cast<void*>(expand_tc_kernel(dtype, tr)));
      smem_e = EXPAND_TC_SMEM;
      per_e = 2;  // see the shrink below
    }
    // expand: the number of 64-column steps per CTA with the shortest estimate (start: 2 steps)
    int status = allow_smem((const void*)expand, smem_e, "cudaFuncSetAttribute(lora expand)");
    if (status) return status;
    const int64_t whole = (a.T + ROWS_L - 1) / ROWS_L, tiles = whole + std::min(a.L, whole) / 2;
    const int64_t nsteps = (a.N + SK - 1) / SK, slots = per_e * resident_clusters((const void*)expand, THREADS, smem_e)[1];
    int steps = 2;
    int64_t best = INT64_MAX;
    for (int s = 2; s <= 16; ++s) {
      const int64_t cost = ((tiles * ((nsteps + s - 1) / s) + slots - 1) / slots) * (s + 2);
      if (cost < best) best = cost, steps = s;
    }
    const int parts = (int)((nsteps + steps - 1) / steps);
    const int64_t blocks = a.lay.max_large * parts;
    if (blocks > (1ll << 31) - 1) return fail(B200Q_ERR_SHAPE, "lora_apply: size too large");
    if constexpr (VEC && RP == 64) {
      // tensor memory instead of register fragments from rank 33 on: D=14336,
      // r=64, 4096 tokens 53 us with it and 61 us without (shrink and expand);
      // D=4096 and N=14336, r=16, 8192 tokens, forward and backward 253 and 250
      const void* kern = shrink_tc_kernel(dtype, tr);
      if ((status = allow_smem(kern, SHRINK_TC_SMEM, "cudaFuncSetAttribute(lora shrink)"))) return status;
      // the occupancy query counts a kernel with tensor memory once per SM; its 64 of 512 columns and its shared memory
      // let two share one
      status = launch_split(reinterpret_cast<ShrinkFn>(const_cast<void*>(kern)), SHRINK_TC_THREADS, SHRINK_TC_SMEM, a, st,
                            resident_clusters(kern, SHRINK_TC_THREADS, SHRINK_TC_SMEM), 2);
    } else {
      auto shrink = tr ? lora_shrink_tile_kernel<T, RP, true, VEC> : lora_shrink_tile_kernel<T, RP, false, VEC>;
      const int smem_s = tr ? ShrinkCfg<RP, true, VEC>::SMEM : ShrinkCfg<RP, false, VEC>::SMEM;
      if ((status = allow_smem((const void*)shrink, smem_s, "cudaFuncSetAttribute(lora shrink)"))) return status;
      status = launch_split(shrink, THREADS, smem_s, a, st, resident_clusters((const void*)shrink, THREADS, smem_s), 1);
    }
    if (status || !a.y) return status;  // no y: mid alone was asked for
    // the expand kernel's start overlaps the shrink kernel's end
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = (size_t)smem_e;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return check_cuda(cudaLaunchKernelEx(&cfg, expand, a, parts, steps), "lora expand launch");
  });
}

}  // namespace lora
}  // namespace b200q
