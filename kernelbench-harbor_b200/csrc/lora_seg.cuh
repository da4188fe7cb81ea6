// Shared pieces of the multi-adapter kernels (lora_plan.cu, lora_small.cu,
// lora_tiles.cu, lora_shrink_tc.cu, lora_grads.cu): adapters of many requests beside one shared
// projection,
//   y[t]  = base[t] + s[id_t] (x[t] . A[id_t]) . B[id_t]
//   dx[t] = base[t] + s[id_t] (dy[t] . B[id_t]^T) . A[id_t]^T
// Both are "shrink" (contract a wide row with a thin matrix, P) and "expand"
// (times a thin matrix, Q, added to a wide row); the backward form takes B and
// A transposed (TR).  Tokens are grouped by adapter (the plan), so a tile of
// rows shares one adapter and the products run on the tensor cores; mid, the
// row between the two (s included), stays in fp32.
//
// Wide rows are read and written once and take 2 r flops per value (r <= 64), so
// memory is the bound.  Most products use mma.sync m16n8k16, whose register
// fragments fit wide rows: of the contraction index, any order serves that both
// operands share, so a thread takes 8 consecutive values of a row (one 16-byte
// load) as its parts of two k16 steps; of the output columns, the order is
// chosen so that a thread ends with 8 consecutive ones.  From rank 33 on the
// fragments of P cost more than the rows, and shrink runs on tcgen05.
#pragma once
#include <type_traits>
#include <utility>

#include "common.cuh"

namespace b200q {
namespace lora {

constexpr int MAX_RANK = 64;
constexpr int MAX_ADAPTERS = 1023;
constexpr int64_t MAX_TOKENS = 1ll << 24;
constexpr int ROWS_S = 16, ROWS_L = 128;  // rows of a small / large tile
constexpr int THREADS = 256, WARPS = THREADS / 32;

// ------------------------------------------------------------------ plan layout (int32 words)
//   [0] small tiles, [1] large tiles, [2..8) unused
//   seg_off [L + 2]: adapter a's rows are order[seg_off[a] .. seg_off[a + 1]);
//                    segment L holds the tokens without an adapter
//   order [T]: token indices, ascending within a segment
//   tiles_s, tiles_l: {adapter or -1, first position in order, rows, 0} each
struct PlanLayout {
  int64_t seg, order, small, large, words, max_small, max_large;
};

inline int64_t max_tiles(int64_t T, int64_t L, int64_t rows) {
  const int64_t n = T / rows + L + 1;
  return n < T ? n : T;
}

inline PlanLayout plan_layout(int64_t T, int64_t L) {
  PlanLayout p;
  auto up4 = [](int64_t v) { return (v + 3) / 4 * 4; };
  p.max_small = max_tiles(T, L, ROWS_S);
  p.max_large = max_tiles(T, L, ROWS_L);
  p.seg = 8;
  p.order = up4(p.seg + L + 2);
  p.small = up4(p.order + T);
  p.large = p.small + 4 * p.max_small;
  p.words = p.large + 4 * p.max_large;
  return p;
}

// Row pitch of mid: the rank rounded up to a multiple of the MMA's 16 that the kernels are built for.
inline int mid_pitch(int64_t r) { return r <= 16 ? 16 : r <= 32 ? 32 : 64; }

// ------------------------------------------------------------------ element types
template <class T>
__device__ __forceinline__ float tf(T v);
template <>
__device__ __forceinline__ float tf<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float tf<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T ft(float v);
template <>
__device__ __forceinline__ __half ft<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 ft<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T>
__device__ __forceinline__ uint32_t pack2(T a, T b) {
  return (uint32_t) * reinterpret_cast<uint16_t*>(&a) | ((uint32_t) * reinterpret_cast<uint16_t*>(&b) << 16);
}

template <class T>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
  T v[2];
  *reinterpret_cast<uint32_t*>(v) = w;
  a = tf<T>(v[0]);
  b = tf<T>(v[1]);
}

// v = hi + lo to twice the type's significand: the products of mid with the
// thin matrix keep a value to 2^-16 (bf16) or 2^-22 (fp16) of itself, in fp16 at
// least to 2^-39 of the largest value that is scaled together with it (scale_of).
// An infinity or NaN stays in hi alone.
template <class T>
__device__ __forceinline__ void split(float v, T& hi, T& lo) {
  hi = ft<T>(v);
  const float rest = v - tf<T>(hi);
  lo = ft<T>(fabsf(rest) < INFINITY ? rest : 0.f);
}

// Power-of-two factor for values up to |v| (finite) and its inverse: fp16 has 5
// exponent bits, and mid may leave their range.  fp16: |v * inv| lies in [2^14,
// 2^15), the last binade but one, so that the smallest step of the halves, 2^-24,
// is 2^-39 of the largest value; the sums of products (below 2^31 each) are
// fp32.  bf16, with fp32's exponents: in [1, 2).  Less for the tiniest v, whose
// factor would be subnormal.
template <class T>
__device__ __forceinline__ void scale_of(float v, float& fac, float& inv) {
  constexpr uint32_t UP = std::is_same<T, __half>::value ? 14 : 0;
  const uint32_t e = min(max((__float_as_uint(v) >> 23) & 0xffu, UP + 1), UP ? 254u : 253u) - UP;
  fac = __uint_as_float(e << 23);
  inv = __uint_as_float((254 - e) << 23);
}

template <class T>
__device__ __forceinline__ void mma16816(float* d, const uint32_t a0, const uint32_t a1, const uint32_t a2,
                                         const uint32_t a3, const uint32_t b0, const uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float* d, const uint32_t a0, const uint32_t a1, const uint32_t a2,
                                                 const uint32_t a3, const uint32_t b0, const uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* d, const uint32_t a0, const uint32_t a1,
                                                        const uint32_t a2, const uint32_t a3, const uint32_t b0,
                                                        const uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Shared-memory accesses at a register plus an immediate: the loops over stages
// are bound by the length of a warp's instruction chain, so no address is
// computed in them that a constant can hold.
template <int OFF = 0>
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4+%5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr), "n"(OFF)
               : "memory");
}
template <int OFF = 0>
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr), "n"(OFF)
               : "memory");
  return v;
}
template <int OFF = 0>
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2+%3];" : "=r"(v.x), "=r"(v.y) : "r"(addr), "n"(OFF) : "memory");
  return v;
}

// f(0), ..., f(N - 1) with the index as a compile-time value
template <int V>
struct Index {
  __host__ __device__ constexpr operator int() const { return V; }
};
template <int... I, class F>
__device__ __forceinline__ void static_for_impl(std::integer_sequence<int, I...>, F&& f) {
  (f(Index<I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_impl(std::make_integer_sequence<int, N>{}, f);
}

// 16 bytes to shared memory, `bytes` of them (16 or 0) from src and zeros for the rest
template <int OFF = 0>
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0+%3], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(OFF) : "memory");
}
// The same for the wide rows: a row's next 128 bytes, the next stage's, come to L2 along with these.
template <int OFF = 0>
__device__ __forceinline__ void cp_async16_ahead(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0+%3], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(OFF) : "memory");
}
template <int OFF = 0>
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0+%3], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(OFF) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------------------------ rows of any width
// VEC: widths and pointers let every piece of a wide row be one aligned 16-byte
// access (D % 8 == 0, N % 8 == 0, and r % 4 == 0, so that A's rows come in
// 8-byte pieces at least).  Otherwise a row may start at any value: 8 values are
// cut out of the one or two aligned 16-byte blocks that hold them, or read one
// by one where such a block would reach past the tensor's end.

// RO: through the read-only path.  Not for base, which may be y itself: another
// CTA may be writing a neighbour's values in the same block (they are dropped).
template <bool RO>
__device__ __forceinline__ uint4 ld16(const uint4* p) {
  if constexpr (RO)
    return __ldg(p);
  else
    return *p;
}

// Up to 8 values from p on, zeros past `left`; `end`: the tensor's end.
template <class T, bool RO = true>
__device__ __forceinline__ uint4 ld8_any(const T* p, int left, const T* end) {
  if (left <= 0) return make_uint4(0, 0, 0, 0);
  const uintptr_t at = reinterpret_cast<uintptr_t>(p), lo = at & ~(uintptr_t)15;
  const int shift = (int)(at & 15);
  const bool two = shift && 2 * min(left, 8) > 16 - shift;
  uint32_t w[8];
  if (lo + (two ? 32 : 16) <= reinterpret_cast<uintptr_t>(end)) {
    const uint4 a = ld16<RO>(reinterpret_cast<const uint4*>(lo));
    const uint4 b = two ? ld16<RO>(reinterpret_cast<const uint4*>(lo) + 1) : make_uint4(0, 0, 0, 0);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    if (shift & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (shift & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (shift & 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (left <= 2 * i) w[i] = 0;
      if (left == 2 * i + 1) w[i] &= 0xffffu;
    }
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (2 * i < left ? (uint32_t)h[2 * i] : 0) | (2 * i + 1 < left ? (uint32_t)h[2 * i + 1] << 16 : 0);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Values [k, k + 8) of a row of K, zeros past its end (VEC: k a multiple of 8, all in or all out).
template <class T, bool VEC, bool RO = true>
__device__ __forceinline__ uint4 ld8(const T* row, int k, int K, const T* end) {
  if constexpr (VEC)
    return k < K ? ld16<RO>(reinterpret_cast<const uint4*>(row + k)) : make_uint4(0, 0, 0, 0);
  else
    return ld8_any<T, RO>(row + k, K - k, end);
}

template <class T, bool VEC>
__device__ __forceinline__ uint2 ld4(const T* row, int k, int K) {
  if constexpr (VEC) {
    return k < K ? __ldg(reinterpret_cast<const uint2*>(row + k)) : make_uint2(0, 0);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t a = k + 2 * i < K ? reinterpret_cast<const uint16_t*>(row)[k + 2 * i] : 0;
      const uint32_t b = k + 2 * i + 1 < K ? reinterpret_cast<const uint16_t*>(row)[k + 2 * i + 1] : 0;
      w[i] = a | (b << 16);
    }
    return make_uint2(w[0], w[1]);
  }
}

// 8 values to p, as many of them as are `left` in the row; otherwise in aligned pairs.
template <class T, bool VEC>
__device__ __forceinline__ void st8(T* p, int left, const uint4 v) {
  if constexpr (VEC) {
    if (left > 0) *reinterpret_cast<uint4*>(p) = v;
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint16_t* h = reinterpret_cast<uint16_t*>(p);
    if (left >= 8) {
      if (reinterpret_cast<uintptr_t>(p) & 2) {
        h[0] = (uint16_t)w[0];
#pragma unroll
        for (int i = 0; i < 3; ++i) *reinterpret_cast<uint32_t*>(h + 1 + 2 * i) = __funnelshift_r(w[i], w[i + 1], 16);
        h[7] = (uint16_t)(w[3] >> 16);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(h + 2 * i) = w[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) h[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

template <int OFF = 0>
__device__ __forceinline__ void sts16(uint32_t dst, const uint4 v) {
  asm volatile("st.shared.v4.u32 [%0+%5], {%1,%2,%3,%4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "n"(OFF) : "memory");
}

// Up to 16 aligned bytes of a row to shared memory, asynchronously, zeros for the
// rest (VEC).  `left`: values of the row from the piece on; `any`: an address
// that may be read.  halves: the row is 8-byte aligned only (A where r % 8 == 4).
template <bool WIDE_ROW, int OFF, class T>
__device__ __forceinline__ void copy16(uint32_t dst, const T* piece, int left, bool in, const T* any, bool halves = false) {
  const bool a = in && left > 0;
  if (WIDE_ROW) {
    cp_async16_ahead<OFF>(dst, a ? piece : any, a ? 16 : 0);
  } else if (!halves) {
    cp_async16<OFF>(dst, a ? piece : any, a ? 16 : 0);
  } else {
    const bool b = in && left > 4;
    cp_async8<OFF>(dst, a ? piece : any, a ? 8 : 0);
    cp_async8<OFF + 8>(dst, b ? piece + 4 : any, b ? 8 : 0);
  }
}

// base + fac * c for the 8 consecutive columns of one row: c[p][h], c[p][h + 1] are columns 2p, 2p + 1
template <class T>
__device__ __forceinline__ uint4 add8(const uint4 b, const float (*c)[4], int h, float fac) {
  const uint32_t w[4] = {b.x, b.y, b.z, b.w};
  uint32_t o[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    float u, v;
    unpack2<T>(w[p], u, v);
    o[p] = pack2<T>(ft<T>(fmaf(fac, c[p][h], u)), ft<T>(fmaf(fac, c[p][h + 1], v)));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Position of contraction row k in shared memory so that one ldmatrix row group
// is what a fragment wants: with 8 consecutive k per thread (32-row groups)
__device__ __forceinline__ int row32(int k) { return (k & ~31) | (((k >> 1) & 3) << 3) | (((k >> 3) & 3) << 1) | (k & 1); }
// and the k at position p when a thread holds 4 consecutive k (16-row groups)
__device__ __forceinline__ int k_of_row16(int p) { return (p & ~15) | (((p >> 1) & 3) << 2) | (((p >> 3) & 1) << 1) | (p & 1); }

// Rows [0, count) of a tile without an adapter: y = base (zeros without one), columns [n0, n1).
template <class T, bool VEC>
__device__ __forceinline__ void copy_rows(const T* base, T* y, const int32_t* rows, int count, int N, int n0, int n1,
                                          const T* end) {
  if (base == y) return;
  // four pieces at a time: their rows are looked up, then loaded, then stored together
  const int g8 = (n1 - n0 + 7) / 8, total = count * g8;
  for (int i0 = threadIdx.x; i0 < total; i0 += 4 * THREADS) {
    size_t off[4];
    int n[4];
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = min(i0 + k * THREADS, total - 1);
      off[k] = (size_t)rows[i / g8] * N;
      n[k] = n0 + i % g8 * 8;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = base ? ld8<T, VEC>(base + off[k], n[k], N, end) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i0 + k * THREADS < total) st8<T, VEC>(y + off[k] + n[k], n1 - n[k], v[k]);
  }
}

struct Args {
  const void *x, *base, *P, *Q;
  const float* scaling;
  const int32_t* plan;
  PlanLayout lay;
  int D, N, r, mp;  // contraction width, output width, rank, mid pitch
  void* y;
  float* mid;
  int64_t T, L;
  int* status;  // or NULL
};

int launch_small(const Args& a, int dtype, bool tr, cudaStream_t st);
int launch_tiles(const Args& a, int dtype, bool tr, cudaStream_t st);

// lora_shrink_tc.cu: ranks 33 to 64, aligned rows
using ShrinkFn = void (*)(const Args, int);
constexpr int SHRINK_TC_THREADS = THREADS + 32, SHRINK_TC_SMEM = 4 * (128 * 128 + 64 * 128) + 1024;
const void* shrink_tc_kernel(int dtype, bool tr);

// lora_expand_tc.cu: the same ranks
using ExpandFn = void (*)(const Args, int, int);
constexpr int EXPAND_TC_SMEM = 2 * 128 * 128 + 3 * (128 * 128 + 64 * 128) + 1024;
const void* expand_tc_kernel(int dtype, bool tr);

inline bool aligned_widths(int64_t D, int64_t N, int64_t r) { return D % 8 == 0 && N % 8 == 0 && r % 4 == 0; }

// Calls f(type, rank, aligned) with compile-time values.
template <class F>
int by_type(int dtype, int64_t r, bool vec, F f) {
  auto rank = [&](auto t) {
    auto width = [&](auto rc) { return vec ? f(t, rc, std::true_type{}) : f(t, rc, std::false_type{}); };
    if (r <= 16) return width(std::integral_constant<int, 16>{});
    if (r <= 32) return width(std::integral_constant<int, 32>{});
    return width(std::integral_constant<int, 64>{});
  };
  return dtype == B200Q_DTYPE_FP16 ? rank(__half{}) : rank(__nv_bfloat16{});
}

}  // namespace lora
}  // namespace b200q
