// Shared by the operators on a key/value cache (kv_rows.cu, kv_search.cu, kv_attend.cu): where the rows of a call stand, 16-bit
// and 8-bit values, warp-wide matrix products, launches.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "internal.h"

namespace fv {

// ---------------------------------------------------------------------------------------------
// host side
int kv_check(const fv_kv* kv, const fv_kv_batch* batch, const char* who);  // kv_rows.cu
inline bool kv_aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
// bytes of a row of a head, and of its scales
inline size_t kv_row_bytes(const fv_kv* kv) { return kv->kind == FV_KV_SAME ? 2 * kv->dim : kv->kind == FV_KV_INT4X32 ? kv->dim / 2 : kv->dim; }
inline size_t kv_scale_bytes(const fv_kv* kv) { return kv->kind == FV_KV_SAME ? 0 : kv->kind == FV_KV_INT4X32 ? kv->dim / 32 : 4; }

// Returns fn<type, kind, dim>(...) for what the cache holds.  kv_check has looked at the three.
#define FV_KV_DISPATCH(kv, fn, ...)                                                                                     \
  do {                                                                                                                  \
    const int _d = int((kv)->dim), _k = (kv)->kind;                                                                     \
    if ((kv)->dtype == FV_KV_BF16) FV_KV_KIND_(__nv_bfloat16, fn, __VA_ARGS__) else FV_KV_KIND_(__half, fn, __VA_ARGS__) \
  } while (0)
#define FV_KV_KIND_(T, fn, ...)                                                     \
  {                                                                                 \
    if (_k == FV_KV_SAME) FV_KV_DIM_(T, FV_KV_SAME, fn, __VA_ARGS__)                \
    else if (_k == FV_KV_INT8) FV_KV_DIM_(T, FV_KV_INT8, fn, __VA_ARGS__)           \
    else if (_k == FV_KV_E4M3) FV_KV_DIM_(T, FV_KV_E4M3, fn, __VA_ARGS__)           \
    else FV_KV_DIM_(T, FV_KV_INT4X32, fn, __VA_ARGS__)                              \
  }
#define FV_KV_DIM_(T, K, fn, ...)                      \
  {                                                    \
    if (_d == 64) return fn<T, K, 64>(__VA_ARGS__);    \
    if (_d == 96) return fn<T, K, 96>(__VA_ARGS__);    \
    return fn<T, K, 128>(__VA_ARGS__);                 \
  }

// Allows a kernel its dynamic shared memory on the current device, once for each device.  Without that it gets 48 KB, its static
// shared memory (up to 18 KB here) among them.
template <auto* kern>
int kv_allow_smem(int device, size_t bytes) {
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = 1ull << (device & 63);
  if (bytes <= 24 * 1024 || (device < 64 && (done.load(std::memory_order_acquire) & bit))) return FV_OK;
  cudaFuncAttributes at;
  FV_CUDA(cudaFuncGetAttributes(&at, kern));
  FV_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - int(at.sharedSizeBytes)));
  done.fetch_or(bit, std::memory_order_release);
  return FV_OK;
}

#ifdef __CUDACC__
// ---------------------------------------------------------------------------------------------
// the batch, as kernels take it
struct KvBatch {
  const int32_t* table;
  size_t table_stride;
  int table_width;
  const int32_t* lens;
  const int32_t* cu;
  int nseq;
  int rows;
  unsigned pages;
  int page_shift;

  __device__ __forceinline__ int cu_at(int b) const {  // rows before sequence b, never outside of the call's tensors
    return cu ? min(max(__ldg(cu + b), 0), rows) : min(b, rows);
  }
  // rows of sequence b.  Less than none are none: a position, n rows before it, stays within 32 bits.
  __device__ __forceinline__ int len(int b) const { return max(__ldg(lens + b), 0); }
  // page of block j of sequence b, or -1
  __device__ __forceinline__ int page(int b, int j) const {
    if (j < 0 || j >= table_width) return -1;
    const int p = __ldg(table + size_t(b) * table_stride + j);
    return unsigned(p) < pages ? p : -1;
  }
};
inline KvBatch kv_batch(const fv_kv* kv, const fv_kv_batch* b) {
  return KvBatch{b->table, b->table_stride, int(b->table_width), b->lens, b->cu, int(b->nseq), int(b->rows),
                 unsigned(kv->pages), __builtin_ctz(kv->page_size)};
}

// The sequence whose work holds item `i` when that of sequence b begins at item cu[b] / per + extra * b: the largest such b.
// Items are handed out without a prefix sum over the sequences that way: floor(x) + floor(y) <= floor(x + y), so a
// sequence of n rows has n / per + extra items at least to itself.  Whole warps call it; 32 sequences are looked at at once.
__device__ __forceinline__ int kv_find(const KvBatch& m, int i, int per, int extra) {
  int lo = 0, n = m.nseq;  // the answer is in lo .. lo + n - 1
  const int lane = lane_id();
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int b = lo + lane * step;
    const bool before = lane * step < n && unsigned(m.cu_at(b)) / unsigned(per) + extra * b <= unsigned(i);
    const int w = 31 - __clz(int(__ballot_sync(FV_FULL, before)) | 1);  // lane 0's begins at item 0
    lo += w * step;
    n = min(step, n - w * step);
  }
  return lo;
}

// ---------------------------------------------------------------------------------------------
// 16-bit values in pairs
template <class T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 to_float(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t from_float(float lo, float hi) {  // to nearest even
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
  }
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ float2 to_float(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t from_float(float lo, float hi) {
    uint32_t w;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
  }
};

// zeros in the halves that are not finite
template <class T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u;
  return w & ~__vcmpeq2(w & e, e);
}
// The smaller and the larger of each half; none of them a NaN.
template <class T>
__device__ __forceinline__ uint32_t min2(uint32_t x, uint32_t y) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  else asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}
template <class T>
__device__ __forceinline__ uint32_t max2(uint32_t x, uint32_t y) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  else asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}

// ---------------------------------------------------------------------------------------------
// 8-bit values.  A code is top * x / most rounded to nearest even, and most, x of 8 or 11 significant bits make the quotient
// either the border of two codes exactly or further from it than half a step of 32 bits: with a correctly rounded division
// the code is that of the true quotient.  Values beyond 2^64 or below 2^-64 are brought nearer to 1 first, by a power of two,
// for top * x and 1 / most to stay finite.
__device__ __forceinline__ float kv_down(float most) { return most > 0x1p64f ? 0x1p-32f : most < 0x1p-64f ? 0x1p64f : 1.0f; }
__device__ __forceinline__ bool kv_finite(float x) { return fabsf(x) < INFINITY; }

// num / den to the nearest whole number, halves to the even one, from inv = 1 / den to within a unit in the last place: num and
// den have at most 21 and 14 significant bits and |num / den| <= 127, so num * inv leads to one of the two nearest, and what that
// leaves of num is exact and says whether the quotient is a half.  A third of the steps of a division.
__device__ __forceinline__ int kv_whole(float num, float den, float inv) {
  const int r = __float2int_rn(num * inv);
  const float left = __fmaf_rn(-float(r), den, num);
  const bool half = fabsf(left) + fabsf(left) == den;
  return half && (r & 1) ? (left > 0.f ? r + 1 : r - 1) : r;
}

template <int KIND>
struct Eight;
template <>
struct Eight<FV_KV_INT8> {
  static constexpr float top = 127.0f;
  // four quotients num / den to four codes, inv = 1 / den
  static __device__ __forceinline__ uint32_t pack(const float* num, float den, float inv) {
    uint32_t hi, w;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(kv_whole(num[3], den, inv)), "r"(kv_whole(num[2], den, inv)));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(w) : "r"(kv_whole(num[1], den, inv)), "r"(kv_whole(num[0], den, inv)), "r"(hi));
    return w;
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float* y) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = float(int32_t(w << (24 - 8 * i)) >> 24);
  }
};
template <>
struct Eight<FV_KV_E4M3> {
  static constexpr float top = 448.0f;
  // The border of two codes has five significant bits.  num * inv is off by less than 2^-22 of itself and a quotient that is
  // no border by more than 2^-20 from the next one: what is nearer than that to a number of eight bits is that number.
  static __device__ __forceinline__ float quotient(float num, float inv) {
    const float y = num * inv, t = __uint_as_float((__float_as_uint(y) + 0x8000u) & 0xFFFF0000u);
    return fabsf(y - t) < fabsf(t) * 0x1p-20f ? t : y;
  }
  static __device__ __forceinline__ uint32_t pack(const float* num, float, float inv) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = quotient(num[i], inv);
    uint16_t a, b;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a) : "f"(y[1]), "f"(y[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(y[3]), "f"(y[2]));
    return uint32_t(a) | uint32_t(b) << 16;
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float* y) {
    uint32_t a, b;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"(uint16_t(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"(uint16_t(w >> 16)));
    const float2 x = Pair<__half>::to_float(a), z = Pair<__half>::to_float(b);
    y[0] = x.x, y[1] = x.y, y[2] = z.x, y[3] = z.y;
  }
};

// ---------------------------------------------------------------------------------------------
// 4-bit values.  A group of 32 neighbouring components has a scale of 5 exponent and 3 mantissa bits without a sign, fp16's upper byte
// moved down by one bit, so fp16 = byte << 7: the smallest one that 7 times is not below any component, at most 9216 (7 times it is
// in fp16's range).  code = rn(x / scale) + 8, from 1 to 15.  scale * (code - 8) has seven significant bits at most and no bit below 2^-17: it is
// exact in fp16, and in bf16.  A quotient of 11 and 4 bits is the border of two codes exactly or further from it than half a
// step of 32 bits, as is a seventh of 11 bits from a scale.
// A row is 8 * groups pieces of 16 bits, four neighbouring components each, the lowest in the lowest bits: first the groups' first
// pieces, then their second ones, and so on.  A quarter of a row has eight neighbours of every group that way, an eighth has four.
struct Four {
  static constexpr float LARGEST = 9216.f;
  static constexpr uint32_t NAN_SCALE = 255;
  // Its byte, of a finite `most`.  A seventh of 11 bits is a scale or further from one than 2^-14 of itself: what is made smaller by 2^-20, and
  // is off by less than that, is rounded up to the same.
  static __device__ __forceinline__ uint32_t scale_of(float most) {
    const float t = most * 0.14285700f;
    if (t < 0x1p-14f) return uint32_t(ceilf(t * 0x1p17f));
    return (min(__float_as_uint(t) + 0xFFFFFu, __float_as_uint(LARGEST)) >> 20) - ((127 - 15) << 3);
  }
  static __device__ __forceinline__ float value(uint32_t byte) { return __half2float(__ushort_as_half(uint16_t(byte << 7))); }
  // Eight codes of neighbouring components, the first in the lowest bits, inv = 1 / scale to within 2^-22 of itself.  A quotient x / scale of
  // 11 and 4 bits from 1/2 on is half a whole number or 2^-13 and more from it, so it is rounded to a multiple of 2^-14 first and then
  // to a whole number, halves to the even one: both by adding a number whose last place that is.  The sum's bits are a constant and
  // the code, and the constants of all eight are taken off together.
  static __device__ __forceinline__ uint32_t pack(const float* x, float inv) {
    uint32_t w = 0u - (0x4B400000u + (0x4B400000u << 4) + (0x4B400000u << 8));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = (x[i] * inv + 0x1.8p9f) - 0x1.8p9f;
      w += __float_as_uint(q + (0x1.8p23f + 8.f)) << (4 * i);
    }
    return w;
  }
  // the eight codes of group g in the NG words of a quarter of a row
  template <int NG>
  static __device__ __forceinline__ uint32_t group(const uint32_t* w, int g) {
    return __byte_perm(w[g / 2], w[(NG + g) / 2], (g & 1 ? 0x32 : 0x10) | ((NG + g) & 1 ? 0x7600 : 0x5400));
  }
  // Eight codes to the pairs (0, 4), (1, 5), (2, 6), (3, 7) of fp16, exactly: a code is added to 1024, or 16 times it to 1024, by its place.
  // (One instruction masks and adds where one of its two constants is in a register; the compiler, which knows both, would take two.)
  static __device__ __forceinline__ uint32_t magic(uint32_t x) {
    uint32_t y;
    asm volatile("mov.b32 %0, %1;" : "=r"(y) : "r"(x));
    return y;
  }
  static __device__ __forceinline__ void halves(uint32_t w, uint32_t* to, uint32_t by_1024, uint32_t by_64) {  // magic(0x64006400), magic(0x54005400)
    const __half2 low = __half2half2(__ushort_as_half(0x6408)), high = __half2half2(__ushort_as_half(0x5480));  // 1032, 72
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t x0, x1;
      asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(x0) : "r"(i ? w >> 8 : w), "r"(by_1024));
      asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(x1) : "r"(i ? w >> 8 : w), "r"(by_64));
      const __half2 u = __hsub2(*reinterpret_cast<const __half2*>(&x0), low), v = __hsub2(*reinterpret_cast<const __half2*>(&x1), high);
      to[2 * i] = *reinterpret_cast<const uint32_t*>(&u), to[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
};

// ---------------------------------------------------------------------------------------------
// attention (kv_attend.cu, kv_prompt.cu)
struct KvAttend {
  const unsigned char* q;
  size_t q_row, q_head;  // bytes
  int heads, group;
  const int32_t* blocks;  // [rows][heads][k], or NULL: all of them
  int k;
  float scale;  // of the products, times log2(e)
  const unsigned char *kp, *vp;
  const float *k_scale, *v_scale;
  unsigned char* out;
  float* lse;
};

// c += a b: 16 x 16 by 16 x 8, sums in 32 bits
template <class T>
__device__ __forceinline__ void mma_16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a b in fp16
__device__ __forceinline__ void mma_16_of(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// Four 8-bit codes as two pairs of fp16, exactly: (0, 1) and (2, 3).
template <int KIND>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& a, uint32_t& b) {
  if constexpr (KIND == FV_KV_E4M3) {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"(uint16_t(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"(uint16_t(w >> 16)));
  } else {  // code + 128 in the low byte of 1024 .. 1279, whose step in fp16 is 1
    w ^= 0x80808080u;
    const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    __half2 u = __hsub2(*reinterpret_cast<const __half2*>(&x), off), v = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
    a = *reinterpret_cast<uint32_t*>(&u), b = *reinterpret_cast<uint32_t*>(&v);
  }
}
__device__ __forceinline__ float exp2_of(float x) {  // to 2 units in the last place; 0 for -inf, NaN for NaN
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // of 8 x 8 values of 16 bits, a row on four lanes
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// The power of two that brings numbers of at most `most` below 2^14, so that they fit fp16 with all their bits.
__device__ __forceinline__ float half_factor(float most) {
  const int e = int(__float_as_uint(most) >> 23);  // biased; 255: not finite
  if (e == 255 || most == 0.f) return 1.f;
  return __uint_as_float(uint32_t(min(max(127 + 13 - (e - 127), 1), 254)) << 23);
}

#endif  // __CUDACC__

}  // namespace fv
