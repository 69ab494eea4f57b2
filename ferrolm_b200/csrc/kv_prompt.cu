// Attention of many rows of a sequence (a prompt, or a piece of one) over blocks of a key/value cache, on the tensor cores.
//
// Every row has a list of blocks of its own, and neighbours have many of them in common.  A CTA has 128 queries (32 rows of a
// group of 4 heads, say) and goes once over the union of their lists in ascending order, 64 rows of the cache at a time:
//
//   S = Q K^T (128 x 64) and O += P V (128 x dim): tcgen05.mma from shared memory into tensor memory, P read from there
//   P = 2^(scale S - max): a thread to a query, which has a whole row of S in its registers: no exchange between lanes
//
// Warps 0-3 turn S into P, warp 4 issues the products, two warps bring keys and four values, each two tiles ahead at most; S has
// two places, so that the next one is worked out while this one becomes P.  P takes the place of its S.  Two CTAs share an SM.
//   4096 rows of 32 heads over all rows before them, bf16: 239 us, 575 TFLOP/s (0.35 of the measured rate); int8: 388 us
//   1687 rows over 16 of up to 266 blocks each: 208 us; 59 blocks on average are in the union of 32 rows' lists
// Where the time of the first goes, by clocks read in the kernel (at 1.8 GHz, which made it 277 us): a tile takes a warp of the weights 2800,
// with another CTA beside it.  1400 are from S to P, 350 to find the rows that it sees, 290 and 190 to load S and to store P, 150 to scale
// O, and 460 are waits, 290 of them for S and 170 for the values; the products take 256, the powers of two 512 (16 an SM and clock).
// A CTA begins in 7800 and ends in 3700, with 98000 between; and a place is empty for 65 of the 277 us: the longest CTAs come first within a
// head, but one head comes after the other, so the last one's are late.  Over int8 a tile takes 4700, 2400 of them from S to P.  With
// lists 2900 and 81 us of 234 without work: 432 CTAs go to 296 places.
// Warps with tiles of their own for every 8 rows, on mma.sync, whose lists have 36 blocks in common but which has a quarter of the
// rate, took 563 and 525 us.
//
// P is rounded to the values' type once, in bf16 to 2^-9 of each weight: the error of a result grows by a tenth of what its own
// rounding leaves (0.0018 of it against 64 bits, 0.0017 with weights in 32), where a second number for the rest would be a second product.
// A maximum that grows by less than a factor of 2 (fp16; 2^0.9 over 8 bits) or 256 (bf16) is left as it was: the weights stay within their type, and
// O, in tensor memory, need not be scaled as often.  Values that are not finite would reach rows that do not see them as
// 0 * inf: they are taken out on their way in, and added by the threads whose rows see them.  In 8 bits the codes become fp16,
// exactly, on their way in; a key's scale multiplies its column of S, a value's its weight (kv_attend.cu), relative to a
// power of two that follows the largest scale that the query itself has seen: what only the others of its tile see costs it no bits.
// The tile's scales come relative to the same for all that the CTA's queries see, which mostly is the query's own power too; a warp
// with a query for which it is not takes the scales as they are (as fast as one power for all: int8, dense 388 us, e4m3, lists 1160).
// In 4 bits code times scale goes into shared memory as fp16, exactly, and the rest is as over 16 bits, but that 2^7 stands for a weight of 1 and
// a maximum may lag behind by 2^8, for O to be scaled as seldom as in bf16 (2.5k rows over up to 6000, 195 GFLOP: 373 us, 428 with 2^14
// and a factor of 2; 396 for bf16 with whole sequences of 6000, 451 in 4 bits).  Taking the codes apart is 1400 of a tile's 3600 instructions.
#include <climits>

#include "kv.cuh"
#include "tc.cuh"

namespace fv {

namespace {

// warps 0-3: weights; 4: products; 6-7: keys; 8-11: values
enum { KV_PROMPT_COLS = 128, KV_PROMPT_THREADS = 384, KV_PROMPT_KEYS = 64, KV_PROMPT_VALUES = 128 };
// Registers: two CTAs share an SM, so a thread starts with 80; the threads of the weights take over what the others give up.
enum { KV_PROMPT_REGS = 80, KV_PROMPT_REGS_MORE = 128, KV_PROMPT_REGS_LESS = 56 };
static_assert(KV_PROMPT_REGS_MORE + 2 * KV_PROMPT_REGS_LESS <= 3 * KV_PROMPT_REGS, "more than a CTA starts with would never come");

// Rows have one scale each, which multiplies scores and weights; in 4 bits the groups' scales go into the fp16 values.
constexpr bool kv_scaled(int kind) { return kind == FV_KV_INT8 || kind == FV_KV_E4M3; }

struct PromptBars {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], pv_done, all_done;
  uint32_t tmem;
  int abort, odd[2][4], entries;
  int2 exponent[2];  // of the largest scale of a value, of the tile and of all tiles up to it
};

template <int KIND, int D>
struct Tile {
  static constexpr int ROWS = 64;                        // of the cache
  static constexpr int HALVES = (D + 63) / 64;           // of 64 components: rows of 128 bytes
  static constexpr int HALF = ROWS * 128;                // bytes
  static constexpr int STAGE = HALVES * HALF;            // keys or values of one tile
  static constexpr int Q_HALF = KV_PROMPT_COLS * 128;
  static constexpr int Q = HALVES * Q_HALF;
  static constexpr int SCALES = !kv_scaled(KIND) ? 0 : 2 * 3 * ROWS * 4;  // [stage][keys, values relative to the largest, values][ROWS]
  static constexpr int K_AT = Q, V_AT = Q + 2 * STAGE, SCALE_AT = Q + 4 * STAGE, BARS_AT = SCALE_AT + SCALES;
  static constexpr int LIST_AT = BARS_AT + (int(sizeof(PromptBars)) + 15) / 16 * 16;
  static constexpr int O_COL = 128;  // columns of tensor memory: S or P 0-63, 64-127, O from 128 on
};

__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// D (tensor memory) += A (tensor memory: two 16-bit values to a column) B (shared memory)
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t to, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(to)
      : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two floats at a time.
__device__ __forceinline__ void fma2(float* x, float by, float add) {  // x[0..1] * by + add
  asm("{\n.reg .b64 a, b, c;\nmov.b64 a, {%0, %1};\nmov.b64 b, {%2, %2};\nmov.b64 c, {%3, %3};\nfma.rn.f32x2 a, a, b, c;\nmov.b64 {%0, %1}, a;\n}\n"
      : "+f"(x[0]), "+f"(x[1])
      : "f"(by), "f"(add));
}
__device__ __forceinline__ void mul2(float* x, float y0, float y1) {
  asm("{\n.reg .b64 a, b;\nmov.b64 a, {%0, %1};\nmov.b64 b, {%2, %3};\nmul.rn.f32x2 a, a, b;\nmov.b64 {%0, %1}, a;\n}\n" : "+f"(x[0]), "+f"(x[1]) : "f"(y0), "f"(y1));
}
__device__ __forceinline__ void add2(float* x, const float* y) {
  asm("{\n.reg .b64 a, b;\nmov.b64 a, {%0, %1};\nmov.b64 b, {%2, %3};\nadd.rn.f32x2 a, a, b;\nmov.b64 {%0, %1}, a;\n}\n" : "+f"(x[0]), "+f"(x[1]) : "f"(y[0]), "f"(y[1]));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// x + 0 * w in both halves: NaN from the first that is not finite on
template <class T>
__device__ __forceinline__ uint32_t watch(uint32_t x, uint32_t w) {
  uint32_t y;
  if constexpr (std::is_same<T, __half>::value) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(w), "r"(0u), "r"(x));
  else asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(w), "r"(0u), "r"(x));
  return y;
}

// What all warps of a CTA know about its work.
struct PromptWork {
  int head, last, pieces, tiles;  // position of the last row; pieces of 16 rows of the cache, tiles of four of them
  int first;                      // 4 bits: tile of the union that is this CTA's first
  const int2* list;               // (block, page) of the union, ascending
  // piece p of the CTA's: where it begins, and its first row in the pages; false: it is none, or has no page
  __device__ __forceinline__ bool piece(const KvAttend& a, const KvBatch& m, int p, int& start, size_t& from) const {
    p += 4 * first;
    if (p >= pieces) return false;
    const int per = m.page_shift - 4, sub = (p & ((1 << per) - 1)) << 4;
    const int2 at = list[p >> per];
    start = (at.x << m.page_shift) + sub;
    from = ((size_t(max(at.y, 0)) * a.heads + head) << m.page_shift) + sub;
    return at.y >= 0;
  }
};

// N threads bring tile i of the keys (or values) to `to`: rows of 128 bytes, 16-byte pieces exchanged by the row's number as the
// tensor cores read them, zeros for rows that are none.  Piece u of a row of 16 bytes in 16 bits, of 8 codes in 8.
template <class T, int KIND, int D, int N>
struct Bring {
  using S = Tile<KIND, D>;
  static constexpr int UNITS = D / 8, PIECE = 16 * UNITS, TIMES = (PIECE + N - 1) / N;  // 16-byte pieces of a row, and of 16 rows
  static __device__ __forceinline__ uint32_t place(int r, int u) { return (u >> 3) * S::HALF + r * 128 + (((u & 7) ^ (r & 7)) << 4); }
  // f(piece of 16 rows, its x-th time, row of the tile, piece of the row, number in the piece), for what thread t has of the tile
  template <class F>
  static __device__ __forceinline__ void each(int t, F&& f) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int x = 0; x < TIMES; ++x) {
        const int n = t + N * x, r = n / UNITS;
        if (PIECE % N && n >= PIECE) continue;
        f(p, x, 16 * p + r, n - r * UNITS, n);
      }
  }

  static __device__ __forceinline__ void start(const KvAttend& a, const KvBatch& m, const PromptWork& w, int i, const unsigned char* src, uint32_t to, int t) {
    const unsigned char* from[4];
    int seen[4];  // rows of the piece that somebody sees
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      int begin = 0;
      size_t at = 0;
      seen[p] = w.piece(a, m, 4 * i + p, begin, at) ? w.last - begin + 1 : 0;
      from[p] = src + (seen[p] ? at * (2 * D) : 0);
    }
    each(t, [&](int p, int, int r, int u, int n) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + place(r, u)), "l"(from[p] + n * 16), "r"((r & 15) < seen[p] ? 16 : 0));
    });
    asm volatile("cp.async.commit_group;");
  }
  // 8 bits: through registers, where the codes become fp16
  static __device__ __forceinline__ void convert(const KvAttend& a, const KvBatch& m, const PromptWork& w, int i, const unsigned char* src, unsigned char* to, int t) {
    uint2 c[4][TIMES];
    const unsigned char* from[4];
    int seen[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      int begin = 0;
      size_t at = 0;
      seen[p] = w.piece(a, m, 4 * i + p, begin, at) ? w.last - begin + 1 : 0;
      from[p] = src + (seen[p] ? at * D : 0);
    }
    each(t, [&](int p, int x, int r, int, int n) {
      c[p][x] = (r & 15) < seen[p] ? __ldg(reinterpret_cast<const uint2*>(from[p] + n * 8)) : make_uint2(0, 0);
    });
    each(t, [&](int p, int x, int r, int u, int) {
      uint4 y;
      codes_to_half<KIND>(c[p][x].x, y.x, y.y);
      codes_to_half<KIND>(c[p][x].y, y.z, y.w);
      *reinterpret_cast<uint4*>(to + place(r, u)) = y;
    });
  }
};

// 4 bits: N threads bring a tile as fp16, code times scale, exactly.  A thread has a quarter of a row, eight neighbouring components of every
// group, in the order 0 4 1 5 2 6 3 7 that the codes come apart in; queries and results are put into it and out of it again.
// Eight lanes that store at one time have rows four apart, whose pieces lie in different banks.  VALUES: a group whose scale is no
// number becomes zeros; whether there was one is returned.
template <int D, int N, bool VALUES>
struct BringFour {
  using S = Tile<FV_KV_INT4X32, D>;
  static constexpr int NG = D / 32, TIMES = 256 / N;
  static __device__ __forceinline__ bool convert(const KvAttend& a, const KvBatch& m, const PromptWork& w, int i, unsigned char* to, int t) {
    const unsigned char* const src = VALUES ? a.vp : a.kp;
    const uint8_t* const scales = reinterpret_cast<const uint8_t*>(VALUES ? a.v_scale : a.k_scale);
    const int quarter = t & 3, r16 = (t >> 5 & 1) * 8 + (t >> 2 & 1) * 4 + (t >> 3 & 3);  // row of the piece
    uint32_t c[TIMES][NG], sc[TIMES];
#pragma unroll
    for (int x = 0; x < TIMES; ++x) {
      const int p = x * (N / 64) + (t >> 6);
      int begin = 0;
      size_t at = 0;
      sc[x] = 0u;
#pragma unroll
      for (int g = 0; g < NG; ++g) c[x][g] = 0u;
      if (!w.piece(a, m, 4 * i + p, begin, at) || begin + r16 > w.last) continue;  // zeros for rows that nobody sees
      const unsigned char* from = src + (at + r16) * (D / 2) + quarter * (4 * NG);
      const uint8_t* s = scales + (at + r16) * NG;
      if constexpr (NG == 4) {
        const uint4 y = __ldg(reinterpret_cast<const uint4*>(from));
        c[x][0] = y.x, c[x][1] = y.y, c[x][2] = y.z, c[x][3] = y.w;
        sc[x] = __ldg(reinterpret_cast<const uint32_t*>(s));
      } else if constexpr (NG == 2) {
        const uint2 y = __ldg(reinterpret_cast<const uint2*>(from));
        c[x][0] = y.x, c[x][1] = y.y;
        sc[x] = __ldg(reinterpret_cast<const uint16_t*>(s));
      } else {
#pragma unroll
        for (int g = 0; g < NG; ++g) c[x][g] = __ldg(reinterpret_cast<const uint32_t*>(from) + g), sc[x] |= uint32_t(__ldg(s + g)) << (8 * g);
      }
    }
    bool odd = false;
    const uint32_t by_1024 = Four::magic(0x64006400u), by_64 = Four::magic(0x54005400u);
#pragma unroll
    for (int x = 0; x < TIMES; ++x) {
      const int r = 16 * (x * (N / 64) + (t >> 6)) + r16;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t byte = sc[x] >> (8 * g) & 255u;
        if (VALUES && byte >= 248u) odd = true, byte = 0u;
        const __half2 by = __half2half2(__ushort_as_half(uint16_t(byte << 7)));
        uint32_t y[4];
        Four::halves(Four::group<NG>(c[x], g), y, by_1024, by_64);
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const __half2 f = __hmul2(*reinterpret_cast<const __half2*>(&y[z]), by);
          y[z] = *reinterpret_cast<const uint32_t*>(&f);
        }
        const int u = 4 * g + quarter;
        *reinterpret_cast<uint4*>(to + (u >> 3) * S::HALF + r * 128 + (((u & 7) ^ (r & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
      }
    }
    return odd;
  }
};

// What brings keys (VALUES: values) to their two places, tile by tile.
template <class T, int KIND, int D, bool VALUES>
__device__ __forceinline__ void bring_all(const KvAttend& a, const KvBatch& m, const PromptWork& work, unsigned char* smem, PromptBars* bars, const AbortCtl& abort, int t) {
  using S = Tile<KIND, D>;
  using B = Bring<T, KIND, D, VALUES ? KV_PROMPT_VALUES : KV_PROMPT_KEYS>;
  const int lane = t & 31;
  uint64_t* const full = VALUES ? bars->v_full : bars->k_full;
  uint64_t* const empty = VALUES ? bars->v_empty : bars->k_empty;
  const unsigned char* const src = VALUES ? a.vp : a.kp;
  unsigned char* const base = smem + (VALUES ? S::V_AT : S::K_AT);
  [[maybe_unused]] int unit = 1;  // 8 bits: scales stand for multiples of 2^(unit - 126), none so far for 2 or more
  for (int i = 0; i < work.tiles; ++i) {
    const uint32_t turn = uint32_t(i >> 1) & 1u;  // of the tile's place
    unsigned char* const to = base + (i & 1) * S::STAGE;
    if (i >= 2 && !__all_sync(FV_FULL, mbar_wait(&empty[i & 1], turn ^ 1u, abort, 32))) break;
    if constexpr (KIND == FV_KV_SAME) {
      B::start(a, m, work, i, src, smem_u32(to), t);
      asm volatile("cp.async.wait_all;");
      if constexpr (VALUES) {  // a thread looks at what it has copied
        uint32_t found = 0u;
        B::each(t, [&](int, int, int r, int u, int) {
          const uint4 v = *reinterpret_cast<const uint4*>(to + B::place(r, u));
          found = watch<T>(watch<T>(watch<T>(watch<T>(found, v.x), v.y), v.z), v.w);
        });
        const bool any = __any_sync(FV_FULL, found != 0u);
        if (any) {
#pragma unroll 1
          for (int p = 0; p < 4; ++p)
            for (int n = t; n < B::PIECE; n += KV_PROMPT_VALUES) {
              const int r = n / B::UNITS;
              uint4* at = reinterpret_cast<uint4*>(to + B::place(16 * p + r, n - r * B::UNITS));
              uint4 v = *at;
              v.x = finite_only<T>(v.x), v.y = finite_only<T>(v.y), v.z = finite_only<T>(v.z), v.w = finite_only<T>(v.w);
              *at = v;
            }
        }
        if (lane == 0) bars->odd[i & 1][t >> 5] = any;
      }
    } else if constexpr (KIND == FV_KV_INT4X32) {
      const bool odd = BringFour<D, VALUES ? KV_PROMPT_VALUES : KV_PROMPT_KEYS, VALUES>::convert(a, m, work, i, to, t);
      if constexpr (VALUES) {
        const bool any = __any_sync(FV_FULL, odd);
        if (lane == 0) bars->odd[i & 1][t >> 5] = any;
      }
    } else {
      B::convert(a, m, work, i, src, to, t);
      if (VALUES && t < 32) {  // the scales of both, which the queries' threads leave together with the values
        float* const sc = reinterpret_cast<float*>(smem + S::SCALE_AT) + (i & 1) * 3 * S::ROWS;
        float vs[2], most = 0.f;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int r = lane + 32 * z;
          int begin = 0;
          size_t from = 0;
          const bool on = work.piece(a, m, 4 * i + (r >> 4), begin, from) && begin + (r & 15) <= work.last;
          sc[r] = on ? __ldg(a.k_scale + from + (r & 15)) : 0.f;
          vs[z] = on ? __ldg(a.v_scale + from + (r & 15)) : 0.f;
          most = fmaxf(most, vs[z]);  // leaves NaN out: it reaches the sums through its weight
        }
        const int e = int(__reduce_max_sync(FV_FULL, __float_as_uint(most)) >> 23);
        unit = e > unit + 1 ? e : unit;
        const float down = __uint_as_float(uint32_t(max(253 - unit, 1)) << 23);
        sc[S::ROWS + lane] = vs[0] * down, sc[S::ROWS + 32 + lane] = vs[1] * down;
        sc[2 * S::ROWS + lane] = vs[0], sc[2 * S::ROWS + 32 + lane] = vs[1];
        const bool any = __any_sync(FV_FULL, !kv_finite(vs[0]) || !kv_finite(vs[1]));
        if (lane == 0) bars->exponent[i & 1] = make_int2(e, unit), bars->odd[i & 1][0] = any;
      }
    }
    fence_async();
    mbar_arrive(&full[i & 1]);
  }
}

// 4 bits: the tiles of a CTA's union are shared out to `count` CTAs where there are few of them, at least KV_PROMPT_LEAST to each, whose
// results [count][rows * heads * group][D] and logarithms to the base of 2 a second kernel joins.
struct PromptParts {
  int count;
  float *out, *lse;
};
enum { KV_PROMPT_LEAST = 6, KV_PROMPT_PLACES = 2 * 148, KV_PROMPT_PARTS = 64 };

template <class T, int KIND, int D>
__global__ void __launch_bounds__(KV_PROMPT_THREADS, 2) kv_prompt_kernel(KvAttend a, KvBatch m, PromptParts parts) {
  using S = Tile<KIND, D>;
  using M = typename std::conditional<KIND == FV_KV_SAME, T, __half>::type;
  constexpr bool HALF = std::is_same<M, __half>::value, FOUR = KIND == FV_KV_INT4X32, SCALED = kv_scaled(KIND);
  constexpr float ONE = FOUR ? 7.f : HALF ? 14.f : 0.f;   // log2 of what stands for a weight of 1
  // log2 of what a maximum may lag behind by; in 8 bits, where the weights meet scales of less than 2, 2^14.9 of them stay in fp16
  constexpr float GROWN = SCALED ? 0.9f : FOUR ? 8.f : HALF ? 1.f : 8.f;
  unsigned char* const smem = dyn_smem();
  PromptBars* const bars = reinterpret_cast<PromptBars*>(smem + S::BARS_AT);
  int2* const list = reinterpret_cast<int2*>(smem + S::LIST_AT);
  const int warp = threadIdx.x >> 5, lane = lane_id(), head = blockIdx.y;

  // which rows of which sequence
  const int tc = KV_PROMPT_COLS / a.group;                // rows of a CTA
  const int item = int(gridDim.x - 1 - blockIdx.x);       // of a head, the rows that see most come first
  const int b = m.cu ? kv_find(m, item, tc, 1) : item;
  const int r0 = m.cu_at(b), r1 = max(m.cu_at(b + 1), r0);
  const int row0 = m.cu ? r0 + (item - (r0 / tc + b)) * tc : r0, rows = min(tc, r1 - row0);
  if (row0 < r0 || rows <= 0) return;
  const int pos0 = m.len(b) - r1 + row0, last = pos0 + rows - 1;  // positions of the first and the last row
  const int blocks = min(m.table_width, last < 0 ? 0 : (last >> m.page_shift) + 1);

  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&bars->tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->k_full[i], KV_PROMPT_KEYS), mbar_init(&bars->k_empty[i], 1), mbar_init(&bars->v_full[i], KV_PROMPT_VALUES), mbar_init(&bars->v_empty[i], 1);
      mbar_init(&bars->s_full[i], 1), mbar_init(&bars->p_full[i], KV_PROMPT_COLS);
    }
    mbar_init(&bars->pv_done, 1), mbar_init(&bars->all_done, 1);
    bars->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // the union of the lists: its bits, where keys will be, then its blocks and their pages in order
  uint32_t* const bits = reinterpret_cast<uint32_t*>(smem + S::K_AT);  // room for 2^18 blocks and more
  if (a.blocks) {
    for (int i = threadIdx.x; i < (blocks + 31) / 32; i += KV_PROMPT_THREADS) bits[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < rows * a.k; i += KV_PROMPT_THREADS) {
      const int r = i / a.k, e = __ldg(a.blocks + (size_t(row0 + r) * a.heads + head) * a.k + (i - r * a.k));
      if (e >= 0 && e < blocks) atomicOr(bits + (e >> 5), 1u << (e & 31));
    }
    __syncthreads();
    if (warp == 5) {
      int n = 0;
      for (int w0 = 0; w0 < (blocks + 31) / 32; w0 += 32) {
        uint32_t x = w0 + lane < (blocks + 31) / 32 ? bits[w0 + lane] : 0u;
        int up = __popc(x);  // up to this lane
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(FV_FULL, up, o);
          if (lane >= o) up += y;
        }
        int at = n + up - __popc(x);
        for (; x; x &= x - 1) list[at++].x = (w0 + lane) * 32 + __ffs(int(x)) - 1;
        n += __shfl_sync(FV_FULL, up, 31);
      }
      if (lane == 0) bars->entries = n;
    }
  } else if (threadIdx.x == 0) {
    bars->entries = blocks;
  }
  // the queries: a thread to a query.  In 8 bits as fp16 times a power of two.  A negative scale turns their sign, 0 makes them 0.
  const int tok = int(threadIdx.x) / a.group, h = int(threadIdx.x) - tok * a.group;  // of a query's thread
  const bool mine = threadIdx.x < KV_PROMPT_COLS && tok < rows;
  float by = a.scale == 0.f ? 1.f : fabsf(a.scale);
  if (warp < 4) {
    const uint4* src = reinterpret_cast<const uint4*>(a.q + size_t(row0 + (mine ? tok : 0)) * a.q_row + size_t(head * a.group + (mine ? h : 0)) * a.q_head);
    float most = 0.f;
    if constexpr (!std::is_same<M, T>::value) {
      for (int u = 0; u < D / 8; ++u) {
        const uint4 x = __ldg(src + u);
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const float2 y = Pair<T>::to_float(reinterpret_cast<const uint32_t*>(&x)[z]);
          most = fmaxf(most, fmaxf(fabsf(y.x), fabsf(y.y)));
        }
      }
    }
    const float f = std::is_same<M, T>::value ? 1.f : half_factor(most);
    by = fmaxf(by / f, __uint_as_float(1u));  // never 0: what is not seen is -inf times it
    const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u, keep = mine && a.scale != 0.f ? ~0u : 0u;
    for (int u = 0; u < D / 8; ++u) {
      uint4 x = __ldg(src + u);
      uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        if constexpr (!std::is_same<M, T>::value) {
          const float2 y = Pair<T>::to_float(w[z]);
          w[z] = Pair<M>::from_float(y.x * f, y.y * f);
        }
        w[z] = (w[z] ^ sign) & keep;
      }
      if constexpr (FOUR)
        x = make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
      const int r = threadIdx.x;
      *reinterpret_cast<uint4*>(smem + (u >> 3) * S::Q_HALF + r * 128 + (((u & 7) ^ (r & 7)) << 4)) = x;
    }
    fence_async();
  }
  __syncthreads();
  PromptWork work;
  work.head = head, work.last = last, work.list = list;
  const int entries = bars->entries;
  for (int i = threadIdx.x; i < entries; i += KV_PROMPT_THREADS) {
    const int block = a.blocks ? list[i].x : i;
    list[i] = make_int2(block, m.page(b, block));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const int per = m.page_shift - 4;
  // of the last block only the pieces up to the last row
  work.pieces = entries ? ((entries - 1) << per) + min(1 << per, ((last - (list[entries - 1].x << m.page_shift)) >> 4) + 1) : 0;
  work.tiles = (work.pieces + 3) / 4;
  work.first = 0;
  if constexpr (FOUR) {
    if (parts.count > 1) {
      const int each = max((work.tiles + parts.count - 1) / parts.count, int(KV_PROMPT_LEAST));
      work.first = int(blockIdx.z) * each;
      work.tiles = min(max(work.tiles - work.first, 0), each);
    }
  }
  const int tiles = work.tiles;
  const uint32_t tmem = bars->tmem;
  const AbortCtl abort{&bars->abort, WAIT_LIMIT_CYCLES};

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(int(KV_PROMPT_REGS_LESS)));
    bring_all<T, KIND, D, true>(a, m, work, smem, bars, abort, threadIdx.x - 256);
  } else if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(int(KV_PROMPT_REGS_LESS)));
    if (warp >= 6) bring_all<T, KIND, D, false>(a, m, work, smem, bars, abort, threadIdx.x - 192);
    if (warp == 4) {  // products
      constexpr uint32_t kind_bits = (1u << 4) | (HALF ? 0u : (1u << 7) | (1u << 10));
      constexpr uint32_t qk = kind_bits | (uint32_t(S::ROWS >> 3) << 17) | (128u >> 4 << 24);
      constexpr uint32_t pv = kind_bits | (1u << 16) | (uint32_t(D >> 3) << 17) | (128u >> 4 << 24);  // values: components along a row
      auto scores = [&](int i) {  // of tile i
        if (!__all_sync(FV_FULL, mbar_wait(&bars->k_full[i & 1], uint32_t(i >> 1) & 1u, abort, 0))) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t q = smem_u32(smem), k = smem_u32(smem + S::K_AT + (i & 1) * S::STAGE);
#pragma unroll
          for (int s = 0; s < D / 16; ++s) {
            const uint32_t at = (s & 3) * 32;
            tc_mma_f16<false>(tmem + (i & 1) * 64, make_desc(desc_lo(q + (s >> 2) * S::Q_HALF + at), DESC_HI_SW128),
                              make_desc(desc_lo(k + (s >> 2) * S::HALF + at), DESC_HI_SW128), qk, s > 0);
          }
          tc_commit<false>(&bars->k_empty[i & 1]);
          tc_commit<false>(&bars->s_full[i & 1]);
        }
        __syncwarp();
        return true;
      };
      bool on = tiles > 0 && scores(0);
      for (int i = 0; on && i < tiles; ++i) {
        if (i + 1 < tiles) {
          // the place of the next scores holds the weights of the tile before this one
          on = __all_sync(FV_FULL, i == 0 || mbar_wait(&bars->pv_done, uint32_t(i - 1) & 1u, abort, 0));
          on = on && scores(i + 1);
          if (!on) break;
        }
        on = __all_sync(FV_FULL, mbar_wait(&bars->v_full[i & 1], uint32_t(i >> 1) & 1u, abort, 0) && mbar_wait(&bars->p_full[i & 1], uint32_t(i >> 1) & 1u, abort, 0));
        if (!on) break;
        tc_fence_after();
        if (elect_one()) {
          // rows of 128 bytes along the components: 8 rows of the cache 1024 bytes apart, 64 components a HALF
          const uint32_t v = smem_u32(smem + S::V_AT + (i & 1) * S::STAGE);
#pragma unroll
          for (int s = 0; s < S::ROWS / 16; ++s) {
            const uint32_t lo = ((v + s * 2048) >> 4) | (uint32_t(S::HALF >> 4) << 16);
            tc_mma_ts(tmem + S::O_COL, tmem + (i & 1) * 64 + s * 8, make_desc(lo, DESC_HI_SW128), pv, 1u);
          }
          tc_commit<false>(&bars->v_empty[i & 1]);
          tc_commit<false>(&bars->pv_done);
          if (i + 1 == tiles) tc_commit<false>(&bars->all_done);
        }
        __syncwarp();
      }
    }
  } else {  // weights
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(int(KV_PROMPT_REGS_MORE)));
    const uint32_t lanes = uint32_t(warp * 32) << 16;
    const int pos = pos0 + tok;
    // the list of the thread's row: the entry that is next, and the one behind it on its way
    const int32_t* const mylist = a.blocks && mine ? a.blocks + (size_t(row0 + tok) * a.heads + head) * a.k : nullptr;
    int entry = -1, ahead = mylist ? __ldg(mylist) : 0, index = 0;
    float top = -INFINITY, sum = 0.f;
    int unit = 0;  // 8 bits: values stand for multiples of 2^(unit - 126), scales the query has seen are below 2 of it; 0: none seen
    bool on = true;
    {
      uint32_t zero[32];
#pragma unroll
      for (int z = 0; z < 32; ++z) zero[z] = 0u;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) tc_st32(tmem + lanes + S::O_COL + c, zero);
      tc_st_wait();
    }
    for (int i = 0; i < tiles; ++i) {
      int seen[4];  // rows of each piece that the query sees
      auto sees = [&](int2 at, int start) {  // whether the query sees the rows from `start` on, of a block of the union
        if (!mine || at.y < 0 || start > pos) return false;
        if (!a.blocks) return true;
        while (entry < at.x) {  // entries that are blocks, each above all before it
          const int e = ahead;
          ++index;
          ahead = index < a.k ? __ldg(mylist + index) : 0;
          if (index > a.k) entry = INT_MAX;
          else if (e > entry && e < blocks && (e << m.page_shift) <= pos) entry = e;
        }
        return entry == at.x;
      };
      if (m.page_shift >= 6) {  // the tile is of one block
        const int more = m.page_shift - 6;
        const int tile = FOUR ? i + work.first : i;
        const int2 at = list[tile >> more];
        const int start = (at.x << m.page_shift) + ((tile & ((1 << more) - 1)) << 6), n = sees(at, start) ? pos - start + 1 : 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) seen[p] = min(max(n - 16 * p, 0), 16);
      } else {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int piece = 4 * (FOUR ? i + work.first : i) + p;
          const int2 at = piece < work.pieces ? list[piece >> per] : make_int2(0, -1);
          const int start = (at.x << m.page_shift) + ((piece & ((1 << per) - 1)) << 4);
          seen[p] = sees(at, start) ? min(pos - start + 1, 16) : 0;
        }
      }
      const bool any = (seen[0] | seen[1] | seen[2] | seen[3]) != 0, all = (seen[0] & seen[1] & seen[2] & seen[3]) == 16;
      const bool whole = ((seen[0] | seen[1] | seen[2] | seen[3]) & 15) == 0;
      const uint32_t turn = uint32_t(i >> 1) & 1u;
      on = __all_sync(FV_FULL, mbar_wait(&bars->s_full[i & 1], turn, abort, 0) && mbar_wait(&bars->v_full[i & 1], turn, abort, 0));
      if (!on) break;
      tc_fence_after();
      const uint32_t place = tmem + lanes + (i & 1) * 64;
      uint32_t p[32];
      bool changed = false;
      float factor = 1.f;
      [[maybe_unused]] const float* const sc = reinterpret_cast<const float*>(smem + S::SCALE_AT) + (i & 1) * 3 * S::ROWS;
      [[maybe_unused]] bool alike = true;  // the tile's scales are relative to the query's unit
      if constexpr (SCALED) {
        const int2 e = bars->exponent[i & 1];
        if (all && (e.x > unit + 1 || unit == 0)) {  // of a tile that the query sees the whole of
          const int own = max(e.x, 1);
          factor = __uint_as_float(uint32_t(max(127 + unit - own, 0)) << 23);
          changed = unit != 0;  // without weights so far the query's O is 0
          unit = own;
        }
        alike = __all_sync(FV_FULL, !any || unit == e.y);
      }
      const bool busy = __any_sync(FV_FULL, any);
      const bool odd = !SCALED ? (bars->odd[i & 1][0] | bars->odd[i & 1][1] | bars->odd[i & 1][2] | bars->odd[i & 1][3]) != 0 : bars->odd[i & 1][0] != 0;
      if (busy) {
        uint32_t r[64];
        tc_ld32_issue(place, r);
        tc_ld32_issue(place + 32, r + 32);
        tc_ld_wait(r);
        tc_ld_wait(r + 32);
        float* s = reinterpret_cast<float*>(r);
        if constexpr (SCALED) {
#pragma unroll
          for (int j = 0; j < 64; j += 4) {
            const float4 ks = *reinterpret_cast<const float4*>(sc + j);
            mul2(s + j, ks.x, ks.y), mul2(s + j + 2, ks.z, ks.w);
          }
        }
        if (!__all_sync(FV_FULL, all)) {
          if (__all_sync(FV_FULL, whole)) {
#pragma unroll
            for (int j = 0; j < 64; ++j) s[j] = seen[j >> 4] ? s[j] : -INFINITY;
          } else {
#pragma unroll
            for (int j = 0; j < 64; ++j) s[j] = (j & 15) < seen[j >> 4] ? s[j] : -INFINITY;
          }
        }
        float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 64; j += 2) y[j >> 1 & 3] = max3(y[j >> 1 & 3], s[j], s[j + 1]);
        const float to = fmaxf(max3(y[0], y[1], y[2]), y[3]) * by;
        if (to > top + GROWN || (top == -INFINITY && to > top)) {
          const float f = exp2_of(top - to);
          factor *= f, sum *= f;
          changed = changed || top != -INFINITY;  // without weights so far the query's O is 0
          top = to;
        }
        const float off = top == -INFINITY ? 0.f : ONE - top;
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 64; j += 2) {
          fma2(s + j, by, off);
          s[j] = exp2_of(s[j]), s[j + 1] = exp2_of(s[j + 1]);
          add2(part + (j & 2), s + j);
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
        if constexpr (SCALED) {
          if (!odd && alike) {
#pragma unroll
            for (int j = 0; j < 64; j += 4) {
              const float4 vs = *reinterpret_cast<const float4*>(sc + S::ROWS + j);
              mul2(s + j, vs.x, vs.y), mul2(s + j + 2, vs.z, vs.w);
            }
          } else {
            const int2 e = bars->exponent[i & 1];
            if (any && (e.x > unit + 1 || unit == 0)) {  // a scale of the tile is above the query's unit: whether it has a weight
              float most = 0.f;  // leaves NaN out
#pragma unroll
              for (int j = 0; j < 64; ++j) most = fmaxf(most, s[j] != 0.f ? sc[2 * S::ROWS + j] : 0.f);
              const int own = max(int(__float_as_uint(most) >> 23), 1);
              if (own > unit + 1 || unit == 0) {
                factor *= __uint_as_float(uint32_t(max(127 + unit - own, 0)) << 23);
                changed = changed || unit != 0;  // without weights so far the query's O is 0
                unit = own;
              }
            }
            const float down = __uint_as_float(uint32_t(max(253 - unit, 1)) << 23);
#pragma unroll  // scales of NaN, and those beyond the query's unit, reach the rows that have a weight for them
            for (int j = 0; j < 64; ++j) s[j] = s[j] != 0.f ? s[j] * (sc[2 * S::ROWS + j] * down) : 0.f;
          }
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) p[j] = Pair<M>::from_float(s[2 * j], s[2 * j + 1]);
        // O, scaled to the new maximum, and values that were taken out of the product
        const bool scale_o = __any_sync(FV_FULL, changed);
        if (!SCALED && odd) {
          on = __all_sync(FV_FULL, i == 0 || mbar_wait(&bars->pv_done, uint32_t(i - 1) & 1u, abort, 0));
          if (!on) break;
          tc_fence_after();
          float w[64];  // where a loop can index them
#pragma unroll
          for (int j = 0; j < 64; ++j) w[j] = s[j];
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tc_ld32_issue(tmem + lanes + S::O_COL + c, o);
            tc_ld_wait(o);
#pragma unroll
            for (int z = 0; z < 32; ++z) o[z] = __float_as_uint(__uint_as_float(o[z]) * factor);
#pragma unroll 1
            for (int j = 0; j < 64; ++j) {
              const float weight = w[j];
              int start = 0;
              size_t from = 0;
              if (weight == 0.f || !work.piece(a, m, 4 * i + (j >> 4), start, from)) continue;
              if constexpr (FOUR) {  // 32 components are a group
                const uint32_t byte = __ldg(reinterpret_cast<const uint8_t*>(a.v_scale) + (from + (j & 15)) * (D / 32) + (c >> 5));
                if (byte >= 248u) {
#pragma unroll
                  for (int z = 0; z < 32; ++z) o[z] = 0x7FFFFFFFu;
                }
                continue;
              }
              const unsigned char* row = a.vp + ((from + (j & 15)) * D + c) * 2;
#pragma unroll
              for (int z = 0; z < 32; z += 2) {
                const float2 v = Pair<T>::to_float(__ldg(reinterpret_cast<const uint32_t*>(row) + z / 2));
                if (!kv_finite(v.x)) o[z] = __float_as_uint(__uint_as_float(o[z]) + weight * v.x);
                if (!kv_finite(v.y)) o[z + 1] = __float_as_uint(__uint_as_float(o[z + 1]) + weight * v.y);
              }
            }
            tc_st32(tmem + lanes + S::O_COL + c, o);
          }
          tc_st_wait();
        } else if (scale_o) {
          on = __all_sync(FV_FULL, i == 0 || mbar_wait(&bars->pv_done, uint32_t(i - 1) & 1u, abort, 0));
          if (!on) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tc_ld32_issue(tmem + lanes + S::O_COL + c, o);
            tc_ld_wait(o);
#pragma unroll
            for (int z = 0; z < 32; ++z) o[z] = __float_as_uint(__uint_as_float(o[z]) * factor);
            tc_st32(tmem + lanes + S::O_COL + c, o);
          }
          tc_st_wait();
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) p[j] = 0u;
      }
      tc_st32(place, p);
      tc_st_wait();
      tc_fence_before();
      mbar_arrive(&bars->p_full[i & 1]);
    }
    // (pv_done may lie one or two phases behind here, which its parity does not tell apart)
    if (on && tiles) on = __all_sync(FV_FULL, mbar_wait(&bars->all_done, 0u, abort, 0));
    tc_fence_after();
    // two factors: their product can be too small for all of its bits where the scales are
    const float f = SCALED ? __uint_as_float(uint32_t(min(unit + 1, 254)) << 23) : 1.f;
    const float down = sum == 0.f ? 0.f : 1.f / sum;
    const size_t query = (size_t(row0 + tok) * a.heads + head) * a.group + h;
    const bool part = FOUR && parts.count > 1;
    const size_t place = part ? size_t(blockIdx.z) * (size_t(m.rows) * a.heads * a.group) + query : 0;
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      uint32_t o[32];
      tc_ld32_issue(tmem + lanes + S::O_COL + c, o);
      tc_ld_wait(o);
      if constexpr (FOUR) {
        if (part) {  // one to be joined: as 32-bit numbers
#pragma unroll
          for (int z = 0; z < 8; ++z) {  // of every eight in their order 0 4 1 5 2 6 3 7
            const int b = 8 * (z >> 1) + (z & 1 ? 1 : 0);
            const float4 x = make_float4(__uint_as_float(o[b]) * down, __uint_as_float(o[b + 2]) * down, __uint_as_float(o[b + 4]) * down, __uint_as_float(o[b + 6]) * down);
            if (mine && sum != 0.f) *reinterpret_cast<float4*>(parts.out + place * D + c + 4 * z) = x;
          }
          continue;
        }
      }
      uint4 w[4];
#pragma unroll
      for (int z = 0; z < 16; ++z) {
        constexpr int order[4] = {0, 4, 1, 5};
        const int z0 = FOUR ? (z & ~3) * 2 + order[z & 3] : 2 * z, z1 = FOUR ? z0 + 2 : 2 * z + 1;
        float u = __uint_as_float(o[z0]) * down, v = __uint_as_float(o[z1]) * down;
        if constexpr (SCALED) u *= f, v *= f;
        // a wait that ran out leaves no result: NaN
        reinterpret_cast<uint32_t*>(w)[z] = !on ? 0x7FFF7FFFu : sum == 0.f ? 0u : Pair<T>::from_float(u, v);
      }
      if (mine) {
#pragma unroll
        for (int z = 0; z < 4; ++z) *reinterpret_cast<uint4*>(a.out + (query * D + c + 8 * z) * 2) = w[z];
      }
    }
    if (part && mine) parts.lse[place] = !on ? __int_as_float(0x7FC00000) : sum == 0.f ? -INFINITY : top - ONE + log2f(sum);
    if (!part && mine && a.lse) a.lse[query] = !on ? __int_as_float(0x7FC00000) : sum == 0.f ? -INFINITY : (top - ONE + log2f(sum)) * 0.693147180559945309f;
  }
  if (warp >= 6) asm volatile("cp.async.wait_all;");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
}

// Joins the parts of a query: a warp to each.
template <class T, int D>
__global__ void __launch_bounds__(256) kv_prompt_join_kernel(KvAttend a, KvBatch m, PromptParts parts) {
  const int lane = lane_id(), heads = a.heads * a.group, row = blockIdx.x;
  const int b = m.cu ? kv_find(m, row, 1, 0) : row;
  if (row < m.cu_at(b) || row >= m.cu_at(b + 1)) return;  // of no sequence
  const size_t all = size_t(m.rows) * heads;
  for (int h = blockIdx.y * 8 + (threadIdx.x >> 5); h < heads; h += gridDim.y * 8) {
    const size_t query = size_t(row) * heads + h;
    float l[2], most = -INFINITY;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      l[z] = lane + 32 * z < parts.count ? parts.lse[(lane + 32 * z) * all + query] : -INFINITY;
      most = fmaxf(most, l[z]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(FV_FULL, most, o));
    float total = 0.f;
#pragma unroll
    for (int z = 0; z < 2; ++z) l[z] = l[z] == -INFINITY ? 0.f : exp2_of(l[z] - (most == -INFINITY ? 0.f : most)), total += l[z];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(FV_FULL, total, o);
    float sum[D / 32] = {};
    for (int z = 0; z < parts.count; ++z) {
      const float w = __shfl_sync(FV_FULL, z < 32 ? l[0] : l[1], z & 31);
      if (w == 0.f) continue;  // nothing seen there: its results are anything
      const float* from = parts.out + (size_t(z) * all + query) * D;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const float2 x = *reinterpret_cast<const float2*>(from + 64 * i + 2 * lane);
        sum[2 * i] = __fmaf_rn(w, x.x, sum[2 * i]), sum[2 * i + 1] = __fmaf_rn(w, x.y, sum[2 * i + 1]);
      }
      if constexpr (D % 64 != 0) sum[D / 32 - 1] = __fmaf_rn(w, from[D - 32 + lane], sum[D / 32 - 1]);
    }
    const float down = total == 0.f ? 0.f : 1.f / total;
    unsigned char* const to = a.out + query * (2 * D);
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
      *reinterpret_cast<uint32_t*>(to + 128 * i + 4 * lane) = total == 0.f ? 0u : Pair<T>::from_float(sum[2 * i] * down, sum[2 * i + 1] * down);
    if constexpr (D % 64 != 0) {
      const uint32_t w = total == 0.f ? 0u : Pair<T>::from_float(sum[D / 32 - 1] * down, 0.f);
      *reinterpret_cast<uint16_t*>(to + 2 * (D - 32 + lane)) = uint16_t(w);
    }
    if (a.lse && lane == 0) a.lse[query] = total == 0.f ? -INFINITY : (most + log2f(total)) * 0.693147180559945309f;
  }
}

size_t prompt_entries(const fv_kv_batch* b, int group, bool lists, size_t k) {
  const size_t most = size_t(KV_PROMPT_COLS / group) * k;
  return lists && most < b->table_width ? most : b->table_width;
}

size_t prompt_items(const fv_kv_batch* b, int group) {
  const int tc = KV_PROMPT_COLS / group;
  return b->cu ? b->rows / tc + b->nseq : b->nseq;
}

// CTAs that the tiles of one's union are shared out to, by the most tiles that a union can have: those that go in the fewest waves of places for
// their size, a part's beginning and end counted as a 25th of the whole.  Where all places are taken anyway CTAs of unequal lengths follow one
// another, and parts only cost (4 groups of 8 key heads, dim 128, us by parts 1/2/3/4/5/8):
//   104 CTAs, 400 rows over 16,000    304/236/251/208/210/219      216 CTAs, 400 rows over 20,000    543/503/512/460/496/517
//   256 CTAs, 1000 rows over 8000     224/246/259/259/279/330      648 CTAs, 3000 rows over 6000     445/506/552/599/649/793
int prompt_parts(const fv_kv* kv, const fv_kv_batch* b, int group, bool lists, size_t k) {
  const size_t ctas = prompt_items(b, group) * kv->heads, tiles = prompt_entries(b, group, lists, k) * kv->page_size / 64;
  if (kv->kind != FV_KV_INT4X32 || ctas == 0 || ctas >= KV_PROMPT_PLACES) return 1;
  int best = 1;
  double least = 1e30;
  for (size_t n = 1; n <= KV_PROMPT_PARTS && (n == 1 || n * KV_PROMPT_LEAST <= tiles); ++n) {
    const double cost = double((ctas * n + KV_PROMPT_PLACES - 1) / KV_PROMPT_PLACES) * (1.0 / double(n) + 0.04);
    if (cost < least) least = cost, best = int(n);
  }
  return best;
}
size_t part_floats(const fv_kv* kv, const fv_kv_batch* b, int group) { return b->rows * kv->heads * group * (kv->dim + 1); }

template <class T, int KIND, int D>
int prompt_of(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a, void* work, size_t work_bytes) {
  using S = Tile<KIND, D>;
  const size_t items = prompt_items(b, a.group);
  const size_t smem = S::LIST_AT + 8 * prompt_entries(b, a.group, a.blocks != nullptr, a.k);
  FV_TRY((kv_allow_smem<kv_prompt_kernel<T, KIND, D>>(kv->device, smem)));
  static std::atomic<int> regs{0};  // a thread's at launch: the kernel waits for more than they add up to
  if (regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes at;
    FV_CUDA(cudaFuncGetAttributes(&at, kv_prompt_kernel<T, KIND, D>));
    regs.store(at.numRegs, std::memory_order_relaxed);
  }
  if (regs.load(std::memory_order_relaxed) < KV_PROMPT_REGS) return fail(FV_ERR_UNSUPPORTED, "fv_kv_attend_dev: built with fewer registers than it shares out");
  PromptParts parts{1, nullptr, nullptr};
  if constexpr (KIND == FV_KV_INT4X32) {
    const size_t floats = part_floats(kv, b, a.group), room = work ? work_bytes / 4 / floats : 0;
    const int n = prompt_parts(kv, b, a.group, a.blocks != nullptr, a.k);
    parts.count = room < 2 ? 1 : size_t(n) < room ? n : int(room);
    parts.out = static_cast<float*>(work), parts.lse = parts.out + size_t(parts.count) * (floats - floats / (D + 1));
  }
  kv_prompt_kernel<T, KIND, D><<<dim3(unsigned(items), kv->heads, parts.count), KV_PROMPT_THREADS, smem, s>>>(a, kv_batch(kv, b), parts);
  FV_CUDA(cudaGetLastError());
  if constexpr (KIND == FV_KV_INT4X32)
    if (parts.count > 1) {
      kv_prompt_join_kernel<T, D><<<dim3(unsigned(b->rows), unsigned((kv->heads * a.group + 7) / 8)), 256, 0, s>>>(a, kv_batch(kv, b), parts);
      FV_CUDA(cudaGetLastError());
    }
  return FV_OK;
}

}  // namespace

// Entries of the union that fit beside the largest tiles.
bool kv_prompt_fits(const fv_kv_batch* b, size_t group, bool lists, size_t k) {
  return prompt_entries(b, int(group), lists, k) <= (226 * 1024 - size_t(Tile<FV_KV_INT8, 128>::LIST_AT)) / 8 && b->table_width <= (1u << 18);
}

// Bytes of work that a call's parts want, whatever its lists.
size_t kv_prompt_work(const fv_kv* kv, const fv_kv_batch* b, size_t group) {
  const int n = prompt_parts(kv, b, int(group), false, 0);  // lists have at most as many tiles
  return n > 1 ? 4 * size_t(n) * part_floats(kv, b, int(group)) : 0;
}

int kv_prompt_attend(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a, void* work, size_t work_bytes) {
  FV_KV_DISPATCH(kv, prompt_of, kv, s, b, a, work, work_bytes);
}

}  // namespace fv
