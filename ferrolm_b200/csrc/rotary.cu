// Rotary positions: pairs of a row's components turned by angles that grow with the row's position.
//
//   y_i = a (x_i cos t - x_j sin t),  y_j = a (x_j cos t + x_i sin t),  t = position * w_i;  components behind the turned part as they are
//
// The angle is kept as a part of a whole turn, a fraction of 2^64: position * (w / 2 pi) modulo 1 is the low half of a product of
// whole numbers, which adds nothing to w's own rounding, however far the position is.  Its upper 32 bits, rounded to 24, are off by less than
// pi 2^-25 + pi 2^-31, and the sine and cosine of that by 2^-24: 2^-22.6 in all.  A row's sines and
// cosines are worked out once and shared by its heads, so the bytes bound it: every row is read once and written once.
#include <climits>

#include "kv.cuh"

namespace fv {
namespace {

enum { ROTARY_THREADS = 256, ROTARY_TENSORS = 4, ROTARY_DIM = 1024 };

struct RotaryRows {
  const unsigned char* in;
  unsigned char* out;
  size_t in_row, in_head, out_row, out_head;  // bytes
  int first;                                  // of its heads among those of all tensors
  bool rest;                                  // what is not turned is to be copied
};
struct Rotary {
  RotaryRows x[ROTARY_TENSORS];
  const unsigned long long* turns;
  const int32_t* positions;
  int heads, half;      // of all tensors; pairs of a head
  int units, turned;    // a thread's pieces of a head, and those of them that are turned
  float a;
  bool back;
};

// A CTA has ROWS rows.  Thread t takes piece t % units of a head: eight pairs of the two halves, or four neighbouring pairs (PAIRS), or
// eight components that stay; it has the pieces of AHEAD heads on their way.  13.6k rows of 40 heads of 128 in halves: 54.0 us, 5.3 TB/s; half of a
// head in neighbours, 48.2 us, 5.9 TB/s, 0.91 of the copy rate (with four on their way, for which fewer CTAs have room, 57.2 and 50.9; with
// eight rows to a CTA 59.9 and 49.9).  24 rows: 2.8 us, dependent loads (lengths, turns, rows).
template <class T, bool PAIRS, int ROWS>
__global__ void __launch_bounds__(ROTARY_THREADS) rotate_kernel(Rotary a, KvBatch m) {
  constexpr int AHEAD = 2;
  float2* const angle = reinterpret_cast<float2*>(dyn_smem());  // [ROWS][half]: cosine, sine
  __shared__ int s_pos[ROWS];
  const int first = blockIdx.x * ROWS;
  if (threadIdx.x < ROWS) {
    const int r = first + threadIdx.x;
    int pos = -1;  // of no row
    if (r < m.rows) {
      if (a.positions) {
        pos = __ldg(a.positions + r);
      } else if (r < m.cu_at(m.nseq)) {
        int lo = 0, n = m.nseq;
        if (m.cu) {
          while (n > 1) {  // the last sequence that begins at or before row r
            const int h = n / 2;
            if (m.cu_at(lo + h) <= r) lo += h, n -= h;
            else n = h;
          }
        } else {
          lo = r;
        }
        if (r >= m.cu_at(lo)) pos = m.len(lo) - max(m.cu_at(lo + 1), r + 1) + r;  // in front of the first there may be rows of no sequence
      }
    }
    s_pos[threadIdx.x] = pos;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * a.half; i += ROTARY_THREADS) {
    const int r = i / a.half;
    const unsigned long long turn = __ldg(a.turns + (i - r * a.half)) * (unsigned long long)(max(s_pos[r], 0));
    float s, c;
    sincospif(float(int(turn >> 32)) * 0x1p-31f, &s, &c);
    angle[i] = make_float2(a.a * c, a.back ? -a.a * s : a.a * s);
  }
  __syncthreads();
  const int step = ROTARY_THREADS / a.units, unit = threadIdx.x % a.units;
  if (int(threadIdx.x) / a.units >= step) return;
  const bool turned = unit < a.turned;
  int row = 0, head = threadIdx.x / a.units;
  while (head >= a.heads) head -= a.heads, ++row;
  // where a piece begins, and for halves its second half
  const int at = turned || PAIRS ? unit * 16 : unit * 16 + a.turned * 16, far = !PAIRS && turned ? a.half * 2 : 0;
  while (row < ROWS) {
    uint4 x[AHEAD][2];
    unsigned char* to[AHEAD];
    int of[AHEAD];
#pragma unroll
    for (int z = 0; z < AHEAD; ++z) {
      of[z] = -1;
      if (row < ROWS && s_pos[row] >= 0) {
        int w = 0;
#pragma unroll
        for (int i = 1; i < ROTARY_TENSORS; ++i) w = head >= a.x[i].first ? i : w;
        const RotaryRows& y = a.x[w];
        if (turned || y.rest) {
          of[z] = row;
          const size_t r = size_t(first) + row, h = head - y.first;
          const unsigned char* from = y.in + r * y.in_row + h * y.in_head + at;
          to[z] = y.out + r * y.out_row + h * y.out_head + at;
          x[z][0] = *reinterpret_cast<const uint4*>(from);
          if (far) x[z][1] = *reinterpret_cast<const uint4*>(from + far);
        }
      }
      head += step;
      while (head >= a.heads) head -= a.heads, ++row;
    }
#pragma unroll
    for (int z = 0; z < AHEAD; ++z) {
      if (of[z] < 0) continue;
      if (turned) {
        uint32_t* const u = reinterpret_cast<uint32_t*>(&x[z][0]);
        uint32_t* const v = reinterpret_cast<uint32_t*>(&x[z][1]);
        if constexpr (PAIRS) {
          const float2* t = angle + of[z] * a.half + unit * 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = Pair<T>::to_float(u[i]), c = t[i];
            u[i] = Pair<T>::from_float(__fmaf_rn(f.x, c.x, -(f.y * c.y)), __fmaf_rn(f.y, c.x, f.x * c.y));
          }
        } else {
          const float2* t = angle + of[z] * a.half + unit * 8;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = Pair<T>::to_float(u[i]), g = Pair<T>::to_float(v[i]), c = t[2 * i], d = t[2 * i + 1];
            u[i] = Pair<T>::from_float(__fmaf_rn(f.x, c.x, -(g.x * c.y)), __fmaf_rn(f.y, d.x, -(g.y * d.y)));
            v[i] = Pair<T>::from_float(__fmaf_rn(g.x, c.x, f.x * c.y), __fmaf_rn(g.y, d.x, f.y * d.y));
          }
        }
      }
      *reinterpret_cast<uint4*>(to[z]) = x[z][0];
      if (far) *reinterpret_cast<uint4*>(to[z] + far) = x[z][1];
    }
  }
}

template <class T, bool PAIRS>
int rotate_of(const Rotary& a, const KvBatch& m, cudaStream_t s) {
  auto go = [&](auto rows_of) {
    constexpr int ROWS = decltype(rows_of)::value;
    rotate_kernel<T, PAIRS, ROWS><<<unsigned((m.rows + ROWS - 1) / ROWS), ROTARY_THREADS, ROWS * a.half * sizeof(float2), s>>>(a, m);
  };
  // a row to a CTA where there are few
  if (m.rows <= 8 * 148) go(std::integral_constant<int, 1>());
  else go(std::integral_constant<int, 4>());
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

}  // namespace
}  // namespace fv

extern "C" int fv_rotate_dev(const fv_rotary* r, void* stream, const fv_rotary_rows* x, size_t count, size_t rows, const int32_t* lens,
                             const int32_t* cu, size_t nseq, const int32_t* positions, int back) {
  using fv::fail;
  const std::string w("fv_rotate_dev");
  if (!r || !x) return fail(FV_ERR_ARG, w + ": NULL description or rows");
  if (r->dtype != FV_KV_BF16 && r->dtype != FV_KV_FP16) return fail(FV_ERR_UNSUPPORTED, w + ": dtype is bf16 or fp16");
  if (r->layout != FV_ROTARY_HALF && r->layout != FV_ROTARY_PAIRS) return fail(FV_ERR_UNSUPPORTED, w + ": layout is half or pairs");
  if (r->dim == 0 || r->dim > fv::ROTARY_DIM || r->dim % 16) return fail(FV_ERR_UNSUPPORTED, w + ": dim is a multiple of 16 up to 1024");
  if (r->part == 0 || r->part > r->dim || r->part % 16) return fail(FV_ERR_UNSUPPORTED, w + ": part is a multiple of 16 up to dim");
  if (!(r->amplitude - r->amplitude == 0.f)) return fail(FV_ERR_ARG, w + ": amplitude is not finite");
  if (r->device < 0) return fail(FV_ERR_ARG, w + ": device index out of range");
  if (count == 0 || count > fv::ROTARY_TENSORS) return fail(FV_ERR_UNSUPPORTED, w + ": one to four tensors");
  if (rows > size_t(INT_MAX) / 2 || nseq > size_t(INT_MAX) / 8) return fail(FV_ERR_UNSUPPORTED, w + ": rows or nseq is too large");
  if (!positions && !cu && rows != nseq) return fail(FV_ERR_ARG, w + ": without cu there is one row for each sequence");
  if (!r->turns || !fv::kv_aligned(r->turns, 8)) return fail(FV_ERR_ARG, w + ": turns is not there or does not begin on 8 bytes");
  if (!fv::kv_aligned(positions, 4) || !fv::kv_aligned(lens, 4) || !fv::kv_aligned(cu, 4)) return fail(FV_ERR_ARG, w + ": positions, lens or cu does not begin on 4 bytes");
  fv::Rotary a = {};
  size_t heads = 0;
  for (size_t i = 0; i < fv::ROTARY_TENSORS; ++i) {
    if (i >= count) {
      a.x[i].first = INT_MAX;
      continue;
    }
    const fv_rotary_rows& y = x[i];
    if (y.heads == 0 || y.heads > 65535) return fail(FV_ERR_UNSUPPORTED, w + ": heads is 1 to 65535");
    if (rows && (!y.in || !y.out)) return fail(FV_ERR_ARG, w + ": NULL rows");
    if (!fv::kv_aligned(y.in, 16) || !fv::kv_aligned(y.out, 16) || ((y.in_row | y.in_head | y.out_row | y.out_head) & 7))
      return fail(FV_ERR_ARG, w + ": rows begin on 16 bytes and strides are multiples of 8 elements");
    const bool same = y.in == y.out && y.in_row == y.out_row && y.in_head == y.out_head;
    a.x[i] = {static_cast<const unsigned char*>(y.in), static_cast<unsigned char*>(y.out), 2 * y.in_row, 2 * y.in_head, 2 * y.out_row, 2 * y.out_head, int(heads), !same};
    heads += y.heads;
  }
  if (rows == 0 || (!positions && nseq == 0)) return FV_OK;
  if (!positions && !lens) return fail(FV_ERR_ARG, w + ": positions or lens");
  a.turns = reinterpret_cast<const unsigned long long*>(r->turns), a.positions = positions;
  a.heads = int(heads), a.half = int(r->part / 2), a.a = r->amplitude, a.back = back != 0;
  a.turned = int(r->layout == FV_ROTARY_PAIRS ? r->part / 8 : r->part / 16);
  a.units = a.turned + int(r->dim - r->part) / 8;
  fv::DeviceGuard g(r->device);
  if (!g.ok) return fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  const fv::KvBatch m{nullptr, 0, 0, lens, cu, int(nseq), int(rows), 0u, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool pairs = r->layout == FV_ROTARY_PAIRS;
  if (r->dtype == FV_KV_BF16) return pairs ? fv::rotate_of<__nv_bfloat16, true>(a, m, s) : fv::rotate_of<__nv_bfloat16, false>(a, m, s);
  return pairs ? fv::rotate_of<__half, true>(a, m, s) : fv::rotate_of<__half, false>(a, m, s);
}
