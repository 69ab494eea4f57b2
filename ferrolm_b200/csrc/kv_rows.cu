// Rows of a key/value cache: written (rounded to 8 bits where the cache holds 8) together with the bounds of their blocks, and
// read back.
//
//   code = rn(top * x / most),  scale = most / top,  most = max |x| over a row of a head
//   lo, hi = componentwise min and max over the block's keys; their codes the same way with one scale for both
//
// Both are a pass over the data with a handful of operations for each value, and bound by the bytes.  94k rows of 8 heads of 128
// read back from e4m3 (605 MB): 95.5 us, 6.3 TB/s, 97% of the copy rate.  14k rows of prompts added as e4m3 (87 MB): 37 us, 2.4
// TB/s: a block's rows pass through one CTA, whose rounding and bounds leave its loads waiting.  24 single rows: 3.7 and 3.2 us.
#include <climits>

#include "kv.cuh"

namespace fv {

int kv_check(const fv_kv* kv, const fv_kv_batch* b, const char* who) {
  const std::string w(who);
  if (!kv || !b) return fail(FV_ERR_ARG, w + ": NULL cache or batch");
  if (kv->dtype != FV_KV_BF16 && kv->dtype != FV_KV_FP16) return fail(FV_ERR_UNSUPPORTED, w + ": dtype is bf16 or fp16");
  if (kv->kind < FV_KV_SAME || kv->kind > FV_KV_E4M3) return fail(FV_ERR_UNSUPPORTED, w + ": kind is same, int8 or e4m3");
  if (kv->dim != 64 && kv->dim != 96 && kv->dim != 128) return fail(FV_ERR_UNSUPPORTED, w + ": dim is 64, 96 or 128");
  if (kv->page_size != 16 && kv->page_size != 32 && kv->page_size != 64 && kv->page_size != 128)
    return fail(FV_ERR_UNSUPPORTED, w + ": page_size is 16, 32, 64 or 128");
  if (kv->heads == 0 || kv->heads > 65535) return fail(FV_ERR_UNSUPPORTED, w + ": heads is 1 to 65535");
  if (kv->pages > size_t(INT_MAX)) return fail(FV_ERR_UNSUPPORTED, w + ": pages does not fit 31 bits");
  if (kv->device < 0) return fail(FV_ERR_ARG, w + ": device index out of range");
  const bool coded = kv->kind != FV_KV_SAME;
  if (kv->pages && (!kv->k || !kv->v || !kv->bounds || !kv->bound_codes || !kv->bound_scale || (coded && (!kv->k_scale || !kv->v_scale))))
    return fail(FV_ERR_ARG, w + ": the cache lacks one of its buffers");
  if (!coded && (kv->k_scale || kv->v_scale)) return fail(FV_ERR_ARG, w + ": a cache of 16 bits has no scales");
  if (!kv_aligned(kv->k, 16) || !kv_aligned(kv->v, 16) || !kv_aligned(kv->bounds, 16) || !kv_aligned(kv->bound_codes, 16))
    return fail(FV_ERR_ARG, w + ": a buffer of the cache does not begin on 16 bytes");
  if (!kv_aligned(kv->k_scale, 4) || !kv_aligned(kv->v_scale, 4) || !kv_aligned(kv->bound_scale, 4))
    return fail(FV_ERR_ARG, w + ": scales do not begin on 4 bytes");
  if (b->rows > size_t(INT_MAX) / 2 || b->nseq > size_t(INT_MAX) / 8 || b->table_width > size_t(1) << 24 || b->table_stride > size_t(1) << 40)
    return fail(FV_ERR_UNSUPPORTED, w + ": rows, nseq or table_width is too large");
  if (b->table_width > size_t(INT_MAX) / kv->page_size) return fail(FV_ERR_UNSUPPORTED, w + ": positions in the table's last block leave 31 bits");
  if (b->rows && b->nseq && (!b->lens || (!b->table && b->table_width))) return fail(FV_ERR_ARG, w + ": NULL table or lens");
  if (!b->cu && b->rows != b->nseq) return fail(FV_ERR_ARG, w + ": without cu there is one row for each sequence");
  if (!kv_aligned(b->table, 4) || !kv_aligned(b->lens, 4) || !kv_aligned(b->cu, 4))
    return fail(FV_ERR_ARG, w + ": table, lens or cu does not begin on 4 bytes");
  return FV_OK;
}

namespace {

struct KvPool {
  unsigned char *k, *v;
  float *k_scale, *v_scale;
  unsigned char* bounds;
  int8_t* bound_codes;
  float* bound_scale;
  int heads, page_shift;
};

KvPool kv_pool(const fv_kv* kv) {
  return KvPool{static_cast<unsigned char*>(kv->k), static_cast<unsigned char*>(kv->v), kv->k_scale, kv->v_scale,
                static_cast<unsigned char*>(kv->bounds), kv->bound_codes, kv->bound_scale, int(kv->heads), __builtin_ctz(kv->page_size)};
}

struct KvInput {
  const unsigned char* p;
  size_t row, head;  // bytes
};

template <int N>
__device__ __forceinline__ float group_max(float x) {  // over N neighbouring lanes
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(FV_FULL, x, o));
  return x;
}

// One row of 8 values a lane over N lanes: codes (or the 16 bits as they are) to dst, the scale to *scale.  `on`: the lane
// has values of a row that is written.
template <class T, int KIND, int N>
__device__ __forceinline__ void write_row(const uint4& raw, bool on, unsigned char* dst, float* scale, bool first_lane) {
  if constexpr (KIND == FV_KV_SAME) {
    if (on) *reinterpret_cast<uint4*>(dst) = raw;
  } else {
    float x[8];
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float most = 0.f;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Pair<T>::to_float(w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
      fine = fine && kv_finite(f.x) && kv_finite(f.y);
      most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
    if (!fine) most = INFINITY;  // also where it is a NaN, which fmaxf drops
    most = group_max<N>(most);
    const bool ok = most < INFINITY, coded = ok && most > 0.f;
    const float down = kv_down(most), den = coded ? most * down : 1.f, up = coded ? Eight<KIND>::top * down : 0.f, inv = __fdiv_rn(1.f, den);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ok ? x[i] * up : 0.f;  // of a row that is not finite, codes of zero
    if (on) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(Eight<KIND>::pack(x, den, inv), Eight<KIND>::pack(x + 4, den, inv));
      if (first_lane) *scale = ok ? __fdiv_rn(most, Eight<KIND>::top) : __int_as_float(0x7FC00000);
    }
  }
}

// An item is the part of one block that this call writes, for one head; WARPS of them share an item (8: prompts, 1: a few rows
// for each sequence, four heads to a CTA).  One owner for each block's bounds means no atomics, and the order of the rows does
// not change a minimum.  N lanes hold a row, 8 values each, so a warp writes 32 / N rows at once.
template <class T, int KIND, int D, int WARPS>
__global__ void __launch_bounds__(WARPS > 1 ? 32 * WARPS : 128, WARPS > 1 ? 3 : 1) kv_add_kernel(KvPool pool, KvBatch m, KvInput kin, KvInput vin) {
  constexpr int N = D <= 64 ? 8 : 16, PER = 32 / N, L = D / 8;
  constexpr int ROW = KIND == FV_KV_SAME ? 2 * D : D, VAL = ROW / D;
  __shared__ float s_lo[WARPS > 1 ? WARPS * D : 1], s_hi[WARPS > 1 ? WARPS * D : 1];
  const int warp = threadIdx.x >> 5, lane = lane_id();
  const int head = WARPS > 1 ? int(blockIdx.y) : int(blockIdx.y) * 4 + warp, part = WARPS > 1 ? warp : 0;
  if (head >= pool.heads) return;  // whole warps, and with WARPS > 1 whole blocks
  const int shift = pool.page_shift, size = 1 << shift, item = blockIdx.x;
  const int b = m.cu ? kv_find(m, item, size, 2) : item;
  const int r0 = m.cu_at(b), r1 = max(m.cu_at(b + 1), r0), len = m.len(b);
  const int pos0 = len - (r1 - r0);  // of row r0
  const int j = (max(pos0, 0) >> shift) + (m.cu ? item - ((r0 >> shift) + 2 * b) : 0);
  const int begin = max(max(pos0, 0), j << shift), end = min(len, (j + 1) << shift);
  if (begin >= end) return;
  const int page = m.page(b, j);
  if (page < 0) return;
  const size_t at = size_t(page) * pool.heads + head;  // of the block's head
  const int sub = lane / N, l = lane % N;
  const bool in_row = l < L;
  float lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
  constexpr int AHEAD = WARPS > 1 ? 2 : 1;  // rows that a lane has on their way
  for (int p0 = begin + part * PER; p0 < end; p0 += AHEAD * WARPS * PER) {
    uint4 kr[AHEAD], vr[AHEAD];
#pragma unroll
    for (int z = 0; z < AHEAD; ++z) {
      const int p = p0 + z * WARPS * PER + sub;
      kr[z] = vr[z] = make_uint4(0, 0, 0, 0);
      if (in_row && p < end) {
        const size_t row = size_t(r0 + (p - pos0));
        kr[z] = __ldg(reinterpret_cast<const uint4*>(kin.p + row * kin.row + head * kin.head + l * 16));
        vr[z] = __ldg(reinterpret_cast<const uint4*>(vin.p + row * vin.row + head * vin.head + l * 16));
      }
    }
#pragma unroll
    for (int z = 0; z < AHEAD; ++z) {
      if (z && p0 + z * WARPS * PER >= end) break;  // whole warps
      const int p = p0 + z * WARPS * PER + sub, slot = p & (size - 1);
      const bool on = in_row && p < end;
      if (on) {
        const uint32_t w[4] = {kr[z].x, kr[z].y, kr[z].z, kr[z].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 f = Pair<T>::to_float(w[i]);
          f.x = kv_finite(f.x) ? f.x : 0.f;
          f.y = kv_finite(f.y) ? f.y : 0.f;
          lo[2 * i] = fminf(lo[2 * i], f.x), hi[2 * i] = fmaxf(hi[2 * i], f.x);
          lo[2 * i + 1] = fminf(lo[2 * i + 1], f.y), hi[2 * i + 1] = fmaxf(hi[2 * i + 1], f.y);
        }
      }
      const size_t row_at = at * size + slot;
      write_row<T, KIND, N>(kr[z], on, pool.k + row_at * ROW + l * 8 * VAL, pool.k_scale + row_at, l == 0);
      write_row<T, KIND, N>(vr[z], on, pool.v + row_at * ROW + l * 8 * VAL, pool.v_scale + row_at, l == 0);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int o = N; o < 32; o <<= 1) {
      lo[i] = fminf(lo[i], __shfl_xor_sync(FV_FULL, lo[i], o));
      hi[i] = fmaxf(hi[i], __shfl_xor_sync(FV_FULL, hi[i], o));
    }
  }
  if constexpr (WARPS > 1) {
    if (lane < L) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s_lo[part * D + lane * 8 + i] = lo[i], s_hi[part * D + lane * 8 + i] = hi[i];
    }
    __syncthreads();
    if (part) return;
    if (lane < L) {
#pragma unroll
      for (int w = 1; w < WARPS; ++w)
#pragma unroll
        for (int i = 0; i < 8; ++i) lo[i] = fminf(lo[i], s_lo[w * D + lane * 8 + i]), hi[i] = fmaxf(hi[i], s_hi[w * D + lane * 8 + i]);
    }
  }
  // with the bounds from before, unless the block begins here; then their codes: lanes 0 .. L-1 have 8 components each
  unsigned char* bounds = pool.bounds + at * (4 * D) + lane * 16;
  float most = 0.f;
  if (lane < L) {
    uint4 was[2];
    if (begin > j << shift) was[0] = *reinterpret_cast<uint4*>(bounds), was[1] = *reinterpret_cast<uint4*>(bounds + 2 * D);
    uint32_t nl[4], nh[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (begin > j << shift) {
        const float2 a = Pair<T>::to_float(reinterpret_cast<uint32_t*>(&was[0])[i]), c = Pair<T>::to_float(reinterpret_cast<uint32_t*>(&was[1])[i]);
        lo[2 * i] = fminf(lo[2 * i], a.x), lo[2 * i + 1] = fminf(lo[2 * i + 1], a.y);
        hi[2 * i] = fmaxf(hi[2 * i], c.x), hi[2 * i + 1] = fmaxf(hi[2 * i + 1], c.y);
      }
      nl[i] = Pair<T>::from_float(lo[2 * i], lo[2 * i + 1]);  // values of T: exact
      nh[i] = Pair<T>::from_float(hi[2 * i], hi[2 * i + 1]);
#pragma unroll
      for (int x = 0; x < 2; ++x) most = fmaxf(most, fmaxf(fabsf(lo[2 * i + x]), fabsf(hi[2 * i + x])));
    }
    *reinterpret_cast<uint4*>(bounds) = make_uint4(nl[0], nl[1], nl[2], nl[3]);
    *reinterpret_cast<uint4*>(bounds + 2 * D) = make_uint4(nh[0], nh[1], nh[2], nh[3]);
  }
  most = group_max<32>(most);
  if (lane < L) {
    const float down = kv_down(most), den = most > 0.f ? most * down : 1.f, up = 127.f * down, inv = __fdiv_rn(1.f, den);
    int8_t* codes = pool.bound_codes + at * (2 * D) + lane * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] *= up, hi[i] *= up;
    using E = Eight<FV_KV_INT8>;
    *reinterpret_cast<uint2*>(codes) = make_uint2(E::pack(lo, den, inv), E::pack(lo + 4, den, inv));
    *reinterpret_cast<uint2*>(codes + D) = make_uint2(E::pack(hi, den, inv), E::pack(hi + 4, den, inv));
    if (lane == 0) pool.bound_scale[at] = __fdiv_rn(most, 127.f);
  }
}

// ROWS rows of the call for all heads: a thread moves 16 bytes of a row of a head at a time, of keys and of values, and has those of
// four rows on their way.  A row's place is looked up once.
template <class T, int KIND, int D, int ROWS>
__global__ void __launch_bounds__(256) kv_vectors_kernel(KvPool pool, KvBatch m, unsigned char* k_out, unsigned char* v_out, bool wide) {
  constexpr int VALUES = KIND == FV_KV_SAME ? 8 : 16, L = D / VALUES, ROW = KIND == FV_KV_SAME ? 2 * D : D, AHEAD = 4;
  __shared__ long long s_at[ROWS];  // page * heads * size + slot: the row in head 0; -1: none
  const int first = blockIdx.x * ROWS;
  if (threadIdx.x < ROWS) {
    const int r = first + threadIdx.x;
    long long at = -1;
    if (r < m.cu_at(m.nseq)) {
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
      const int pos = m.len(lo) - max(m.cu_at(lo + 1), r + 1) + r;
      if (pos >= 0) {
        const int page = m.page(lo, pos >> pool.page_shift);
        if (page >= 0) at = ((long long)(page) * pool.heads << pool.page_shift) + (pos & ((1 << pool.page_shift) - 1));
      }
    }
    s_at[threadIdx.x] = at;
  }
  __syncthreads();
  const unsigned per_row = unsigned(pool.heads) * L, all = per_row * ROWS;
  for (unsigned i0 = threadIdx.x; i0 < all; i0 += AHEAD * 256) {
    uint4 in[AHEAD][2];
    float scale[AHEAD][2];
    size_t to[AHEAD];
    bool on[AHEAD];
#pragma unroll
    for (int z = 0; z < AHEAD; ++z) {
      const unsigned i = i0 + z * 256, r = i / per_row, x = i - r * per_row, head = x / L, l = x - head * L;
      const long long at0 = i < all ? s_at[r] : -1;
      on[z] = at0 >= 0;
      if (!on[z]) continue;
      const size_t at = size_t(at0) + (size_t(head) << pool.page_shift);
      to[z] = ((size_t(first) + r) * per_row + x) * (2 * VALUES);
      in[z][0] = __ldg(reinterpret_cast<const uint4*>(pool.k + at * ROW + l * 16));
      in[z][1] = __ldg(reinterpret_cast<const uint4*>(pool.v + at * ROW + l * 16));
      if constexpr (KIND != FV_KV_SAME) scale[z][0] = __ldg(pool.k_scale + at), scale[z][1] = __ldg(pool.v_scale + at);
    }
#pragma unroll
    for (int z = 0; z < AHEAD; ++z) {
      if (!on[z]) continue;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        uint4* const out = reinterpret_cast<uint4*>((which ? v_out : k_out) + to[z]);
        const uint4 c = in[z][which];
        if constexpr (KIND == FV_KV_SAME) {
          *out = c;
        } else {
          const float s = scale[z][which];
          const uint32_t codes[4] = {c.x, c.y, c.z, c.w};
          uint32_t w[8];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float y[4];
            Eight<KIND>::unpack(codes[x], y);
            w[2 * x] = Pair<T>::from_float(y[0] * s, y[1] * s), w[2 * x + 1] = Pair<T>::from_float(y[2] * s, y[3] * s);
          }
          if (wide)  // the results begin on 32 bytes: one store, where two would each leave half of every sector
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                         "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
          else
            out[0] = make_uint4(w[0], w[1], w[2], w[3]), out[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
    }
  }
}

template <class T, int KIND, int D>
int add_of(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvInput& k, const KvInput& v) {
  const KvBatch m = kv_batch(kv, b);
  const KvPool pool = kv_pool(kv);
  const size_t items = b->cu ? b->rows / kv->page_size + 2 * b->nseq : b->nseq;
  // a warp for a block where a sequence brings a few rows, eight where it brings a prompt
  if (b->rows <= 8 * b->nseq)
    kv_add_kernel<T, KIND, D, 1><<<dim3(unsigned(items), (kv->heads + 3) / 4), 128, 0, s>>>(pool, m, k, v);
  else
    kv_add_kernel<T, KIND, D, 8><<<dim3(unsigned(items), kv->heads), 256, 0, s>>>(pool, m, k, v);
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

template <class T, int KIND, int D>
int vectors_of(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, void* k, void* v) {
  const bool wide = kv_aligned(k, 32) && kv_aligned(v, 32);
  auto go = [&](auto rows_of) {
    constexpr int ROWS = decltype(rows_of)::value;
    kv_vectors_kernel<T, KIND, D, ROWS><<<unsigned((b->rows + ROWS - 1) / ROWS), 256, 0, s>>>(
        kv_pool(kv), kv_batch(kv, b), static_cast<unsigned char*>(k), static_cast<unsigned char*>(v), wide);
  };
  // few rows: a CTA for four of them, so that more SMs have some (24 rows of 8 heads in int8: 3.2 us, 5.2 by sixteens)
  if (b->rows <= 16 * 148) go(std::integral_constant<int, 4>());
  else go(std::integral_constant<int, 16>());
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

}  // namespace

}  // namespace fv

extern "C" int fv_kv_add_dev(const fv_kv* kv, void* stream, const fv_kv_batch* batch, const void* k, size_t k_row, size_t k_head,
                             const void* v, size_t v_row, size_t v_head) {
  FV_TRY(fv::kv_check(kv, batch, "fv_kv_add_dev"));
  if (batch->rows == 0 || batch->nseq == 0 || kv->pages == 0) return FV_OK;
  if (!k || !v) return fv::fail(FV_ERR_ARG, "fv_kv_add_dev: NULL rows");
  if (!fv::kv_aligned(k, 16) || !fv::kv_aligned(v, 16) || ((k_row | k_head | v_row | v_head) & 7))
    return fv::fail(FV_ERR_ARG, "fv_kv_add_dev: rows begin on 16 bytes and strides are multiples of 8 elements");
  fv::DeviceGuard g(kv->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  const fv::KvInput ki{static_cast<const unsigned char*>(k), 2 * k_row, 2 * k_head}, vi{static_cast<const unsigned char*>(v), 2 * v_row, 2 * v_head};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FV_KV_DISPATCH(kv, fv::add_of, kv, s, batch, ki, vi);
}

extern "C" int fv_kv_vectors_dev(const fv_kv* kv, void* stream, const fv_kv_batch* batch, void* k_out, void* v_out) {
  FV_TRY(fv::kv_check(kv, batch, "fv_kv_vectors_dev"));
  if (batch->rows == 0 || batch->nseq == 0 || kv->pages == 0) return FV_OK;
  if (!k_out || !v_out) return fv::fail(FV_ERR_ARG, "fv_kv_vectors_dev: NULL rows");
  if (!fv::kv_aligned(k_out, 16) || !fv::kv_aligned(v_out, 16)) return fv::fail(FV_ERR_ARG, "fv_kv_vectors_dev: rows begin on 16 bytes");
  fv::DeviceGuard g(kv->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FV_KV_DISPATCH(kv, fv::vectors_of, kv, s, batch, k_out, v_out);
}
