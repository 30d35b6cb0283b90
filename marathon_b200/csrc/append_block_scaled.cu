// append_block_scaled.cu — new keys and values into a paged e4m3 cache with one
// scale for each block and head.
//
// For a (block, head) that receives rows x of a request:
//     want = the least power of two s with max|x| <= 448 s   (finite values only)
//     new  = want, or max(old, want) if the block holds earlier tokens of the request
//     code = e4m3(x / new), earlier codes become e4m3(code * old / new) if new > old
// A power of two costs e4m3 nothing (its step is relative, so only the subnormal
// end moves by up to one binade) and makes division, growth and the attention's
// dequantisation exact but for codes that fall below 2^-6 * new.
//
// Bound by HBM: each row is read once, each code written once.  One warp has one (block,
// head), K and V: it keeps the block's rows in registers between the maximum and the rounding, so
// nothing is read twice for blocks of 16 tokens of up to 512 bytes a row; longer blocks
// are walked twice, the second time from L2.  Both sides' loads are issued before either is used, since
// what comes before them (the request, its length, its table) is a chain of dependent reads.
// Heads are neighbouring warps, which makes a CTA's reads and writes whole rows of
// the NHD layout.  No atomics, no workspace: a block's tokens are consecutive rows
// of one request, so the warp sees all of them.
//
// 28,608 tokens of 8 heads of 128 in bf16, from inside a block on: 38 us for 176 MB, 4.6 TB/s, bound by the
// chain of dependent reads before each warp's 12 KB; 72 us with a warp a side.  In fp32 77 us for 293 MB, 3.8
// TB/s: the kept rows' 170 registers leave one CTA an SM.
#include "serve_common.cuh"

namespace mshift {
namespace serve {
namespace {

constexpr int kAppWarps = 8;

struct AppArgs {
  const void* k;
  const void* v;
  int64_t k_tok, k_head, v_tok, v_head;  // elements
  int rows, heads;
  uint8_t* kc;
  uint8_t* vc;
  int64_t blk, off, head;  // cache strides, bytes
  int64_t num_blocks;
  int bs;
  float* ks;
  float* vs;
  int64_t ks_blk, ks_head, vs_blk, vs_head;
  const int32_t* tables;
  int64_t tab_stride;
  int width;
  const int32_t* qs;
  const int32_t* lens;
  int reqs;
  int64_t items;
  uint32_t* err;
};

// The least power of two s with amax <= 448 s, at least 2^-64: 448 = 0.875 * 2^9.
__device__ __forceinline__ float scale_for(float amax) {
  if (!(amax >= kScaleFloor)) return kScaleFloor;
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 126;  // amax = m 2^e, m in [1/2, 1)
  const int s = (b & 0x7fffffu) <= 0x600000u ? e - 9 : e - 8;
  return fmaxf(__uint_as_float((uint32_t)(max(s, -64) + 127) << 23), kScaleFloor);
}

// N elements (one 16-byte load) of a row.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& w, float* f) {
  constexpr int kPer = Elem<T>::kPer;
  Elem<T>::unpack(w.x, f);
  Elem<T>::unpack(w.y, f + kPer);
  Elem<T>::unpack(w.z, f + 2 * kPer);
  Elem<T>::unpack(w.w, f + 3 * kPer);
}

template <typename T, int D>
__global__ void __launch_bounds__(kAppWarps * 32) append_kernel(const AppArgs a) {
  constexpr int kVec = 16 / sizeof(T);        // elements of a 16-byte load
  constexpr int kVecs = D / kVec;             // loads of a row
  constexpr int kLanes = kVecs < 32 ? kVecs : 32;  // lanes of a row
  constexpr int kPerLane = kVecs / kLanes;    // loads of a lane in a row
  constexpr int kRows = 32 / kLanes;          // rows of one warp-wide load
  constexpr int kKeep = kPerLane == 1 && kRows == 1 ? 16 : 8;  // loads kept in registers
  constexpr int kChunk = kKeep / kPerLane * kRows;  // rows kept in registers

  if (blockIdx.x == gridDim.x - 1) {  // one CTA more than the work's looks the step over
    for (int r = threadIdx.x; r < a.reqs; r += kAppWarps * 32) {
      const int begin = a.qs[r], end = a.qs[r + 1], q0 = inside(begin, a.rows);
      if (begin < 0 || end < begin || end > a.rows ||
          (end > begin && a.lens[r] < (long long)end - q0))
        flag(a.err, MSHIFT_ERR_LENGTHS);
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kAppWarps + (threadIdx.x >> 5);
  const int h = (int)(w % a.heads);
  const int64_t item = w / a.heads;
  if (item >= a.items) return;

  // a request of n tokens touches at most n / bs + 2 blocks, and
  // floor(q_r / bs) + 2 r numbers its items without a scan over the requests
  const int r = find_request(a.reqs, item, [&](int i) {
    return (long long)row_start(a.qs, i, a.rows) / a.bs + 2ll * i;
  });
  const int end = a.qs[r + 1], q0 = row_start(a.qs, r, a.rows), n = inside(end, a.rows) - q0;
  if (n <= 0) return;
  // the last row's place is the length's, whether the call holds that row or not
  const long long start = a.lens[r] - ((long long)end - q0), stop = start + n;
  const long long base = (long long)q0 / a.bs + 2ll * r;
  if (item < base) return;
  const long long first = max(start, 0ll);  // rows before position 0 are not written
  const long long col = first / a.bs + (item - base);
  const long long lo = max(first, col * a.bs), hi = min(stop, (col + 1) * a.bs);
  if (lo >= hi) return;
  int block = -1;
  if (col < a.width) block = a.tables[(int64_t)r * a.tab_stride + col];
  if (block < 0 || block >= a.num_blocks) {
    if (lane == 0) flag(a.err, col < a.width ? MSHIFT_EBIT_SLOT : MSHIFT_ERR_POOL);
    return;
  }

  const int count = (int)(hi - lo), off0 = (int)(lo - col * a.bs);
  const int sub = lane / kLanes, part = (lane % kLanes) * kPerLane;  // row of the load, place in it
  const T* k_src = static_cast<const T*>(a.k) + (q0 + (lo - start)) * a.k_tok + h * a.k_head;
  const T* v_src = static_cast<const T*>(a.v) + (q0 + (lo - start)) * a.v_tok + h * a.v_head;
  const int64_t page = block * a.blk + h * a.head;

  auto load = [&](uint4* keep, const T* src, int64_t tok, int row0) {
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const int row = row0 + (i / kPerLane) * kRows + sub;
      keep[i] = make_uint4(0, 0, 0, 0);
      if (row < count)
        keep[i] = *reinterpret_cast<const uint4*>(src + row * tok + (part + i % kPerLane) * kVec);
    }
  };
  // Largest magnitude as its bits, which order as the values do: both halves of a word of 16-bit
  // elements at once.
  auto largest = [&](const uint4* keep, uint32_t top) {
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const uint32_t w[4] = {keep[i].x, keep[i].y, keep[i].z, keep[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        top = kVec == 8 ? __vmaxu2(top, w[e] & 0x7fff7fffu) : max(top, w[e] & 0x7fffffffu);
    }
    return top;
  };
  // The same without infinities and NaN, for rows that have some.
  auto largest_finite = [&](const T* src, int64_t tok) {
    float amax = 0.0f;
#pragma unroll 1
    for (int i = lane; i < count * D; i += 32) {
      const float m = fabsf(Elem<T>::get(src[i / D * tok + i % D]));
      if (m <= 3.402823466e38f) amax = fmaxf(amax, m);
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    return amax;
  };
  // The block's new scale; earlier codes follow it.
  auto rescale = [&](uint8_t* rows, float* scale, uint32_t top, const T* src, int64_t tok) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
      const uint32_t o = __shfl_xor_sync(0xffffffffu, top, d);
      top = kVec == 8 ? __vmaxu2(top, o) : max(top, o);
    }
    if (kVec == 8) top = __vmaxu2(top, top >> 16) & 0xffffu;
    float f[2];
    Elem<T>::unpack(top, f);
    const float amax = f[0] <= 3.402823466e38f ? f[0] : largest_finite(src, tok);
    float s = scale_for(amax);
    if (off0 > 0) {  // the block holds earlier tokens of the request
      const float old = *scale;
      s = fmaxf(old, s);
      if (s != old) {
        const float ratio = old / s;
        constexpr int kWords = D / 4;
#pragma unroll 1
        for (int i = lane; i < off0 * kWords; i += 32) {
          uint32_t* p = reinterpret_cast<uint32_t*>(rows + (i / kWords) * a.off) + i % kWords;
          const uint32_t c = *p;
          const uint32_t lo2 = e4m3x2_to_f16x2((uint16_t)c);
          const uint32_t hi2 = e4m3x2_to_f16x2((uint16_t)(c >> 16));
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo2));
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi2));
          *p = f32x2_to_e4m3x2(x.x * ratio, x.y * ratio) |
               ((uint32_t)f32x2_to_e4m3x2(y.x * ratio, y.y * ratio) << 16);
        }
      }
    }
    __syncwarp();  // every lane has read the old scale
    if (lane == 0) *scale = s;
    return s;
  };
  auto store = [&](const uint4* keep, uint8_t* rows, float s, int row0) {
    // x / s: the scales written here are powers of two, whose reciprocal is exact
    const float inv = 1.0f / s;
    uint8_t* to = rows + (off0 + row0 + sub) * a.off + part * kVec;
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      float f[kVec];
      unpack16<T>(keep[i], f);
      uint32_t o[kVec / 4];
#pragma unroll
      for (int e = 0; e < kVec / 4; ++e)
        o[e] = f32x2_to_e4m3x2(f[4 * e] * inv, f[4 * e + 1] * inv) |
               ((uint32_t)f32x2_to_e4m3x2(f[4 * e + 2] * inv, f[4 * e + 3] * inv) << 16);
      if (row0 + (i / kPerLane) * kRows + sub < count) {
        uint32_t* p = reinterpret_cast<uint32_t*>(to + (i / kPerLane) * kRows * a.off + i % kPerLane * kVec);
        if constexpr (kVec == 8)
          *reinterpret_cast<uint2*>(p) = make_uint2(o[0], o[1]);
        else
          *p = o[0];
      }
    }
  };
  // A scale of another origin, kept because it is large enough, takes the division.
  auto store_divided = [&](const T* src, int64_t tok, uint8_t* rows, float s) {
#pragma unroll 1
    for (int i = lane; i < count * (D / 2); i += 32) {
      const T* x = src + i / (D / 2) * tok + i % (D / 2) * 2;
      *reinterpret_cast<uint16_t*>(rows + (off0 + i / (D / 2)) * a.off + i % (D / 2) * 2) =
          f32x2_to_e4m3x2(Elem<T>::get(x[0]) / s, Elem<T>::get(x[1]) / s);
    }
  };
  auto power_of_two = [](float s) { return (__float_as_uint(s) & 0x7fffffu) == 0; };

  float* k_scale = a.ks + block * a.ks_blk + h * a.ks_head;
  float* v_scale = a.vs + block * a.vs_blk + h * a.vs_head;
  uint8_t *k_rows = a.kc + page, *v_rows = a.vc + page;
  if (count <= kChunk) {
    uint4 kk[kKeep], vv[kKeep];
    load(kk, k_src, a.k_tok, 0);
    load(vv, v_src, a.v_tok, 0);
    const float ks = rescale(k_rows, k_scale, largest(kk, 0), k_src, a.k_tok);
    if (power_of_two(ks))
      store(kk, k_rows, ks, 0);
    else
      store_divided(k_src, a.k_tok, k_rows, ks);
    const float vs = rescale(v_rows, v_scale, largest(vv, 0), v_src, a.v_tok);
    if (power_of_two(vs))
      store(vv, v_rows, vs, 0);
    else
      store_divided(v_src, a.v_tok, v_rows, vs);
    return;
  }
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const T* src = side ? v_src : k_src;
    const int64_t tok = side ? a.v_tok : a.k_tok;
    uint8_t* rows = side ? v_rows : k_rows;
    uint4 keep[kKeep];
    uint32_t top = 0;
#pragma unroll 1
    for (int row0 = 0; row0 < count; row0 += kChunk) {
      load(keep, src, tok, row0);
      top = largest(keep, top);
    }
    const float s = rescale(rows, side ? v_scale : k_scale, top, src, tok);
    if (!power_of_two(s)) {
      store_divided(src, tok, rows, s);
      continue;
    }
#pragma unroll 1
    for (int row0 = 0; row0 < count; row0 += kChunk) {
      load(keep, src, tok, row0);
      store(keep, rows, s, row0);
    }
  }
}

template <typename T>
int launch_append(const AppArgs& a, int head_size, cudaStream_t stream) {
  const int64_t warps = a.items * a.heads;
  const int64_t grid = (warps + kAppWarps - 1) / kAppWarps + 1;
  if (grid > INT32_MAX) return MSHIFT_EINVAL;
  const dim3 g((unsigned)grid), b(kAppWarps * 32);
  switch (head_size) {
    case 64: append_kernel<T, 64><<<g, b, 0, stream>>>(a); break;
    case 128: append_kernel<T, 128><<<g, b, 0, stream>>>(a); break;
    case 256: append_kernel<T, 256><<<g, b, 0, stream>>>(a); break;
    default: return MSHIFT_EUNSUPPORTED;
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MSHIFT_OK : cuda_fail(e);
}

}  // namespace
}  // namespace serve
}  // namespace mshift

extern "C" int mshift_append_block_scaled(
    int32_t dtype, const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok,
    int64_t v_head, int32_t rows, const mshift_paged* paged, void* k_base, void* v_base,
    float* k_scale, int64_t ks_blk, int64_t ks_head, float* v_scale, int64_t vs_blk,
    int64_t vs_head, const int32_t* block_tables, int64_t table_stride, int32_t width,
    const int32_t* query_start, const int32_t* seq_lens, int32_t reqs, uint32_t* err,
    void* stream) {
  using namespace mshift;
  using namespace mshift::serve;
  if (paged == nullptr || rows < 0 || reqs < 0 || width < 0 || table_stride < width)
    return MSHIFT_EINVAL;
  if (paged->dtype != MSHIFT_E4M3) return MSHIFT_EUNSUPPORTED;
  if (paged->heads <= 0 || paged->block_size <= 0 || paged->num_blocks < 0) return MSHIFT_EINVAL;
  if (rows == 0 || reqs == 0) return MSHIFT_OK;
  if (k == nullptr || v == nullptr || k_base == nullptr || v_base == nullptr ||
      k_scale == nullptr || v_scale == nullptr || (width > 0 && block_tables == nullptr) ||
      query_start == nullptr || seq_lens == nullptr || err == nullptr)
    return MSHIFT_EINVAL;
  const int64_t vec = dtype == MSHIFT_F32 ? 4 : 8;
  const auto odd = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
  if (odd(k) || odd(v) || odd(k_base) || odd(v_base) || k_tok % vec || k_head % vec ||
      v_tok % vec || v_head % vec || paged->blk_stride % 16 || paged->off_stride % 16 ||
      paged->head_stride % 16)
    return MSHIFT_EINVAL;
  const AppArgs a{k, v, k_tok, k_head, v_tok, v_head, rows, paged->heads,
                  static_cast<uint8_t*>(k_base), static_cast<uint8_t*>(v_base),
                  paged->blk_stride, paged->off_stride, paged->head_stride, paged->num_blocks,
                  paged->block_size, k_scale, v_scale, ks_blk, ks_head, vs_blk, vs_head,
                  block_tables, table_stride, width, query_start, seq_lens, reqs,
                  (int64_t)rows / paged->block_size + 2ll * reqs, err};
  auto s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case MSHIFT_BF16: return launch_append<__nv_bfloat16>(a, paged->head_size, s);
    case MSHIFT_F16: return launch_append<__half>(a, paged->head_size, s);
    case MSHIFT_F32: return launch_append<float>(a, paged->head_size, s);
    default: return MSHIFT_EUNSUPPORTED;
  }
}
