// rotary_axes.cu — rotary positions with several axes, queries and keys in one launch.
//
// Frequency i of a token turns by a = positions[axes[i]][token] * inv_freq[i]:
//     out[i]        = x[i] * cos a - x[i + half] * sin a
//     out[i + half] = x[i + half] * cos a + x[i] * sin a
// (NeoX half-split pairs; sin changes sign for the inverse).  The path is bound by
// HBM: each element is read once and written once, in 16-byte vectors that are
// rotary partners, so a thread holds both halves of its pairs.
//
// The angle.  A far position times an fp32 frequency has an fp32 rounding of up to 0.06 rad at a
// million, so the angle is formed in turns, modulo one, in fixed point: inv_freq / 2pi is an integer
// product with 2^k / 2pi, of which the bits behind the point are kept, and position times those wraps modulo
// one turn (Payne and Hanek 1983 reduce large arguments so).  What is left, in [-1/2, 1/2) turns, goes to
// fp32 sincospi.  Positions below 2^31 with frequencies below 32 take 64 bits, which leave an error below 2^-27
// turns; others take 128 of a product with 2^192 / 2pi: |position| (inv_freq 2^-192 + 2^-128) + 2^-62.  So
// the fp32 rounding, 2^-25, is the larger part at every 64-bit position for frequencies up to 2^64.  The
// long form is a call, which costs the short one nothing (the prefill below 128.3 us with and without it;
// 128 bits for all: 130).  One sin and cos a (token, frequency), shared by
// all heads through shared memory; they cost nothing that shows.
//
// Neighbouring threads have neighbouring vectors, then neighbouring heads, then tokens, so a CTA reads
// and writes whole rows; one pair of loads a thread at a time, since more
// registers cost more threads than they bring loads (30,720 tokens of 40 + 8 heads in bf16: 127 us
// against 133 with heads strided over the CTA, 148 with two pairs in flight, 208 with four and no
// shared memory; 756 MB at 5.9 TB/s).
#include <type_traits>

#include "serve_common.cuh"

namespace mshift {
namespace serve {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 8;      // most tokens of a CTA
constexpr int kRotMaxHalf = 256;   // frequencies: rotary up to 512
// 2^192 / 2pi, the lowest word first
constexpr uint64_t kTurn0 = 0x36d8a5664f10e410ull, kTurn1 = 0x7f09d5f47d4d3770ull, kTurn2 = 0x28be60db9391054aull;

struct RotArgs {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int64_t q_tok, q_head, k_tok, k_head, qo_tok, qo_head, ko_tok, ko_head;  // elements
  int64_t n;
  int hq, hk, head_size, half;
  const void* positions;
  int64_t pos_axis;  // elements between axes
  int pos64, n_axes;
  const float* inv_freq;
  const int32_t* axes;
  float sign;
  int tokens, slices;  // tokens a CTA, head slices
  uint32_t* err;
};

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
  T x[VEC];
};

// far * m 2^(e - 150) / pi half turns, modulo two, by way of m 2^192 / 2pi in four words, of which the bits
// from 214 - e on are 128 behind the point.  NaN for a frequency that is no number.
__device__ __noinline__ float far_half_turns(uint64_t m, int e, uint64_t far) {
  if (e == 255) return __int_as_float(0x7fffffff);
  const uint64_t p0 = m * kTurn0, c0 = __umul64hi(m, kTurn0);
  const uint64_t p1 = m * kTurn1 + c0, c1 = __umul64hi(m, kTurn1) + (p1 < c0);
  const uint64_t p2 = m * kTurn2 + c1, p3 = __umul64hi(m, kTurn2) + (p2 < c1);
  const int from = 214 - e, word = from >> 6, bit = from & 63;
  auto at = [&](int i) { return i == 0 ? p0 : i == 1 ? p1 : i == 2 ? p2 : i == 3 ? p3 : 0; };
  const uint64_t w0 = at(word), w1 = at(word + 1), w2 = at(word + 2);
  const uint64_t lo = w0 >> bit | w1 << 1 << (63 - bit), hi = w1 >> bit | w2 << 1 << (63 - bit);
  return (float)(int64_t)(far * hi + __umul64hi(far, lo)) * 0x1p-63f;
}

// position * inv_freq / pi half turns, modulo two.
__device__ __forceinline__ float half_turns(float inv, int64_t position) {
  const uint32_t b = __float_as_uint(inv);
  const int e = max((int)(b >> 23 & 0xff), 1);
  const uint64_t m = (b & 0x7fffffu) | (b & 0x7f800000u ? 0x800000u : 0u);  // |inv| = m 2^(e - 150)
  const uint64_t far = position < 0 ? 0 - (uint64_t)position : (uint64_t)position;
  float t;
  if (far >> 31 == 0 && e < 132) {
    const uint64_t lo = m * kTurn2, hi = __umul64hi(m, kTurn2);
    const int right = 150 - e;
    const uint64_t f = right < 64 ? lo >> right | hi << (64 - right) : right < 128 ? hi >> (right - 64) : 0;
    t = (float)(int64_t)(far * f) * 0x1p-63f;
  } else {
    t = far_half_turns(m, e, far);
  }
  return (position < 0) != (b >> 31 != 0) ? -t : t;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kRotThreads) rotary_axes_kernel(const RotArgs a) {
  __shared__ float2 s_cs[kRotTokens * kRotMaxHalf];
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int here = (int)min((int64_t)a.tokens, a.n - t0);
  for (int u = threadIdx.x; u < here * a.half; u += kRotThreads) {
    const int tok = u / a.half, i = u - tok * a.half;
    int axis = a.axes != nullptr ? a.axes[i] : 0;
    if (axis < 0 || axis >= a.n_axes) {
      flag(a.err, MSHIFT_EBIT_TABLE);
      axis = 0;
    }
    const int64_t at = axis * a.pos_axis + t0 + tok;
    const int64_t pos = a.pos64 ? static_cast<const int64_t*>(a.positions)[at]
                                : static_cast<const int32_t*>(a.positions)[at];
    float sn, cs;
    sincospif(half_turns(a.inv_freq[i], pos), &sn, &cs);
    s_cs[u] = make_float2(cs, sn * a.sign);
  }
  __syncthreads();

  using P = Pack<T, VEC>;
  using E = Elem<T>;
  const int rot = a.half / VEC;  // vectors of pairs in a head
  // the tail past the rotary is copied where the result goes elsewhere
  const int tail = (a.head_size - 2 * a.half) / VEC;
  const int per = rot + tail;
  const int heads = a.hq + a.hk;
  for (int u = threadIdx.x; u < here * per * a.slices; u += kRotThreads) {
    const int j = u % per, rest = u / per;
    const int slice = rest % a.slices, tok = rest / a.slices;
    const int64_t t = t0 + tok;
    float2 cs[VEC];
    if (j < rot) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) cs[e] = s_cs[tok * a.half + j * VEC + e];
    }
#pragma unroll 1
    for (int h = slice; h < heads; h += a.slices) {
      const T* src;
      T* dst;
      if (h < a.hq) {
        src = static_cast<const T*>(a.q) + t * a.q_tok + h * a.q_head;
        dst = static_cast<T*>(a.q_out) + t * a.qo_tok + h * a.qo_head;
      } else {
        src = static_cast<const T*>(a.k) + t * a.k_tok + (h - a.hq) * a.k_head;
        dst = static_cast<T*>(a.k_out) + t * a.ko_tok + (h - a.hq) * a.ko_head;
      }
      if (j >= rot) {
        const int at = 2 * a.half + (j - rot) * VEC;
        if (dst != src) *reinterpret_cast<P*>(dst + at) = *reinterpret_cast<const P*>(src + at);
        continue;
      }
      const P x = *reinterpret_cast<const P*>(src + j * VEC);
      const P y = *reinterpret_cast<const P*>(src + a.half + j * VEC);
      P xo, yo;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float xf = E::get(x.x[e]), yf = E::get(y.x[e]);
        xo.x[e] = E::put(xf * cs[e].x - yf * cs[e].y);
        yo.x[e] = E::put(yf * cs[e].x + xf * cs[e].y);
      }
      *reinterpret_cast<P*>(dst + j * VEC) = xo;
      *reinterpret_cast<P*>(dst + a.half + j * VEC) = yo;
    }
  }
}

template <typename T>
cudaError_t launch_rotary(RotArgs a, cudaStream_t stream) {
  constexpr int kVec = 16 / sizeof(T);
  auto whole = [](const void* p, int64_t tok, int64_t head) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && tok % kVec == 0 &&
                            head % kVec == 0);
  };
  // 16-byte vectors where every row starts on one and the halves split into
  // whole vectors; element by element otherwise (odd strides or frequencies)
  const bool vec = whole(a.q, a.q_tok, a.q_head) && whole(a.k, a.k_tok, a.k_head) &&
                   whole(a.q_out, a.qo_tok, a.qo_head) && whole(a.k_out, a.ko_tok, a.ko_head) &&
                   a.half % kVec == 0 && a.head_size % kVec == 0;
  // one token a CTA, so that a few thousand tokens still give every SM many CTAs; eight, which share
  // a CTA's start-up, once there are enough for that.  In us, one against eight, the launches back to back:
  //   tokens                     2,048      4,099      8,192     16,384     30,720
  //   40 + 8 heads of 128, bf16  15 16      27 22      49 40      93 70    169 125
  //   16 + 8 of 128, fp32, half  19 34      32 39      58 72    109 114    197 171
  //   8 + 1 of 64, bf16           6  4      11  5      19  7      42 14      79 25
  //   32 + 8 of 256, fp16        23 25      40 35      72 66    138 114
  // so the border is late for many rows and early for that fp32 case; two or four tokens a CTA, which no
  // rule here takes, lie between or below in most of these places
  a.tokens = a.n >= 16384 ? kRotTokens : 1;
  const int v = vec ? kVec : 1;
  const int per = a.half / v + (a.head_size - 2 * a.half) / v;
  a.slices = max(1, min(a.hq + a.hk, kRotThreads / (a.tokens * max(per, 1))));
  const int64_t grid = (a.n + a.tokens - 1) / a.tokens;
  if (vec)
    rotary_axes_kernel<T, kVec><<<(unsigned)grid, kRotThreads, 0, stream>>>(a);
  else
    rotary_axes_kernel<T, 1><<<(unsigned)grid, kRotThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace serve
}  // namespace mshift

extern "C" int mshift_rotary_axes(int32_t dtype, const void* q, int64_t q_tok, int64_t q_head,
                                  void* q_out, int64_t qo_tok, int64_t qo_head, int32_t hq,
                                  const void* k, int64_t k_tok, int64_t k_head, void* k_out,
                                  int64_t ko_tok, int64_t ko_head, int32_t hk, int64_t n,
                                  int32_t head_size, int32_t rotary, const void* positions,
                                  int64_t pos_axis_stride, int32_t pos_is_64, int32_t n_axes,
                                  const float* inv_freq, const int32_t* axes, int32_t inverse,
                                  uint32_t* err, void* stream) {
  using namespace mshift;
  using namespace mshift::serve;
  if (n < 0 || n > INT32_MAX || hq < 0 || hk < 0 || head_size <= 0 || rotary < 0 ||
      rotary % 2 != 0 || rotary > head_size || n_axes <= 0 || head_size > 1024)
    return MSHIFT_EINVAL;
  if (rotary > 2 * kRotMaxHalf) return MSHIFT_EUNSUPPORTED;
  if (n == 0 || hq + hk == 0) return MSHIFT_OK;
  if ((hq > 0 && (q == nullptr || q_out == nullptr)) ||
      (hk > 0 && (k == nullptr || k_out == nullptr)) || positions == nullptr || err == nullptr ||
      (rotary > 0 && inv_freq == nullptr))
    return MSHIFT_EINVAL;
  const RotArgs a{hq ? q : nullptr, hk ? k : nullptr, hq ? q_out : nullptr, hk ? k_out : nullptr,
                  q_tok, q_head, k_tok, k_head, qo_tok, qo_head, ko_tok, ko_head, n, hq, hk,
                  head_size, rotary / 2, positions, pos_axis_stride, pos_is_64, n_axes, inv_freq,
                  axes, inverse ? -1.0f : 1.0f, 1, 1, err};
  auto s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (dtype) {
    case MSHIFT_BF16: e = launch_rotary<__nv_bfloat16>(a, s); break;
    case MSHIFT_F16: e = launch_rotary<__half>(a, s); break;
    case MSHIFT_F32: e = launch_rotary<float>(a, s); break;
    default: return MSHIFT_EUNSUPPORTED;
  }
  return e == cudaSuccess ? MSHIFT_OK : cuda_fail(e);
}
