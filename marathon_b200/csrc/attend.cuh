// attend.cuh — arguments and bookkeeping shared by the attention kernels over a
// block-scaled cache (few rows: attend_block_scaled.cu, many: attend_rows.cu).
//
// Mathematics.  For a query row m at position x_m, keys j of its request:
//     s_j = scale * ks[b(j), h] * (q_m . kcode_j)         natural-log score
//     o   = sum_j e^{s_j} vs[b(j), h] vcode_j / sum_j e^{s_j}
// The value scale is moved into the exponent: with t_j = s_j log2 e + log2 vs_j and
// any reference M near max t_j,
//     P_j = 2^(t_j - M),   acc = sum P_j vcode_j,   l = sum P_j / vs_j,   o = acc / l.
// P_j is then in [0, 256] whatever the scales are and goes to f16 (11 bits) for the
// matrix product without ever losing the row's largest term; l, acc and M are fp32.
// One pass over the keys, by the running softmax (Milakov and Gimelshein 2018) in a known refinement: M
// follows the maximum only when it is passed by more than 2^8 (f16 holds that), and acc and l
// are rescaled only then.
//
// e4m3 codes convert to f16 exactly.  A query row is brought to f16 by a power of two
// that takes its largest element to [1, 2): a bf16 element keeps all its bits unless it is
// below 2^-14 of that, and loses at most 2^-25 of the largest then.  An fp16 element keeps its bits
// likewise.  The roundings to fewer than 32 bits are these, of P and of Q, which are what the f16 products
// ask for (tf32 ones run at half their rate), and the result's own: P's is 2^-11 of each weight, against
// the result's 2^-8 in bf16 and 2^-11 in fp16 (errors against 64 bits of 1.7e-3 and 2.5e-4; 32-bit weights
// give 1.7e-3 and 2.1e-4).  Below 2^-14 P is subnormal and off by up to 2^-25 of M's unit: an element to which
// only keys with such weights contribute, the heavier keys' values being zero there, has that absolute
// error and no relative one.
#pragma once

#include "serve_common.cuh"

namespace mshift {
namespace serve {

constexpr float kLazy = 8.0f;            // log2 of how far P may pass 1 before a rescale
constexpr float kNoKey = -3.402823466e38f;  // M of a row that has seen no key: below every score
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.4426950408889634f;

struct AttendArgs {
  const void* q;
  int64_t q_tok, q_head;  // elements
  int rows;               // rows of q
  const uint8_t* k;
  const uint8_t* v;
  int64_t blk, off, head;  // cache strides, bytes
  int64_t num_blocks;
  int bs;
  uint32_t bs_mul, bs_shift;  // t / bs = (high word of t * mul, + t) >> shift for t below 2^31
  const float* ks;
  const float* vs;
  int64_t ks_blk, ks_head, vs_blk, vs_head;
  const int32_t* tables;
  int64_t tab_stride;
  int width;
  const int32_t* qs;
  const int32_t* lens;
  int reqs, hq, hk, group;
  int max_len;
  float scale_log2;  // softmax scale * log2 e
  int causal, window;
  void* out;
  int64_t o_tok, o_head;
  float* lse;  // [rows, hq] or null
  // Requests of at most few_rows (token, group) rows go to the few-rows kernel, the others to
  // the many-rows one; each cuts the keys into splits of its own.  More than one: partial
  // results acc [split][D] and (M, l) [split] for each (row, head), joined afterwards.
  int few_rows;
  int chunk, nsplit;
  int64_t cap;  // rows a (request, head) has in part_o, or 0: part_o goes by (row of q, head)
  float* part_o;
  float2* part_ml;
  int rchunk, rsplit;
  float* rpart_o;  // by (row of q, head)
  float2* rpart_ml;
  int zero_tail;
  int max_q;     // the caller's bound on a request's tokens
  uint32_t* err;
};

// Division by the block size as a multiplication by its rounded-up reciprocal (Granlund and
// Montgomery 1994): exact for every t below 2^31.
inline void set_block_size(AttendArgs& a, int bs) {
  a.bs = bs;
  a.bs_shift = 0;
  while ((1ll << a.bs_shift) < bs) ++a.bs_shift;
  a.bs_mul = (uint32_t)((((1ull << a.bs_shift) - (uint64_t)bs) << 32) / (uint64_t)bs + 1);
}
__device__ __forceinline__ int block_column(const AttendArgs& a, int t) {
  return (int)((__umulhi((uint32_t)t, a.bs_mul) + (uint32_t)t) >> a.bs_shift);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// What a value scale adds to the scores and multiplies the weights' sum with.  One below 2^-64 reads as 2^-64;
// NaN goes to the scores alone, where the rows that do not see the key mask it.
__device__ __forceinline__ float value_log2(float vs) { return __log2f(max_nan(vs, kScaleFloor)); }
__device__ __forceinline__ float value_inverse(float vs) { return __frcp_rn(fmaxf(vs, kScaleFloor)); }

// One request's lengths, bounded by what the call's arrays hold.  Rows past the caller's bound have
// no place in the workspace, which the bound sized: no kernel sees them.
struct Request {
  int q0, n, seq;
  int past;         // rows left out behind its n
  long long start;  // position of its first row
};

__device__ __forceinline__ Request request_of(const AttendArgs& a, int r, bool report) {
  Request x;
  const int begin = a.qs[r], end = a.qs[r + 1];
  x.q0 = inside(begin, a.rows);
  const int n = max(inside(end, a.rows) - x.q0, 0);
  x.n = min(n, a.max_q);
  x.past = n - x.n;
  const int len = a.lens[r];
  x.start = len - ((long long)end - x.q0);  // the last row's place is the length's, whether q holds it or not
  const long long held = (long long)a.width * a.bs;
  x.seq = (int)min((long long)min(max(len, 0), a.max_len), held);
  if (report) {
    if (len > a.max_len || len < 0 || n > a.max_q || x.start < 0 || begin < 0 || end < begin ||
        end > a.rows)
      flag(a.err, MSHIFT_ERR_LENGTHS);
    if (len > held) flag(a.err, MSHIFT_ERR_POOL);
  }
  return x;
}

// Keys [lo, hi) that the row at position x sees.
__device__ __forceinline__ int2 seen(const AttendArgs& a, const Request& rq, long long x) {
  const long long hi = a.causal ? min(x + 1, (long long)rq.seq) : rq.seq;
  const long long lo = a.window > 0 ? max(x - a.window + 1, 0ll) : 0;
  if (x < 0 || hi <= lo) return make_int2(0, 0);
  return make_int2((int)lo, (int)hi);
}

// The keys [lo, hi) that some of a tile's rows see, those at positions first to last: later rows see later
// keys at both ends.  The last row's window may be empty where an earlier row's is not, behind a length
// that was cut.
__device__ __forceinline__ int2 seen_by_tile(const AttendArgs& a, const Request& rq, long long first,
                                             long long last) {
  const long long hi = a.causal ? min(last + 1, (long long)rq.seq) : rq.seq;
  const long long lo = a.window > 0 ? max(max(first, 0ll) - a.window + 1, 0ll) : 0;
  if (last < 0 || hi <= lo) return make_int2(0, 0);
  return make_int2((int)lo, (int)hi);
}

// Whether a row with this M and l has seen a key.  No comparison passes for NaN, so a row whose scores
// all are leaves M where it was, but its l is NaN then: it gets NaN, not the zeros of a row without keys.
__device__ __forceinline__ bool has_key(float M, float l) { return M > kNoKey || l != l; }

}  // namespace serve
}  // namespace mshift
