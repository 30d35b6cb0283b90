// attend_block_scaled.cu — attention over a block-scaled e4m3 paged cache: the kernel for
// few query rows (decoding), the join of split results, and the entry point.
//
// A CTA has one (request, kv head, tile of NT * 8 query rows, split of the keys); its four
// warps take 16-token steps in turn and join through shared memory at the end.
// The rows are the request's (token, query head of the group) pairs, so the heads that
// share a KV head read it once.
//
// Bound by HBM: 2 D bytes a (token, KV head) against 2 * 16 * D * 8 NT operations, so the
// rows ride the narrow side of m16n8k16 and keys and values, as the wide side, go to the matrix
// instructions without being rearranged:
//   scores  S^T[16 tokens x 8 rows] += K[16 x 16 dims] Q^T.  The order of the dims in a
//           product is free, so lane (g, c) loads 16 contiguous codes of tokens g and g+8 at
//           dims 64 u + 16 c, and Q is laid out to match once.
//   values  O^T[16 dims x 8 rows] += V^T[16 dims x 16 tokens] P^T.  Lane (g, c) loads the
//           codes of tokens 2c, 2c+1, 2c+8, 2c+9 at D/8 contiguous dims from g D/8; byte pairs of two
//           tokens are the f16 pairs that the fragment wants.
// P^T's fragment is S^T's transposed, which movmatrix does in registers.  Codes and scales come
// through a ring of three stages in shared memory that each warp fills for itself with asynchronous
// copies, two steps (8 KB at D = 128) ahead of the one it works on; chunks of 16 bytes are swizzled
// so that the fragments' reads hit every bank once.
//
// 64 sessions of 2k-32k tokens, 32 query heads over 8 of 128: 358-396 us by the box, 4.8-5.3 TB/s, 0.73-0.81
// of the copy peak (head size 64: 249, 256: 705; blocks of 24 tokens: 385).  58 % of the issue slots are
// used, by some 210 instructions a step, half of them conversions and products; the rest of the time a
// scheduler's four warps wait, each for its own chain.
// Four stages leave three CTAs an SM instead of four: 447 us; five: 569; the next step's codes in registers
// instead of the ring: 502; five or six CTAs an SM with spilled registers: 403, 412.
#include "attend.cuh"

namespace mshift {
namespace serve {

template <int D, typename T>
cudaError_t launch_attend_rows(const AttendArgs& a, cudaStream_t stream);

namespace {

constexpr int kWarps = 4;

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

__device__ __forceinline__ void copy16(void* to, const void* from, bool take) {  // or zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(to))),
               "l"(from), "r"(take ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(to))),
               "l"(from)
               : "memory");
}

// One 16-token step of a warp.
template <int D>
struct Stage {
  uint8_t k[16 * D], v[16 * D];
  float ks[16], vs[16];  // a block's at its first token's place, or each token's
  static constexpr int kCopies = D / 32;  // 16-byte copies a lane, K or V
  // place of 16-byte chunk c of token t
  __device__ static int k_at(int t, int c) { return t * D + ((c ^ (D > 64 ? (t & 1) * 4 : 0)) << 4); }
  __device__ static int v_at(int t, int c) {
    return t * D + ((c ^ (D > 64 ? (t >> 1 & 3) * 2 : (t >> 1 & 1) * 2)) << 4);
  }
};
template <int D>
constexpr int kStages = D == 256 ? 2 : 3;

template <int D, int NT, bool PAGE16, typename T>
__global__ void __launch_bounds__(kWarps * 32) attend_few_kernel(const AttendArgs a, int tiles) {
  constexpr int kRows = NT * 8;
  constexpr int kMt = D / 16;  // 16-dim tiles of O^T
  constexpr int kS = kStages<D>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  float(*s_o)[kRows][D + 4] = reinterpret_cast<float(*)[kRows][D + 4]>(ring);  // after the last step

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  // with zero_tail the result is new memory: rows that nothing else writes become zeros
  auto clear = [&](int64_t row, int head, int heads) {
    for (int i = threadIdx.x; i < heads * D; i += kWarps * 32)
      static_cast<T*>(a.out)[row * a.o_tok + (head + i / D) * a.o_head + i % D] = Elem<T>::put(0.0f);
    for (int i = threadIdx.x; i < heads && a.lse != nullptr; i += kWarps * 32)
      a.lse[row * a.hq + head + i] = -INFINITY;
  };
  if (a.zero_tail) {  // rows of no request
    const int before = row_start(a.qs, 0, a.rows), behind = row_start(a.qs, a.reqs, a.rows);
    const int64_t none = before + (int64_t)a.rows - behind;
    for (int64_t i = blockIdx.x; i < none; i += gridDim.x)
      clear(i < before ? i : i - before + behind, 0, a.hq);
  }
  asm volatile("griddepcontrol.launch_dependents;");  // the join may be made ready
  // heads fastest: in the NHD layouts neighbouring CTAs read neighbouring bytes
  int64_t id = blockIdx.x;
  const int h = (int)(id % a.hk);
  id /= a.hk;
  const int tile = (int)(id % tiles);
  id /= tiles;
  const int split = (int)(id % a.nsplit);
  const int r = (int)(id / a.nsplit);
  const Request rq = request_of(a, r, threadIdx.x == 0 && h == 0 && tile == 0 && split == 0);
  if (a.zero_tail && tile == 0 && split == 0)  // rows past the caller's bound
    for (int i = 0; i < rq.past; ++i) clear(rq.q0 + rq.n + i, h * a.group, a.group);
  const int all = rq.n * a.group, m0 = tile * kRows;
  if (all > a.few_rows || m0 >= all) return;
  const int live = min(kRows, all - m0);

  // what this lane's rows 8 nt + 2c, 8 nt + 2c + 1 see, and the keys of the whole tile
  int2 mine[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int m = i * 8 + 2 * c + e;
      mine[i][e] = m < live ? seen(a, rq, rq.start + (m0 + m) / a.group) : make_int2(0, 0);
    }
  const long long first_at = rq.start + m0 / a.group, last_at = rq.start + (m0 + live - 1) / a.group;
  const int2 tile_see = seen_by_tile(a, rq, first_at, last_at);
  const int2 head = seen(a, rq, max(first_at, 0ll)), last = seen(a, rq, last_at);
  const int lo = max(tile_see.x, split * a.chunk);
  const int hi = min(tile_see.y, split * a.chunk + a.chunk);
  const int full_lo = max(last.x, lo);  // keys that every row sees
  const int full_hi = min(a.causal ? min(head.y, last.y) : last.y, hi);
  const bool all_live = first_at >= 0;

  const int32_t* table = a.tables + (int64_t)r * a.tab_stride;
  const uint8_t* kh = a.k + h * a.head;
  const uint8_t* vh = a.v + h * a.head;
  const float* ksh = a.ks + h * a.ks_head;
  const float* vsh = a.vs + h * a.vs_head;
  const int first = lo < hi ? lo / 16 : 0, steps = lo < hi ? (hi + 15) / 16 - first : 0;

  Stage<D>* stage = reinterpret_cast<Stage<D>*>(ring) + (threadIdx.x >> 5) * kS;
  // Where step st's tokens lie: the step's block (PAGE16), or that of token lane & 15; -1 for
  // a bad block or nothing to read.
  auto block_of = [&](int st) -> int {
    const int t = (first + st) * 16 + (PAGE16 ? 0 : lane & 15);
    if (st >= steps || (!PAGE16 && (t < lo || t >= hi))) return -1;
    const int b = table[block_column(a, t)];
    if (b >= 0 && b < a.num_blocks) return b;
    flag(a.err, MSHIFT_EBIT_SLOT);
    return -1;
  };
  // Starts the copies of step st; tokens outside [lo, hi) or in a bad block are zeros, and a bad
  // block's value scale is -inf.
  auto fetch = [&](int st, int b) {
    if (st < steps) {
      Stage<D>& x = stage[st / kWarps % kS];
      const int t0 = (first + st) * 16, mine = t0 + (PAGE16 ? 0 : lane & 15);
      const long long base = b * a.blk + (mine - block_column(a, mine) * a.bs) * a.off;
      unsigned in = PAGE16 ? (b >= 0 ? 0xffffu : 0u) : __ballot_sync(0xffffffffu, b >= 0) & 0xffffu;
      if (t0 < lo) in &= 0xffffu << (lo - t0);
      if (t0 + 16 > hi) in &= 0xffffu >> (t0 + 16 - hi);
#pragma unroll
      for (int i = 0; i < Stage<D>::kCopies; ++i) {
        const int q = lane + 32 * i, t = q / (D / 16), c = q % (D / 16);
        const bool take = (in >> t) & 1;
        const long long at =
            (PAGE16 ? base + t * a.off : __shfl_sync(0xffffffffu, base, t)) + 16 * c;
        copy16(x.k + Stage<D>::k_at(t, c), take ? kh + at : kh, take);
        copy16(x.v + Stage<D>::v_at(t, c), take ? vh + at : vh, take);
      }
      if (PAGE16 ? lane < 2 : true) {
        const bool is_v = PAGE16 ? lane == 1 : lane >= 16;
        float* to = (is_v ? x.vs : x.ks) + (PAGE16 ? 0 : lane & 15);
        if (b >= 0)
          copy4(to, is_v ? vsh + b * a.vs_blk : ksh + b * a.ks_blk);
        else
          *to = is_v ? -INFINITY : 0.0f;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  int ahead = block_of(warp);
#pragma unroll 1
  for (int i = 0; i < kS - 1; ++i) {
    fetch(warp + i * kWarps, ahead);
    ahead = block_of(warp + (i + 1) * kWarps);
  }
  // queries: f16 after a power of two for each row
  uint32_t qf[NT][D / 16][2];
  float rf[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int m = i * 8 + g;
    float x[D / 4];
    float top = 0.0f;
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {  // 8 elements of 16 bits
        uint4 w = make_uint4(0, 0, 0, 0);
        if (m < live) {
          const T* src = static_cast<const T*>(a.q) + (rq.q0 + (m0 + m) / a.group) * a.q_tok +
                         (h * a.group + (m0 + m) % a.group) * a.q_head + 64 * u + 16 * c + 8 * p;
          w = *reinterpret_cast<const uint4*>(src);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) Elem<T>::unpack(word(w, e), x + 16 * u + 8 * p + 2 * e);
      }
    }
#pragma unroll
    for (int e = 0; e < D / 4; ++e) top = fmaxf(top, fabsf(x[e]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // exponent of the largest element; rows of zeros, infinities or NaN as they are
    int e2 = (int)(__float_as_uint(top) >> 23) - 127;
    if (e2 < -126 || e2 > 126) e2 = 0;
    const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
    const float up = __uint_as_float((uint32_t)(127 + e2) << 23) * a.scale_log2;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const float* y = x + 16 * (s / 4) + 4 * (s % 4);
      qf[i][s][0] = pack_f16x2(y[0] * down, y[1] * down);
      qf[i][s][1] = pack_f16x2(y[2] * down, y[3] * down);
    }
    rf[i][0] = __shfl_sync(0xffffffffu, up, 8 * c);
    rf[i][1] = __shfl_sync(0xffffffffu, up, 8 * c + 4);
  }

  float M[NT][2], l[NT][2], o[NT][kMt][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    M[i][0] = M[i][1] = kNoKey;
    l[i][0] = l[i][1] = 0.0f;
#pragma unroll
    for (int j = 0; j < kMt; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.0f;
  }

#pragma unroll 1
  for (int st = warp; st < steps; st += kWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kS - 2) : "memory");
    __syncwarp();
    fetch(st + (kS - 1) * kWarps, ahead);
    ahead = block_of(st + kS * kWarps);
    const Stage<D>& cur = stage[st / kWarps % kS];
    const int t0 = (first + st) * 16;

    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      const uint4 k0 = *reinterpret_cast<const uint4*>(cur.k + Stage<D>::k_at(g, 4 * u + c));
      const uint4 k1 = *reinterpret_cast<const uint4*>(cur.k + Stage<D>::k_at(g + 8, 4 * u + c));
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint32_t w0 = word(k0, d), w1 = word(k1, d);
        const uint32_t f[4] = {e4m3x2_to_f16x2((uint16_t)w0), e4m3x2_to_f16x2((uint16_t)w1),
                               e4m3x2_to_f16x2((uint16_t)(w0 >> 16)),
                               e4m3x2_to_f16x2((uint16_t)(w1 >> 16))};
#pragma unroll
        for (int i = 0; i < NT; ++i) mma_f16(s[i], f, qf[i][4 * u + d]);
      }
    }

    // t = S ks rf + log2 vs, masked
    float ks[2], lv[2], rv[2];
    bool good[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int t = PAGE16 ? 0 : g + 8 * e;
      ks[e] = cur.ks[t];
      good[e] = cur.vs[t] != -INFINITY;
      lv[e] = value_log2(cur.vs[t]);
      rv[e] = value_inverse(cur.vs[t]);
    }
    const bool whole = __all_sync(0xffffffffu, all_live && t0 >= full_lo && t0 + 16 <= full_hi &&
                                                   good[0] && good[1]);
    bool passed = false;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float t = fmaf(s[i][e] * rf[i][e & 1], ks[e >> 1], lv[e >> 1]);
        if (!whole) {
          const int key = t0 + g + 8 * (e >> 1);
          const int2 see = mine[i][e & 1];
          if (!good[e >> 1] || key < max(see.x, lo) || key >= min(see.y, hi)) t = -INFINITY;
        }
        s[i][e] = t;
        passed |= t > M[i][e & 1] + kLazy;
      }
    if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(M[i][e], fmaxf(s[i][e], s[i][e + 2]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float by = ex2(M[i][e] - top);
          M[i][e] = top;
          l[i][e] *= by;
#pragma unroll
          for (int j = 0; j < kMt; ++j) {
            o[i][j][e] *= by;
            o[i][j][e + 2] *= by;
          }
        }
    }
    uint32_t p[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = ex2(s[i][e] - M[i][e & 1]);
        l[i][e & 1] = fmaf(s[i][e], rv[e >> 1], l[i][e & 1]);
      }
      p[i][0] = transpose8x8(pack_f16x2(s[i][0], s[i][1]));
      p[i][1] = transpose8x8(pack_f16x2(s[i][2], s[i][3]));
    }
    // two 16-bit pairs of a word: dims 2j (rows g) and 2j + 1 (rows g + 8) of tokens
    // (2c, 2c+1) and (2c+8, 2c+9)
    constexpr int kWords = D == 64 ? 2 : 4;  // words of a lane's V row in one read
#pragma unroll
    for (int u = 0; u < (D == 256 ? 2 : 1); ++u) {
      uint4 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = 2 * c + (e & 1) + 8 * (e >> 1);
        if constexpr (D == 64) {
          const uint2 w =
              *reinterpret_cast<const uint2*>(cur.v + Stage<D>::v_at(t, g >> 1) + 8 * (g & 1));
          v[e] = make_uint4(w.x, w.y, 0, 0);
        } else {
          v[e] = *reinterpret_cast<const uint4*>(cur.v + Stage<D>::v_at(t, 8 * u + g));
        }
      }
#pragma unroll
      for (int b = 0; b < 2 * kWords; ++b) {
        const uint32_t sel = b % 2 == 0 ? 0x5140 : 0x7362;
        const uint32_t x = __byte_perm(word(v[0], b / 2), word(v[1], b / 2), sel);
        const uint32_t y = __byte_perm(word(v[2], b / 2), word(v[3], b / 2), sel);
        const uint32_t f[4] = {e4m3x2_to_f16x2((uint16_t)x), e4m3x2_to_f16x2((uint16_t)(x >> 16)),
                               e4m3x2_to_f16x2((uint16_t)y), e4m3x2_to_f16x2((uint16_t)(y >> 16))};
#pragma unroll
        for (int i = 0; i < NT; ++i) mma_f16(o[i][8 * u + b], f, p[i]);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();  // the ring becomes the place where the warps join

  // join the warps
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[i][e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      const int m = i * 8 + 2 * c + e;
      if (g == 0) {
        s_m[warp][m] = M[i][e];
        s_l[warp][m] = x;
      }
#pragma unroll
      for (int j = 0; j < kMt; ++j) {
        const int dim = D == 64 ? 8 * g + 2 * j : 128 * (j / 8) + 16 * g + 2 * (j % 8);
        *reinterpret_cast<float2*>(&s_o[warp][m][dim]) = make_float2(o[i][j][e], o[i][j][e + 2]);
      }
    }
  __syncthreads();
  for (int at = threadIdx.x; at < live * (D / 4); at += kWarps * 32) {
    const int m = at / (D / 4), d = at % (D / 4) * 4;
    float top = s_m[0][m];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][m]);
    float sum = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float by = ex2(s_m[w][m] - top);
      sum = fmaf(s_l[w][m], by, sum);
      const float4 y = *reinterpret_cast<const float4*>(&s_o[w][m][d]);
      x[0] = fmaf(y.x, by, x[0]);
      x[1] = fmaf(y.y, by, x[1]);
      x[2] = fmaf(y.z, by, x[2]);
      x[3] = fmaf(y.w, by, x[3]);
    }
    const int64_t row = rq.q0 + (m0 + m) / a.group;
    const int hq = h * a.group + (m0 + m) % a.group;
    if (a.nsplit > 1) {
      const int64_t part =
          (a.cap ? (((int64_t)r * a.hk + h) * a.cap + m0 + m) : row * a.hq + hq) * a.nsplit + split;
      *reinterpret_cast<float4*>(a.part_o + part * D + d) = make_float4(x[0], x[1], x[2], x[3]);
      if (d == 0) a.part_ml[part] = make_float2(top, sum);
    } else {
      const bool any = has_key(top, sum);
      const float by = any ? 1.0f / sum : 0.0f;
      T* dst = static_cast<T*>(a.out) + row * a.o_tok + hq * a.o_head + d;
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[e] = Elem<T>::put(any ? x[e] * by : 0.0f);
      if (d == 0 && a.lse != nullptr)
        a.lse[row * a.hq + hq] = any ? (top + log2f(sum)) * kLn2 : -INFINITY;
    }
  }
}

// o = sum_s 2^(M_s - M) acc_s / sum_s 2^(M_s - M) l_s over the splits of one (row, head), which WPR
// warps share: one where there are few splits (a chunk's many rows), eight where a few rows
// have many (decoding over a long cache).  ROWS: of the many-rows kernel.
constexpr int kJoinWarps = 8;
template <int D, typename T, bool ROWS, int WPR>
__global__ void __launch_bounds__(kJoinWarps * 32) attend_join_kernel(const AttendArgs a, int64_t total) {
  constexpr int kVec = D / 32;  // dims of a lane
  constexpr unsigned kAll = 0xffffffffu;
  __shared__ float s_x[WPR > 1 ? kJoinWarps : 1][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part_of = warp % WPR;
  const int chunk = ROWS ? a.rchunk : a.chunk, nsplit = ROWS ? a.rsplit : a.nsplit;
  const int64_t id = (int64_t)blockIdx.x * (kJoinWarps / WPR) + warp / WPR;
  int64_t row = -1;
  int hq = 0;
  Request rq{};
  if (id < total) {
    if (!ROWS && a.cap) {
      const int64_t m = id % a.cap, rh = id / a.cap;
      rq = request_of(a, (int)(rh / a.hk), false);
      if (m < (int64_t)rq.n * a.group) row = rq.q0 + m / a.group;
      hq = (int)(rh % a.hk) * a.group + (int)(m % a.group);
    } else if (id / a.hq < row_start(a.qs, a.reqs, a.rows)) {
      row = id / a.hq;
      hq = (int)(id % a.hq);
      const int r =
          find_request(a.reqs, row, [&](int i) { return (long long)row_start(a.qs, i, a.rows); });
      rq = request_of(a, r, false);
      if (row < rq.q0 || row >= rq.q0 + rq.n) row = -1;
    }
    if (((int64_t)rq.n * a.group > a.few_rows) != ROWS) row = -1;
  }
  // nothing the kernel before wrote has been read so far
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (WPR == 1 && row < 0) return;  // else the row's warps, all alike, still meet below

  const int2 see = row < 0 ? make_int2(0, 0) : seen(a, rq, rq.start + (row - rq.q0));
  // splits that hold a key of this row; at least one, for a row without keys
  const int s0 = see.x / chunk, s1 = row < 0 ? s0 : max((see.y + chunk - 1) / chunk, s0 + 1);
  const int64_t part = id * nsplit;
  const float2* ml = (ROWS ? a.rpart_ml : a.part_ml) + part;
  const float* acc = (ROWS ? a.rpart_o : a.part_o) + part * D + lane * kVec;
  float top = kNoKey;
  for (int s = s0 + lane; s < s1; s += 32) top = fmaxf(top, ml[s].x);
#pragma unroll
  for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(kAll, top, d));
  float sum = 0.0f;
  for (int s = s0 + lane; s < s1; s += 32) {
    const float2 y = ml[s];
    sum = fmaf(y.y, ex2(y.x - top), sum);
  }
#pragma unroll
  for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(kAll, sum, d);
  float x[kVec];
#pragma unroll
  for (int e = 0; e < kVec; ++e) x[e] = 0.0f;
#pragma unroll 4
  for (int s = s0 + part_of; s < s1; s += WPR) {
    const float by = ex2(ml[s].x - top);
    const float* y = acc + (int64_t)s * D;
    float f[kVec];
    if constexpr (kVec == 2) {
      const float2 z = *reinterpret_cast<const float2*>(y);
      f[0] = z.x;
      f[1] = z.y;
    } else {
#pragma unroll
      for (int e = 0; e < kVec; e += 4) {
        const float4 z = *reinterpret_cast<const float4*>(y + e);
        f[e] = z.x;
        f[e + 1] = z.y;
        f[e + 2] = z.z;
        f[e + 3] = z.w;
      }
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[e] = fmaf(f[e], by, x[e]);
  }
  if constexpr (WPR > 1) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) s_x[warp][lane * kVec + e] = x[e];
    __syncthreads();
    if (part_of > 0 || row < 0) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w)
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[e] += s_x[warp + w][lane * kVec + e];
  }
  const bool any = has_key(top, sum);
  T* dst = static_cast<T*>(a.out) + row * a.o_tok + hq * a.o_head + lane * kVec;
#pragma unroll
  for (int e = 0; e < kVec; ++e) x[e] = any ? x[e] / sum : 0.0f;
#pragma unroll
  for (int e = 0; e < kVec; e += 2) reinterpret_cast<uint32_t*>(dst)[e / 2] = Elem<T>::pack(x + e);
  if (lane == 0 && a.lse != nullptr)
    a.lse[row * a.hq + hq] = any ? (top + log2f(sum)) * kLn2 : -INFINITY;
}

template <int D, int NT, typename T>
cudaError_t launch_few(const AttendArgs& a, int64_t most_rows, cudaStream_t stream) {
  // at least one, for the rows of no request
  const int tiles = most_rows > 0 ? (int)((most_rows + NT * 8 - 1) / (NT * 8)) : 1;
  const int64_t grid = (int64_t)a.reqs * a.nsplit * tiles * a.hk;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  // whole 16-token steps inside one block need one table entry; other block
  // sizes look each token up
  const auto fn = a.bs % 16 == 0 ? attend_few_kernel<D, NT, true, T> : attend_few_kernel<D, NT, false, T>;
  const int ring = kWarps * kStages<D> * (int)sizeof(Stage<D>);
  const int join = kWarps * NT * 8 * (D + 4) * (int)sizeof(float);
  const int bytes = ring > join ? ring : join;
  // every call: the attribute belongs to the current device, and setting it is cheap
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  fn<<<(unsigned)grid, kWarps * 32, bytes, stream>>>(a, tiles);
  return cudaGetLastError();
}

template <int D, typename T, bool ROWS>
cudaError_t launch_join(const AttendArgs& a, cudaStream_t stream) {
  const int64_t total = !ROWS && a.cap ? (int64_t)a.reqs * a.hk * a.cap : (int64_t)a.rows * a.hq;
  // a warp a row while that is one round of reads, or where the rows alone fill the GPU
  const int nsplit = ROWS ? a.rsplit : a.nsplit;
  const bool one = nsplit <= 4 || total >= 148 * 64;
  const int64_t grid = one ? (total + kJoinWarps - 1) / kJoinWarps : total;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return one ? cudaLaunchKernelEx(&cfg, attend_join_kernel<D, T, ROWS, 1>, a, total)
             : cudaLaunchKernelEx(&cfg, attend_join_kernel<D, T, ROWS, kJoinWarps>, a, total);
}

template <int D, typename T>
cudaError_t launch_all(const AttendArgs& a, cudaStream_t stream) {
  const int64_t all = (int64_t)min(a.max_q, a.rows) * a.group;
  const int64_t few = min(all, (int64_t)a.few_rows);
  // 8 rows a tile, or 16 where a request has more: twice the rows for the same codes
  cudaError_t e;
  if constexpr (D == 256)
    e = launch_few<D, 1, T>(a, few, stream);
  else
    e = few <= 8 ? launch_few<D, 1, T>(a, few, stream) : launch_few<D, 2, T>(a, few, stream);
  if (e == cudaSuccess && a.nsplit > 1) e = launch_join<D, T, false>(a, stream);
  if constexpr (D <= 128) {
    if (e == cudaSuccess && all > a.few_rows) {
      e = launch_attend_rows<D, T>(a, stream);
      if (e == cudaSuccess && a.rsplit > 1) e = launch_join<D, T, true>(a, stream);
    }
  }
  return e;
}

template <typename T>
int attend_dispatch(const AttendArgs& a, int head_size, cudaStream_t stream) {
  cudaError_t e;
  switch (head_size) {
    case 64: e = launch_all<64, T>(a, stream); break;
    case 128: e = launch_all<128, T>(a, stream); break;
    case 256: e = launch_all<256, T>(a, stream); break;
    default: return MSHIFT_EUNSUPPORTED;
  }
  return e == cudaSuccess ? MSHIFT_OK : cuda_fail(e);
}

// Rows of a request up to which the few-rows kernel is the faster: 64 requests of 32 rows over 8,192 keys take
// it 514 us and the other 621, of 64 rows 999 and 657; 4 requests of 32 rows 66 and 72, of 64 rows 104 and 76.
constexpr int kFewRows = 32;

// Keys of a split of the few-rows kernel, a multiple of 128.  Enough splits that the CTAs of all units
// fill the 148 SMs' four places each; none shorter than 256, whose start-up would show, nor longer than
// 4,096, so that requests far shorter than the bound still end together; but past what fills the GPU
// never more than 32, nor than 1 GB of partial results (`bytes` a split) allow, since those go by
// the bound and not by the lengths.
int few_chunk(int64_t units, int max_len, int64_t bytes) {
  const int64_t fill = units > 0 ? (148 * 4 + units - 1) / units : 1;
  int64_t most = bytes > 0 ? (1ll << 30) / bytes : 32;
  most = most > 32 ? 32 : most;
  most = most < fill ? fill : most;
  int64_t chunk = ((int64_t)max_len + fill - 1) / fill;
  chunk = chunk < 256 ? 256 : chunk > 4096 ? 4096 : chunk;
  const int64_t floor = ((int64_t)max_len + most - 1) / most;
  if (chunk < floor) chunk = floor;
  return (int)((chunk + 127) / 128 * 128);
}

// Keys of a split of the many-rows kernel.  One CTA an SM: `units` CTAs a split run in rounds of
// 148, each as long as its tiles of 128 keys and five more for starting and writing back (a tile takes
// 2.3 us at head size 128, both measured; by the whole kernel's times 2.1 at 64, and 3.6 in blocks that are no
// multiple of 16).  Splitting fills the last round, and costs the partial results' way to memory and
// back and the join's launch; the cheapest count is taken.  Measured both ways: 64-244 tokens over eight
// histories 483 us whole, 506 in three, 457 in four; 1,024 tokens over 16,384 297 us whole, 370 in seven; 244
// over 30,720 654 us whole, 250-260 in seven to fifteen.
int rows_chunk(int64_t units, int max_len, int64_t elements) {
  const int64_t tiles = ((int64_t)max_len + 127) / 128;
  const double part = (double)elements * 8 / 6.5e12 / 2.3e-6;  // of a split, in tiles
  int64_t best = 1;
  double least = 0.0;
  // at most 64 splits, of at least 8 tiles, with at most 1 GB of partial results
  for (int64_t s = 1; s <= 64 && (s == 1 || (tiles / s >= 8 && s * elements * 4 <= 1ll << 30)); ++s) {
    const double rounds = (double)((units * s + 147) / 148);
    const double cost = rounds * ((double)((tiles + s - 1) / s) + 5.0) + (s > 1 ? (double)s * part + 3.0 : 0.0);
    if (s == 1 || cost < least) {
      least = cost;
      best = s;
    }
  }
  return best == 1 ? 1 << 30 : (int)((tiles + best - 1) / best * 128);
}

struct Plan {
  int few_rows, chunk, nsplit, rchunk, rsplit;
  int64_t cap;
  int64_t parts, rparts;  // partial results of each kernel
};

Plan plan(int32_t rows, int32_t hq, int32_t hk, int32_t head_size, int32_t reqs, int32_t max_q,
          int32_t max_len) {
  Plan p{};
  const int64_t group = hq / hk, all = (int64_t)(max_q < rows ? max_q : rows) * group;
  p.few_rows = head_size > 128 ? INT32_MAX : kFewRows;
  const int64_t few = all < p.few_rows ? all : p.few_rows;
  const int64_t tiles = few <= 8 ? 1 : (few + 15) / 16;
  p.cap = (int64_t)reqs * hk * few <= (int64_t)rows * hq ? few : 0;
  const int64_t partial = p.cap ? (int64_t)reqs * hk * p.cap : (int64_t)rows * hq;
  p.chunk = few_chunk((int64_t)reqs * hk * tiles, max_len, partial * (head_size + 2) * 4);
  p.nsplit = max_len > 0 ? (int)(((int64_t)max_len + p.chunk - 1) / p.chunk) : 1;
  if (p.nsplit > 1) p.parts = partial * p.nsplit;
  p.rchunk = 1 << 30;
  p.rsplit = 1;
  if (all > p.few_rows) {
    const int64_t items = (int64_t)rows * group / 256 + reqs;
    p.rchunk = rows_chunk(items * hk, max_len, (int64_t)rows * hq * head_size);
    p.rsplit = max_len > 0 ? (int)(((int64_t)max_len + p.rchunk - 1) / p.rchunk) : 1;
    if (p.rsplit > 1) p.rparts = (int64_t)rows * hq * p.rsplit;
  }
  return p;
}

}  // namespace
}  // namespace serve
}  // namespace mshift

static constexpr int32_t kMaxSeqLen = 1 << 30;  // key positions and their sums stay within int32

extern "C" {

int64_t mshift_attend_workspace(int32_t rows, int32_t hq, int32_t hk, int32_t head_size,
                                int32_t reqs, int32_t max_query_len, int32_t max_seq_len) {
  if (rows < 0 || hq <= 0 || hk <= 0 || hq % hk != 0 || head_size <= 0 || reqs < 0 ||
      max_query_len < 0 || max_seq_len < 0 || max_seq_len > kMaxSeqLen)
    return -1;
  if (rows == 0 || reqs == 0) return 0;
  const auto p = mshift::serve::plan(rows, hq, hk, head_size, reqs, max_query_len, max_seq_len);
  return (p.parts + p.rparts) * (head_size + 2) * 4;
}

int mshift_attend_block_scaled(
    int32_t dtype, const void* q, int64_t q_tok, int64_t q_head, int32_t rows, int32_t hq,
    const mshift_paged* paged, const void* k_base, const void* v_base, const float* k_scale,
    int64_t ks_blk, int64_t ks_head, const float* v_scale, int64_t vs_blk, int64_t vs_head,
    const int32_t* block_tables, int64_t table_stride, int32_t width, const int32_t* query_start,
    const int32_t* seq_lens, int32_t reqs, int32_t max_query_len, int32_t max_seq_len, float scale,
    int32_t causal, int32_t window, void* out, int64_t o_tok, int64_t o_head, float* lse,
    int32_t zero_tail, void* workspace, int64_t workspace_bytes, uint32_t* err, void* stream) {
  using namespace mshift;
  using namespace mshift::serve;
  if (paged == nullptr || rows < 0 || reqs < 0 || hq <= 0 || width < 0 || table_stride < width ||
      max_query_len < 0 || max_seq_len < 0 || max_seq_len > kMaxSeqLen || window < 0)
    return MSHIFT_EINVAL;
  if (paged->dtype != MSHIFT_E4M3 || (dtype != MSHIFT_BF16 && dtype != MSHIFT_F16))
    return MSHIFT_EUNSUPPORTED;
  if (paged->heads <= 0 || hq % paged->heads != 0 || paged->block_size <= 0 ||
      paged->num_blocks < 0)
    return MSHIFT_EINVAL;
  if (rows == 0 || reqs == 0) return MSHIFT_OK;
  if (q == nullptr || k_base == nullptr || v_base == nullptr || k_scale == nullptr ||
      v_scale == nullptr || (width > 0 && block_tables == nullptr) || query_start == nullptr ||
      seq_lens == nullptr || out == nullptr || err == nullptr)
    return MSHIFT_EINVAL;
  const auto odd = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
  if (odd(q) || odd(out) || odd(k_base) || odd(v_base) || o_tok % 8 || o_head % 8 || q_tok % 8 || q_head % 8 || paged->blk_stride % 16 ||
      paged->off_stride % 16 || paged->head_stride % 16)
    return MSHIFT_EINVAL;
  const Plan p = plan(rows, hq, paged->heads, paged->head_size, reqs, max_query_len, max_seq_len);
  const int64_t d = paged->head_size;
  if (p.parts + p.rparts > 0 &&
      (workspace == nullptr || odd(workspace) ||
       workspace_bytes < (p.parts + p.rparts) * (d + 2) * 4))
    return MSHIFT_EINVAL;
  AttendArgs a{};
  a.q = q;
  a.q_tok = q_tok;
  a.q_head = q_head;
  a.rows = rows;
  a.k = static_cast<const uint8_t*>(k_base);
  a.v = static_cast<const uint8_t*>(v_base);
  a.blk = paged->blk_stride;
  a.off = paged->off_stride;
  a.head = paged->head_stride;
  a.num_blocks = paged->num_blocks;
  set_block_size(a, paged->block_size);
  a.ks = k_scale;
  a.vs = v_scale;
  a.ks_blk = ks_blk;
  a.ks_head = ks_head;
  a.vs_blk = vs_blk;
  a.vs_head = vs_head;
  a.tables = block_tables;
  a.tab_stride = table_stride;
  a.width = width;
  a.qs = query_start;
  a.lens = seq_lens;
  a.reqs = reqs;
  a.hq = hq;
  a.hk = paged->heads;
  a.group = hq / paged->heads;
  a.max_len = max_seq_len;
  a.scale_log2 = scale * kLog2e;
  a.causal = causal;
  a.window = window;
  a.out = out;
  a.o_tok = o_tok;
  a.o_head = o_head;
  a.lse = lse;
  a.few_rows = p.few_rows;
  a.chunk = p.chunk;
  a.nsplit = p.nsplit;
  a.cap = p.cap;
  a.rchunk = p.rchunk;
  a.rsplit = p.rsplit;
  a.part_o = static_cast<float*>(workspace);
  a.rpart_o = a.part_o + p.parts * d;
  a.part_ml = reinterpret_cast<float2*>(a.rpart_o + p.rparts * d);
  a.rpart_ml = a.part_ml + p.parts;
  a.zero_tail = zero_tail;
  a.max_q = max_query_len;
  a.err = err;
  auto s = static_cast<cudaStream_t>(stream);
  return dtype == MSHIFT_BF16 ? attend_dispatch<__nv_bfloat16>(a, paged->head_size, s)
                              : attend_dispatch<__half>(a, paged->head_size, s);
}

}  // extern "C"
