// block_maps.cu — block tables and slot maps of one step, from request lengths.
//
// need(r) = ceil((cached + new) / bs) - ceil(cached / bs); exclusive sums of
// `new` and `need` over the requests give every request's first token row and
// its first block of the free list.  A token at position p then lives in the
// table's block p / bs, or, if p / bs is past the blocks held, in a free one.
//
// The work is a few bytes a token and the call is bound by latency, so it is one
// launch with nothing between CTAs: every CTA scans all requests itself (a few
// KB from L2) and writes its own 1,024 tokens.  A new block's table entry is
// written by the token at the block's first position, which is always new.
// 64 requests of one token, or 512 of up to 128 (33,000 tokens): 4-5 us on the GPU, of which a launch is
// half; a call costs the host 19 us.
#include "serve_common.cuh"

namespace mshift {
namespace serve {
namespace {

constexpr int kMapThreads = 1024;  // tokens per CTA, requests per scan pass

struct MapArgs {
  const int32_t* cached;
  const int32_t* fresh;
  int reqs;
  int32_t* tables;
  int64_t tab_stride;
  int width;
  const int32_t* free_blocks;
  int free_len;
  const int32_t* free_head;
  int bs, tokens;
  int32_t* query_start;
  int32_t* seq_lens;
  int64_t* slots;
  int64_t* positions;
  int32_t* free_head_out;
  uint32_t* err;
};

__device__ __forceinline__ long long warp_inclusive(long long v) {
  const int lane = threadIdx.x & 31;
  for (int d = 1; d < 32; d *= 2) {
    const long long o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

__global__ void __launch_bounds__(kMapThreads) block_maps_kernel(const MapArgs a) {
  // the request that owns the tokens from a place of this CTA's tile on
  __shared__ int s_req[kMapThreads];
  __shared__ int s_cached[kMapThreads];
  __shared__ long long s_start[kMapThreads], s_end[kMapThreads], s_block[kMapThreads];
  __shared__ long long s_warp[2][32];
  __shared__ int s_scan[32];
  __shared__ long long s_used;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long t0 = (long long)blockIdx.x * kMapThreads;
  const int head = *a.free_head;
  s_req[tid] = -1;
  if (tid == 0) s_used = 0;
  __syncthreads();

  // 64-bit sums: lengths come from the device and are not trusted to be small
  long long tok_base = 0, blk_base = 0;
  for (int r0 = 0; r0 < a.reqs; r0 += kMapThreads) {
    const int r = r0 + tid;
    int cached = 0, fresh = 0;
    if (r < a.reqs) {
      cached = a.cached[r];
      fresh = a.fresh[r];
      if ((cached < 0 || fresh < 0 || (long long)cached + fresh > INT32_MAX) && blockIdx.x == 0)
        flag(a.err, MSHIFT_ERR_LENGTHS);
      cached = max(cached, 0);
      fresh = max(fresh, 0);
    }
    const long long total = (long long)cached + fresh;
    const long long need = (total + a.bs - 1) / a.bs - ((long long)cached + a.bs - 1) / a.bs;
    const long long tok_in = warp_inclusive(fresh), blk_in = warp_inclusive(need);
    if (lane == 31) {
      s_warp[0][warp] = tok_in;
      s_warp[1][warp] = blk_in;
    }
    __syncthreads();
    if (warp < 2) s_warp[warp][lane] = warp_inclusive(s_warp[warp][lane]);
    __syncthreads();
    const long long tok0 = tok_base + tok_in - fresh + (warp ? s_warp[0][warp - 1] : 0);
    const long long blk0 = blk_base + blk_in - need + (warp ? s_warp[1][warp - 1] : 0);
    if (r < a.reqs) {
      if (blockIdx.x == 0) {
        // tokens past the caller's bound are dropped from the lengths too, so a
        // request's rows still stand at its last positions
        const long long q0 = min(tok0, (long long)a.tokens);
        const long long q1 = min(tok0 + fresh, (long long)a.tokens);
        a.query_start[r] = (int)q0;
        a.seq_lens[r] = (int)min(cached + q1 - q0, (long long)INT32_MAX);
        // the request in which the bound falls: what is dropped takes no blocks
        if (tok0 < a.tokens && tok0 + fresh >= a.tokens)
          s_used = blk0 + (cached + q1 - q0 + a.bs - 1) / a.bs - ((long long)cached + a.bs - 1) / a.bs;
      }
      // requests tile the token axis, so at most one of them starts at, or
      // reaches into the tile at, each place
      const long long lo = max(tok0, t0), hi = min(tok0 + fresh, t0 + kMapThreads);
      if (lo < hi) {
        const int at = (int)(lo - t0);
        s_req[at] = r;
        s_cached[at] = cached;
        s_start[at] = tok0;
        s_end[at] = tok0 + fresh;
        s_block[at] = blk0;
      }
    }
    tok_base += s_warp[0][31];
    blk_base += s_warp[1][31];
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.query_start[a.reqs] = (int)min(tok_base, (long long)a.tokens);
    const long long end = (long long)head + (tok_base > a.tokens ? s_used : blk_base);
    a.free_head_out[0] = (int)min(max(end, 0ll), (long long)a.free_len);
    if (tok_base > a.tokens) flag(a.err, MSHIFT_ERR_LENGTHS);
    if (head < 0 || end > a.free_len) flag(a.err, MSHIFT_ERR_POOL);
  }
  __syncthreads();  // the places marked in the last pass (or, with no requests, the clearing)

  // the nearest marked place at or before this token: an inclusive running maximum
  int src = s_req[tid] >= 0 ? tid : -1;
  for (int d = 1; d < 32; d *= 2) {
    const int o = __shfl_up_sync(0xffffffffu, src, d);
    if (lane >= d) src = max(src, o);
  }
  if (lane == 31) s_scan[warp] = src;
  __syncthreads();
  for (int w = 0; w < warp; ++w) src = max(src, s_scan[w]);

  const long long t = t0 + tid;
  if (t >= a.tokens) return;
  if (src < 0 || t >= s_end[src]) {  // behind the last request
    a.slots[t] = -1;
    a.positions[t] = 0;
    return;
  }
  const long long p = s_cached[src] + (t - s_start[src]);
  const long long col = p / a.bs, off = p - col * a.bs;
  const long long have = ((long long)s_cached[src] + a.bs - 1) / a.bs;
  int32_t* row = a.tables + (int64_t)s_req[src] * a.tab_stride;
  int block = -1;
  if (col >= have) {
    const long long f = head + s_block[src] + (col - have);
    if (head >= 0 && f < a.free_len) {
      block = a.free_blocks[f];
      if (block < 0) flag(a.err, MSHIFT_EBIT_SLOT);
    }
    if (off == 0 && col < a.width) row[col] = block;
  } else if (col < a.width) {
    block = row[col];
    if (block < 0) flag(a.err, MSHIFT_EBIT_SLOT);
  }
  if (col >= a.width) {
    flag(a.err, MSHIFT_ERR_POOL);
    block = -1;
  }
  a.slots[t] = block < 0 ? -1 : (int64_t)block * a.bs + off;
  a.positions[t] = p;
}

}  // namespace
}  // namespace serve
}  // namespace mshift

extern "C" int mshift_block_maps(const int32_t* cached_lens, const int32_t* new_lens, int32_t reqs,
                                 int32_t* block_tables, int64_t table_stride, int32_t width,
                                 const int32_t* free_blocks, int32_t free_len,
                                 const int32_t* free_head, int32_t block_size, int32_t tokens,
                                 int32_t* query_start, int32_t* seq_lens, int64_t* slots,
                                 int64_t* positions, int32_t* free_head_out, uint32_t* err,
                                 void* stream) {
  using namespace mshift;
  using namespace mshift::serve;
  if (reqs < 0 || width < 0 || free_len < 0 || block_size <= 0 || tokens < 0 ||
      table_stride < width)
    return MSHIFT_EINVAL;
  if (free_head == nullptr || query_start == nullptr || free_head_out == nullptr || err == nullptr)
    return MSHIFT_EINVAL;
  if (free_head == free_head_out) return MSHIFT_EINVAL;  // read by every CTA
  if (reqs > 0 && (cached_lens == nullptr || new_lens == nullptr || seq_lens == nullptr ||
                   (width > 0 && block_tables == nullptr)))
    return MSHIFT_EINVAL;
  if (free_len > 0 && free_blocks == nullptr) return MSHIFT_EINVAL;
  if (tokens > 0 && (slots == nullptr || positions == nullptr)) return MSHIFT_EINVAL;
  const MapArgs a{cached_lens, new_lens,   reqs,   block_tables, table_stride, width,
                  free_blocks, free_len,   free_head, block_size, tokens,      query_start,
                  seq_lens,    slots,      positions, free_head_out, err};
  const int grid = tokens > 0 ? (int)(((int64_t)tokens + kMapThreads - 1) / kMapThreads) : 1;
  block_maps_kernel<<<grid, kMapThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MSHIFT_OK : cuda_fail(e);
}
