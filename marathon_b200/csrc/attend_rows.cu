// attend_rows.cu — attention over a block-scaled e4m3 paged cache: the kernel for
// many query rows (chunks and prefills), on the fifth-generation tensor cores.
//
// A CTA has 256 (token, head of the group) rows of one request and KV head, as two tiles of
// 128, and walks the keys they see in tiles of 128 (attend.cuh has the mathematics):
//     S_t = Q_t K^T        tcgen05.mma 128 x 64 x D, Q and K f16 in shared memory, S in TMEM
//     P_t = 2^(t - M)      a thread a row: TMEM -> registers -> f16 -> TMEM, in place of S
//     O_t += P_t V         tcgen05.mma 128 x D x 64, P from TMEM, V f16 in shared memory
// Warps 0-3 and 4-7 are the rows of tile 0 and 1, warps 8-11 bring the codes in, warps 12 and 13
// issue the products of tile 0 and 1, warps 14 and 15 look up where the next tiles' keys lie.
//
// e4m3 has no matrix product with f16, so the loaders convert: 16 codes a 16-byte load,
// exactly, into the 128-byte-swizzled tiles that the descriptors name.  K and V have the
// same layout in shared memory (rows of tokens, 64 dims a swizzle atom); K is read with its dims as the
// contraction (K-major), V with its tokens (MN-major), so no tile is transposed.
// A code is converted once for 256 rows.
//
// The keys of a tile are taken in halves of 64, each with its own S (then P) columns: while the
// softmax has one half, the other's products run.  TMEM columns: S of row tile t, half b at
// 128 t + 64 b, O of tile t at 256 + D t.  O is rescaled in place when a row's maximum passes its
// reference by 2^8, after the product before has completed; that is rare after the first tiles.
//
// What bounds it.  8,192 causal tokens of 32 heads over 8 (550 GFLOP) take 615-645 us by the box, 850-890
// TFLOP/s, 0.52-0.54 of cuBLAS's rate; of head size 64, whose softmax is the same for half the products,
// 550; in blocks of 24 tokens, where every key has a scale of its own, 950.  A half of 64 keys for 256
// rows takes about 2,000 cycles; the products need 1,280 of them (50 cycles a 16-deep step of scores, which
// N = 64 leaves bound by shared memory, 66 of values), the exponentials 770, and the rest is the softmax
// warps' own latency: two of them a scheduler, in step with each other.  With work left out: products
// alone 397 us, softmax alone 575, loads alone 383.  Measured and not kept: the row tiles' softmax in turns (618-665 of then
// 626), sixteen softmax warps (743), scores given back early with P in columns of its own (668 of 643),
// all exponentials on the special-function units (626 of 598), 128 keys at once (762 of 693).
//
// Registers: 512 threads are launched with 128 each; the softmax warps take 176
// (64 scores of a row at once), the loaders 112 (two tiles' codes in flight) and the rest 48,
// which is the launch's sum.  Loops stay rolled but for the tiles' own: at 147 KB of code
// the roles evicted each other's instructions.
//
// Every wait is bounded: one that runs out sets MSHIFT_EBIT_TIMEOUT, every role leaves
// its loop, issued products are waited for, TMEM is freed and the CTA returns.
#include "attend.cuh"

namespace mshift {
namespace serve {
namespace {

constexpr int kTile = 128;  // keys of a tile, rows of a row tile
constexpr int kHalf = 64;   // keys whose scores a softmax thread holds at once
constexpr int kByHand = 4;  // of 16 exponentials, those that the FMA units work out
constexpr int kCta = 512;
constexpr int kRing = 4;  // tiles whose places and scales are held
constexpr uint32_t kRounds = 1u << 18;  // try_wait rounds of a wait

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
// One arrival for a warp whose lanes have all fenced what they wrote: a barrier takes them
// one by one.
__device__ __forceinline__ void warp_arrive(uint64_t* b) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) bar_arrive(b);
}
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
// False once the wait, or another role's, has run out.
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, volatile int* gone,
                                         uint32_t* err) {
  if (bar_try(b, parity)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < kRounds; ++i) {
    if (bar_try(b, parity)) return true;
    if (*gone) return false;
  }
  *gone = 1;
  flag(err, MSHIFT_EBIT_TIMEOUT);
  return false;
}

// One lane, and the compiler knows that it is one: what it issues is uniform.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ void commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(b))
               : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_smem() {  // generic stores, then the tensor core's reads
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Shared-memory descriptor of a 128-byte-swizzled tile: groups of 8 rows are 1,024 bytes
// apart; `lead` is the distance between 64-element columns where they are the rows of
// the operand (MN-major), unused otherwise.
__device__ __forceinline__ uint64_t descriptor(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(lead >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// f16 x f16 -> f32, M = 128; bit 16: B is MN-major.
__device__ constexpr uint32_t instruction(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                         bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}

// 32 columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_loaded() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// What was loaded may be used from here on: keeps the compiler from moving arithmetic on the
// registers to before the wait.
template <int N>
__device__ __forceinline__ void tmem_use(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_stored() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of a pair without the special-function unit, by the textbook reduction: x = n + f with n the nearest
// whole number (from adding 1.5 * 2^23, whose low bits then hold n), 2^f by a polynomial of degree 5 fitted
// here for the least relative error on [-1/2, 1/2] (1.6e-7 with its coefficients in fp32, 2.2e-7 with every
// rounding), and n added to its exponent.  Below -126, masked keys' -inf among it, the result
// is 2^-126, which f16 rounds to zero; NaN stays NaN.
__device__ __forceinline__ float2 exp2_pair(float x0, float x1) {
  constexpr float kMagic = 12582912.0f;
  const uint64_t x = pair(max_nan(x0, -126.0f), max_nan(x1, -126.0f));
  const uint64_t t = add2(x, pair(kMagic, kMagic));
  const uint64_t f = add2(x, fma2(t, pair(-1.0f, -1.0f), pair(kMagic, kMagic)));
  uint64_t r = fma2(f, pair(0x1.5c08e2p-10f, 0x1.5c08e2p-10f), pair(0x1.3d0c54p-7f, 0x1.3d0c54p-7f));
  r = fma2(r, f, pair(0x1.c6b6e6p-5f, 0x1.c6b6e6p-5f));
  r = fma2(r, f, pair(0x1.ebf918p-3f, 0x1.ebf918p-3f));
  r = fma2(r, f, pair(0x1.62e428p-1f, 0x1.62e428p-1f));
  r = fma2(r, f, pair(0x1.000002p+0f, 0x1.000002p+0f));
  const float2 y = unpair(r), n = unpair(t);
  return unpair(fma2(x, pair(0.0f, 0.0f),
                     pair(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(n.x) << 23)),
                          __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(n.y) << 23)))));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int D>
struct alignas(1024) Smem {
  static constexpr int kBytes = kTile * D * 2;  // an f16 tile
  uint8_t q[2][kBytes];
  uint8_t k[2][kBytes];
  uint8_t v[2][kBytes];
  float4 scale[kRing][kTile];  // of each key: ks, log2 vs, 1 / vs
  long long at[kRing][kTile];  // byte offset of each key in the cache, -1: not read
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], place_full[kRing],
      place_empty[kRing], s_full[2][2], p_full[2][2], o_done[2], done;
  float up[2][kTile];  // of each row: what its scores are multiplied with, log2 e among it
  uint32_t tmem;
  int gone;
};

// Byte offset of 16-byte chunk `c` (8 dims) of row `row` in a swizzled tile.
template <int D>
__device__ __forceinline__ uint32_t tile_at(int row, int c) {
  return (c >> 3) * (kTile * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}

// Keys [lo, hi) of this CTA, from tile-aligned `first`, in `tiles` tiles.
struct Span {
  int lo, hi, first, tiles;
};

// A loader thread has 16 codes of rows tid / 4 + 32 j, at dims 16 (tid % 4) + 64 u: eight
// neighbouring lanes store to two rows of one swizzle atom, all banks once.
template <int D>
__device__ __forceinline__ void load_codes(const uint8_t* base, const long long* at, uint4* w) {
  const int tid = threadIdx.x - 256;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long long off = at[tid / 4 + 32 * j];
    const uint8_t* p = base + off + (tid & 3) * 16;
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      w[j * (D / 64) + u] = make_uint4(0, 0, 0, 0);
      if (off >= 0) w[j * (D / 64) + u] = __ldg(reinterpret_cast<const uint4*>(p + 64 * u));
    }
  }
}

template <int D>
__device__ __forceinline__ void store_f16(uint8_t* tile, const uint4* w) {
  const int tid = threadIdx.x - 256, row = tid / 4, c = 2 * (tid & 3);
  uint8_t* at0 = tile + tile_at<D>(row, c);
  uint8_t* at1 = tile + tile_at<D>(row, c + 1);
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      const uint4 x = w[j * (D / 64) + u];
      const uint32_t in[4] = {x.x, x.y, x.z, x.w};
      uint32_t f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = e4m3x2_to_f16x2((uint16_t)in[e]);
        f[2 * e + 1] = e4m3x2_to_f16x2((uint16_t)(in[e] >> 16));
      }
      const int to = j * 32 * 128 + u * kTile * 128;
      *reinterpret_cast<uint4*>(at0 + to) = make_uint4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<uint4*>(at1 + to) = make_uint4(f[4], f[5], f[6], f[7]);
    }
}

// Warps 14 and 15: where the keys of each tile lie and their blocks' scales, two keys a lane.
// A tile's look-ups are three iterations' work, block, scales and entry, so that none waits for
// the one before.
template <int D, bool PAGE16>
__device__ __forceinline__ void finder(const AttendArgs& a, Smem<D>& s, int r, int h, const Span sp) {
  const int first = threadIdx.x - 14 * 32;
  const int32_t* table = a.tables + (int64_t)r * a.tab_stride;
  const float* ksh = a.ks + h * a.ks_head;
  const float* vsh = a.vs + h * a.vs_head;
  auto block_of = [&](int it, int i) -> int {
    const int key = sp.first + it * kTile + first + 64 * i;
    // PAGE16 reads the scales of 16 keys at the first of them, which may itself be outside
    if (it >= sp.tiles ||
        (PAGE16 ? (key | 15) < sp.lo || (key & ~15) >= sp.hi : key < sp.lo || key >= sp.hi))
      return -1;
    const int b = table[block_column(a, key)];
    if (b >= 0 && b < a.num_blocks) return b;
    flag(a.err, MSHIFT_EBIT_SLOT);
    return -1;
  };
  int b1[2], b2[2];
  float ks[2], vs[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    b1[i] = block_of(0, i);
    b2[i] = block_of(1, i);
    ks[i] = vs[i] = 0.0f;
    if (b1[i] >= 0) {
      ks[i] = ksh[b1[i] * a.ks_blk];
      vs[i] = vsh[b1[i] * a.vs_blk];
    }
  }
#pragma unroll 1
  for (int it = 0; it < sp.tiles; ++it) {
    const int ring = it % kRing;
    if (!__all_sync(0xffffffffu,
                    bar_wait(&s.place_empty[ring], ((it / kRing) & 1) ^ 1, &s.gone, a.err)))
      return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = first + 64 * i, key = sp.first + it * kTile + at, b = b1[i];
      s.at[ring][at] = b >= 0 && key >= sp.lo && key < sp.hi ? b * a.blk + (key - block_column(a, key) * a.bs) * a.off : -1ll;
      s.scale[ring][at] = b >= 0 ? make_float4(ks[i], value_log2(vs[i]), value_inverse(vs[i]), 0.0f)
                                 : make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
    }
    warp_arrive(&s.place_full[ring]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      b1[i] = b2[i];
      if (b1[i] >= 0) {
        ks[i] = ksh[b1[i] * a.ks_blk];
        vs[i] = vsh[b1[i] * a.vs_blk];
      }
      b2[i] = block_of(it + 2, i);
    }
  }
}

template <int D>
__device__ __forceinline__ void loader(const AttendArgs& a, Smem<D>& s, int h, int tiles) {
  const uint8_t* kh = a.k + h * a.head;
  const uint8_t* vh = a.v + h * a.head;
  uint4 kw[D / 16], vw[D / 16];
  auto all = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
  auto placed = [&](int it) {
    return all(bar_wait(&s.place_full[it % kRing], (it / kRing) & 1, &s.gone, a.err));
  };
  if (!placed(0)) return;
  load_codes<D>(kh, s.at[0], kw);
  load_codes<D>(vh, s.at[0], vw);
  warp_arrive(&s.place_empty[0]);
#pragma unroll 1
  for (int it = 0; it < tiles; ++it) {
    const int st = it & 1;
    const uint32_t free = ((it >> 1) & 1) ^ 1;
    const bool more = it + 1 < tiles;
    // the codes of a tile are loaded an iteration before they are converted
    if (!all(bar_wait(&s.k_empty[st], free, &s.gone, a.err))) return;
    store_f16<D>(s.k[st], kw);
    fence_smem();
    warp_arrive(&s.k_full[st]);
    if (more) {
      if (!placed(it + 1)) return;
      load_codes<D>(kh, s.at[(it + 1) % kRing], kw);
    }
    if (!all(bar_wait(&s.v_empty[st], free, &s.gone, a.err))) return;
    store_f16<D>(s.v[st], vw);
    fence_smem();
    warp_arrive(&s.v_full[st]);
    if (more) {
      load_codes<D>(vh, s.at[(it + 1) % kRing], vw);
      warp_arrive(&s.place_empty[(it + 1) % kRing]);
    }
  }
}

// The products of row tile t, issued by one lane.  Each tile has a warp of its own: the products wait in
// a queue and their operands' registers with them, so a warp that issues cannot prepare the next ones
// until they start; two warps keep the tensor core supplied between them.
template <int D>
__device__ __forceinline__ void issuer(const AttendArgs& a, Smem<D>& s, int tiles, int t) {
  constexpr uint32_t kScore = instruction(kHalf, false), kValue = instruction(D, true);
  const uint32_t s_at = s.tmem + t * kTile, o_at = s.tmem + 256 + t * D;
  const uint64_t q_desc = descriptor(smem_u32(s.q[t]), 16), k_desc = descriptor(smem_u32(s.k[0]), 16),
                 v_desc = descriptor(smem_u32(s.v[0]), kTile * 128);
  // half n of the keys: rows 64 (n % 2) of stage (n / 2) % 2, columns 64 (n % 2)
  auto stage = [](int n) -> uint32_t {
    return (((n >> 1) & 1) * Smem<D>::kBytes + (n & 1) * (kHalf * 128)) >> 4;
  };
  auto scores = [&](int n) {
    const uint64_t kd = k_desc + stage(n);
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {  // 16 dims: 32 bytes of a 128-byte row
      const uint32_t in = ((d >> 2) * (kTile * 128) + (d & 3) * 32) >> 4;
      mma_smem(s_at + (n & 1) * kHalf, q_desc + in, kd + in, kScore, d > 0);
    }
    commit(&s.s_full[t][n & 1]);
  };
  auto values = [&](int n) {
    const uint64_t vd = v_desc + stage(n);
#pragma unroll
    for (int k = 0; k < kHalf / 16; ++k)  // 16 keys: two groups of 8 rows
      mma_tmem(o_at, s_at + (n & 1) * kHalf + k * 8, vd + (k * 2048 >> 4), kValue, n > 0 || k > 0);
    commit(&s.o_done[t]);
  };
  bool ok = bar_wait(&s.q_full, 0, &s.gone, a.err) && bar_wait(&s.k_full[0], 0, &s.gone, a.err);
  fence_after();
  if (ok) {
    scores(0);
    scores(1);
    commit(&s.k_empty[0]);
  }
#pragma unroll 1
  for (int it = 0; ok && it < tiles; ++it) {
    const int st = it & 1;
    const bool more = it + 1 < tiles;
    ok = bar_wait(&s.v_full[st], (it >> 1) & 1, &s.gone, a.err);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      ok = ok && bar_wait(&s.p_full[t][b], it & 1, &s.gone, a.err);
      if (!ok) break;
      fence_after();
      values(2 * it + b);
      if (b == 1) commit(&s.v_empty[st]);
      if (!more) continue;
      if (b == 0) ok = bar_wait(&s.k_full[st ^ 1], ((it + 1) >> 1) & 1, &s.gone, a.err);
      if (!ok) break;
      scores(2 * it + 2 + b);
      if (b == 1) commit(&s.k_empty[st ^ 1]);
    }
  }
  // also after a wait ran out: what was issued completes before TMEM is freed
  commit(&s.done);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const float f[2] = {lo, hi};
  return Elem<T>::pack(f);
}

// Whether one of the keys lies in a block of the cache.  Only rows of NaN ask.
__device__ __forceinline__ bool any_block(const AttendArgs& a, int r, int2 see) {
  bool any = false;
#pragma unroll 1
  for (int key = see.x; !any && key < see.y; key = (block_column(a, key) + 1) * a.bs) {
    const int b = a.tables[(int64_t)r * a.tab_stride + block_column(a, key)];
    any = b >= 0 && b < a.num_blocks;
  }
  return any;
}

// Rows 32 * (warp % 4) + lane of tile t.
template <int D, bool PAGE16, typename T>
__device__ __forceinline__ void softmax(const AttendArgs& a, Smem<D>& s, const Request& rq, int r,
                                        int h, int m0, int split, const Span sp, int all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = warp >> 2, row = (warp & 3) * 32 + lane;
  const int m = m0 + t * kTile + row;
  const bool live = m < all;
  const int64_t tok = rq.q0 + (live ? m / a.group : 0);
  const int hq = h * a.group + (live ? m % a.group : 0);
  const int mine = all - (m - lane);  // the warp's live rows, or more than 32
  int2 see = live ? seen(a, rq, rq.start + (tok - rq.q0)) : make_int2(0, 0);
  see.x = max(see.x, sp.lo);
  see.y = min(see.y, sp.hi);

  // The warp's query rows, a row on D / 8 lanes: copied as they are, then made f16 after a power of two
  // in place.  The loops stay rolled: this code runs once a CTA, and fetching it costs more than it.
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;  // lanes of a row, rows of a warp-wide load
  const int64_t q_row = tok * a.q_tok + hq * a.q_head;  // of this lane's row; others' by shuffle
  constexpr int kBatch = 4;
#pragma unroll 4
  for (int i = 0; i < 32; i += kRows) {
    const int from = i + lane / kLanes;
    const T* src = static_cast<const T*>(a.q) + __shfl_sync(0xffffffffu, q_row, from) + lane % kLanes * 8;
    // rows past the last are zeros: a copy of no bytes fills with them
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(
                     s.q[t] + tile_at<D>((warp & 3) * 32 + from, lane % kLanes))),
                 "l"(src), "r"(from < mine ? 16 : 0)
                 : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
  for (int i = 0; i < 32; i += kBatch * kRows) {
    uint4 w[kBatch];
    float top[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      w[j] = *reinterpret_cast<const uint4*>(
          s.q[t] + tile_at<D>((warp & 3) * 32 + i + j * kRows + lane / kLanes, lane % kLanes));
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      // the largest magnitude: both 16-bit types order as their bits do without the sign
      uint32_t m = __vmaxu2(__vmaxu2(w[j].x & 0x7fff7fff, w[j].y & 0x7fff7fff),
                            __vmaxu2(w[j].z & 0x7fff7fff, w[j].w & 0x7fff7fff));
#pragma unroll
      for (int d = kLanes / 2; d > 0; d /= 2) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, d));
      float f[2];
      Elem<T>::unpack(__vmaxu2(m, m >> 16), f);
      top[j] = f[0];
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int r = (warp & 3) * 32 + i + j * kRows + lane / kLanes;
      int e2 = (int)(__float_as_uint(top[j]) >> 23) - 127;
      if (e2 < -126 || e2 > 126) e2 = 0;
      const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
      const uint32_t in[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
      uint32_t to[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[2];
        Elem<T>::unpack(in[e], f);
        to[e] = pack_f16x2(f[0] * down, f[1] * down);
      }
      *reinterpret_cast<uint4*>(s.q[t] + tile_at<D>(r, lane % kLanes)) =
          make_uint4(to[0], to[1], to[2], to[3]);
      if (lane % kLanes == 0)
        s.up[t][r] = __uint_as_float((uint32_t)(127 + e2) << 23) * a.scale_log2;
    }
  }
  fence_smem();
  warp_arrive(&s.q_full);
  const float rf = s.up[t][row];  // its own warp's
  if (m0 + t * kTile >= all) return;  // a tile without rows

  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const uint32_t s_at = s.tmem + lanes + t * kTile, o_at = s.tmem + lanes + 256 + t * D;
  float M = kNoKey, l = 0.0f;
  bool ok = true;
#pragma unroll 1
  for (int n = 0; n < 2 * sp.tiles; ++n) {
    const int it = n >> 1, b = n & 1, key0 = sp.first + n * kHalf;
    if (b == 0) ok = bar_wait(&s.place_full[it % kRing], (it / kRing) & 1, &s.gone, a.err);
    ok = ok && bar_wait(&s.s_full[t][b], it & 1, &s.gone, a.err);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    fence_after();
    const float4* sc = s.scale[it % kRing] + b * kHalf;
    const uint32_t sb_at = s_at + b * kHalf;
    uint32_t x[kHalf];
    tmem_load32(sb_at, x);
    tmem_load32(sb_at + 32, x + 32);
    // x = t - M
    const float ref = M == kNoKey ? 0.0f : M;
    tmem_loaded();
    tmem_use<kHalf>(x);
    if constexpr (PAGE16) {  // one scale for 16 keys
#pragma unroll
      for (int c = 0; c < kHalf; c += 16) {
        const float4 y = sc[c];
        const float by = rf * y.x, plus = y.y - ref;
        const uint64_t by2 = pair(by, by), plus2 = pair(plus, plus);
#pragma unroll
        for (int e = c; e < c + 16; e += 2) {
          const float2 z =
              unpair(fma2(pair(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), by2, plus2));
          x[e] = __float_as_uint(z.x);
          x[e + 1] = __float_as_uint(z.y);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < kHalf; ++e) {
        const float4 y = sc[e];
        x[e] = __float_as_uint(fmaf(__uint_as_float(x[e]), rf * y.x, y.y - ref));
      }
    }
    if (!__all_sync(0xffffffffu, see.x <= key0 && see.y >= key0 + kHalf)) {
      const int lo = see.x - key0, hi = see.y - key0;
#pragma unroll
      for (int e = 0; e < kHalf; ++e)
        if (e < lo || e >= hi) x[e] = __float_as_uint(-INFINITY);
    }
    float top = -INFINITY, top2 = -INFINITY;
#pragma unroll
    for (int e = 0; e < kHalf; e += 4) {
      top = max3(top, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
      top2 = max3(top2, __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
    }
    top = fmaxf(top, top2);
    const bool passed = M == kNoKey ? top > -INFINITY : top > kLazy;
    if (__any_sync(0xffffffffu, passed)) {
      const float up = passed ? top : 0.0f;
      const float by = !passed ? 1.0f : M == kNoKey ? 0.0f : ex2(-up);
      if (passed) M = ref + up;
      l *= by;
#pragma unroll
      for (int e = 0; e < kHalf; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) - up);
      if (n > 0) {  // O holds every half before this one once the last product is done
        ok = __all_sync(0xffffffffu, bar_wait(&s.o_done[t], (n - 1) & 1, &s.gone, a.err));
        if (!ok) break;
        fence_after();
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          uint32_t o[32];
          tmem_load32(o_at + d, o);
          tmem_loaded();
          tmem_use<32>(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
          tmem_store32(o_at + d, o);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < kHalf; q += 32) {
      uint32_t p[16];
#pragma unroll
      for (int c = q; c < q + 32; c += 16) {
        uint64_t sum = 0;
#pragma unroll
        for (int e = c; e < c + 16; e += 2) {
          float p0, p1;
          if (e % 16 >= 16 - kByHand) {
            const float2 z = exp2_pair(__uint_as_float(x[e]), __uint_as_float(x[e + 1]));
            p0 = z.x;
            p1 = z.y;
          } else {
            p0 = ex2(__uint_as_float(x[e]));
            p1 = ex2(__uint_as_float(x[e + 1]));
          }
          if constexpr (PAGE16)
            sum = add2(sum, pair(p0, p1));
          else
            l = fmaf(p1, sc[e + 1].z, fmaf(p0, sc[e].z, l));
          p[(e - q) / 2] = pack_f16x2(p0, p1);
        }
        if constexpr (PAGE16) {
          const float2 z = unpair(sum);
          l = fmaf(z.x + z.y, sc[c].z, l);
        }
      }
      tmem_store16(sb_at + q / 2, p);
    }
    tmem_stored();
    fence_before();
    warp_arrive(&s.p_full[t][b]);
    if (b == 1) warp_arrive(&s.place_empty[it % kRing]);
  }

  if (ok) ok = __all_sync(0xffffffffu, bar_wait(&s.done, 0, &s.gone, a.err));
  if (!ok || s.gone) return;
  fence_after();
  // keys in bad blocks are unseen by a row of NaN too, whose product with their zeros is NaN
  if (M == kNoKey && l != l && !any_block(a, r, see)) l = 0.0f;
  const bool any = has_key(M, l);
  const float by = any ? 1.0f / l : 0.0f;
  const int64_t part = (tok * a.hq + hq) * a.rsplit + split;
  if (live && a.rsplit > 1)
    a.rpart_ml[part] = make_float2(M, l);
  else if (live && a.lse != nullptr)
    a.lse[tok * a.hq + hq] = any ? (M + log2f(l)) * kLn2 : -INFINITY;
  // Rows go through shared memory (K's and V's, done with), so that whole rows are written: 32 rows of
  // D words a warp, 16-byte chunks swizzled by row.
  float4* stage = reinterpret_cast<float4*>((t ? s.v : s.k)[0]) + (warp & 3) * (32 * D / 4);
#pragma unroll 1
  for (int c = 0; c < D; c += 32) {
    uint32_t o[32];
    tmem_load32(o_at + c, o);
    tmem_loaded();
    tmem_use<32>(o);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      stage[lane * (D / 4) + ((c / 4 + e) ^ (lane & 7))] =
          make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                      __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
  }
  __syncwarp();
  constexpr int kLanesOut = D / 4;  // lanes of a row of float4
  const bool parts = a.rsplit > 1;
  const int64_t o_row = parts ? part * D : tok * a.o_tok + hq * a.o_head;
  const float mul = !any ? 0.0f : parts ? 1.0f : by;
  T* out = static_cast<T*>(a.out) + lane % kLanesOut * 4;
  float* part_o = a.rpart_o + lane % kLanesOut * 4;
#pragma unroll 1
  for (int i = 0; i < kLanesOut; i += kBatch) {
    float4 y[kBatch];
    int64_t to[kBatch];
    float scale[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int from = (i + j) * (32 / kLanesOut) + lane / kLanesOut;
      y[j] = stage[from * kLanesOut + (lane % kLanesOut ^ (from & 7))];
      to[j] = __shfl_sync(0xffffffffu, o_row, from);
      scale[j] = __shfl_sync(0xffffffffu, mul, from);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int from = (i + j) * (32 / kLanesOut) + lane / kLanesOut;
      // a row without keys is zeros, whatever the values beside it were
      const float4 z = scale[j] == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                        : make_float4(y[j].x * scale[j], y[j].y * scale[j],
                                                      y[j].z * scale[j], y[j].w * scale[j]);
      if (from < mine) {
        if (parts)
          *reinterpret_cast<float4*>(part_o + to[j]) = z;
        else
          *reinterpret_cast<uint2*>(out + to[j]) = make_uint2(pack2<T>(z.x, z.y), pack2<T>(z.z, z.w));
      }
    }
  }
}

// Rows without a key in this CTA's span: an empty part, or zeros.
template <int D, typename T>
__device__ __forceinline__ void nothing(const AttendArgs& a, const Request& rq, int h, int m0,
                                        int split, int all) {
#pragma unroll 1
  for (int i = threadIdx.x; i < min(2 * kTile, all - m0); i += kCta) {
    const int m = m0 + i;
    const int64_t tok = rq.q0 + m / a.group;
    const int hq = h * a.group + m % a.group;
    if (a.rsplit > 1) {
      a.rpart_ml[(tok * a.hq + hq) * a.rsplit + split] = make_float2(kNoKey, 0.0f);
      continue;
    }
    T* dst = static_cast<T*>(a.out) + tok * a.o_tok + hq * a.o_head;
#pragma unroll 1
    for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
    if (a.lse != nullptr) a.lse[tok * a.hq + hq] = -INFINITY;
  }
}

template <int D, bool PAGE16, typename T>
__global__ void __launch_bounds__(kCta, 1) attend_rows_kernel(const AttendArgs a, int items) {
  extern __shared__ uint8_t raw[];
  Smem<D>& s = *reinterpret_cast<Smem<D>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5;
  int64_t id = blockIdx.x;
  const int h = (int)(id % a.hk);
  id /= a.hk;
  const int split = (int)(id % a.rsplit);
  id /= a.rsplit;
  // a request's later rows see more keys: the longest tiles first
  const long long item = items - 1 - id;
  // a request of n rows has at most ceil(n / 256) tiles, and floor(q_r / 256) + r numbers
  // them without a scan over the requests
  const int r = find_request(a.reqs, item, [&](int i) {
    return (long long)row_start(a.qs, i, a.rows) * a.group / (2 * kTile) + i;
  });
  const Request rq = request_of(a, r, threadIdx.x == 0 && h == 0 && split == 0);
  const long long base = (long long)rq.q0 * a.group / (2 * kTile) + r;
  const long long rows = (long long)rq.n * a.group;
  if (item < base || rows <= a.few_rows || (item - base) * 2 * kTile >= rows) return;
  const int m0 = (int)(item - base) * 2 * kTile, all = (int)rows;
  const int last_m = min(m0 + 2 * kTile, all) - 1;
  Span sp;
  {
    const int2 see = seen_by_tile(a, rq, rq.start + m0 / a.group, rq.start + last_m / a.group);
    sp.lo = max(see.x, split * a.rchunk);
    sp.hi = (int)min((long long)see.y, (long long)split * a.rchunk + a.rchunk);
    sp.first = sp.lo / kTile * kTile;
    sp.tiles = sp.hi > sp.lo ? (sp.hi - sp.first + kTile - 1) / kTile : 0;
  }
  if (sp.tiles == 0) {
    nothing<D, T>(a, rq, h, m0, split, all);
    return;
  }
  const bool two = m0 + kTile < all;

  if (threadIdx.x == 0) {
    bar_init(&s.q_full, 8);  // one arrival a warp
    for (int i = 0; i < 2; ++i) {
      bar_init(&s.k_full[i], 4);
      bar_init(&s.k_empty[i], two ? 2 : 1);  // an arrival a row tile
      bar_init(&s.v_full[i], 4);
      bar_init(&s.v_empty[i], two ? 2 : 1);
      for (int b = 0; b < 2; ++b) {
        bar_init(&s.s_full[i][b], 1);
        bar_init(&s.p_full[i][b], 4);
      }
      bar_init(&s.o_done[i], 1);
    }
    for (int i = 0; i < kRing; ++i) {
      bar_init(&s.place_full[i], 2);
      bar_init(&s.place_empty[i], two ? 12 : 8);  // softmax warps of live tiles, loaders
    }
    bar_init(&s.done, two ? 2 : 1);
    s.gone = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&s.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();

  // 256 * 176 + 128 * 112 + 128 * 48 = 512 * 128 registers
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    softmax<D, PAGE16, T>(a, s, rq, r, h, m0, split, sp, all);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    loader<D>(a, s, h, sp.tiles);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp < 14) {
      if ((warp == 12 || two) && elect_one()) {
        issuer<D>(a, s, sp.tiles, warp - 12);
        // after a wait that ran out nobody else waits for the products
#pragma unroll 1
        for (uint32_t i = 0; i < kRounds && !bar_try(&s.done, 0); ++i) {
        }
      }
      __syncwarp();
    } else {
      finder<D, PAGE16>(a, s, r, h, sp);
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 12)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(s.tmem));
}

template <int D, bool PAGE16, typename T>
cudaError_t launch(const AttendArgs& a, int items, cudaStream_t stream) {
  const int bytes = (int)sizeof(Smem<D>) + 1024;
  const auto fn = attend_rows_kernel<D, PAGE16, T>;
  // the roles' register shares add up to 512 * 128: a build that launched with fewer would
  // wait for the difference for good
  static const int regs = [fn] {
    cudaFuncAttributes at{};
    return cudaFuncGetAttributes(&at, fn) == cudaSuccess ? at.numRegs : 0;
  }();
  if (regs != 128) return cudaErrorLaunchOutOfResources;
  // every call: the attribute belongs to the current device, and setting it is cheap
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  const int64_t grid = (int64_t)items * a.rsplit * a.hk;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  fn<<<(unsigned)grid, kCta, bytes, stream>>>(a, items);
  return cudaGetLastError();
}

}  // namespace

template <int D, typename T>
cudaError_t launch_attend_rows(const AttendArgs& a, cudaStream_t stream) {
  const int items = (int)((int64_t)a.rows * a.group / (2 * kTile)) + a.reqs;
  return a.bs % 16 == 0 ? launch<D, true, T>(a, items, stream) : launch<D, false, T>(a, items, stream);
}

template cudaError_t launch_attend_rows<64, __nv_bfloat16>(const AttendArgs&, cudaStream_t);
template cudaError_t launch_attend_rows<64, __half>(const AttendArgs&, cudaStream_t);
template cudaError_t launch_attend_rows<128, __nv_bfloat16>(const AttendArgs&, cudaStream_t);
template cudaError_t launch_attend_rows<128, __half>(const AttendArgs&, cudaStream_t);

}  // namespace serve
}  // namespace mshift
