// Softmax attention's gradients on the tensor cores, 16-bit types.
//
//   P = exp2(S c - lse log2 e),  S = Q K^T,  c = scale log2 e;   dP = dO V^T,  D = rowsum(dO o O)
//   dS = P o (dP - D);   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K
//
// A first kernel takes D and lse log2 e per row. One launch then runs two kinds of blocks. A key block
// keeps 128 keys of one key head and passes over the queries that see them, of all the heads that share
// the key head: it computes S^T = K Q^T and dP^T = V dO^T, a thread per key and half of the queries, and
// adds P^T dO and dS^T Q in TMEM. A query block keeps 128 queries and passes over the keys: S, dP and
// dS K. So S and dP are computed twice (7 products where 5 would do), and in return dK, dV and dQ are
// each summed by one block in one order: no atomics, no second pass over a 32-bit dQ in memory, and
// the gradients of a shared key head need no reduction.
// Both kinds run the same pipeline. Per step, T1 = S (or S^T) and T2 = dP (or dP^T) lie in TMEM; P
// overwrites T1 and dS overwrites T2 as 16-bit operands. The products of one step and the scores of the
// next are issued as their operands get ready: while the threads take the exponentials of T1, the
// tensor core adds dS and computes the next T2; while they form dS, it adds P and computes the next T1.
// Sixteen warps share a tile's scores, 32 columns a thread: with eight the waits on TMEM and on the special
// function units showed more (1267 us to 1170 when changed). 4 x 16 heads x 4096 x 64, no mask: 1130 us, 608 TFLOP/s
// of the five products; dim 128: 1918 us, 716.
// P and dS are rounded to 16 bits for the products: half a step of each term, which leaves the gradients with a relative error
// of 0.0024 in bf16 and 0.0003 in fp16, at 8 keys as at 4096, where the rounding of the results alone makes 0.0017 and
// 0.0002. In rows of n keys D adds to that: o was rounded, and computed from a rounded P, which makes 2 / n of
// what dS's rounding does. It is the first rows of a causal sequence that this shows in, at any length, since they
// make up most of the gradients' size. So blocks of rows with at most kFewKeys keys (query tiles; key tiles that such
// rows begin at) multiply dS in two parts, the rounded value and what that left. Over a causal training step of 1000
// tokens dq is then off by 1.24 to 1.41 times what rounding the result alone makes, 1.44 to 1.58 without; it is at
// most two tiles of a sequence that pay for it.
// In fp16 P is taken times 2^10 (at most 1024), so that rows over thousands of keys stay above its smallest normal
// value; dV is scaled back. dS has no size of its own
// (loss-scaled gradients pass fp16's largest value, small ones over many keys lie among its smallest), so in fp16
// it is taken times 2^x, one x for a key head and the query heads that share it, from
//   |dS| <= |dO_i| (max |v_j| + |o_i|) <= B = 2 max |dO_i| max |v_j|,   2^13 <= 2^x B < 2^14,
// over the rows that are seen and finite: nothing overflows, and what is lost lies 2^-38 below B. The kernel that takes D
// leaves the largest of each tile, and every block takes the largest of those again (8 x 16 heads x 1024 x 64 causal: 146.7 us,
// 141.6 in bf16; dS unscaled lost a tenth of dq at dout of 1e-4 on 8192 keys, and overflowed beyond 65504).
#include <type_traits>

#include "attention_sm100.cuh"

namespace lsr {
namespace {

constexpr int PARTS = 4;  // warpgroups on the scores, each with 128 / PARTS columns
constexpr int COLS = kRows / PARTS;
constexpr int BWD_THREADS = PARTS * 128 + 128;  // then the loader, the issuer, one for the size of dS (kSized) and an idle warp
constexpr int LOADER = 4 * PARTS, ISSUER = LOADER + 1, SIZER = ISSUER + 1;
// Registers a thread after the split, within the 96 that five warpgroups are launched with: 5 x 96 = 4 x 104 + 64.
constexpr int kScoreRegs = 104, kRestRegs = 64;

// Of more keys D's part is under 2% of dS's own rounding.
constexpr int kFewKeys = 128;

// Whether dS is scaled to a size of the data.
template <typename T>
constexpr bool kSized = false;
template <>
constexpr bool kSized<__half> = true;

// Extra power of two in P.
template <typename T>
constexpr int kExtra = 0;
template <>
constexpr int kExtra<__half> = 10;

struct BwdParams {
  AttnParams a;
  CUtensorMap mq, mk, mv, mdo;
  float* stats;  // [batch][heads][query tiles][2][128]: lse log2 e - extra (plus infinity: no probability), D
  // kSized: the largest |dout row|^2 of each tile, [batch][heads][q_tiles], then the largest |v row|^2 among its keys that are
  // seen, [batch][kv_heads][kv_tiles]; rows that are not finite do not count
  float* sizes;
  long long size_rows, size_keys;  // tiles of each
  int2* seen;                      // [batch] with a mask: the first key that is seen, and how many are
  int q_tiles, kv_tiles;
  long long kv_blocks;
  // blocks that the steps of 128 keys, and of 128 queries, are dealt to; with more than one their sums go here
  int split_k, split_q;
  float *part_dk, *part_dv, *part_dq;  // [split][batch][head][position][dim]
};

template <int PANELS, bool MASK>
struct BwdSmem {
  static constexpr int TILE = PANELS * kPanel;
  static constexpr int STAGES = PANELS == 1 ? 8 : 4;  // tiles in the ring, two per step
  static constexpr int STATS = (2 + STAGES) * TILE;   // 1 KB per step in the ring
  static constexpr int BITS = STATS + STAGES / 2 * 1024;
  static constexpr int BARS = BITS + (MASK ? kMaskTiles * 16 : 0);
  static constexpr int TOTAL = BARS + 256 + 1024;  // and room to align the tiles
};

template <typename T>
__device__ __forceinline__ float dot8(const uint4& x, const uint4& y, float s) {
  const T *xe = reinterpret_cast<const T*>(&x), *ye = reinterpret_cast<const T*>(&y);
#pragma unroll
  for (int k = 0; k < 8; ++k) s = fmaf(attn_to_f(xe[k]), attn_to_f(ye[k]), s);
  return s;
}

// A sum over the eight lanes of a row.
__device__ __forceinline__ float row_sum(float s) {
#pragma unroll
  for (int w = 4; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
  return s;
}

// Row statistics: a tile of 128 rows per block, eight lanes per row, four rows per thread in flight (one row per thread and
// 32 per block: 23.5 us at 8 x 16 heads x 1024 x 64 in fp16, now 12.8). kSized: the blocks after those of the
// queries take the sizes of the values. The last blocks look the masks over, one each.
template <typename T>
__global__ void __launch_bounds__(256) attn_stats_kernel(const __grid_constant__ BwdParams p) {
  __shared__ unsigned tops[8];
  launch_dependents();
  if (blockIdx.x >= p.size_rows + p.size_keys) {
    __shared__ unsigned counts[8];
    const unsigned b = blockIdx.x - (unsigned)(p.size_rows + p.size_keys);
    const unsigned char* mask = p.a.mask + b * p.a.mask_stride;
    unsigned first = p.a.kv_len, count = 0;
#pragma unroll 8
    for (int j = threadIdx.x; j < p.a.kv_len; j += 256)
      if (mask[j]) first = min(first, (unsigned)j), ++count;
    first = __reduce_min_sync(0xffffffffu, first);
    count = __reduce_add_sync(0xffffffffu, count);
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = first, counts[threadIdx.x / 32] = count;
    __syncthreads();
    if (threadIdx.x) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) first = min(first, tops[w]), count += counts[w];
    p.seen[b] = make_int2((int)first, (int)count);
    return;
  }
  const bool keys = kSized<T> && blockIdx.x >= p.size_rows;
  const long long id = blockIdx.x - (keys ? p.size_rows : 0);
  const int tiles = keys ? p.kv_tiles : p.q_tiles, heads = keys ? p.a.kv_heads : p.a.heads;
  const int part = threadIdx.x % 8, sub = threadIdx.x / 8;
  const int row0 = (int)(id % tiles) * kRows + sub, h = (int)(id / tiles % heads), b = (int)(id / tiles / heads);
  float s[4] = {}, z[4] = {};  // dout . out (not of keys), and the row's own square (kSized)
  if (keys) {
    const T* v = attn_at<T>(p.a.v, p.a.sv, b, h);
    const unsigned char* mask = p.a.mask ? p.a.mask + b * p.a.mask_stride : nullptr;
    for (int e = part * 8; e < p.a.head_dim; e += 64) {
      uint4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = row0 + 32 * k;
        x[k] = j < p.a.kv_len && (!mask || mask[j]) ? *reinterpret_cast<const uint4*>(v + j * p.a.sv.s + e) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) z[k] = dot8<T>(x[k], x[k], z[k]);
    }
  } else {
    const T *o = attn_at<T>(p.a.out, p.a.so, b, h), *d = attn_at<T>(p.a.dout, p.a.sdo, b, h);
    const float* from = p.a.lse + ((long long)b * p.a.heads + h) * p.a.q_len;
    float lse[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) lse[k] = row0 + 32 * k < p.a.q_len ? from[row0 + 32 * k] : -INFINITY;
    for (int e = part * 8; e < p.a.head_dim; e += 64) {
      uint4 x[4], y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = row0 + 32 * k;
        const bool in = i < p.a.q_len;
        x[k] = in ? *reinterpret_cast<const uint4*>(o + i * p.a.so.s + e) : make_uint4(0, 0, 0, 0);
        y[k] = in ? *reinterpret_cast<const uint4*>(d + i * p.a.sdo.s + e) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[k] = dot8<T>(x[k], y[k], s[k]);
        if (kSized<T>) z[k] = dot8<T>(y[k], y[k], z[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float delta = row_sum(s[k]);
      if (part == 0) {
        float* dst = p.stats + id * 256 + sub + 32 * k;
        dst[0] = lse[k] != -INFINITY ? fmaf(lse[k], kLog2e, -(float)kExtra<T>) : INFINITY;
        dst[128] = delta;
      }
    }
  }
  if (!kSized<T>) return;
  unsigned top = 0;  // of the finite ones: values >= 0 are ordered as their bits are
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float x = row_sum(z[k]);
    top = max(top, x < INFINITY ? __float_as_uint(x) : 0u);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
  if (threadIdx.x) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) top = max(top, tops[w]);
  p.sizes[blockIdx.x] = __uint_as_float(top);
}

// The power of two that dS of a key head is taken times, the same for a whole warp.
template <typename T>
__device__ __forceinline__ float ds_scale(const BwdParams& p, int b, int hk, int lane) {
  if (!kSized<T>) return 1.f;
  const long long at = (long long)b * p.a.kv_heads + hk, rows = (long long)p.q_tiles * p.a.group, keys = p.kv_tiles;
  const float *of_rows = p.sizes + at * rows, *of_keys = p.sizes + p.size_rows + at * keys;
  unsigned d2 = 0, v2 = 0;
  for (long long k = lane; k < rows; k += 32) d2 = max(d2, __float_as_uint(of_rows[k]));
  for (long long k = lane; k < keys; k += 32) v2 = max(v2, __float_as_uint(of_keys[k]));
  const float bound = 2.f * sqrtf(__uint_as_float(__reduce_max_sync(0xffffffffu, d2))) *
                      sqrtf(__uint_as_float(__reduce_max_sync(0xffffffffu, v2)));
  // 2^-47 to 2^41, or 0
  return bound > 0.f ? __uint_as_float((2 * 127 + 13 - (__float_as_uint(bound) >> 23)) << 23) : 1.f;
}

// Query tiles before this one have rows of few keys, as far as causality and the first key that a mask leaves tell (or none).
template <bool MASK>
__device__ __forceinline__ int few_key_tiles(const BwdParams& p, int b) {
  const int2 seen = MASK ? p.seen[b] : make_int2(0, p.a.kv_len);
  if (seen.y <= kFewKeys) return 0x7fffffff;
  // the row that sees kFewKeys keys from that first one on
  const int last = seen.x + kFewKeys - 1 - (p.a.kv_len - p.a.q_len);
  return p.a.causal && last >= 0 ? last / kRows + 1 : 0;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Rows of an accumulator (32 columns at a time) to [position][entry], times `mul`; zeros where !any.
template <typename T>
__device__ __forceinline__ void store_rows(T* dst, uint32_t at, int col0, int col1, int dim, bool live, bool any, float mul) {
  for (int q = col0; q < col1; q += 32) {
    uint32_t o[32];
    tmem_ld32(at + q, o);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; e += 8)
      if (live && q + e < dim) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (any) {
          v.x = pack2<T>(__uint_as_float(o[e]) * mul, __uint_as_float(o[e + 1]) * mul);
          v.y = pack2<T>(__uint_as_float(o[e + 2]) * mul, __uint_as_float(o[e + 3]) * mul);
          v.z = pack2<T>(__uint_as_float(o[e + 4]) * mul, __uint_as_float(o[e + 5]) * mul);
          v.w = pack2<T>(__uint_as_float(o[e + 6]) * mul, __uint_as_float(o[e + 7]) * mul);
        }
        *reinterpret_cast<uint4*>(dst + q + e) = v;
      }
  }
}

// The same in 32 bits.
__device__ __forceinline__ void store_part(float* dst, uint32_t at, int col0, int col1, int dim, bool live, bool any, float mul) {
  for (int q = col0; q < col1; q += 32) {
    uint32_t o[32];
    tmem_ld32(at + q, o);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; e += 4)
      if (live && q + e < dim)
        *reinterpret_cast<float4*>(dst + q + e) =
            any ? make_float4(__uint_as_float(o[e]) * mul, __uint_as_float(o[e + 1]) * mul, __uint_as_float(o[e + 2]) * mul,
                              __uint_as_float(o[e + 3]) * mul)
                : make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

template <typename T, int PANELS, bool MASK, bool KEYS>
__device__ __forceinline__ void bwd_block(const BwdParams& p, unsigned x, uint8_t* smem) {
  using L = BwdSmem<PANELS, MASK>;
  constexpr int STAGES = L::STAGES;
  uint8_t *r1 = smem, *r2 = smem + L::TILE, *ring = smem + 2 * L::TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t *fixed = bars, *full = fixed + 1, *empty = full + STAGES, *t1_full = empty + STAGES, *t2_full = t1_full + 1,
           *p_ready = t2_full + 1, *ds_ready = p_ready + 1, *done = ds_ready + 1, *sized = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sized + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* size_slot = reinterpret_cast<float*>(tmem_slot + 2);
  // the same in all lanes, and known to be: the roles below then run as uniform code
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int off = p.a.kv_len - p.a.q_len;  // under causality query i sees keys up to i + off
  int* status = p.a.status;

  // the block's rows, and the tiles of the other side that it passes over
  const int splits = KEYS ? p.split_k : p.split_q;
  int split = 0;
  if (splits > 1) {
    split = (int)(x % splits);
    x /= splits;
  }
  int tile, h, b, first = 0, tiles;
  if (KEYS) {
    tile = (int)(x % p.kv_tiles);  // under causality the first keys are seen by the most queries
    x /= p.kv_tiles;
    h = (int)(x % p.a.kv_heads);
    b = (int)(x / p.a.kv_heads);
    if (p.a.causal) first = min(p.q_tiles, max(0, tile * kRows - off) / kRows);
    tiles = p.q_tiles - first;
  } else {
    tile = p.q_tiles - 1 - (int)(x % p.q_tiles);
    x /= p.q_tiles;
    h = (int)(x % p.a.heads);
    b = (int)(x / p.a.heads);
    const int keys = p.a.causal ? max(0, min(p.a.kv_len, min((tile + 1) * kRows, p.a.q_len) + off)) : p.a.kv_len;
    tiles = (keys + kRows - 1) / kRows;
  }
  const int row0 = tile * kRows;
  const unsigned char* mask = MASK ? p.a.mask + b * p.a.mask_stride : nullptr;

  if (warp == LOADER && lane == 0) {
    mbar_init(fixed, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    mbar_init(t1_full, 1);
    mbar_init(t2_full, 1);
    mbar_init(p_ready, 4 * PARTS);
    mbar_init(ds_ready, 4 * PARTS);
    mbar_init(done, 1);
    mbar_init(sized, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  // steps: query tiles of every head of the group, or tiles of keys of which some are seen
  int steps = KEYS ? tiles * p.a.group : tiles, begin = 0;
  if (splits > 1) {  // this block's share of them
    const int share = (steps + splits - 1) / splits;
    begin = min(steps, split * share);
    steps = min(steps, begin + share);
  }
  auto load_fixed = [&] {
    mbar_arrive_expect_tx(fixed, 2 * L::TILE);
#pragma unroll
    for (int i = 0; i < PANELS; ++i) {
      tma_load_4d(r1 + i * kPanel, KEYS ? &p.mk : &p.mq, fixed, i * 64, row0, h, b);
      tma_load_4d(r2 + i * kPanel, KEYS ? &p.mv : &p.mdo, fixed, i * 64, row0, h, b);
    }
  };
  // operand k (0: queries with their statistics, or keys; 1: dout, or values) of step j, into a stage
  auto load_step = [&](int j, int k, int s) {
    const int t = KEYS ? first + j % tiles : j, hh = KEYS ? h * p.a.group + j / tiles : h / p.a.group;
    const bool stats = KEYS && k == 0;
    mbar_arrive_expect_tx(full + s, L::TILE + (stats ? 1024 : 0));
    const CUtensorMap* map = KEYS ? (k ? &p.mdo : &p.mq) : (k ? &p.mv : &p.mk);
#pragma unroll
    for (int i = 0; i < PANELS; ++i) tma_load_4d(ring + s * L::TILE + i * kPanel, map, full + s, i * 64, t * kRows, hh, b);
    if (stats)
      bulk_load(smem + L::STATS + s / 2 * 1024, p.stats + (((long long)b * p.a.heads + hh) * p.q_tiles + t) * 256, 1024,
                full + s);
  };
  if (MASK && !KEYS)
    pack_key_bits(reinterpret_cast<uint32_t*>(smem + L::BITS) - begin * 4, mask, begin, steps, p.a.kv_len, warp, BWD_THREADS / 32, lane);
  if (warp == ISSUER) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  bool dead_key = false;  // this thread's key row is masked
  if (MASK && KEYS) {
    const int j = row0 + (int)threadIdx.x % kRows;
    dead_key = j < p.a.kv_len && !mask[j];
  }
  tc_fence_before();
  // a tile of masked keys alone has nothing to do
  if (MASK && KEYS) {
    if (!__syncthreads_or(!dead_key && row0 + (int)threadIdx.x % kRows < p.a.kv_len)) steps = begin;
  } else {
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, t1 = tmem, t2 = tmem + 128, acc1 = tmem + 256, acc2 = tmem + 256 + 64 * PANELS;
  const KeyBits bits{MASK && !KEYS ? reinterpret_cast<const uint4*>(smem + L::BITS) - begin : nullptr};
  const int start = bits.next(begin, steps);

  if (warp >= LOADER) {
    regs_dec<kRestRegs>();
    if (warp == LOADER) {
      if (lane == 0 && start < steps) {
        load_fixed();
        if (KEYS) wait_dependency();
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int j = start; ok && j < steps; j = bits.next(j + 1, steps)) {
          for (int k = 0; k < 2; ++k) {
            if (!(ok = mbar_wait(empty + s, ph ^ 1, abort_flag, status, ST_ATTN_LOAD))) break;
            load_step(j, k, s);
            if (++s == STAGES) s = 0, ph ^= 1;
          }
        }
        drain_loads<STAGES>(full, s, ph, status);
        drain_loads<1>(fixed, 1, 0, status);
      }
      __syncwarp();
    } else if (warp == ISSUER) {
      // The whole warp runs along, so that addresses and descriptors stay in uniform registers; one lane issues.
      const int ksteps = (p.a.head_dim + 15) / 16;
      const uint32_t idesc_t = make_idesc(128, 128, umma_format<T>(), 0, 0);
      const uint32_t idesc_a = make_idesc(128, ksteps * 16, umma_format<T>(), 0, 1);
      const uint32_t ra1 = smem_u32(r1), ra2 = smem_u32(r2), xa = smem_u32(ring);
      if (MASK) wait_dependency();
      const bool low = (KEYS ? first : tile) < few_key_tiles<MASK>(p, b);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && warp_wait(bar, parity, abort_flag, status, ST_ATTN_MMA);
        tc_fence_after();
        return ok;
      };
      int s = 0;  // stage of the step's first tile; the second lies in the next (the stage count is even)
      uint32_t ph = 0, pph = 0, more = 0;
      auto scores1 = [&] {
        mma_scores<PANELS>(t1, ra1, xa + s * L::TILE, idesc_t, ksteps);
        umma_commit(t1_full);
      };
      auto scores2 = [&] {
        mma_scores<PANELS>(t2, ra2, xa + (s + 1) * L::TILE, idesc_t, ksteps);
        umma_commit(t2_full);
        if (!KEYS) umma_commit(empty + s + 1);
      };
      int j = start;
      if (j < steps && wait(fixed, 0) && wait(full, 0)) {
        if (elect_one()) scores1();
        __syncwarp();
        if (wait(full + 1, 0)) {
          if (elect_one()) scores2();
          __syncwarp();
        }
      }
      while (ok && j < steps) {
        const uint32_t x1 = xa + s * L::TILE, x2 = x1 + L::TILE;
        uint64_t* left = empty + s;
        s += 2;
        if (s == STAGES) s = 0, ph ^= 1;
        const int jn = bits.next(j + 1, steps);
        if (jn < steps && !wait(full + s, ph)) break;
        if (!wait(p_ready, pph)) break;
        if (elect_one()) {
          if (KEYS) {
            mma_probs<128, COLS, COLS>(acc1, t1, x2, idesc_a, more);
            umma_commit(left + 1);
          }
          if (jn < steps) scores1();
        }
        __syncwarp();
        if (jn < steps && !wait(full + s + 1, ph)) break;
        if (!wait(ds_ready, pph)) break;
        if (elect_one()) {
          mma_probs<128, COLS, COLS>(acc2, t2, x1, idesc_a, more);
          if (low) mma_probs<128, COLS, COLS>(acc2, t2 + COLS / 2, x1, idesc_a, 1);
          umma_commit(left);
          if (jn < steps) scores2();
        }
        __syncwarp();
        more = 1;
        pph ^= 1;
        j = jn;
      }
      // the sums are whole, and no product may be writing TMEM when it is released
      if (elect_one()) umma_commit(done);
      __syncwarp();
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(done, 0))
        if (globaltimer_ns() - t0 > LSR_WAIT_TIMEOUT_NS) {
          set_status(status, ST_ATTN_DONE);
          *abort_flag = 1;
          break;
        }
      __syncwarp();
    } else if (kSized<T> && warp == SIZER) {
      wait_dependency();
      const float up = ds_scale<T>(p, b, KEYS ? h : h / p.a.group, lane);
      if (lane == 0) {
        *size_slot = up;
        mbar_arrive(sized);
      }
    }
  } else {
    regs_inc<kScoreRegs>();
    const int part = warp / 4, r = warp % 4 * 32 + lane, row = row0 + r;
    const uint32_t quarter = (uint32_t)(warp % 4 * 32) << 16;
    const uint32_t my1 = t1 + part * COLS + quarter, my2 = t2 + part * COLS + quarter;
    const float c = p.a.scale * kLog2e;
    const uint64_t c2 = pair(c, c);
    bool ok = true;
    uint32_t ph = 0;
    int cur = 0;  // stage of the step's first tile
    uint32_t sph = 0;
    float lse = 0.f, delta = 0.f;
    if (MASK || !KEYS) wait_dependency();
    const bool low = (KEYS ? first : tile) < few_key_tiles<MASK>(p, b);
    if (!KEYS) {
      const float* st = p.stats + (((long long)b * p.a.heads + h) * p.q_tiles + tile) * 256 + r;
      lse = st[0] + (float)kExtra<T>;
      delta = st[128];
    }
    if (kSized<T>) ok = warp_wait(sized, 0, abort_flag, status, ST_ATTN_SOFTMAX);
    auto run = [&](auto parts) {
      for (int j = start; ok && j < steps; j = bits.next(j + 1, steps)) {
        const int t0 = (KEYS ? first + j % tiles : j) * kRows + part * COLS;  // position of the thread's first column
        // the statistics come with the step's first tile
        if (KEYS && !(ok = warp_wait(full + cur, sph, abort_flag, status, ST_ATTN_SOFTMAX))) break;
        const float4* stat = reinterpret_cast<const float4*>(smem + L::STATS + cur / 2 * 1024) + part * (COLS / 4);
        if (!(ok = warp_wait(t1_full, ph, abort_flag, status, ST_ATTN_SOFTMAX))) break;
        tc_fence_after();
        uint32_t s[COLS];
        tmem_ld32(my1, s);
        tmem_ld_wait();
        uint32_t word = ~0u;  // which of the thread's keys are seen
        if (MASK && !KEYS) word = reinterpret_cast<const uint32_t*>(bits.bits + j)[part];
        if (KEYS) {
          if (p.a.causal && row0 + kRows - 1 > t0 + off) {
            const int from = row - off - t0;  // queries before it do not see the key
#pragma unroll
            for (int e = 0; e < COLS; ++e)
              if (e < from) s[e] = 0xff800000u;
          }
        } else {
          warp_arrive(p_ready, lane);  // T1 is in registers
          const int sees = min(p.a.kv_len, p.a.causal ? row + off + 1 : p.a.kv_len) - t0;
          if (word != ~0u || t0 + COLS > p.a.kv_len || (p.a.causal && t0 + COLS - 1 > row0 + off)) {
#pragma unroll
            for (int e = 0; e < COLS; ++e)
              if (e >= sees || (MASK && !((word >> e) & 1))) s[e] = 0xff800000u;
          }
        }
#pragma unroll
        for (int e = 0; e < COLS; e += 4) {
          const float4 v = KEYS ? stat[e / 4] : make_float4(lse, lse, lse, lse);
          float x[4];
          unpair(fma2(pair(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, pair(-v.x, -v.y)), x[0], x[1]);
          unpair(fma2(pair(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])), c2, pair(-v.z, -v.w)), x[2], x[3]);
#pragma unroll
          for (int k = 0; k < 4; ++k) s[e + k] = __float_as_uint(ex2(x[k]));
        }
        if (KEYS) {
          uint32_t pr[COLS / 2];
#pragma unroll
          for (int e = 0; e < COLS / 2; ++e) pr[e] = pack2<T>(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
          tmem_st16(my1, pr);
          tmem_st_wait();
          warp_arrive(p_ready, lane);
        }
        if (!(ok = warp_wait(t2_full, ph, abort_flag, status, ST_ATTN_SOFTMAX))) break;
        tc_fence_after();
        uint32_t d[COLS], pr[COLS / 2];
        tmem_ld32(my2, d);
        tmem_ld_wait();
        if (word != ~0u) {  // what a hidden key's values hold must not reach 0 times it
#pragma unroll
          for (int e = 0; e < COLS; ++e)
            if (!((word >> e) & 1)) d[e] = 0;
        }
        // kSized: P times 2^x (read again in every step: there are no registers to spare), and without its extra power
        const float up = kSized<T> ? *size_slot : 1.f;
        const uint64_t by = pair(up * (1.f / (1 << (KEYS ? kExtra<T> : 0))), up * (1.f / (1 << (KEYS ? kExtra<T> : 0))));
#pragma unroll
        for (int e = 0; e < COLS; e += 4) {
          const float4 v = KEYS ? stat[32 + e / 4] : make_float4(delta, delta, delta, delta);
          uint64_t p0 = pair(__uint_as_float(s[e]), __uint_as_float(s[e + 1]));
          uint64_t p1 = pair(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
          if (kSized<T>) p0 = mul2(p0, by), p1 = mul2(p1, by);
          float x[4];
          unpair(mul2(add2(pair(__uint_as_float(d[e]), __uint_as_float(d[e + 1])), pair(-v.x, -v.y)), p0), x[0], x[1]);
          unpair(mul2(add2(pair(__uint_as_float(d[e + 2]), __uint_as_float(d[e + 3])), pair(-v.z, -v.w)), p1), x[2], x[3]);
          pr[e / 2] = pack2<T>(x[0], x[1]);
          pr[e / 2 + 1] = pack2<T>(x[2], x[3]);
          if (parts.value == 2) {
#pragma unroll
            for (int k = 0; k < 4; ++k) d[e + k] = __float_as_uint(x[k]);
          }
        }
        tmem_st16(my2, pr);
        if (parts.value == 2) {  // what the rounding left, beside it
#pragma unroll
          for (int e = 0; e < COLS / 2; ++e) {
            const float2 hi = unpack2<T>(pr[e]);
            pr[e] = pack2<T>(__uint_as_float(d[2 * e]) - hi.x, __uint_as_float(d[2 * e + 1]) - hi.y);
          }
          tmem_st16(my2 + COLS / 2, pr);
        }
        if (MASK && !KEYS) {  // nor what its keys hold
          const uint32_t seen = reinterpret_cast<const uint32_t*>(bits.bits + j)[r / 32];
          if (!((seen >> lane) & 1) && part < PANELS) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(ring + cur * L::TILE + part * kPanel + r * 128 + e * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tmem_st_wait();
        warp_arrive(ds_ready, lane);
        ph ^= 1;
        cur += 2;
        if (cur == STAGES) cur = 0, sph ^= 1;
      }
    };
    if (low) run(std::integral_constant<int, 2>());  // two bodies: the common one keeps nothing for the second part
    else run(std::integral_constant<int, 1>());
    if (ok) ok = warp_wait(done, 0, abort_flag, status, ST_ATTN_SOFTMAX);
    tc_fence_after();
    if (ok) {
      const bool any = start < steps && !dead_key;
      const float back = kSized<T> ? 1.f / *size_slot : 1.f;
      constexpr int SHARE = 64 * PANELS / (PARTS / 2);  // half of the warpgroups store dv, half dk
      const bool second = part >= PARTS / 2;
      const int col = part % (PARTS / 2) * SHARE;
      if (splits > 1) {
        const int len = KEYS ? p.a.kv_len : p.a.q_len, heads = KEYS ? p.a.kv_heads : p.a.heads;
        float* to = (KEYS ? (second ? p.part_dk : p.part_dv) : p.part_dq) +
                    ((((long long)split * p.a.batch + b) * heads + h) * len + row) * p.a.head_dim;
        if (KEYS) store_part(to, (second ? acc2 : acc1) + quarter, col, col + SHARE, p.a.head_dim, row < len, any,
                             second ? back : 1.f);
        else if (part < 2 * PANELS) store_part(to, acc2 + quarter, part * 32, part * 32 + 32, p.a.head_dim, row < len, any, back);
      } else if (KEYS) {
        const bool live = row < p.a.kv_len;
        if (!second)
          store_rows(attn_at<T>(p.a.dv, p.a.sdv, b, h) + row * p.a.sdv.s, acc1 + quarter, col, col + SHARE, p.a.head_dim, live, any,
                     1.f / (1 << kExtra<T>));
        else
          store_rows(attn_at<T>(p.a.dk, p.a.sdk, b, h) + row * p.a.sdk.s, acc2 + quarter, col, col + SHARE, p.a.head_dim, live, any,
                     p.a.scale * back);
      } else if (part < 2 * PANELS) {
        store_rows(attn_at<T>(p.a.dq, p.a.sdq, b, h) + row * p.a.sdq.s, acc2 + quarter, part * 32, part * 32 + 32, p.a.head_dim,
                   row < p.a.q_len, any, p.a.scale * back);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == ISSUER) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int PANELS, bool MASK>
__global__ void __launch_bounds__(BWD_THREADS, 1) attn_bwd_kernel(const __grid_constant__ BwdParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (1024 - (smem_u32(smem_raw) & 1023)) % 1024;
  if (blockIdx.x < p.kv_blocks) bwd_block<T, PANELS, MASK, true>(p, blockIdx.x, smem);
  else bwd_block<T, PANELS, MASK, false>(p, blockIdx.x - (unsigned)p.kv_blocks, smem);
}

// The sums of several blocks added in order and rounded, a warp per row of dq, dk or dv.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_grads_kernel(const __grid_constant__ BwdParams p) {
  const long long rq = p.split_q > 1 ? (long long)p.a.batch * p.a.heads * p.a.q_len : 0;
  const long long rk = p.split_k > 1 ? (long long)p.a.batch * p.a.kv_heads * p.a.kv_len : 0;
  long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  if (row >= rq + 2 * rk) return;
  const int which = row < rq ? 0 : row < rq + rk ? 1 : 2;  // dq, dk, dv
  row -= which == 0 ? 0 : which == 1 ? rq : rq + rk;
  const int len = which ? p.a.kv_len : p.a.q_len, heads = which ? p.a.kv_heads : p.a.heads;
  const int splits = which ? p.split_k : p.split_q, e = threadIdx.x % 32 * 4;
  if (e >= p.a.head_dim) return;
  const float* from = (which == 0 ? p.part_dq : which == 1 ? p.part_dk : p.part_dv) + row * p.a.head_dim + e;
  const long long step = (which ? rk : rq) * p.a.head_dim;
  float x[4] = {};
  for (int s = 0; s < splits; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(from + s * step);
    x[0] += v.x;
    x[1] += v.y;
    x[2] += v.z;
    x[3] += v.w;
  }
  const float mul = which == 2 ? 1.f / (1 << kExtra<T>) : p.a.scale;
  const int i = (int)(row % len), h = (int)(row / len % heads), b = (int)(row / len / heads);
  const AttnStride& sd = which == 0 ? p.a.sdq : which == 1 ? p.a.sdk : p.a.sdv;
  T* dst = attn_at<T>(which == 0 ? p.a.dq : which == 1 ? p.a.dk : p.a.dv, sd, b, h) + i * sd.s + e;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(x[0] * mul, x[1] * mul), pack2<T>(x[2] * mul, x[3] * mul));
}

template <typename T, int PANELS, bool MASK>
int launch(BwdParams& p, cudaStream_t st) {
  using L = BwdSmem<PANELS, MASK>;
  static_assert(L::TOTAL <= 232448, "shared memory budget exceeded");
  const long long blocks = p.kv_blocks + (long long)p.q_tiles * p.a.heads * p.a.batch * p.split_q;
  const long long stat_blocks = p.size_rows + p.size_keys + (MASK ? p.a.batch : 0);
  if (blocks > 0x7fffffffll || stat_blocks > 0x7fffffffll) return LSR_ERR_SHAPE;
  {
    ProfScope prof(PK_EW_OTHER, st);
    attn_stats_kernel<T><<<(unsigned)stat_blocks, 256, 0, st>>>(p);
    if (cudaGetLastError() != cudaSuccess) return LSR_ERR_LAUNCH;
  }
  auto kernel = attn_bwd_kernel<T, PANELS, MASK>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL) != cudaSuccess)
    return LSR_ERR_LAUNCH;
  {
    ProfScope prof(PK_GEMM_OTHER, st);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(BWD_THREADS);
    cfg.dynamicSmemBytes = L::TOTAL;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the blocks are set up while the statistics are taken
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) return LSR_ERR_LAUNCH;
  }
  const long long joined = (p.split_q > 1 ? (long long)p.a.batch * p.a.heads * p.a.q_len : 0) +
                           (p.split_k > 1 ? 2ll * p.a.batch * p.a.kv_heads * p.a.kv_len : 0);
  if (joined == 0) return LSR_OK;
  ProfScope prof(PK_EW_OTHER, st);
  attn_join_grads_kernel<T><<<(unsigned)((joined + 7) / 8), 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? LSR_OK : LSR_ERR_LAUNCH;
}

// Blocks that the steps of one set of rows are dealt to: one, unless they are one and a half times what an SM
// has on average or more (few keys under many queries, or few queries over many keys), and four steps at least.
int split_count(long long steps, long long mean) {
  mean = std::max<long long>(mean, 4);
  return 2 * steps >= 3 * mean ? (int)std::min<long long>((steps + mean - 1) / mean, 64) : 1;
}

void set_splits(BwdParams& p) {
  p.q_tiles = cdiv(p.a.q_len, kRows);
  p.kv_tiles = cdiv(p.a.kv_len, kRows);
  const long long k_sets = (long long)p.kv_tiles * p.a.kv_heads * p.a.batch, k_steps = (long long)p.q_tiles * p.a.group;
  const long long q_sets = (long long)p.q_tiles * p.a.heads * p.a.batch, q_steps = p.kv_tiles;
  const long long sms = device_sm_count(), mean = (k_sets * k_steps + q_sets * q_steps + sms - 1) / sms;
  p.split_k = split_count(k_steps, mean);
  p.split_q = std::max(split_count(q_steps, mean), mask_splits(p.a));
}

template <typename T>
int backward(BwdParams& p, cudaStream_t st) {
  if (p.a.head_dim > 64) return p.a.mask ? launch<T, 2, true>(p, st) : launch<T, 2, false>(p, st);
  return p.a.mask ? launch<T, 1, true>(p, st) : launch<T, 1, false>(p, st);
}

// Where the workspace's parts begin, each on 16 bytes; the partial sums come last. The floats before those.
size_t place(BwdParams& p, int dtype, void* ws) {
  const auto up4 = [](size_t n) { return (n + 3) / 4 * 4; };
  p.size_rows = (long long)p.q_tiles * p.a.heads * p.a.batch;
  p.size_keys = dtype == LSR_DTYPE_F16 ? (long long)p.kv_tiles * p.a.kv_heads * p.a.batch : 0;
  p.stats = static_cast<float*>(ws);
  const size_t sizes = (size_t)p.size_rows * 256;
  const size_t seen = sizes + (dtype == LSR_DTYPE_F16 ? up4(p.size_rows + p.size_keys) : 0);
  p.sizes = p.stats + sizes;
  p.seen = reinterpret_cast<int2*>(p.stats + seen);
  return seen + (p.a.mask ? up4(2 * (size_t)p.a.batch) : 0);
}

}  // namespace

size_t attention_backward_sm100_ws(const AttnParams& a, int dtype) {
  BwdParams p{};
  p.a = a;
  set_splits(p);
  size_t floats = place(p, dtype, nullptr);
  if (p.split_k > 1) floats += (size_t)p.split_k * 2 * a.batch * a.kv_heads * a.kv_len * a.head_dim;
  if (p.split_q > 1) floats += (size_t)p.split_q * a.batch * a.heads * a.q_len * a.head_dim;
  return floats * sizeof(float);
}

int attention_backward_sm100(const AttnParams& a, int dtype, void* ws, cudaStream_t st) {
  BwdParams p{};
  p.a = a;
  set_splits(p);
  p.part_dk = static_cast<float*>(ws) + place(p, dtype, ws);
  const size_t kv = p.split_k > 1 ? (size_t)p.split_k * a.batch * a.kv_heads * a.kv_len * a.head_dim : 0;
  p.part_dv = p.part_dk + kv;
  p.part_dq = p.part_dv + kv;
  p.kv_blocks = (long long)p.kv_tiles * a.kv_heads * a.batch * p.split_k;
  int rc = encode_rows(&p.mq, a.q, a.sq, a.batch, a.heads, a.q_len, a.head_dim, dtype);
  if (rc == LSR_OK) rc = encode_rows(&p.mdo, a.dout, a.sdo, a.batch, a.heads, a.q_len, a.head_dim, dtype);
  if (rc == LSR_OK) rc = encode_rows(&p.mk, a.k, a.sk, a.batch, a.kv_heads, a.kv_len, a.head_dim, dtype);
  if (rc == LSR_OK) rc = encode_rows(&p.mv, a.v, a.sv, a.batch, a.kv_heads, a.kv_len, a.head_dim, dtype);
  if (rc != LSR_OK) return rc;
  return dtype == LSR_DTYPE_BF16 ? backward<__nv_bfloat16>(p, st) : backward<__half>(p, st);
}

}  // namespace lsr
