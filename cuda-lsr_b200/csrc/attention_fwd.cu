// Softmax attention's forward pass on the tensor cores, 16-bit types.
//
//   per key tile:  S = Q K^T;  m' = max(m, rowmax S);  P = exp2((S - m') c);  l = l 2^((m - m') c) + rowsum P;
//                  O = O 2^((m - m') c) + P V;      c = scale log2 e
//   at the end:    out = O / l,  lse = (m c + log2 l) ln 2
//
// A block owns NQ tiles of 128 queries of one head and passes once over its keys. Warp 4 NQ loads
// (TMA, a ring of key and value tiles), the warps after it issue the products, and one warpgroup per
// query tile does the softmax, a thread per query: a row's maximum and sum need no exchange. S and O
// stay in TMEM; P goes back to TMEM as the 16-bit operand of P V, so scores and probabilities never
// touch shared memory. While one query tile is in its softmax the tensor core works for the other.
// What bounds it: per 128 x 128 tile the exponentials take 1024 cycles of the special function units and
// the products 1024 cycles of the tensor core at dim 128, 512 at dim 64. Measured (bf16, 4 x 16 heads x
// 4096, no mask): dim 128 464 to 499 us from run to run, 1100 to 1185 TFLOP/s; dim 64 350 to 367 us, 749 to
// 786 TFLOP/s, where those units take instructions in 75% of the cycles and the tensor core works in 37%. Exponentials by polynomial on the FMA
// units for one pair in eight made it slower (413 us): issue slots and latency, not the units, are short.
// O is rescaled only when a row's maximum has grown by more than 2^8 since it last was: until then P is
// taken against the old maximum, which fp32 sums and 16-bit P (at most 2^8) hold without loss, and O /
// l is the same. P is rounded to 16 bits for the product (l adds it unrounded).
// A row that sees no key has l = 0: out 0, lse minus infinity.
#include "attention_sm100.cuh"

namespace lsr {
namespace {

constexpr float kLazy = 8.f;  // log2 of the growth that the running maximum may be behind by

struct FwdParams {
  AttnParams a;
  CUtensorMap mq, mk, mv;
  int q_blocks, splits;
  float* part_out;  // [split][row][dim], splits > 1
  float* part_lse;  // [split][row]
};

template <int PANELS, int NQ, bool MASK>
struct FwdSmem {
  static constexpr int TILE = PANELS * kPanel;
  static constexpr int STAGES = NQ == 2 ? (PANELS == 1 ? 8 : 4) : (PANELS == 1 ? 4 : 2);
  static constexpr int BARS = (NQ + STAGES) * TILE;
  static constexpr int BITS = BARS + 256;  // 16 bytes per key tile of the block
  // With room to align the tiles. A launch asks for the key tiles that it has, so that masked blocks of one query
  // tile, too, share an SM (3 rows on 4097 keys, 4 x 12 heads: 34 us with room for the longest mask, now 24).
  static constexpr int total(int tiles) { return BITS + (MASK ? tiles * 16 : 0) + 1024; }
  static constexpr int TOTAL = total(kMaskTiles);
};

// Queries [i0, i0 + 128): how many tiles of keys they see, at most.
__device__ __forceinline__ int key_tiles(const AttnParams& p, int i0) {
  if (i0 >= p.q_len) return 0;
  const int last = min(i0 + kRows, p.q_len) - 1 + (p.kv_len - p.q_len);  // the last key of the last query
  const int keys = p.causal ? max(0, min(p.kv_len, last + 1)) : p.kv_len;
  return (keys + kRows - 1) / kRows;
}

// The softmax warpgroups hold a row of 128 scores a thread and take the registers that the last
// warpgroup, of the loader and the issuer, does not need: 2 x 128 = 208 + 48, 3 x 168 = 2 x 224 + 56.
constexpr int kSoftRegs(int nq) { return nq == 1 ? 208 : 224; }
constexpr int kRestRegs(int nq) { return nq == 1 ? 48 : 56; }

template <typename T, int PANELS, int NQ, bool MASK>
__global__ void __launch_bounds__(NQ * 128 + 128, NQ == 1 ? 2 : 1) attn_fwd_kernel(const __grid_constant__ FwdParams p) {
  using L = FwdSmem<PANELS, NQ, MASK>;
  constexpr int STAGES = L::STAGES;
  constexpr bool APART = PANELS == 1;  // P beside S: the next scores are computed while this tile is in its softmax
  // With room for P beside S the query tiles' products need no common order, and a warp issues for each: the
  // waits of one do not hold up the other (4 x 16 heads x 4096 x 64: 361 us, 381 with one issuer). Without it
  // one issuer keeps them in turn; two would interleave their products and finish both late (dim 128: 563 us, 499).
  constexpr int ISSUERS = APART ? NQ : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (1024 - (smem_u32(smem_raw) & 1023)) % 1024;
  uint8_t* sq = smem;
  uint8_t* skv = smem + NQ * L::TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t *q_full = bars, *full = q_full + NQ, *empty = full + STAGES, *s_full = empty + STAGES, *s_free = s_full + NQ,
           *p_ready = s_free + NQ, *pv_done = p_ready + NQ, *done = pv_done + NQ;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // the same in all lanes, and known to be: the roles below then run as uniform code
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  constexpr int LOADER = 4 * NQ, ISSUER = 4 * NQ + 1;

  unsigned x = blockIdx.x;
  const int split = (int)(x % p.splits);
  x /= p.splits;
  const int qb = p.q_blocks - 1 - (int)(x % p.q_blocks);  // under causality the longest first
  x /= p.q_blocks;
  const int h = (int)(x % p.a.heads), b = (int)(x / p.a.heads), hk = h / p.a.group;
  const int i0 = qb * NQ * kRows;
  int n[NQ], first = 0, most = 0;
#pragma unroll
  for (int w = 0; w < NQ; ++w) {
    n[w] = key_tiles(p.a, i0 + w * kRows);
    most = max(most, n[w]);
  }
  if (p.splits > 1) {  // this block's share of the key tiles
    const int per = (most + p.splits - 1) / p.splits;
    first = split * per;
    most = min(most, first + per);
#pragma unroll
    for (int w = 0; w < NQ; ++w) n[w] = min(n[w], most);
  }

  if (warp == LOADER && lane == 0) {
    for (int w = 0; w < NQ; ++w) {
      mbar_init(q_full + w, 1);
      mbar_init(s_full + w, 1);
      mbar_init(s_free + w, 4);
      mbar_init(p_ready + w, 4);
      mbar_init(pv_done + w, 1);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, ISSUERS);
    }
    mbar_init(done, ISSUERS);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (MASK)
    pack_key_bits(reinterpret_cast<uint32_t*>(smem + L::BITS) - first * 4, p.a.mask + b * p.a.mask_stride, first, most, p.a.kv_len, warp,
                  NQ * 4 + 4, lane);
  if (warp == ISSUER) {
    tmem_alloc(tmem_slot, NQ == 2 ? 512 : 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // columns: S of each query tile, O of each, and P of its own if there is room, else over S
  const uint32_t tmem = *tmem_slot;
  auto s_at = [&](int w) { return tmem + w * 128; };
  auto o_at = [&](int w) { return tmem + NQ * 128 + w * 64 * PANELS; };
  auto p_at = [&](int w) { return APART ? tmem + NQ * 192 + w * 64 : tmem + w * 128; };
  const KeyBits bits{MASK ? reinterpret_cast<const uint4*>(smem + L::BITS) - first : nullptr};

  if (warp >= LOADER) {
    regs_dec<kRestRegs(NQ)>();
    if (warp == LOADER) {
      if (lane == 0) {
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        const int j0 = bits.next(first, most);
        for (int w = 0; w < NQ; ++w)
          if (n[w] > j0) load_rows<PANELS>(sq + w * L::TILE, &p.mq, q_full + w, i0 + w * kRows, h, b);
        for (int j = j0; ok && j < most; j = bits.next(j + 1, most)) {
          for (int kv = 0; kv < 2; ++kv) {
            if (!(ok = mbar_wait(empty + s, ph ^ 1, abort_flag, p.a.status, ST_ATTN_LOAD))) break;
            load_rows<PANELS>(skv + s * L::TILE, kv ? &p.mv : &p.mk, full + s, j * kRows, hk, b);
            if (++s == STAGES) s = 0, ph ^= 1;
          }
        }
        drain_loads<STAGES>(full, s, ph, p.a.status);
        for (int w = 0; w < NQ; ++w)
          if (n[w] > j0) drain_loads<1>(q_full + w, 1, 0, p.a.status);
      }
      __syncwarp();
    } else if (warp < ISSUER + ISSUERS) {
      // The whole warp runs along, so that addresses and descriptors stay in uniform registers; one lane issues.
      const int ksteps = (p.a.head_dim + 15) / 16;
      const uint32_t idesc_s = make_idesc(128, 128, umma_format<T>(), 0, 0);
      const uint32_t idesc_o = make_idesc(128, ksteps * 16, umma_format<T>(), 0, 1);
      const uint32_t qa = smem_u32(sq), kva = smem_u32(skv);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && warp_wait(bar, parity, abort_flag, p.a.status, ST_ATTN_MMA);
        tc_fence_after();
        return ok;
      };
      auto scores = [&](int w, int s) {
        mma_scores<PANELS>(s_at(w), qa + w * L::TILE, kva + s * L::TILE, idesc_s, ksteps);
        umma_commit(s_full + w);
      };
      const int me = warp - ISSUER;
      auto mine = [&](int w) { return ISSUERS == 1 || w == me; };
      auto last = [&](int w) { return ISSUERS > 1 || w == NQ - 1; };  // of this issuer's: the stage is done with
      // stage and phase of the tile's keys; its values lie in the next stage (the stage count is even)
      int s = 0;
      uint32_t ph = 0, pph = 0;
      bool more = false;
      int j = bits.next(first, most);
      if (j < most && wait(full, 0)) {
#pragma unroll
        for (int w = 0; w < NQ; ++w) {
          if (!mine(w) || (j < n[w] && !wait(q_full + w, 0))) continue;
          if (elect_one()) {
            if (j < n[w]) scores(w, 0);
            if (last(w)) umma_commit(empty);
          }
          __syncwarp();
        }
      }
      while (ok && j < most) {
        const int vs = s + 1;
        const uint32_t vph = ph;
        s += 2;
        if (s == STAGES) s = 0, ph ^= 1;
        const int jn = bits.next(j + 1, most);
        if (APART && jn < most && wait(full + s, ph)) {
#pragma unroll
          for (int w = 0; w < NQ; ++w) {
            if (!mine(w) || (jn < n[w] && !wait(s_free + w, pph))) continue;
            if (elect_one()) {
              if (jn < n[w]) scores(w, s);
              if (last(w)) umma_commit(empty + s);
            }
            __syncwarp();
          }
        }
        if (!ok || !wait(full + vs, vph)) break;
#pragma unroll
        for (int w = 0; w < NQ; ++w) {
          if (!mine(w) || (j < n[w] && !wait(p_ready + w, pph))) continue;
          if (elect_one()) {
            if (j < n[w]) {
              mma_probs<128, 128, 0>(o_at(w), p_at(w), kva + vs * L::TILE, idesc_o, more);
              if (APART || jn >= n[w]) umma_commit(pv_done + w);
            }
            if (last(w)) umma_commit(empty + vs);
          }
          __syncwarp();
          if (!APART && jn < most && wait(full + s, ph)) {
            if (elect_one()) {
              if (jn < n[w]) scores(w, s);
              if (last(w)) umma_commit(empty + s);
            }
            __syncwarp();
          }
        }
        more = true;
        pph ^= 1;
        j = jn;
      }
      // no product may be writing TMEM when it is released
      if (elect_one()) umma_commit(done);
      __syncwarp();
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(done, 0))
        if (globaltimer_ns() - t0 > LSR_WAIT_TIMEOUT_NS) {
          set_status(p.a.status, ST_ATTN_DONE);
          break;
        }
      __syncwarp();
    }
  } else {
    regs_inc<kSoftRegs(NQ)>();
    const int w = warp / 4, r = (warp % 4) * 32 + lane, i = i0 + w * kRows + r;
    const int nw = NQ == 1 ? n[0] : (w ? n[NQ - 1] : n[0]);
    const bool idle = i0 + w * kRows + (warp % 4) * 32 >= p.a.q_len;  // none of the warp's rows exists
    const uint32_t at = (uint32_t)(warp % 4 * 32) << 16;
    const uint32_t st = s_at(w) + at, ot = o_at(w) + at, pt = p_at(w) + at;
    const float c = p.a.scale * kLog2e;
    // keys that the row sees, counted from the first
    const int sees = p.a.causal ? max(0, min(p.a.kv_len, i + 1 + p.a.kv_len - p.a.q_len)) : p.a.kv_len;
    const int sees_all = p.a.causal ? i0 + w * kRows + (warp % 4) * 32 + 1 + p.a.kv_len - p.a.q_len : p.a.kv_len;  // the warp's first row
    float m = -INFINITY, l = 0.f;
    bool ok = true, started = false;
    uint32_t ph = 0;
    int vs = 1;        // stage of the tile's values
    uint32_t vph = 0;  // and its phase
    for (int j = bits.next(first, nw); j < nw; j = bits.next(j + 1, nw)) {
      if (!(ok = warp_wait(s_full + w, ph, abort_flag, p.a.status, ST_ATTN_SOFTMAX))) break;
      tc_fence_after();
      uint4 word = make_uint4(~0u, ~0u, ~0u, ~0u);
      if (MASK) word = bits.bits[j];
      const bool holes = MASK && (word.x & word.y & word.z & word.w) != ~0u;
      if (!idle) {
        uint32_t sr[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(st + q * 32, sr[q]);
        tmem_ld_wait();
        if (APART) warp_arrive(s_free + w, lane);
        const int j0 = j * kRows;
        if (j0 + kRows > sees_all || j0 + kRows > p.a.kv_len || holes) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t wq = q == 0 ? word.x : q == 1 ? word.y : q == 2 ? word.z : word.w;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (j0 + q * 32 + e >= sees || (MASK && !((wq >> e) & 1))) sr[q][e] = 0xff800000u;
          }
        }
        float top[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          top[q] = fmaxf(__uint_as_float(sr[q][0]), __uint_as_float(sr[q][1]));
#pragma unroll
          for (int e = 2; e < 32; e += 2) top[q] = max3(top[q], __uint_as_float(sr[q][e]), __uint_as_float(sr[q][e + 1]));
        }
        const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const bool grown = (mx - m) * c > kLazy;  // false for NaN, as of two minus infinities
        // the product before has read P, and O may be rescaled (without P of its own the scores' wait said so)
        if (APART && started && !(ok = warp_wait(pv_done + w, ph ^ 1, abort_flag, p.a.status, ST_ATTN_SOFTMAX))) break;
        if (APART) tc_fence_after();
        if (__any_sync(0xffffffffu, grown)) {
          const float keep = grown ? ex2((m - mx) * c) : 1.f;
          if (grown) m = mx;
          l *= keep;
          if (started) {
#pragma unroll
            for (int q = 0; q < 2 * PANELS; ++q) {
              uint32_t o[32];
              tmem_ld32(ot + q * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
              tmem_st32(ot + q * 32, o);
            }
          }
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
        const uint64_t c2 = pair(c, c), mc2 = pair(-mc, -mc);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t pr[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const uint32_t* v = &sr[2 * q + e / 16][e % 16 * 2];
            const uint64_t x = fma2(pair(__uint_as_float(v[0]), __uint_as_float(v[1])), c2, mc2);
            float a0, a1;
            unpair(x, a0, a1);
            a0 = ex2(a0);
            a1 = ex2(a1);
            sum[e % 2] = add2(sum[e % 2], pair(a0, a1));
            pr[e] = pack2<T>(a0, a1);
          }
          tmem_st32(pt + q * 32, pr);
        }
        float l0, l1, l2, l3;
        unpair(sum[0], l0, l1);
        unpair(sum[1], l2, l3);
        l += (l0 + l1) + (l2 + l3);
        tmem_st_wait();
      } else if (APART) {
        warp_arrive(s_free + w, lane);
        // as the other warps, or its arrival for this tile could stand for theirs for the one before
        if (started && !(ok = warp_wait(pv_done + w, ph ^ 1, abort_flag, p.a.status, ST_ATTN_SOFTMAX))) break;
      }
      started = true;
      if (holes) {  // a hidden key's probability is 0, but 0 times what its values hold need not be
        if (!(ok = warp_wait(full + vs, vph, abort_flag, p.a.status, ST_ATTN_SOFTMAX))) break;
        const uint32_t wq = r < 32 ? word.x : r < 64 ? word.y : r < 96 ? word.z : word.w;
        if (!((wq >> lane) & 1)) {
#pragma unroll
          for (int d = 0; d < PANELS; ++d)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(skv + vs * L::TILE + d * kPanel + r * 128 + e * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      vs += 2;
      if (vs > STAGES) vs = 1, vph ^= 1;
      ph ^= 1;
      warp_arrive(p_ready + w, lane);
    }
    if (ok && started) ok = warp_wait(pv_done + w, APART ? ph ^ 1 : 0, abort_flag, p.a.status, ST_ATTN_SOFTMAX);
    tc_fence_after();
    if (ok && !idle) {
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      const long long row = ((long long)b * p.a.heads + h) * p.a.q_len + i;
      const float lse = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m * p.a.scale) + log2f(l) * kLn2;
      const bool live = i < p.a.q_len;
      if (p.splits > 1) {
        const long long rows = (long long)p.a.batch * p.a.heads * p.a.q_len;
        float* dst = p.part_out + (split * rows + row) * p.a.head_dim;
        if (live) p.part_lse[split * rows + row] = lse;
#pragma unroll
        for (int q = 0; q < 2 * PANELS; ++q) {
          uint32_t o[32];
          if (started) tmem_ld32(ot + q * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (live && q * 32 + e < p.a.head_dim) {
              float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
              if (started)
                v = make_float4(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv, __uint_as_float(o[e + 2]) * inv,
                                __uint_as_float(o[e + 3]) * inv);
              *reinterpret_cast<float4*>(dst + q * 32 + e) = v;
            }
        }
      } else {
        T* dst = attn_at<T>(p.a.out, p.a.so, b, h) + i * p.a.so.s;
        if (live) p.a.lse[row] = lse;
#pragma unroll
        for (int q = 0; q < 2 * PANELS; ++q) {
          uint32_t o[32];
          if (started) tmem_ld32(ot + q * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            if (live && q * 32 + e < p.a.head_dim) {
              uint4 v = make_uint4(0, 0, 0, 0);
              if (started) {
                v.x = pack2<T>(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
                v.y = pack2<T>(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
                v.z = pack2<T>(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
                v.w = pack2<T>(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
              }
              *reinterpret_cast<uint4*>(dst + q * 32 + e) = v;
            }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == ISSUER) {
    tc_fence_after();
    tmem_dealloc(tmem, NQ == 2 ? 512 : 256);
  }
}

// Rows of several splits joined: lse = log sum exp lse_s, out = sum exp(lse_s - lse) out_s; a warp per row.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ FwdParams p) {
  const long long rows = (long long)p.a.batch * p.a.heads * p.a.q_len;
  const long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  if (row >= rows) return;
  const int i = (int)(row % p.a.q_len), h = (int)(row / p.a.q_len % p.a.heads), b = (int)(row / p.a.q_len / p.a.heads);
  const int lane = threadIdx.x % 32;
  float top = -INFINITY;
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.part_lse[s * rows + row]);
  const float base = top == -INFINITY ? 0.f : top;
  float total = 0.f, o[4] = {};
  for (int s = 0; s < p.splits; ++s) {
    const float wgt = expf(p.part_lse[s * rows + row] - base);
    total += wgt;
    if (lane * 4 < p.a.head_dim) {
      const float4 v = *reinterpret_cast<const float4*>(p.part_out + (s * rows + row) * p.a.head_dim + lane * 4);
      o[0] = fmaf(wgt, v.x, o[0]);
      o[1] = fmaf(wgt, v.y, o[1]);
      o[2] = fmaf(wgt, v.z, o[2]);
      o[3] = fmaf(wgt, v.w, o[3]);
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (lane == 0) p.a.lse[row] = total == 0.f ? -INFINITY : base + logf(total);
  if (lane * 4 < p.a.head_dim) {
    T* dst = attn_at<T>(p.a.out, p.a.so, b, h) + i * p.a.so.s + lane * 4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
  }
}

template <typename T, int PANELS, int NQ, bool MASK>
int launch(FwdParams& p, cudaStream_t st) {
  using L = FwdSmem<PANELS, NQ, MASK>;
  static_assert(L::TOTAL <= 232448, "shared memory budget exceeded");
  p.q_blocks = cdiv(p.a.q_len, NQ * kRows);
  const long long blocks = (long long)p.q_blocks * p.a.heads * p.a.batch * p.splits;
  if (blocks > 0x7fffffffll) return LSR_ERR_SHAPE;
  auto kernel = attn_fwd_kernel<T, PANELS, NQ, MASK>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL) != cudaSuccess)
    return LSR_ERR_LAUNCH;
  ProfScope prof(PK_GEMM_OTHER, st);
  const int tiles = cdiv(cdiv(p.a.kv_len, kRows), p.splits);  // of a block's share, at most
  kernel<<<(unsigned)blocks, NQ * 128 + 128, L::total(tiles), st>>>(p);
  return cudaGetLastError() == cudaSuccess ? LSR_OK : LSR_ERR_LAUNCH;
}

template <typename T, int PANELS, int NQ>
int launch_mask(FwdParams& p, cudaStream_t st) {
  return p.a.mask ? launch<T, PANELS, NQ, true>(p, st) : launch<T, PANELS, NQ, false>(p, st);
}

// Two query tiles a block share the loads of keys and values and hide each other's softmax; with one
// the grid is twice as large.
int query_tiles(const AttnParams& p) {
  return (long long)cdiv(p.q_len, 2 * kRows) * p.heads * p.batch >= device_sm_count() ? 2 : 1;
}

// Blocks that the key tiles of a block's queries are dealt to when there are few queries: as many as
// the SMs have room for, with four tiles each at least, so that the join does not cost more than it saves. And as many
// as a long mask's bits take.
int split_count(const AttnParams& p) {
  const int pair = query_tiles(p), room = (pair == 2 ? 1 : 2) * device_sm_count();
  const long long blocks = (long long)cdiv(p.q_len, pair * kRows) * p.heads * p.batch;
  const int tiles = cdiv(p.kv_len, kRows);
  return (int)std::max<long long>(mask_splits(p), std::min<long long>(std::min<long long>(room / blocks, tiles / 4), 64));
}

template <typename T>
int forward(FwdParams& p, cudaStream_t st) {
  const bool wide = p.a.head_dim > 64;
  int rc;
  if (query_tiles(p.a) == 2) rc = wide ? launch_mask<T, 2, 2>(p, st) : launch_mask<T, 1, 2>(p, st);
  else rc = wide ? launch_mask<T, 2, 1>(p, st) : launch_mask<T, 1, 1>(p, st);
  if (rc != LSR_OK || p.splits == 1) return rc;
  const long long rows = (long long)p.a.batch * p.a.heads * p.a.q_len;
  ProfScope prof(PK_EW_OTHER, st);
  attn_join_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? LSR_OK : LSR_ERR_LAUNCH;
}

}  // namespace

bool rows_ok(const void* base, const AttnStride& s, int batch, int heads, int len, int dim) {
  const auto fits = [](long long st, int size) { return size == 1 || (st > 0 && st % 8 == 0 && st < (1ll << 36)); };
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && dim % 8 == 0 && fits(s.b, batch) && fits(s.s, len) &&
         fits(s.h, heads);
}

int encode_rows(CUtensorMap* map, const void* base, const AttnStride& s, int batch, int heads, int len, int dim, int dtype) {
  // the stride of a dimension of one entry says nothing; the map wants a valid one all the same
  const uint64_t any = (uint64_t)dim * 2;
  const uint64_t dims[4] = {(uint64_t)dim, (uint64_t)len, (uint64_t)heads, (uint64_t)batch};
  const uint64_t strides[3] = {len == 1 ? any : (uint64_t)s.s * 2, heads == 1 ? any : (uint64_t)s.h * 2,
                               batch == 1 ? any : (uint64_t)s.b * 2};
  const uint32_t box[4] = {64, kRows, 1, 1};
  return encode_tmap_4d(map, dtype == LSR_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        base, dims, strides, box);
}

size_t attention_forward_sm100_ws(const AttnParams& p) {
  const int splits = split_count(p);
  if (splits == 1) return 0;
  return (size_t)splits * p.batch * p.heads * p.q_len * (p.head_dim + 1) * sizeof(float) + 16;
}

int attention_forward_sm100(const AttnParams& a, int dtype, void* ws, cudaStream_t st) {
  FwdParams p{};
  p.a = a;
  p.splits = split_count(a);
  p.part_out = static_cast<float*>(ws);
  p.part_lse = p.part_out + (size_t)p.splits * a.batch * a.heads * a.q_len * a.head_dim;
  int rc = encode_rows(&p.mq, a.q, a.sq, a.batch, a.heads, a.q_len, a.head_dim, dtype);
  if (rc == LSR_OK) rc = encode_rows(&p.mk, a.k, a.sk, a.batch, a.kv_heads, a.kv_len, a.head_dim, dtype);
  if (rc == LSR_OK) rc = encode_rows(&p.mv, a.v, a.sv, a.batch, a.kv_heads, a.kv_len, a.head_dim, dtype);
  if (rc != LSR_OK) return rc;
  return dtype == LSR_DTYPE_BF16 ? forward<__nv_bfloat16>(p, st) : forward<__half>(p, st);
}

}  // namespace lsr
