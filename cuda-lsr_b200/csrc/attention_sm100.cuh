// What the tensor-core attention kernels share: 128-row tiles in shared memory, the products on them
// and the moves between registers and TMEM.
//
// A tile is 128 rows (positions of one head) by up to 128 entries, as one or two panels of 128 rows x
// 64 entries: rows of 128 bytes, 128-byte swizzled, 16 KB a panel, loaded by TMA with zeros past the
// tensor's end in either direction. The same bytes serve as an operand with its rows along M or N and
// the head's entries along K (K-major: scores), and with its rows along K and the entries along N
// (MN-major: products that take probabilities), so nothing is ever transposed.
#pragma once

#include "attention.cuh"

namespace lsr {

constexpr int kRows = 128;                 // of a tile
constexpr int kPanel = kRows * 128;        // bytes
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Status codes of waits that ran out (lsr_device_status).
enum : int { ST_ATTN_LOAD = 120, ST_ATTN_MMA = 121, ST_ATTN_SOFTMAX = 122, ST_ATTN_DONE = 123 };

// One lane of the warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
}

// D[tmem] (+)= A[tmem] * B[smem]: A is 128 lanes of 16-bit pairs, 8 columns per 16-deep step.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Store 32 consecutive 32-bit columns of this warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Give up or take registers, for a whole warpgroup (the block's total stays within what it was launched with).
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// mbar_wait of a whole warp: one answer for all lanes, which the .aligned TMEM moves after it need.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  const bool ok = mbar_wait(bar, parity, abort_flag, status, code);
  return __all_sync(0xffffffffu, ok);
}

// Before a block ends, also after a wait that ran out: its copies into shared memory have landed (`bars` count
// them, a ring of N; the next copy would have gone to stage s in phase ph). Bounded like every wait.
template <int N>
__device__ __forceinline__ void drain_loads(uint64_t* bars, int s, uint32_t ph, int* status) {
  const uint64_t t0 = globaltimer_ns();
  for (int i = 0; i < N; ++i)
    while (!mbar_try_wait(bars + i, i < s ? ph : ph ^ 1))
      if (globaltimer_ns() - t0 > LSR_WAIT_TIMEOUT_NS) {
        set_status(status, ST_ATTN_DONE);
        return;
      }
}

// One arrival for a whole warp, after what its lanes did before (moves to and from TMEM included).
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// Two floats as one 32-bit pair of the 16-bit type, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

template <typename T>
constexpr uint32_t umma_format();
template <>
constexpr uint32_t umma_format<__nv_bfloat16>() { return 1; }
template <>
constexpr uint32_t umma_format<__half>() { return 0; }

// D (128 x N) = A B^T over the heads' entries: both tiles K-major, B from its row `b_row` on, `steps` 16-entry steps.
template <int PANELS>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a_smem, uint32_t b_smem, uint32_t idesc, int steps,
                                           int b_row = 0) {
  const uint64_t a = smem_desc_sw128(a_smem, 16, 1024), b = smem_desc_sw128(b_smem + b_row * 128, 16, 1024);
#pragma unroll
  for (int k = 0; k < 4 * PANELS; ++k) {
    if (k >= steps) break;
    const uint64_t off = (uint64_t)((k >> 2) * (kPanel >> 4) + (k & 3) * 2);
    umma_bf16(d, a + off, b + off, idesc, k > 0);
  }
}

// D (128 x entries) (+)= P B over ROWS rows of the tile B, from `row` on: P in TMEM at p_tmem, the operands of
// each PER rows APART columns after those of the ones before.
template <int ROWS, int PER, int APART>
__device__ __forceinline__ void mma_probs(uint32_t d, uint32_t p_tmem, uint32_t b_smem, uint32_t idesc, uint32_t accumulate,
                                          int row = 0) {
  const uint64_t b = smem_desc_sw128(b_smem + row * 128, kPanel, 1024);
#pragma unroll
  for (int k = 0; k < ROWS / 16; ++k)
    umma_ts(d, p_tmem + (k * 16 / PER) * APART + (k * 16 % PER) / 2, b + (uint64_t)(k * (2048 >> 4)), idesc, accumulate || k > 0);
}

// One tile of [position][entry], panel by panel.
template <int PANELS>
__device__ __forceinline__ void load_rows(void* dst, const CUtensorMap* map, uint64_t* bar, int row0, int h, int b) {
  mbar_arrive_expect_tx(bar, PANELS * kPanel);
#pragma unroll
  for (int i = 0; i < PANELS; ++i) tma_load_4d(static_cast<uint8_t*>(dst) + i * kPanel, map, bar, i * 64, row0, h, b);
}

// Which of the keys of a tile are seen, 128 bits, kept for every tile of the batch entry.
struct KeyBits {
  const uint4* bits;
  // the first tile in [j, n) with a key that is seen
  __device__ __forceinline__ int next(int j, int n) const {
    if (bits)
      for (; j < n; ++j) {
        const uint4 w = bits[j];
        if (w.x | w.y | w.z | w.w) break;
      }
    return j;
  }
};
constexpr int kMaskTiles = 1536;  // that a block has room for, 24 KB of bits: of more than 196608 masked keys each block takes a share
inline int mask_splits(const AttnParams& p) { return p.mask ? cdiv(cdiv(p.kv_len, kRows), kMaskTiles) : 1; }

// Every warp packs its share of the mask's bytes for the key tiles [first, end), as far as there are keys.
__device__ __forceinline__ void pack_key_bits(uint32_t* words, const unsigned char* mask, int first, int end, int len,
                                              int warp, int warps, int lane) {
#pragma unroll 4
  for (int w = first * 4 + warp; w < end * 4; w += warps) {
    const int j = w * 32 + lane;
    const uint32_t v = __ballot_sync(0xffffffffu, j < len && mask[j] != 0);
    if (lane == 0) words[w] = v;
  }
}

// [batch][head][position][entry] map of a tensor with boxes of 128 positions x 64 entries.
int encode_rows(CUtensorMap* map, const void* base, const AttnStride& s, int batch, int heads, int len, int dim, int dtype);
// Whether encode_rows can take the tensor.
bool rows_ok(const void* base, const AttnStride& s, int batch, int heads, int len, int dim);

int attention_forward_sm100(const AttnParams& p, int dtype, void* ws, cudaStream_t st);
size_t attention_forward_sm100_ws(const AttnParams& p);
int attention_backward_sm100(const AttnParams& p, int dtype, void* ws, cudaStream_t st);
size_t attention_backward_sm100_ws(const AttnParams& p, int dtype);

}  // namespace lsr
