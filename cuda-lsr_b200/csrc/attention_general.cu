// Softmax attention and its gradients in 32-bit arithmetic on the CUDA cores: every type, head
// dimension up to 128, stride and alignment.
//
//   s_ij = scale q_i . k_j (minus infinity where i does not see j),  lse_i = log sum_j exp s_ij
//   p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//   D_i  = do_i . o_i,  ds_ij = scale p_ij (do_i . v_j - D_i)
//   dv_j = sum_i p_ij do_i,  dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i   (i over the group's heads too)
//
// Bound by the FFMA rate and the shared-memory reads that feed it. A block of 8 warps is WR x G: WR sets of
// 16 rows (queries in the forward pass and for dq, keys for dk and dv), and G shares of the columns of each
// tile of the other side that the block passes over. The fewer rows there are, the more the columns are
// shared, so that a short sequence or few key heads still fill the SMs; the shares' results are joined in
// shared memory at the end, in order. A warp is 4 x 8 lanes; a lane holds 4 rows by CW / 8 columns of the
// scores and 4 rows by dim / 8 entries of the results. Rows of a tile are dim + 4 floats apart, which puts
// lanes that read consecutive rows on different banks. A row's maximum and sum are exchanged by shuffles
// among 8 lanes. The forward pass keeps a running maximum
// and sum per row; the backward pass computes p again from lse. dq and dk/dv come from two passes, each of
// which sums in one fixed order: no atomics.
// A masked key's row of k and v is taken as zeros, so that nothing in it reaches a result.
// fp32, 8 x 32 heads (8 key heads) x 1500 x 128: forward 6.83 ms, 43 TFLOP/s; backward 28.2 ms, 37 TFLOP/s of its
// seven products (26 of five).
#include <algorithm>
#include <cmath>

#include "attention.cuh"

namespace lsr {
namespace {

// A lane's row (of 4) and column (of 8) in the warp's tile. Neighbours share a column, and lanes two apart a row, so
// that of either operand the 16 bytes each that half a warp reads are taken in one pass over the banks (lanes 0-7 in
// one row instead: 7% longer forward and 9% backward at 4 x 16 heads x 1024 x 64 causal).
__device__ __forceinline__ int lane_row() { return (threadIdx.x & 1) | (threadIdx.x >> 3 & 2); }
__device__ __forceinline__ int lane_col() { return threadIdx.x >> 1 & 7; }

// out[r][c] = sum_d A[4 r][d] * B[tx + 8 c][d]: A the first of the lane's rows, four apart, B a tile, rows LD
// apart. Even and odd entries are summed apart, two to an instruction.
template <int LD, int C>
__device__ __forceinline__ void mm_nt(const float* A, const float* B, int tx, float (&out)[4][C]) {
  uint64_t acc[4][C] = {};
#pragma unroll 2
  for (int d = 0; d < LD - 4; d += 4) {
    ulonglong2 a[4], b[C];
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = *reinterpret_cast<const ulonglong2*>(A + 4 * r * LD + d);
#pragma unroll
    for (int c = 0; c < C; ++c) b[c] = *reinterpret_cast<const ulonglong2*>(B + (tx + 8 * c) * LD + d);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        acc[r][c] = fma2(a[r].x, b[c].x, acc[r][c]);
        acc[r][c] = fma2(a[r].y, b[c].y, acc[r][c]);
      }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float even, odd;
      unpair(acc[r][c], even, odd);
      out[r][c] = even + odd;
    }
}

// A lane's part of a result: 4 rows by DIM / 8 entries, as pairs.
template <int CH>
using Sums = uint64_t[CH][4][2];

// acc[ch][r][e] += sum_k P[4 r][k] * B[k][ch*32 + tx*4 + e] over the COLS rows of the tile B.
template <int LD, int COLS, int CH>
__device__ __forceinline__ void mm_nn(const float* P, const float* B, int tx, Sums<CH>& acc) {
#pragma unroll 2
  for (int k = 0; k < COLS; k += 4) {
    float4 a[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = *reinterpret_cast<const float4*>(P + 4 * r * (COLS + 4) + k);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint64_t x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = kk == 0 ? a[r].x : kk == 1 ? a[r].y : kk == 2 ? a[r].z : a[r].w;
        x[r] = pair(v, v);
      }
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(B + (k + kk) * LD + ch * 32 + tx * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[ch][r][0] = fma2(x[r], b.x, acc[ch][r][0]);
          acc[ch][r][1] = fma2(x[r], b.y, acc[ch][r][1]);
        }
      }
    }
  }
}

// `rows` rows from row0 on of a [len][D] matrix with rows `stride` apart, zeros past len, past D and in
// rows that `mask` hides. vec (fp32 rows on 16-byte boundaries, D a multiple of 4): copied asynchronously, done
// when the group that the caller commits is.
template <typename T, int LD>
__device__ __forceinline__ void load_tile(float* dst, int rows, const T* src, long long stride, int row0, int len, int D,
                                          const unsigned char* mask, bool vec) {
  constexpr int W = LD - 4;
  if (vec) {
    for (int i = threadIdx.x; i < rows * (W / 4); i += blockDim.x) {
      const int r = i / (W / 4), d = i % (W / 4) * 4, g = row0 + r;
      const bool in = g < len && d < D && (!mask || mask[g]);
      const float* from = reinterpret_cast<const float*>(src) + (in ? (long long)g * stride + d : 0);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + r * LD + d)), "l"(from), "r"(in ? 16 : 0)
                   : "memory");
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * W; i += blockDim.x) {
      const int r = i / W, d = i % W, g = row0 + r;
      float x = 0.f;
      if (g < len && d < D && (!mask || mask[g])) x = attn_to_f(src[(long long)g * stride + d]);
      dst[r * LD + d] = x;
    }
  }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Wait until at most N of this thread's latest groups are on their way.
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The lane's four rows of a result.
template <typename T, int CH>
__device__ __forceinline__ void store_rows(T* dst, long long stride, int row0, int len, int D, int tx,
                                           const Sums<CH>& acc, const float (&mul)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int g = row0 + 4 * r;
    if (g >= len) continue;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      float x[4];
      unpair(acc[ch][r][0], x[0], x[1]);
      unpair(acc[ch][r][1], x[2], x[3]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = ch * 32 + tx * 4 + c;
        if (d < D) dst[(long long)g * stride + d] = attn_from_f<T>(x[c] * mul[r]);
      }
    }
  }
}

// The block's (row tile, head, batch), heads fastest. With a causal rule the tiles that see most come first (the last
// queries, the first keys), so that short blocks fill the end of the launch.
struct Place {
  int tile, h, b;
  __device__ __forceinline__ Place(int tiles, int heads, int batch, bool backwards) {
    unsigned x = blockIdx.x;
    h = (int)(x % heads);
    x /= heads;
    b = (int)(x % batch);
    tile = (int)(x / batch);
    if (backwards) tile = tiles - 1 - tile;
  }
};

// Keys that the rows before i_end can see, at most.
__device__ __forceinline__ int key_end(const AttnParams& p, int i_end) {
  return p.causal ? max(0, min(p.kv_len, min(i_end, p.q_len) + (p.kv_len - p.q_len))) : p.kv_len;
}

// The G column shares of the block's rows, summed in order: every lane writes its part, then the block
// adds and stores row by row.
template <typename T, int DIM, int WR, int G>
__device__ __forceinline__ void store_joined(float* room, T* dst, long long stride, int row0, int len, int D, int mine, int tx,
                                             int share, const Sums<DIM / 32>& acc, const float (&mul)[4]) {
  constexpr int ROWS = 16 * WR;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int ch = 0; ch < DIM / 32; ++ch)
      *reinterpret_cast<ulonglong2*>(room + (share * ROWS + mine + 4 * r) * DIM + ch * 32 + tx * 4) =
          make_ulonglong2(mul2(acc[ch][r][0], pair(mul[r], mul[r])), mul2(acc[ch][r][1], pair(mul[r], mul[r])));
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * DIM; i += blockDim.x) {
    const int r = i / DIM, d = i % DIM;
    if (row0 + r >= len || d >= D) continue;
    float x = room[i];
#pragma unroll
    for (int g = 1; g < G; ++g) x += room[g * ROWS * DIM + i];
    dst[(long long)(row0 + r) * stride + d] = attn_from_f<T>(x);
  }
}

constexpr int GTHREADS = 256;

template <int DIM, int WR, int G>
struct FwdGeneral {
  static constexpr int ROWS = 16 * WR, CW = G == 1 ? 64 : 32, COLS = CW * G, LD = DIM + 4;
  static constexpr int FLOATS = ROWS * LD + 2 * COLS * LD + 8 * 16 * (CW + 4) + 2 * G * ROWS;
  static constexpr int SMEM = FLOATS * 4;
  static_assert(WR * G == 8 && G * ROWS * DIM <= ROWS * LD + 2 * COLS * LD, "the shares' results take the tiles' room");
};

template <typename T, int DIM, int WR, int G>
__global__ void __launch_bounds__(GTHREADS, 1) attn_fwd_general_kernel(const AttnParams p, bool vec) {
  using L = FwdGeneral<DIM, WR, G>;
  constexpr int ROWS = L::ROWS, CW = L::CW, COLS = L::COLS, LD = L::LD, CH = DIM / 32, C = CW / 8;
  extern __shared__ float sm[];
  float *Q = sm, *K = Q + ROWS * LD, *V = K + COLS * LD, *PS = V + COLS * LD, *stat = PS + 8 * 16 * (CW + 4);
  const Place at((p.q_len + ROWS - 1) / ROWS, p.heads, p.batch, true);
  const int warp = threadIdx.x / 32, ty = lane_row(), tx = lane_col(), D = p.head_dim;
  const int i0 = at.tile * ROWS, mine = warp / G * 16 + ty;  // and every fourth row after it
  const int share = warp % G, x0 = share * CW;               // the warp's columns of a tile
  float* P = PS + (warp * 16 + ty) * (CW + 4);
  const unsigned char* mask = p.mask ? p.mask + at.b * p.mask_stride : nullptr;
  const T* k = attn_at<T>(p.k, p.sk, at.b, at.h / p.group);
  const T* v = attn_at<T>(p.v, p.sv, at.b, at.h / p.group);
  const int jend = key_end(p, i0 + ROWS), off = p.kv_len - p.q_len;
  load_tile<T, LD>(Q, ROWS, attn_at<T>(p.q, p.sq, at.b, at.h), p.sq.s, i0, p.q_len, D, nullptr, vec);
  if (jend > 0) load_tile<T, LD>(K, COLS, k, p.sk.s, 0, p.kv_len, D, mask, vec);
  copies_commit();
  if (jend > 0) load_tile<T, LD>(V, COLS, v, p.sv.s, 0, p.kv_len, D, mask, vec);
  copies_commit();
  Sums<CH> o = {};
  float m[4], l[4] = {};
#pragma unroll
  for (int r = 0; r < 4; ++r) m[r] = -INFINITY;
  for (int j0 = 0; j0 < jend; j0 += COLS) {
    copies_wait<1>();
    __syncthreads();
    float s[4][C];
    mm_nt<LD, C>(Q + mine * LD, K + x0 * LD, tx, s);
    __syncthreads();
    // the next keys arrive during the softmax and the product with the values, the next values during the next scores
    if (j0 + COLS < jend) load_tile<T, LD>(K, COLS, k, p.sk.s, j0 + COLS, p.kv_len, D, mask, vec);
    copies_commit();
    if (j0 + COLS > p.kv_len || mask || (p.causal && j0 + COLS - 1 > i0 + off)) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int j = j0 + x0 + tx + 8 * c;
        const bool ok = j < p.kv_len && (!mask || mask[j]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!ok || (p.causal && j > i0 + mine + 4 * r + off)) s[r][c] = -INFINITY;
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        // (not times the scale where hidden: it may be 0 or negative)
        s[r][c] = s[r][c] == -INFINITY ? s[r][c] : s[r][c] * p.scale;
        top = fmaxf(top, s[r][c]);
      }
#pragma unroll
      for (int w = 8; w > 1; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float mn = fmaxf(m[r], top), base = mn == -INFINITY ? 0.f : mn;
      const float keep = expf(m[r] - base);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float e = expf(s[r][c] - base);
        sum += e;
        P[4 * r * (CW + 4) + tx + 8 * c] = e;
      }
#pragma unroll
      for (int w = 8; w > 1; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      l[r] = l[r] * keep + sum;
      m[r] = mn;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int c = 0; c < 2; ++c) o[ch][r][c] = mul2(o[ch][r][c], pair(keep, keep));
    }
    copies_wait<1>();
    __syncthreads();
    mm_nn<LD, CW, CH>(P, V + x0 * LD, tx, o);
    __syncthreads();
    if (j0 + COLS < jend) load_tile<T, LD>(V, COLS, v, p.sv.s, j0 + COLS, p.kv_len, D, mask, vec);
    copies_commit();
  }
  copies_wait<0>();
  float mul[4];
  if (G > 1) {  // the row's maximum and sum over all shares
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (tx == 0) {
        stat[share * ROWS + mine + 4 * r] = m[r];
        stat[(G + share) * ROWS + mine + 4 * r] = l[r];
      }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float top = m[r], total = l[r];
    mul[r] = 1.f;
    if (G > 1) {
      const float* at_row = stat + mine + 4 * r;
      top = -INFINITY;
#pragma unroll
      for (int g = 0; g < G; ++g) top = fmaxf(top, at_row[g * ROWS]);
      const float base = top == -INFINITY ? 0.f : top;
      total = 0.f;
#pragma unroll
      for (int g = 0; g < G; ++g) total += at_row[(G + g) * ROWS] * expf(at_row[g * ROWS] - base);
      mul[r] = expf(m[r] - base);
    }
    mul[r] *= total > 0.f || total != total ? 1.f / total : 0.f;
    const int g = i0 + mine + 4 * r;
    if (tx == 0 && share == 0 && g < p.q_len)
      p.lse[((long long)at.b * p.heads + at.h) * p.q_len + g] = top + logf(total);
  }
  T* dst = attn_at<T>(p.out, p.so, at.b, at.h);
  if constexpr (G == 1) store_rows<T, CH>(dst, p.so.s, i0 + mine, p.q_len, D, tx, o, mul);
  else store_joined<T, DIM, WR, G>(sm, dst, p.so.s, i0, p.q_len, D, mine, tx, share, o, mul);
}

// delta[row] = dout . out, one warp per row.
template <typename T>
__global__ void __launch_bounds__(256) attn_delta_kernel(const AttnParams p) {
  const long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  if (row >= (long long)p.batch * p.heads * p.q_len) return;
  const int i = (int)(row % p.q_len), h = (int)(row / p.q_len % p.heads), b = (int)(row / p.q_len / p.heads);
  const T* o = attn_at<T>(p.out, p.so, b, h) + i * p.so.s;
  const T* d = attn_at<T>(p.dout, p.sdo, b, h) + i * p.sdo.s;
  float s = 0.f;
  for (int e = threadIdx.x % 32; e < p.head_dim; e += 32) s = fmaf(attn_to_f(o[e]), attn_to_f(d[e]), s);
#pragma unroll
  for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
  if (threadIdx.x % 32 == 0) p.delta[row] = s;
}

template <int DIM, int WR, int G, bool KEYS>
struct BwdGeneral {
  static constexpr int ROWS = 16 * WR, CW = 32, COLS = CW * G, LD = DIM + 4;
  static constexpr int BUFS = G <= 2 ? 2 : 1;  // of the first operand's tile: the next one arrives during the step
  static constexpr int FLOATS = 2 * ROWS * LD + (BUFS + 1) * COLS * LD + (KEYS ? 2 : 1) * 8 * 16 * (CW + 4) + BUFS * 2 * COLS;
  static constexpr int SMEM = FLOATS * 4;
  static_assert(WR * G == 8 && G * ROWS * DIM <= FLOATS, "the shares' results take the tiles' room");
};

// KEYS: the rows are keys and the columns queries of every head of the group (dv and dk); else rows are
// queries and columns keys (dq).
template <typename T, int DIM, int WR, int G, bool KEYS>
__global__ void __launch_bounds__(GTHREADS, 1) attn_bwd_general_kernel(const AttnParams p, bool vec) {
  using L = BwdGeneral<DIM, WR, G, KEYS>;
  constexpr int ROWS = L::ROWS, CW = L::CW, COLS = L::COLS, LD = L::LD, CH = DIM / 32, C = CW / 8, BUFS = L::BUFS;
  extern __shared__ float sm[];
  float *R1 = sm, *R2 = R1 + ROWS * LD, *X1 = R2 + ROWS * LD, *X2 = X1 + BUFS * COLS * LD, *SS = X2 + COLS * LD;
  float *PS = SS + 8 * 16 * (CW + 4), *stat = KEYS ? PS + 8 * 16 * (CW + 4) : PS;  // PS: only KEYS multiplies it
  const int rows_len = KEYS ? p.kv_len : p.q_len, cols_len = KEYS ? p.q_len : p.kv_len;
  const Place at((rows_len + ROWS - 1) / ROWS, KEYS ? p.kv_heads : p.heads, p.batch, !KEYS);
  if (KEYS) launch_dependents();
  const int warp = threadIdx.x / 32, ty = lane_row(), tx = lane_col(), D = p.head_dim;
  const int row0 = at.tile * ROWS, mine = warp / G * 16 + ty;  // and every fourth row after it
  const int share = warp % G, x0 = share * CW;                 // the warp's columns of a tile
  float *P = PS + (warp * 16 + ty) * (CW + 4), *S = SS + (warp * 16 + ty) * (CW + 4);
  const int hk = KEYS ? at.h : at.h / p.group;
  const unsigned char* mask = p.mask ? p.mask + at.b * p.mask_stride : nullptr;
  const T *k = attn_at<T>(p.k, p.sk, at.b, hk), *v = attn_at<T>(p.v, p.sv, at.b, hk);
  const int off = p.kv_len - p.q_len;
  float lse[4], delta[4];
  if (KEYS) {
    load_tile<T, LD>(R1, ROWS, k, p.sk.s, row0, p.kv_len, D, mask, vec);
    load_tile<T, LD>(R2, ROWS, v, p.sv.s, row0, p.kv_len, D, mask, vec);
  } else {
    load_tile<T, LD>(R1, ROWS, attn_at<T>(p.q, p.sq, at.b, at.h), p.sq.s, row0, p.q_len, D, nullptr, vec);
    load_tile<T, LD>(R2, ROWS, attn_at<T>(p.dout, p.sdo, at.b, at.h), p.sdo.s, row0, p.q_len, D, nullptr, vec);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int g = row0 + mine + 4 * r;
      const long long row = ((long long)at.b * p.heads + at.h) * p.q_len + g;
      lse[r] = g < p.q_len ? p.lse[row] : 0.f;
      delta[r] = g < p.q_len ? p.delta[row] : 0.f;
    }
  }
  Sums<KEYS ? CH : 1> acc1 = {};
  Sums<CH> acc2 = {};
  // queries before `first` see none of the block's keys; keys from `end` on are seen by none of its queries
  const int first = KEYS && p.causal ? max(0, row0 - off) / CW * CW : 0;
  const int end = KEYS ? cols_len : key_end(p, row0 + ROWS);
  const int tiles = max(0, (end - first + COLS - 1) / COLS), steps = KEYS ? tiles * p.group : tiles;
  // the tile that step t passes over, as the first operand (q or k; with the queries' statistics) and the second (dout or v)
  auto load1 = [&](int t) {
    float* dst = X1 + t % BUFS * COLS * LD;
    if (KEYS) {
      const int h = at.h * p.group + t / tiles, c0 = first + t % tiles * COLS;
      load_tile<T, LD>(dst, COLS, attn_at<T>(p.q, p.sq, at.b, h), p.sq.s, c0, p.q_len, D, nullptr, vec);
      for (int x = threadIdx.x; x < COLS; x += GTHREADS) {
        const int i = c0 + x;
        const long long row = ((long long)at.b * p.heads + h) * p.q_len + i;
        stat[t % BUFS * 2 * COLS + x] = i < p.q_len ? p.lse[row] : 0.f;
        stat[t % BUFS * 2 * COLS + COLS + x] = i < p.q_len ? p.delta[row] : 0.f;
      }
    } else {
      load_tile<T, LD>(dst, COLS, k, p.sk.s, t * COLS, p.kv_len, D, mask, vec);
    }
  };
  auto load2 = [&](int t) {
    if (KEYS)
      load_tile<T, LD>(X2, COLS, attn_at<T>(p.dout, p.sdo, at.b, at.h * p.group + t / tiles), p.sdo.s, first + t % tiles * COLS,
                       p.q_len, D, nullptr, vec);
    else load_tile<T, LD>(X2, COLS, v, p.sv.s, t * COLS, p.kv_len, D, mask, vec);
  };
  if (steps > 0) load1(0);
  copies_commit();
  if (steps > 0) load2(0);
  copies_commit();
  for (int t = 0; t < steps; ++t) {
    const float* x1 = X1 + (t % BUFS * COLS + x0) * LD;
    const float* st = stat + t % BUFS * 2 * COLS + x0;
    const int c0 = first + (KEYS ? t % tiles : t) * COLS + x0;
    if (BUFS == 2 && t + 1 < steps) load1(t + 1);
    if (BUFS == 2) copies_commit();
    copies_wait<BUFS>();
    __syncthreads();
    float s[4][C], dp[4][C];
    mm_nt<LD, C>(R1 + mine * LD, x1, tx, s);
    copies_wait<BUFS - 1>();
    __syncthreads();
    mm_nt<LD, C>(R2 + mine * LD, X2 + x0 * LD, tx, dp);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int x = c0 + tx + 8 * c;
      const bool in = x < cols_len && (KEYS || !mask || mask[x]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int a = row0 + mine + 4 * r;
        const float ls = KEYS ? st[tx + 8 * c] : lse[r], dl = KEYS ? st[COLS + tx + 8 * c] : delta[r];
        // 0 where i does not see j (a row that sees nothing has lse = minus infinity); masked rows are left out at the end
        const bool ok = in && (!p.causal || (KEYS ? a <= x + off : x <= a + off));
        const float e = ok ? expf(s[r][c] * p.scale - ls) : 0.f;
        if (KEYS) P[4 * r * (CW + 4) + tx + 8 * c] = e;
        S[4 * r * (CW + 4) + tx + 8 * c] = ok ? e * (dp[r][c] - dl) : 0.f;
      }
    }
    __syncwarp();  // the warp's rows of P and S are its own
    if constexpr (KEYS) mm_nn<LD, CW, CH>(P, X2 + x0 * LD, tx, acc1);
    __syncthreads();
    if (t + 1 < steps) load2(t + 1);
    copies_commit();
    mm_nn<LD, CW, CH>(S, x1, tx, acc2);
    __syncthreads();
    if (BUFS == 1) {
      if (t + 1 < steps) load1(t + 1);
      copies_commit();
      copies_commit();  // an empty group, so that the wait for all but one covers both operands
    }
  }
  copies_wait<0>();
  float one[4], sc[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int a = row0 + mine + 4 * r;
    const bool hidden = KEYS && mask && a < p.kv_len && !mask[a];  // a masked key has no gradient
    if (KEYS && hidden) {
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int c = 0; c < 2; ++c) acc1[KEYS ? ch : 0][r][c] = acc2[ch][r][c] = 0;
    }
    one[r] = 1.f;
    sc[r] = p.scale;
  }
  auto store = [&](void* base, const AttnStride& sd, const Sums<CH>& acc, const float(&mul)[4]) {
    T* dst = attn_at<T>(base, sd, at.b, at.h);
    if constexpr (G == 1) store_rows<T, CH>(dst, sd.s, row0 + mine, rows_len, D, tx, acc, mul);
    else store_joined<T, DIM, WR, G>(sm, dst, sd.s, row0, rows_len, D, mine, tx, share, acc, mul);
  };
  if constexpr (KEYS) {
    store(p.dv, p.sdv, acc1, one);
    store(p.dk, p.sdk, acc2, sc);
  } else {
    store(p.dq, p.sdq, acc2, sc);
    wait_dependency();  // the launch ends after that of dk and dv
  }
}

// Whether fp32 rows can be read as 16-byte vectors.
bool vec_ok(const void* base, const AttnStride& s, int batch, int heads, int len, int dim) {
  const auto fits = [](long long st, int size) { return size <= 1 || st % 4 == 0; };
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && dim % 4 == 0 && fits(s.b, batch) && fits(s.s, len) && fits(s.h, heads);
}

// early: blocks start as soon as those of the launch before have all started and leave room.
template <typename K, typename... A>
int launch(K kernel, long long blocks, int threads, int smem, cudaStream_t st, bool early, A... args) {
  if (blocks == 0) return LSR_OK;
  if (blocks > 0x7fffffffll) return LSR_ERR_SHAPE;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return LSR_ERR_LAUNCH;
  ProfScope prof(PK_GEMM_OTHER, st);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = early;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? LSR_OK : LSR_ERR_LAUNCH;
}

// Sets of 16 rows per block in the backward pass: the most whose blocks still fill the SMs (its tails are filled: the
// blocks of dq follow those of dk and dv).
int row_sets(long long rows, long long heads, int least) {
  for (int w = 8; w > least; w /= 2)
    if ((rows + 16 * w - 1) / (16 * w) * heads >= device_sm_count()) return w;
  return least;
}

// Sets of 16 rows per block in the forward pass: the number for which the blocks that run one after the other on an SM
// take least. Fewer rows make finer blocks, but each reads its columns for fewer rows. Measured on 4 x 16 heads x 1024 x
// 64, per row: 1, 1.17, 1.45 and 2.08 with 8, 4, 2 and 1 sets (128 wide: 1, 1.19, 1.33). Causal blocks differ in
// length and the short ones come last, so that they fill the end: half a block more than their mean.
int forward_sets(const AttnParams& p, int least) {
  const double heads = (double)p.heads * p.batch, sms = device_sm_count();
  const double seen = !p.causal || p.kv_len == 0 ? 1. : p.q_len <= p.kv_len ? 1. - .5 * p.q_len / p.kv_len : .5 * p.kv_len / p.q_len;
  int best = 8;
  double time = 0.;
  for (int w = 8; w >= least; w /= 2) {
    const double waves = (double)cdiv(p.q_len, 16 * w) * heads / sms;
    const double turns = p.causal ? std::max(1., waves * seen + .5) : std::ceil(waves);
    const double t = turns * w * (w == 8 ? 1. : w == 4 ? 1.17 : w == 2 ? 1.45 : 2.08);
    if (w == 8 || t < time) time = t, best = w;
  }
  return best;
}

template <typename T, int DIM, int WR>
int forward_w(const AttnParams& p, bool vec, cudaStream_t st) {
  using L = FwdGeneral<DIM, WR, 8 / WR>;
  static_assert(L::SMEM <= 232448, "shared memory budget exceeded");
  return launch(attn_fwd_general_kernel<T, DIM, WR, 8 / WR>, (long long)cdiv(p.q_len, L::ROWS) * p.heads * p.batch, GTHREADS,
                L::SMEM, st, false, p, vec);
}

template <typename T, int DIM, int WR, bool KEYS>
int backward_w(const AttnParams& p, bool vec, cudaStream_t st) {
  using L = BwdGeneral<DIM, WR, 8 / WR, KEYS>;
  static_assert(L::SMEM <= 232448, "shared memory budget exceeded");
  return launch(attn_bwd_general_kernel<T, DIM, WR, 8 / WR, KEYS>,
                (long long)cdiv(KEYS ? p.kv_len : p.q_len, L::ROWS) * (KEYS ? p.kv_heads : p.heads) * p.batch, GTHREADS,
                L::SMEM, st, !KEYS && p.kv_len > 0, p, vec);
}

constexpr int least_sets(int dim) { return dim == 64 ? 1 : 2; }  // eight shares of wider tiles do not fit

template <typename T, int DIM>
int forward(const AttnParams& p, bool vec, cudaStream_t st) {
  switch (forward_sets(p, least_sets(DIM))) {
    case 8: return forward_w<T, DIM, 8>(p, vec, st);
    case 4: return forward_w<T, DIM, 4>(p, vec, st);
    case 2: return forward_w<T, DIM, 2>(p, vec, st);
    default: return forward_w<T, DIM, least_sets(DIM)>(p, vec, st);
  }
}

template <typename T, int DIM, bool KEYS>
int gradients(const AttnParams& p, bool vec, cudaStream_t st) {
  switch (row_sets(KEYS ? p.kv_len : p.q_len, (long long)(KEYS ? p.kv_heads : p.heads) * p.batch, least_sets(DIM))) {
    case 8: return backward_w<T, DIM, 8, KEYS>(p, vec, st);
    case 4: return backward_w<T, DIM, 4, KEYS>(p, vec, st);
    case 2: return backward_w<T, DIM, 2, KEYS>(p, vec, st);
    default: return backward_w<T, DIM, least_sets(DIM), KEYS>(p, vec, st);
  }
}

template <typename T, int DIM>
int backward(const AttnParams& p, bool vec, cudaStream_t st) {
  const long long rows = (long long)p.batch * p.heads * p.q_len;
  int rc = launch(attn_delta_kernel<T>, (rows + 7) / 8, 256, 0, st, false, p);
  if (rc == LSR_OK) rc = gradients<T, DIM, true>(p, vec, st);
  return rc == LSR_OK ? gradients<T, DIM, false>(p, vec, st) : rc;
}

// Tiles of 64, 96 or 128 entries, with zeros past the head dimension. (4 x 16 heads x 1000 x 96 causal: forward 365 us,
// backward 1391; in tiles of 128 they took 458 and 1773.)
template <typename T>
int forward_t(const AttnParams& p, bool vec, cudaStream_t st) {
  return p.head_dim > 96 ? forward<T, 128>(p, vec, st) : p.head_dim > 64 ? forward<T, 96>(p, vec, st) : forward<T, 64>(p, vec, st);
}
template <typename T>
int backward_t(const AttnParams& p, bool vec, cudaStream_t st) {
  return p.head_dim > 96 ? backward<T, 128>(p, vec, st) : p.head_dim > 64 ? backward<T, 96>(p, vec, st) : backward<T, 64>(p, vec, st);
}

}  // namespace

int attention_forward_general(const AttnParams& p, int dtype, cudaStream_t st) {
  const bool vec = dtype == LSR_DTYPE_F32 && vec_ok(p.q, p.sq, p.batch, p.heads, p.q_len, p.head_dim) &&
                   vec_ok(p.k, p.sk, p.batch, p.kv_heads, p.kv_len, p.head_dim) &&
                   vec_ok(p.v, p.sv, p.batch, p.kv_heads, p.kv_len, p.head_dim);
  if (dtype == LSR_DTYPE_F32) return forward_t<float>(p, vec, st);
  return dtype == LSR_DTYPE_BF16 ? forward_t<__nv_bfloat16>(p, vec, st) : forward_t<__half>(p, vec, st);
}

int attention_backward_general(const AttnParams& p, int dtype, cudaStream_t st) {
  const bool vec = dtype == LSR_DTYPE_F32 && vec_ok(p.q, p.sq, p.batch, p.heads, p.q_len, p.head_dim) &&
                   vec_ok(p.k, p.sk, p.batch, p.kv_heads, p.kv_len, p.head_dim) &&
                   vec_ok(p.v, p.sv, p.batch, p.kv_heads, p.kv_len, p.head_dim) &&
                   vec_ok(p.dout, p.sdo, p.batch, p.heads, p.q_len, p.head_dim);
  if (dtype == LSR_DTYPE_F32) return backward_t<float>(p, vec, st);
  return dtype == LSR_DTYPE_BF16 ? backward_t<__nv_bfloat16>(p, vec, st) : backward_t<__half>(p, vec, st);
}

}  // namespace lsr
