// Softmax attention and its gradients in 32-bit arithmetic on the CUDA cores: every type, head
// dimension up to 128, stride and alignment.
//
//   s_ij = scale q_i . k_j (minus infinity where i does not see j),  lse_i = log sum_j exp s_ij
//   p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//   D_i  = do_i . o_i,  ds_ij = scale p_ij (do_i . v_j - D_i)
//   dv_j = sum_i p_ij do_i,  dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i   (i over the group's heads too)
//
// Bound by the FFMA rate. A block of 256 threads owns 64 rows (queries in the forward pass and for
// dq, keys for dk and dv) and passes over the other side in tiles of 64; each thread holds a 4 x 4
// piece of the 64 x 64 scores and of the 64 x dim results, so a product reads two 16-byte vectors of
// shared memory per 16 multiply-adds. Rows of a tile are dim + 4 floats apart: eight lanes that
// read the same column of consecutive rows then fall on different banks. The forward pass keeps a
// running maximum and sum per row; the backward pass computes p again from lse. dq and dk/dv come
// from two passes, each of which sums in one fixed order: no atomics.
// A masked key's row of k and v is taken as zeros, so that nothing in it reaches a result.
#include "attention.cuh"

namespace lsr {
namespace {

constexpr int AT = 64;        // rows and columns of a tile
constexpr int ATHREADS = 256;
constexpr int PLD = AT + 4;   // row of the score tile in shared memory

// acc[r][c] += sum_d A[ty*4 + r][d] * B[tx + 16 c][d]   (both row-major, rows LD apart)
template <int LD>
__device__ __forceinline__ void mm_nt(const float* A, const float* B, int D, int ty, int tx, float (&acc)[4][4]) {
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    float4 a[4], b[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = *reinterpret_cast<const float4*>(A + (ty * 4 + r) * LD + d);
#pragma unroll
    for (int c = 0; c < 4; ++c) b[c] = *reinterpret_cast<const float4*>(B + (tx + 16 * c) * LD + d);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        acc[r][c] = fmaf(a[r].x, b[c].x, acc[r][c]);
        acc[r][c] = fmaf(a[r].y, b[c].y, acc[r][c]);
        acc[r][c] = fmaf(a[r].z, b[c].z, acc[r][c]);
        acc[r][c] = fmaf(a[r].w, b[c].w, acc[r][c]);
      }
  }
}

// acc[ch][r][c] += sum_k P[ty*4 + r][k] * B[k][ch*64 + tx*4 + c]
template <int LD, int CH>
__device__ __forceinline__ void mm_nn(const float* P, const float* B, int ty, int tx, float (&acc)[CH][4][4]) {
#pragma unroll 2
  for (int k = 0; k < AT; k += 4) {
    float4 a[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = *reinterpret_cast<const float4*>(P + (ty * 4 + r) * PLD + k);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const float4 b = *reinterpret_cast<const float4*>(B + (k + kk) * LD + ch * 64 + tx * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = kk == 0 ? a[r].x : kk == 1 ? a[r].y : kk == 2 ? a[r].z : a[r].w;
          acc[ch][r][0] = fmaf(x, b.x, acc[ch][r][0]);
          acc[ch][r][1] = fmaf(x, b.y, acc[ch][r][1]);
          acc[ch][r][2] = fmaf(x, b.z, acc[ch][r][2]);
          acc[ch][r][3] = fmaf(x, b.w, acc[ch][r][3]);
        }
      }
  }
}

// acc[ch][r][c] += sum_k P[k][ty*4 + r] * B[k][ch*64 + tx*4 + c]
template <int LD, int CH>
__device__ __forceinline__ void mm_tn(const float* P, const float* B, int ty, int tx, float (&acc)[CH][4][4]) {
#pragma unroll 4
  for (int k = 0; k < AT; ++k) {
    const float4 a = *reinterpret_cast<const float4*>(P + k * PLD + ty * 4);
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const float4 b = *reinterpret_cast<const float4*>(B + k * LD + ch * 64 + tx * 4);
      const float x[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        acc[ch][r][0] = fmaf(x[r], b.x, acc[ch][r][0]);
        acc[ch][r][1] = fmaf(x[r], b.y, acc[ch][r][1]);
        acc[ch][r][2] = fmaf(x[r], b.z, acc[ch][r][2]);
        acc[ch][r][3] = fmaf(x[r], b.w, acc[ch][r][3]);
      }
    }
  }
}

// Rows [row0, row0 + 64) of a [len][D] matrix with rows `stride` apart, zeros past len, past D and in
// rows that `mask` hides.
template <typename T, int LD>
__device__ __forceinline__ void load_tile(float* dst, const T* src, long long stride, int row0, int len, int D,
                                          const unsigned char* mask) {
  constexpr int W = LD - 4;
  for (int i = threadIdx.x; i < AT * W; i += ATHREADS) {
    const int r = i / W, d = i % W, g = row0 + r;
    float x = 0.f;
    if (g < len && d < D && (!mask || mask[g])) x = attn_to_f(src[(long long)g * stride + d]);
    dst[r * LD + d] = x;
  }
}

template <typename T, int CH>
__device__ __forceinline__ void store_tile(T* dst, long long stride, int row0, int len, int D, int ty, int tx,
                                           const float (&acc)[CH][4][4], const float (&mul)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int g = row0 + ty * 4 + r;
    if (g >= len) continue;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = ch * 64 + tx * 4 + c;
        if (d < D) dst[(long long)g * stride + d] = attn_from_f<T>(acc[ch][r][c] * mul[r]);
      }
  }
}

// The block's (row tile, head, batch), row tiles fastest.
struct Place {
  int tile, h, b;
  __device__ __forceinline__ Place(int tiles, int heads) {
    unsigned x = blockIdx.x;
    tile = (int)(x % tiles);
    x /= tiles;
    h = (int)(x % heads);
    b = (int)(x / heads);
  }
};

__device__ __forceinline__ bool sees(const AttnParams& p, const unsigned char* mask, int i, int j) {
  return i < p.q_len && j < p.kv_len && (!p.causal || j <= i + (p.kv_len - p.q_len)) && (!mask || mask[j]);
}

// Keys that the rows before i_end can see, at most.
__device__ __forceinline__ int key_end(const AttnParams& p, int i_end) {
  return p.causal ? max(0, min(p.kv_len, min(i_end, p.q_len) + (p.kv_len - p.q_len))) : p.kv_len;
}

template <typename T, int CH>
__global__ void __launch_bounds__(ATHREADS) attn_fwd_general_kernel(const AttnParams p) {
  constexpr int LD = CH * 64 + 4;
  extern __shared__ float sm[];
  float *Q = sm, *K = Q + AT * LD, *V = K + AT * LD, *P = V + AT * LD;
  const Place at((p.q_len + AT - 1) / AT, p.heads);
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16, D = p.head_dim, i0 = at.tile * AT;
  const unsigned char* mask = p.mask ? p.mask + at.b * p.mask_stride : nullptr;
  const T* k = attn_at<T>(p.k, p.sk, at.b, at.h / p.group);
  const T* v = attn_at<T>(p.v, p.sv, at.b, at.h / p.group);
  load_tile<T, LD>(Q, attn_at<T>(p.q, p.sq, at.b, at.h), p.sq.s, i0, p.q_len, D, nullptr);
  float o[CH][4][4] = {}, m[4], l[4] = {};
#pragma unroll
  for (int r = 0; r < 4; ++r) m[r] = -INFINITY;
  const int jend = key_end(p, i0 + AT);
  for (int j0 = 0; j0 < jend; j0 += AT) {
    __syncthreads();
    load_tile<T, LD>(K, k, p.sk.s, j0, p.kv_len, D, mask);
    load_tile<T, LD>(V, v, p.sv.s, j0, p.kv_len, D, mask);
    __syncthreads();
    float s[4][4] = {};
    mm_nt<LD>(Q, K, CH * 64, ty, tx, s);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = sees(p, mask, i0 + ty * 4 + r, j0 + tx + 16 * c) ? s[r][c] * p.scale : -INFINITY;
        top = fmaxf(top, s[r][c]);
      }
#pragma unroll
      for (int w = 8; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float mn = fmaxf(m[r], top), base = mn == -INFINITY ? 0.f : mn;
      const float keep = expf(m[r] - base);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float e = expf(s[r][c] - base);
        sum += e;
        P[(ty * 4 + r) * PLD + tx + 16 * c] = e;
      }
#pragma unroll
      for (int w = 8; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      l[r] = l[r] * keep + sum;
      m[r] = mn;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[ch][r][c] *= keep;
    }
    __syncthreads();
    mm_nn<LD, CH>(P, V, ty, tx, o);
  }
  float inv[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    inv[r] = l[r] > 0.f || l[r] != l[r] ? 1.f / l[r] : 0.f;
    const int g = i0 + ty * 4 + r;
    if (tx == 0 && g < p.q_len) p.lse[((long long)at.b * p.heads + at.h) * p.q_len + g] = m[r] + logf(l[r]);
  }
  store_tile<T, CH>(attn_at<T>(p.out, p.so, at.b, at.h), p.so.s, i0, p.q_len, D, ty, tx, o, inv);
}

// delta[row] = dout . out, one warp per row.
template <typename T>
__global__ void __launch_bounds__(ATHREADS) attn_delta_kernel(const AttnParams p) {
  const long long row = (long long)blockIdx.x * (ATHREADS / 32) + threadIdx.x / 32;
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

// exp(s - lse), 0 where i does not see j (a row that sees nothing has lse = minus infinity).
__device__ __forceinline__ float prob(const AttnParams& p, const unsigned char* mask, int i, int j, float s, float lse) {
  return sees(p, mask, i, j) ? expf(s * p.scale - lse) : 0.f;
}

template <typename T, int CH>
__global__ void __launch_bounds__(ATHREADS) attn_dq_general_kernel(const AttnParams p) {
  constexpr int LD = CH * 64 + 4;
  extern __shared__ float sm[];
  float *Q = sm, *DO = Q + AT * LD, *K = DO + AT * LD, *V = K + AT * LD, *P = V + AT * LD;
  const Place at((p.q_len + AT - 1) / AT, p.heads);
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16, D = p.head_dim, i0 = at.tile * AT;
  const unsigned char* mask = p.mask ? p.mask + at.b * p.mask_stride : nullptr;
  const T* k = attn_at<T>(p.k, p.sk, at.b, at.h / p.group);
  const T* v = attn_at<T>(p.v, p.sv, at.b, at.h / p.group);
  load_tile<T, LD>(Q, attn_at<T>(p.q, p.sq, at.b, at.h), p.sq.s, i0, p.q_len, D, nullptr);
  load_tile<T, LD>(DO, attn_at<T>(p.dout, p.sdo, at.b, at.h), p.sdo.s, i0, p.q_len, D, nullptr);
  float lse[4], delta[4], acc[CH][4][4] = {}, mul[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int g = i0 + ty * 4 + r;
    const long long row = ((long long)at.b * p.heads + at.h) * p.q_len + g;
    lse[r] = g < p.q_len ? p.lse[row] : 0.f;
    delta[r] = g < p.q_len ? p.delta[row] : 0.f;
    mul[r] = p.scale;
  }
  const int jend = key_end(p, i0 + AT);
  for (int j0 = 0; j0 < jend; j0 += AT) {
    __syncthreads();
    load_tile<T, LD>(K, k, p.sk.s, j0, p.kv_len, D, mask);
    load_tile<T, LD>(V, v, p.sv.s, j0, p.kv_len, D, mask);
    __syncthreads();
    float s[4][4] = {}, dp[4][4] = {};
    mm_nt<LD>(Q, K, CH * 64, ty, tx, s);
    mm_nt<LD>(DO, V, CH * 64, ty, tx, dp);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        P[(ty * 4 + r) * PLD + tx + 16 * c] =
            prob(p, mask, i0 + ty * 4 + r, j0 + tx + 16 * c, s[r][c], lse[r]) * (dp[r][c] - delta[r]);
    __syncthreads();
    mm_nn<LD, CH>(P, K, ty, tx, acc);
  }
  store_tile<T, CH>(attn_at<T>(p.dq, p.sdq, at.b, at.h), p.sdq.s, i0, p.q_len, D, ty, tx, acc, mul);
}

template <typename T, int CH>
__global__ void __launch_bounds__(ATHREADS) attn_dkv_general_kernel(const AttnParams p) {
  constexpr int LD = CH * 64 + 4;
  extern __shared__ float sm[];
  float *K = sm, *V = K + AT * LD, *Q = V + AT * LD, *DO = Q + AT * LD, *P = DO + AT * LD, *S = P + AT * PLD;
  const Place at((p.kv_len + AT - 1) / AT, p.kv_heads);
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16, D = p.head_dim, j0 = at.tile * AT;
  const unsigned char* mask = p.mask ? p.mask + at.b * p.mask_stride : nullptr;
  load_tile<T, LD>(K, attn_at<T>(p.k, p.sk, at.b, at.h), p.sk.s, j0, p.kv_len, D, mask);
  load_tile<T, LD>(V, attn_at<T>(p.v, p.sv, at.b, at.h), p.sv.s, j0, p.kv_len, D, mask);
  float dk[CH][4][4] = {}, dv[CH][4][4] = {};
  const int first = p.causal ? max(0, j0 - (p.kv_len - p.q_len)) / AT * AT : 0;  // rows before it see none of these keys
  for (int h = at.h * p.group; h < (at.h + 1) * p.group; ++h) {
    const T* q = attn_at<T>(p.q, p.sq, at.b, h);
    const T* dout = attn_at<T>(p.dout, p.sdo, at.b, h);
    const long long row = ((long long)at.b * p.heads + h) * p.q_len;
    for (int i0 = first; i0 < p.q_len; i0 += AT) {
      __syncthreads();
      load_tile<T, LD>(Q, q, p.sq.s, i0, p.q_len, D, nullptr);
      load_tile<T, LD>(DO, dout, p.sdo.s, i0, p.q_len, D, nullptr);
      __syncthreads();
      float s[4][4] = {}, dp[4][4] = {};
      mm_nt<LD>(Q, K, CH * 64, ty, tx, s);
      mm_nt<LD>(DO, V, CH * 64, ty, tx, dp);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + ty * 4 + r;
        const float lse = i < p.q_len ? p.lse[row + i] : 0.f, delta = i < p.q_len ? p.delta[row + i] : 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float e = prob(p, mask, i, j0 + tx + 16 * c, s[r][c], lse);
          P[(ty * 4 + r) * PLD + tx + 16 * c] = e;
          S[(ty * 4 + r) * PLD + tx + 16 * c] = e * (dp[r][c] - delta);
        }
      }
      __syncthreads();
      mm_tn<LD, CH>(P, DO, ty, tx, dv);
      mm_tn<LD, CH>(S, Q, ty, tx, dk);
    }
  }
  const float one[4] = {1.f, 1.f, 1.f, 1.f}, sc[4] = {p.scale, p.scale, p.scale, p.scale};
  store_tile<T, CH>(attn_at<T>(p.dv, p.sdv, at.b, at.h), p.sdv.s, j0, p.kv_len, D, ty, tx, dv, one);
  store_tile<T, CH>(attn_at<T>(p.dk, p.sdk, at.b, at.h), p.sdk.s, j0, p.kv_len, D, ty, tx, dk, sc);
}

template <typename K>
int launch(K kernel, const AttnParams& p, long long blocks, int smem, cudaStream_t st) {
  if (blocks == 0) return LSR_OK;
  if (blocks > 0x7fffffffll) return LSR_ERR_SHAPE;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return LSR_ERR_LAUNCH;
  ProfScope prof(PK_GEMM_OTHER, st);
  kernel<<<(unsigned)blocks, ATHREADS, smem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? LSR_OK : LSR_ERR_LAUNCH;
}

template <typename T, int CH>
int forward(const AttnParams& p, cudaStream_t st) {
  const int tile = AT * (CH * 64 + 4) * 4, score = AT * PLD * 4;
  return launch(attn_fwd_general_kernel<T, CH>, p, (long long)cdiv(p.q_len, AT) * p.heads * p.batch, 3 * tile + score, st);
}

template <typename T, int CH>
int backward(const AttnParams& p, cudaStream_t st) {
  const int tile = AT * (CH * 64 + 4) * 4, score = AT * PLD * 4;
  const long long rows = (long long)p.batch * p.heads * p.q_len;
  int rc = launch(attn_delta_kernel<T>, p, (rows + ATHREADS / 32 - 1) / (ATHREADS / 32), 0, st);
  if (rc != LSR_OK) return rc;
  rc = launch(attn_dkv_general_kernel<T, CH>, p, (long long)cdiv(p.kv_len, AT) * p.kv_heads * p.batch,
              4 * tile + 2 * score, st);
  if (rc != LSR_OK) return rc;
  return launch(attn_dq_general_kernel<T, CH>, p, (long long)cdiv(p.q_len, AT) * p.heads * p.batch, 4 * tile + score, st);
}

}  // namespace

int attention_forward_general(const AttnParams& p, int dtype, cudaStream_t st) {
  const bool wide = p.head_dim > 64;
  if (dtype == LSR_DTYPE_F32) return wide ? forward<float, 2>(p, st) : forward<float, 1>(p, st);
  if (dtype == LSR_DTYPE_BF16) return wide ? forward<__nv_bfloat16, 2>(p, st) : forward<__nv_bfloat16, 1>(p, st);
  return wide ? forward<__half, 2>(p, st) : forward<__half, 1>(p, st);
}

int attention_backward_general(const AttnParams& p, int dtype, cudaStream_t st) {
  const bool wide = p.head_dim > 64;
  if (dtype == LSR_DTYPE_F32) return wide ? backward<float, 2>(p, st) : backward<float, 1>(p, st);
  if (dtype == LSR_DTYPE_BF16) return wide ? backward<__nv_bfloat16, 2>(p, st) : backward<__nv_bfloat16, 1>(p, st);
  return wide ? backward<__half, 2>(p, st) : backward<__half, 1>(p, st);
}

}  // namespace lsr
