// The weights that a prompt's queries give its keys (gfx950).
//
// w[j] = sum over the query heads of a key-value head and over the last W tokens i of a prompt of exp(s_ij - lse_i), with
// s_ij = scale q_i.k_j for keys j up to the query's own token and lse_i = log sum_j exp(s_ij): column sums of the attention
// matrix, which is never stored.  The sums need every row's lse first, so the product is made twice: once for the lse of each
// (query, head), called a column here, and once for the sums.  Both times a tile of it is K Q^T (MFMA 32x32x16, 32 keys as rows,
// 32 columns): lane l has column l % 32 and the keys 8 (i / 4) + 4 (l / 32) + i % 4 of its 16 accumulators i, so that maxima and
// sums over keys (first kernel), and sums over columns (second), stay in the lane until all tiles are done.
#include <math.h>

#include "ri_common.h"

#define WG_WAVES 4
#define WG_LOG2E 1.4426950408889634f

typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct WeighParams {
  const uint16_t* q;      // [B, W, heads * gs, D]
  const uint16_t* key;    // [B, T, heads, D]
  int64_t qb, qt, qh, kb, kt, kh;
  const int32_t* lens;    // [B] or null: T each
  float* out;             // [B, heads, T]
  float* lse;             // [B * heads, W * gs], units of ln 2; +inf: the column has no keys
  float* part;            // [B * heads, S, W * gs, 2] maximum and sum
  int heads, gs, W, T, S, rows;   // rows: keys of a split
  float scale2;           // scale / ln 2
};

__device__ __forceinline__ int weigh_len(const WeighParams& P, int b) { return P.lens ? min(max(P.lens[b], 0), P.T) : P.T; }

template <bool HALF>
__device__ __forceinline__ f32x16_t weigh_mfma(uint4 a, uint4 b, f32x16_t c) {
  return HALF ? __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0)
              : __builtin_amdgcn_mfma_f32_32x32x16_bf16(ri_as_bf16x8(a), ri_as_bf16x8(b), c, 0, 0, 0);
}

__device__ __forceinline__ int weigh_key_of(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }

// lane's operand of a column tile: the query row of column col, dims 8 (lane / 32) + 16 kk
template <int D>
__device__ __forceinline__ void weigh_query(const WeighParams& P, int b, int head, int col, uint4* q) {
  const int lane = threadIdx.x & 63, c = min(col, P.W * P.gs - 1), i = c / P.gs;
  const uint16_t* at = P.q + b * P.qb + i * P.qt + (head * P.gs + c - i * P.gs) * P.qh + 8 * (lane >> 5);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) q[kk] = ri_ld16(at + 16 * kk);
}

// Grid (ceil(W * gs / (32 * WG_WAVES)), B * heads, S): a wave has 32 columns and the keys of the split.
template <int D, bool HALF>
__global__ __launch_bounds__(64 * WG_WAVES) void weigh_lse_kernel(WeighParams P) {
  constexpr int KK = D / 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = blockIdx.y, b = g / P.heads, head = g - b * P.heads, cols = P.W * P.gs;
  const int col0 = (blockIdx.x * WG_WAVES + wave) * 32, col = col0 + (lane & 31);
  if (col0 >= cols) return;
  const int n = weigh_len(P, b);
  const int mine = n - P.W + min(col, cols - 1) / P.gs;                  // the column's own token: its last key
  const int top = n - P.W + min(col0 + 31, cols - 1) / P.gs;             // of the tile's columns the last one's
  uint4 q[KK];
  weigh_query<D>(P, b, head, col, q);
  const uint16_t* const kb = P.key + b * P.kb + head * P.kh + 8 * (lane >> 5);
  float m = -INFINITY, l = 0.f;
  const int j1 = min((int)(blockIdx.z + 1) * P.rows, top + 1);
  for (int j0 = blockIdx.z * P.rows; j0 < j1; j0 += 32) {
    const uint16_t* at = kb + min(j0 + (lane & 31), n - 1) * P.kt;
    f32x16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) s = weigh_mfma<HALF>(ri_ld16(at + 16 * kk), q[kk], s);
    float t = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = j0 + weigh_key_of(i, lane) <= mine ? s[i] * P.scale2 : -INFINITY;
      t = fmaxf(t, s[i]);
    }
    const float mn = fmaxf(m, t);
    if (mn == -INFINITY) continue;
    l *= __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
    for (int i = 0; i < 16; ++i) l += __builtin_amdgcn_exp2f(s[i] - mn);
    m = mn;
  }
  const float M = ri_xor_max<32>(m);
  const float L = ri_xor_sum<32>(m == -INFINITY ? 0.f : l * __builtin_amdgcn_exp2f(m - M));
  if (lane < 32 && col < cols) {
    if (P.S == 1) {
      P.lse[(size_t)g * cols + col] = L > 0.f ? M + __log2f(L) : INFINITY;
    } else {
      float* const at = P.part + (((size_t)g * P.S + blockIdx.z) * cols + col) * 2;
      at[0] = M;
      at[1] = L;
    }
  }
}

// Grid (ceil(W * gs / 256), B * heads): a thread joins the splits of a column.
__global__ __launch_bounds__(256) void weigh_join_kernel(WeighParams P) {
  const int g = blockIdx.y, cols = P.W * P.gs, col = blockIdx.x * 256 + threadIdx.x;
  if (col >= cols) return;
  const float* const at = P.part + ((size_t)g * P.S * cols + col) * 2;
  float M = -INFINITY, L = 0.f;
  for (int s = 0; s < P.S; ++s) {
    const float m = at[(size_t)s * cols * 2], l = at[(size_t)s * cols * 2 + 1];
    const float mn = fmaxf(M, m);
    if (mn == -INFINITY) continue;
    L = L * __builtin_amdgcn_exp2f(M - mn) + l * __builtin_amdgcn_exp2f(m - mn);
    M = mn;
  }
  P.lse[(size_t)g * cols + col] = L > 0.f ? M + __log2f(L) : INFINITY;
}

// Grid (ceil(T / (32 * WG_WAVES)), B * heads): a wave has 32 keys and goes over the columns that see them.
template <int D, bool HALF>
__global__ __launch_bounds__(64 * WG_WAVES) void weigh_sum_kernel(WeighParams P) {
  constexpr int KK = D / 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = blockIdx.y, b = g / P.heads, head = g - b * P.heads, cols = P.W * P.gs;
  const int j0 = (blockIdx.x * WG_WAVES + wave) * 32, n = weigh_len(P, b);
  if (j0 >= P.T) return;
  float sum[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) sum[i] = 0.f;
  if (j0 < n) {
    uint4 k[KK];
    const uint16_t* const at = P.key + b * P.kb + min(j0 + (lane & 31), n - 1) * P.kt + head * P.kh + 8 * (lane >> 5);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) k[kk] = ri_ld16(at + 16 * kk);
    const int i0 = max(j0 - (n - P.W), 0);      // the first query that sees a key of the tile
    for (int c0 = i0 * P.gs / 32 * 32; c0 < cols; c0 += 32) {
      const int col = c0 + (lane & 31);
      uint4 q[KK];
      weigh_query<D>(P, b, head, col, q);
      const float lse = col < cols ? P.lse[(size_t)g * cols + col] : INFINITY;
      const int mine = n - P.W + min(col, cols - 1) / P.gs;
      f32x16_t s;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) s = weigh_mfma<HALF>(k[kk], q[kk], s);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (j0 + weigh_key_of(i, lane) <= mine && lse != INFINITY) sum[i] += __builtin_amdgcn_exp2f(s[i] * P.scale2 - lse);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float x = ri_xor_sum<1>(ri_xor_sum<2>(ri_xor_sum<4>(ri_xor_sum<8>(ri_xor_sum<16>(sum[i])))));
    const int j = j0 + weigh_key_of(i, lane);
    if ((lane & 31) == 0 && j < P.T) P.out[(size_t)g * P.T + j] = j < n ? x : 0.f;
  }
}

// ------------------------------------------------------------------------------------ host side
// Keys of a split of the first kernel: enough workgroups for the compute units.
static int weigh_rows(int64_t groups, int cols, int T) {
  const int64_t blocks = groups * ((cols + 32 * WG_WAVES - 1) / (32 * WG_WAVES));
  const int64_t splits = blocks >= 1024 ? 1 : (1024 + blocks - 1) / blocks;
  const int64_t rows = (T + splits - 1) / splits;
  return (int)(rows < 256 ? 256 : (rows + 31) / 32 * 32);
}

extern "C" size_t ri_attention_weights_workspace_bytes(int B, int heads, int gs, int W, int T) {
  if (B <= 0 || heads <= 0 || gs <= 0 || gs > 16 || W <= 0 || T < W || T > 1 << 24 || (int64_t)B * heads > 65535) return 0;
  const int rows = weigh_rows((int64_t)B * heads, W * gs, T), S = (T + rows - 1) / rows;
  return (size_t)B * heads * W * gs * (S > 1 ? 2 * (size_t)S + 1 : 1) * sizeof(float);
}

static int attention_weights_impl(const void* q, const void* key, const int32_t* seqlens, float* out, int64_t q_batch_stride,
                                  int64_t q_token_stride, int64_t q_head_stride, int64_t key_batch_stride,
                                  int64_t key_token_stride, int64_t key_head_stride, int B, int W, int T, int heads, int gs,
                                  int dim, float scale, void* workspace, size_t workspace_bytes, bool half, ri_stream_t stream) {
  if (!q || !key || !out || !workspace || ri_any_misaligned16(q, key, workspace)) return RI_ERR_ARG;
  const size_t need = ri_attention_weights_workspace_bytes(B, heads, gs, W, T);
  if (!need || (dim != 64 && dim != 128)) return RI_ERR_ARG;
  for (const int64_t s : {q_batch_stride, q_token_stride, q_head_stride, key_batch_stride, key_token_stride, key_head_stride})
    if (s < 0 || s % 8) return RI_ERR_ARG;
  if (workspace_bytes < need) return RI_ERR_WORKSPACE;
  const int cols = W * gs, groups = B * heads;
  WeighParams P = {(const uint16_t*)q, (const uint16_t*)key, q_batch_stride, q_token_stride, q_head_stride, key_batch_stride,
                   key_token_stride, key_head_stride, seqlens, out, (float*)workspace, (float*)workspace + (size_t)groups * cols,
                   heads, gs, W, T, 1, weigh_rows(groups, cols, T), scale * WG_LOG2E};
  P.S = (T + P.rows - 1) / P.rows;
  hipStream_t s = (hipStream_t)stream;
  const int tile = 32 * WG_WAVES;
  const dim3 first((cols + tile - 1) / tile, groups, P.S), second((T + tile - 1) / tile, groups);
  auto* lse = dim == 64 ? half ? weigh_lse_kernel<64, true> : weigh_lse_kernel<64, false>
                        : half ? weigh_lse_kernel<128, true> : weigh_lse_kernel<128, false>;
  auto* sum = dim == 64 ? half ? weigh_sum_kernel<64, true> : weigh_sum_kernel<64, false>
                        : half ? weigh_sum_kernel<128, true> : weigh_sum_kernel<128, false>;
  lse<<<first, 64 * WG_WAVES, 0, s>>>(P);
  if (P.S > 1) weigh_join_kernel<<<dim3((cols + 255) / 256, groups), 256, 0, s>>>(P);
  sum<<<second, 64 * WG_WAVES, 0, s>>>(P);
  RI_HIP_CHECK_LAUNCH();
  return RI_OK;
}

extern "C" int ri_attention_weights(const void* q, const void* key, const int32_t* seqlens, float* out, int64_t q_batch_stride,
                                    int64_t q_token_stride, int64_t q_head_stride, int64_t key_batch_stride,
                                    int64_t key_token_stride, int64_t key_head_stride, int B, int W, int T, int heads, int gs,
                                    int dim, float scale, void* workspace, size_t workspace_bytes, ri_stream_t stream) {
  return attention_weights_impl(q, key, seqlens, out, q_batch_stride, q_token_stride, q_head_stride, key_batch_stride,
                                key_token_stride, key_head_stride, B, W, T, heads, gs, dim, scale, workspace, workspace_bytes,
                                false, stream);
}

extern "C" int ri_attention_weights_f16(const void* q, const void* key, const int32_t* seqlens, float* out, int64_t q_batch_stride,
                                        int64_t q_token_stride, int64_t q_head_stride, int64_t key_batch_stride,
                                        int64_t key_token_stride, int64_t key_head_stride, int B, int W, int T, int heads, int gs,
                                        int dim, float scale, void* workspace, size_t workspace_bytes, ri_stream_t stream) {
  return attention_weights_impl(q, key, seqlens, out, q_batch_stride, q_token_stride, q_head_stride, key_batch_stride,
                                key_token_stride, key_head_stride, B, W, T, heads, gs, dim, scale, workspace, workspace_bytes,
                                true, stream);
}
