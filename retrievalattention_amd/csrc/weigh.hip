// The weights that a prompt's queries give its keys (gfx950).
//
// w[j] = sum over the query heads of a key-value head and over the last W tokens i of a prompt of exp(s_ij - lse_i), with
// s_ij = scale q_i.k_j for keys j up to the query's own token and lse_i = log sum_j exp(s_ij): column sums of the attention
// matrix, which is never stored.  The sums need every row's lse first, so the product is made twice: once for the lse of each
// (query, head), called a column here, and once for the sums.  Both times a tile of it is K Q^T (MFMA 32x32x16, 32 keys as rows,
// 32 columns): lane l has column l % 32 and the keys 8 (i / 4) + 4 (l / 32) + i % 4 of its 16 accumulators i, so that the sums
// over keys (first kernel), and those over columns (second), stay in the lane until all tiles are done.
//
// A wave keeps two tiles of one operand in registers (64 columns, then 64 keys) and a workgroup of four streams the other one
// through LDS, 64 rows at a time straight from memory, two steps ahead.
#include <math.h>

#include "ri_common.h"

#define WG_WAVES 4
#define WG_BLOCK (64 * WG_WAVES)   // columns, then keys, of a workgroup
#define WG_TILE 64                 // rows of a streamed tile
#define WG_BUFFERS 3
#define WG_LOG2E 1.4426950408889634f

typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct WeighParams {
  const uint16_t* q;      // [B, W, heads * gs, D]
  const uint16_t* key;    // [B, T, heads, D]
  int64_t qb, qt, qh, kb, kt, kh;
  const int32_t* lens;    // [B] or null: T each
  float* out;             // [B, heads, T]
  float* lse;             // [B * heads, cols_pad], units of ln 2; +inf: the column has no keys
  float* part;            // [B * heads, S, W * gs, 2] maximum and sum, then [B * heads, S2, T] sums
  int heads, gs, W, T, cols, cols_pad;
  int S, rows;            // splits of the keys in the first kernel, keys of one
  int S2, cols2;          // splits of the columns in the second, columns of one
  float scale2;           // scale / ln 2
};

__device__ __forceinline__ int weigh_len(const WeighParams& P, int b) { return P.lens ? min(max(P.lens[b], 0), P.T) : P.T; }

template <bool HALF>
__device__ __forceinline__ f32x16_t weigh_mfma(uint4 a, uint4 b, f32x16_t c) {
  return HALF ? __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0)
              : __builtin_amdgcn_mfma_f32_32x32x16_bf16(ri_as_bf16x8(a), ri_as_bf16x8(b), c, 0, 0, 0);
}

__device__ __forceinline__ int weigh_key_of(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }

// 16 or 4 bytes per lane from memory straight into LDS, lane l behind lane l - 1 from lds_base on; `at`: the lane's byte offset.
// The caller waits (vmcnt).
__device__ __forceinline__ uint32_t weigh_lds(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
__device__ __forceinline__ void weigh_dma16(const void* base, uint32_t at, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(at), "s"(base), "s"(lds_base) : "memory", "m0");
}
__device__ __forceinline__ void weigh_dma4(const void* base, uint32_t at, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(at), "s"(base), "s"(lds_base) : "memory", "m0");
}
template <int V>
__device__ __forceinline__ void weigh_wait() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(V) : "memory"); }
__device__ __forceinline__ void weigh_barrier() { asm volatile("s_barrier" ::: "memory"); }

// A streamed tile in LDS: row r's piece p (16 bytes) lies at place p ^ (r % pieces) of the row, so that neither the 32 rows that
// a wave reads a piece of nor the loads, a row by a row's lanes, meet in a bank.  offset(r): byte offset of row r's start in
// memory from `base`; a wave loads a quarter of the rows, WG_LOADS<D> instructions.
template <int D>
constexpr int WG_LOADS = WG_TILE * D * 2 / (1024 * WG_WAVES);
template <int D, typename Offset>
__device__ __forceinline__ void weigh_stage(const void* base, uint16_t* tile, int wave, Offset&& offset) {
  constexpr int PP = D / 8, RW = 64 / PP;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < WG_LOADS<D>; ++i) {
    const int r0 = (wave * WG_LOADS<D> + i) * RW, r = r0 + lane / PP;
    weigh_dma16(base, offset(r) + (((lane % PP) ^ (r % PP)) << 4), __builtin_amdgcn_readfirstlane(weigh_lds(tile + r0 * D)));
  }
}
// lane's operand kk of the 32 rows from `sub` on: row sub + lane % 32, dims 16 kk + 8 (lane / 32) ..
template <int D>
__device__ __forceinline__ uint4 weigh_operand(const uint16_t* tile, int sub, int kk) {
  constexpr int PP = D / 8;
  const int lane = threadIdx.x & 63, r = lane & 31;
  return *reinterpret_cast<const uint4*>(tile + (sub + r) * D + (((2 * kk + (lane >> 5)) ^ (r % PP)) << 3));
}

// Waits for a wave's own operand, so that no wait for it stands between the counted ones for the tiles.
template <int KK>
__device__ __forceinline__ void weigh_arrived(uint4 (&x)[2][KK]) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) asm volatile("" : "+v"(x[t][kk].x), "+v"(x[t][kk].y), "+v"(x[t][kk].z), "+v"(x[t][kk].w));
  weigh_wait<0>();
}

// Grid (B * heads, ceil(cols / WG_BLOCK), S): a wave has 64 columns, the workgroup the keys of the split.
// m and l of a lane: its reference and sum of exponentials relative to it, over its own keys.  The reference is the maximum of
// the first tile that the column sees, and moves only where a tile's sum passes 2^100: until then neither the sums nor their
// precision suffer, and a score costs a product with its offset, an exponential and an addition.
template <int D, bool HALF>
__global__ __launch_bounds__(64 * WG_WAVES, 2) void weigh_lse_kernel(WeighParams P) {
  constexpr int KK = D / 16;
  __shared__ __attribute__((aligned(16))) uint16_t sh[WG_BUFFERS][WG_TILE * D];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x, b = g / P.heads, head = g - b * P.heads;
  const int block = gridDim.y - 1 - blockIdx.y;                     // (the columns that see most keys first)
  const int n = weigh_len(P, b), first = n - P.W;                   // first: the first query's token
  const int colw = block * WG_BLOCK + wave * 64;
  const int block_top = first + min(block * WG_BLOCK + WG_BLOCK - 1, P.cols - 1) / P.gs;   // the workgroup's last key
  const int j0 = blockIdx.z * P.rows, j1 = min(j0 + P.rows, block_top + 1);
  int mine[2], low[2], top[2];   // last key of the lane's column; of the tile's first and last column
  float m[2], l[2];
  uint4 q[2][KK];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int c = colw + 32 * t, col = min(c + (lane & 31), P.cols - 1), i = col / P.gs;
    mine[t] = first + i;
    low[t] = first + min(c, P.cols - 1) / P.gs;
    top[t] = first + min(c + 31, P.cols - 1) / P.gs;
    m[t] = -INFINITY;
    l[t] = 0.f;
    const uint16_t* at = P.q + b * P.qb + i * P.qt + (head * P.gs + col - i * P.gs) * P.qh + 8 * (lane >> 5);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) q[t][kk] = ri_ld16(at + 16 * kk);
  }
  if (j0 < j1) {
    const int tiles = (j1 - j0 + WG_TILE - 1) / WG_TILE;
    const uint16_t* const keys = P.key + b * P.kb + head * P.kh;
    const uint32_t stride = (uint32_t)P.kt * 2;
    const auto stage = [&](int t) {
      const int j = j0 + t * WG_TILE;
      weigh_stage<D>(keys + j * P.kt, sh[t % WG_BUFFERS], wave, [&](int r) { return (uint32_t)min(r, n - 1 - j) * stride; });
    };
    weigh_arrived(q);
    stage(0);
    if (tiles > 1) stage(1);
    for (int t = 0; t < tiles; ++t) {
      if (t + 1 < tiles) weigh_wait<WG_LOADS<D>>();
      else weigh_wait<0>();
      weigh_barrier();
      if (t + 2 < tiles) stage(t + 2);
      const uint16_t* const tile = sh[t % WG_BUFFERS];
#pragma unroll
      for (int sub = 0; sub < WG_TILE; sub += 32) {
        const int j = j0 + t * WG_TILE + sub;
        if (j > top[1] || j >= j1) continue;
        f32x16_t s[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) s[0][i] = s[1][i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          const uint4 a = weigh_operand<D>(tile, sub, kk);
          s[0] = weigh_mfma<HALF>(a, q[0][kk], s[0]);
          s[1] = weigh_mfma<HALF>(a, q[1][kk], s[1]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float scale2 = P.scale2;
          if (j + 31 > low[c]) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[c][i] = j + weigh_key_of(i, lane) > mine[c] ? -INFINITY : s[c][i] * scale2;
            scale2 = 1.f;
          }
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f(fmaf(s[c][i], scale2, -m[c]));
          if (__builtin_amdgcn_ballot_w64(!(sum < 0x1p100f))) {
            float x = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) x = fmaxf(x, s[c][i] * scale2);
            const float mn = fmaxf(m[c], x), ref = mn == -INFINITY ? 0.f : mn;
            l[c] *= __builtin_amdgcn_exp2f(m[c] - ref);
            m[c] = mn;
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f(fmaf(s[c][i], scale2, -ref));
          }
          l[c] += sum;
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int col = colw + 32 * t + (lane & 31);
    const float M = ri_xor_max<32>(m[t]);
    const float L = ri_xor_sum<32>(m[t] == -INFINITY ? l[t] : l[t] * __builtin_amdgcn_exp2f(m[t] - M));
    if (lane < 32 && col < P.cols_pad) {
      if (P.S == 1) {
        P.lse[(size_t)g * P.cols_pad + col] = col < P.cols && L != 0.f ? M + __log2f(L) : INFINITY;
      } else if (col < P.cols) {
        float* const at = P.part + (((size_t)g * P.S + blockIdx.z) * P.cols + col) * 2;
        at[0] = M;
        at[1] = L;
      }
    }
  }
}

// Grid (ceil(cols_pad / 256), B * heads): a thread joins the splits of a column.
__global__ __launch_bounds__(256) void weigh_join_kernel(WeighParams P) {
  const int g = blockIdx.y, col = blockIdx.x * 256 + threadIdx.x;
  if (col >= P.cols_pad) return;
  float M = -INFINITY, L = 0.f;
  if (col < P.cols) {
    const float* const at = P.part + ((size_t)g * P.S * P.cols + col) * 2;
    for (int s = 0; s < P.S; ++s) {
      const float m = at[(size_t)s * P.cols * 2], l = at[(size_t)s * P.cols * 2 + 1];
      const float mn = fmaxf(M, m), ref = mn == -INFINITY ? 0.f : mn;
      L = L * __builtin_amdgcn_exp2f(M - ref) + l * __builtin_amdgcn_exp2f(m - ref);
      M = mn;
    }
  }
  P.lse[(size_t)g * P.cols_pad + col] = L != 0.f ? M + __log2f(L) : INFINITY;
}

// The first column that sees a key of the workgroup's block of keys from j0 on, rounded down to a streamed tile.
__device__ __forceinline__ int weigh_first_col(const WeighParams& P, int n, int j0) {
  return max(j0 - (n - P.W), 0) * P.gs / WG_TILE * WG_TILE;
}

// Grid (B * heads, ceil(T / WG_BLOCK), S2): a wave has 64 keys, the workgroup the columns of the split that see any of them.
template <int D, bool HALF>
__global__ __launch_bounds__(64 * WG_WAVES, 2) void weigh_sum_kernel(WeighParams P) {
  constexpr int KK = D / 16;
  __shared__ __attribute__((aligned(16))) uint16_t sh[WG_BUFFERS][WG_TILE * D];
  __shared__ __attribute__((aligned(16))) float sh_lse[WG_BUFFERS][WG_WAVES][WG_TILE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x, b = g / P.heads, head = g - b * P.heads;
  const int n = weigh_len(P, b), first = n - P.W, jb = blockIdx.y * WG_BLOCK, jw = jb + wave * 64;
  const int c0 = max(weigh_first_col(P, n, jb), (int)blockIdx.z * P.cols2), c1 = min(((int)blockIdx.z + 1) * P.cols2, P.cols);
  f32x16_t sum[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) sum[0][i] = sum[1][i] = 0.f;
  if (jb < n && c0 < c1) {
    uint4 k[2][KK];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t* const at = P.key + b * P.kb + min(jw + 32 * t + (lane & 31), n - 1) * P.kt + head * P.kh + 8 * (lane >> 5);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) k[t][kk] = ri_ld16(at + 16 * kk);
    }
    const int tiles = (c1 - c0 + WG_TILE - 1) / WG_TILE;
    const uint16_t* const queries = P.q + b * P.qb + head * P.gs * P.qh;
    const float* const lse = P.lse + (size_t)g * P.cols_pad;
    const auto stage = [&](int t) {
      const int c = c0 + t * WG_TILE, i0 = c / P.gs;
      weigh_stage<D>(queries + i0 * P.qt, sh[t % WG_BUFFERS], wave, [&](int r) {
        const int col = min(c + r, P.cols - 1), i = col / P.gs;
        return ((uint32_t)(i - i0) * (uint32_t)P.qt + (uint32_t)(col - i * P.gs) * (uint32_t)P.qh) * 2;
      });
      weigh_dma4(lse + c, lane * 4, __builtin_amdgcn_readfirstlane(weigh_lds(sh_lse[t % WG_BUFFERS][wave])));
    };
    weigh_arrived(k);
    stage(0);
    if (tiles > 1) stage(1);
    for (int t = 0; t < tiles; ++t) {
      if (t + 1 < tiles) weigh_wait<WG_LOADS<D> + 1>();
      else weigh_wait<0>();
      weigh_barrier();
      if (t + 2 < tiles) stage(t + 2);
      const uint16_t* const tile = sh[t % WG_BUFFERS];
#pragma unroll
      for (int sub = 0; sub < WG_TILE; sub += 32) {
        const int c = c0 + t * WG_TILE + sub;
        const int low = first + c / P.gs, top = first + min(c + 31, P.cols - 1) / P.gs;   // last keys of the first and last column
        if (c >= P.cols || top < jw) continue;
        f32x16_t s[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) s[0][i] = s[1][i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          const uint4 a = weigh_operand<D>(tile, sub, kk);
          s[0] = weigh_mfma<HALF>(k[0][kk], a, s[0]);
          s[1] = weigh_mfma<HALF>(k[1][kk], a, s[1]);
        }
        const float off = sh_lse[t % WG_BUFFERS][wave][sub + (lane & 31)];
        const bool all = low >= jw + 63;    // every column sees every key (and the first one is there)
        float scale2 = P.scale2;
        if (!all) {
          const int mine = first + min(c + (lane & 31), P.cols - 1) / P.gs;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = jw + 32 * u + weigh_key_of(i, lane) > mine ? -INFINITY : s[u][i] * scale2;
          scale2 = 1.f;
        }
        // (a column without keys, and one past the last, has an lse of inf: -inf less it weighs 0)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[u][i] += __builtin_amdgcn_exp2f(fmaf(s[u][i], scale2, -off));
      }
    }
  } else if (P.S2 > 1) {
    return;   // (not read)
  }
  float* const to = P.S2 > 1 ? P.part + ((size_t)g * P.S2 + blockIdx.z) * P.T : P.out + (size_t)g * P.T;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = ri_xor_sum<1>(ri_xor_sum<2>(ri_xor_sum<4>(ri_xor_sum<8>(ri_xor_sum<16>(sum[u][i])))));
      const int j = jw + 32 * u + weigh_key_of(i, lane);
      if ((lane & 31) == 0 && j < P.T) to[j] = j < n ? x : 0.f;
    }
}

// Grid (ceil(T / 256), B * heads): a thread adds the splits of a key.
__global__ __launch_bounds__(256) void weigh_add_kernel(WeighParams P) {
  const int g = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x, n = weigh_len(P, g / P.heads);
  if (j >= P.T) return;
  float x = 0.f;
  if (j < n)
    for (int s = weigh_first_col(P, n, j / WG_BLOCK * WG_BLOCK) / P.cols2; s < P.S2; ++s) x += P.part[((size_t)g * P.S2 + s) * P.T + j];
  P.out[(size_t)g * P.T + j] = x;
}

// ------------------------------------------------------------------------------------ host side
// Splits of the keys in the first kernel and of the columns in the second: enough workgroups for the compute units.
struct WeighPlan { int S, rows, S2, cols2, cols_pad; };
static int weigh_up(int64_t n, int to) { return (int)((n + to - 1) / to * to); }
static WeighPlan weigh_plan(int64_t groups, int cols, int T) {
  const auto split = [&](int64_t blocks, int64_t n, int* S, int* per) {
    const int64_t want = blocks >= 1024 ? 1 : (1024 + blocks - 1) / blocks;
    *per = weigh_up(max((n + want - 1) / want, (int64_t)512), WG_TILE);
    *S = (int)((n + *per - 1) / *per);
  };
  WeighPlan p;
  split(groups * ((cols + WG_BLOCK - 1) / WG_BLOCK), T, &p.S, &p.rows);
  split(groups * ((T + WG_BLOCK - 1) / WG_BLOCK), cols, &p.S2, &p.cols2);
  p.cols_pad = weigh_up(cols, WG_TILE);
  return p;
}

extern "C" size_t ri_attention_weights_workspace_bytes(int B, int heads, int gs, int W, int T) {
  if (B <= 0 || heads <= 0 || gs <= 0 || gs > 16 || W <= 0 || T < W || T > 1 << 24 || (int64_t)B * heads > 65535) return 0;
  const WeighPlan p = weigh_plan((int64_t)B * heads, W * gs, T);
  const size_t first = p.S > 1 ? 2 * (size_t)p.S * W * gs : 0, second = p.S2 > 1 ? (size_t)p.S2 * T : 0;
  return (size_t)B * heads * (p.cols_pad + (first > second ? first : second)) * sizeof(float);
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
  // (a tile's rows are addressed by 32-bit offsets from its first)
  if (key_token_stride > 1 << 23 || q_token_stride > 1 << 23 || q_head_stride > 1 << 25) return RI_ERR_ARG;
  if (workspace_bytes < need) return RI_ERR_WORKSPACE;
  const int cols = W * gs, groups = B * heads;
  const WeighPlan p = weigh_plan(groups, cols, T);
  const WeighParams P = {(const uint16_t*)q, (const uint16_t*)key, q_batch_stride, q_token_stride, q_head_stride, key_batch_stride,
                         key_token_stride, key_head_stride, seqlens, out, (float*)workspace,
                         (float*)workspace + (size_t)groups * p.cols_pad, heads, gs, W, T, cols, p.cols_pad, p.S, p.rows, p.S2,
                         p.cols2, scale * WG_LOG2E};
  hipStream_t s = (hipStream_t)stream;
  const dim3 first(groups, (cols + WG_BLOCK - 1) / WG_BLOCK, P.S), second(groups, (T + WG_BLOCK - 1) / WG_BLOCK, P.S2);
  auto* lse = dim == 64 ? half ? weigh_lse_kernel<64, true> : weigh_lse_kernel<64, false>
                        : half ? weigh_lse_kernel<128, true> : weigh_lse_kernel<128, false>;
  auto* sum = dim == 64 ? half ? weigh_sum_kernel<64, true> : weigh_sum_kernel<64, false>
                        : half ? weigh_sum_kernel<128, true> : weigh_sum_kernel<128, false>;
  lse<<<first, 64 * WG_WAVES, 0, s>>>(P);
  if (P.S > 1) weigh_join_kernel<<<dim3((p.cols_pad + 255) / 256, groups), 256, 0, s>>>(P);
  sum<<<second, 64 * WG_WAVES, 0, s>>>(P);
  if (P.S2 > 1) weigh_add_kernel<<<dim3((T + 255) / 256, groups), 256, 0, s>>>(P);
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
