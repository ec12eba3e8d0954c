// The weights that a prompt's queries give its keys (gfx950).
//
// w[j] = sum over the query heads of a key-value head and over the last W tokens i of a prompt of exp(s_ij - lse_i), with
// s_ij = scale q_i.k_j for keys j up to the query's own token and lse_i = log sum_j exp(s_ij): column sums of the attention
// matrix, which is never stored.  The sums need every row's lse first, so the product is made twice: once for the lse of each
// (query, head), called a column here, and once for the sums.  A tile of it is 32 keys by 32 columns (MFMA 32x32x16), whose lane
// l holds one column of the product, l % 32, and of its rows 8 (i / 4) + 4 (l / 32) + i % 4 as accumulator i: with the columns as
// columns the sums over keys stay in the lane until all tiles are done, with the keys as columns those over columns do.
//
// A wave keeps 64 columns in registers, and a workgroup of four streams the keys through LDS, 64 at a time straight from memory,
// three tiles ahead.  The matrix cores (32 cycles to an instruction) and the exponentials (8, and 4 each for the product with
// its offset and the addition) take the same time, 256 cycles for a tile of 128 dims, so one tile's products are issued between
// the exponentials of the tile before.
#include <math.h>

#include "ri_common.h"

#define WG_WAVES 4
#define WG_BLOCK (64 * WG_WAVES)   // columns of a workgroup
#define WG_TILE 64                 // rows of a streamed tile
#define WG_BUFFERS 3
#define WG_ROWS 1024               // keys of a split at most
#define WG_LOG2E 1.4426950408889634f

typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct WeighParams {
  const uint16_t* q;      // [B, W, heads * gs, D]
  const uint16_t* key;    // [B, T, heads, D]
  int64_t qb, qt, qh, kb, kt, kh;
  const int32_t* lens;    // [B] or null: T each
  float* out;             // [B, heads, T]
  float* stats;           // [B * heads, S, cols_pad, 2] maximum (units of ln 2) and sum of the splits
  float* lse;             // [B * heads, cols_pad], units of ln 2; +inf: the column has no keys
  float* part;            // [B * heads, supers, T] sums of `per` blocks of columns each
  int heads, gs, W, T, cols, cols_pad;
  int S, rows;            // splits of the keys, keys of one
  int per, supers;
  int joined;             // whether lse is filled before the second kernel
  float scale2;           // scale / ln 2
};

// The lse of a column from its splits, of which this thread takes `part`, part + of, ...; `of` neighbouring lanes together.
__device__ __forceinline__ float weigh_join(const WeighParams& P, int g, int col, int part, int of) {
  const float* const at = P.stats + ((size_t)g * P.S * P.cols_pad + col) * 2;
  float M = -INFINITY, L = 0.f;
#pragma unroll 4
  for (int s = part; s < P.S; s += of) {
    const float2 x = *reinterpret_cast<const float2*>(at + (size_t)s * P.cols_pad * 2);
    const float mn = fmaxf(M, x.x), ref = mn == -INFINITY ? 0.f : mn;
    L = L * __builtin_amdgcn_exp2f(M - ref) + x.y * __builtin_amdgcn_exp2f(x.x - ref);
    M = mn;
  }
  for (int d = 1; d < of; d <<= 1) {
    const float m = __shfl_xor(M, d), l = __shfl_xor(L, d), mn = fmaxf(M, m), ref = mn == -INFINITY ? 0.f : mn;
    L = L * __builtin_amdgcn_exp2f(M - ref) + l * __builtin_amdgcn_exp2f(m - ref);
    M = mn;
  }
  return L != 0.f ? M + __log2f(L) : INFINITY;
}

__device__ __forceinline__ int weigh_len(const WeighParams& P, int b) { return P.lens ? min(max(P.lens[b], 0), P.T) : P.T; }

template <bool HALF>
__device__ __forceinline__ f32x16_t weigh_mfma(uint4 a, uint4 b, f32x16_t c) {
  return HALF ? __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0)
              : __builtin_amdgcn_mfma_f32_32x32x16_bf16(ri_as_bf16x8(a), ri_as_bf16x8(b), c, 0, 0, 0);
}

__device__ __forceinline__ int weigh_key_of(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }

// 16 bytes per lane from memory straight into LDS, lane l behind lane l - 1 from lds_base on; `at`: the lane's byte offset.
// The caller waits (vmcnt).
__device__ __forceinline__ uint32_t weigh_lds(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
__device__ __forceinline__ void weigh_dma16(const void* base, uint32_t at, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(at), "s"(base), "s"(lds_base) : "memory", "m0");
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

// The product of one tile beside the exponentials of the one before: eight (D = 64: four) matrix instructions, each followed by
// a share of the sixteen exponentials and their additions.
template <int KK>
__device__ __forceinline__ void weigh_interleave() {
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);             // matrix product
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);             // LDS read
    __builtin_amdgcn_sched_group_barrier(0x400, 16 / KK, 0);       // exponentials
    __builtin_amdgcn_sched_group_barrier(0x002, 2 * 16 / KK, 0);   // their products and sums
  }
}

// One pass over the keys [j0, j1) of split blockIdx.z of group blockIdx.x.
// SUM false: the lse.  Columns of block gridDim.y - 1 - blockIdx.y (those that see most keys first), as columns of the product;
// m and l of a lane: its reference and the sum of exponentials relative to it, over its own keys.  The reference is the maximum of
// the first tile that the column sees, and moves only where a tile's sum passes 2^100: until then neither the sums nor their
// precision suffer, and a score costs a product with its offset, an exponential and an addition.
// SUM true: the sums over the columns of `per` blocks from blockIdx.y * per on, as rows of the product, so that the columns add
// up in the lane; a wave keeps its sums of the split's keys in LDS.
template <int D, bool HALF, bool SUM>
__global__ __launch_bounds__(64 * WG_WAVES, 2) void weigh_kernel(WeighParams P) {
  constexpr int KK = D / 16, L = WG_LOADS<D>;
  __shared__ __attribute__((aligned(16))) uint16_t sh[WG_BUFFERS][WG_TILE * D];
  __shared__ __attribute__((aligned(16))) float sh_lse[SUM ? WG_BLOCK : 4];
  extern __shared__ float sh_sum[];   // [WG_WAVES][rows]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x, b = g / P.heads, head = g - b * P.heads;
  const int n = weigh_len(P, b), first = n - P.W;                   // first: the first query's token
  const int blocks = P.cols_pad / WG_BLOCK;
  const int block0 = SUM ? blockIdx.y * P.per : gridDim.y - 1 - blockIdx.y, block1 = SUM ? min(block0 + P.per, blocks) : block0 + 1;
  const int j0 = blockIdx.z * P.rows, jn = min(j0 + P.rows, n);
  const uint16_t* const keys = P.key + b * P.kb + head * P.kh;
  const uint32_t stride = (uint32_t)P.kt * 2;
  const auto stage = [&](int t) {
    const int j = j0 + t * WG_TILE;
    weigh_stage<D>(keys + j * P.kt, sh[t % WG_BUFFERS], wave, [&](int r) { return (uint32_t)min(r, n - 1 - j) * stride; });
  };
  float* const mine_sum = sh_sum + wave * P.rows;
  if (SUM)
    for (int i = lane; i < P.rows; i += 64) mine_sum[i] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  for (int block = block0; block < block1; ++block) {
    const int colw = block * WG_BLOCK + wave * 64;
    const int j1 = min(jn, first + min(block * WG_BLOCK + WG_BLOCK - 1, P.cols - 1) / P.gs + 1);   // (the last key of the block)
    if (j0 >= j1) continue;
    const int tiles = (j1 - j0 + WG_TILE - 1) / WG_TILE, subs = (j1 - j0 + 31) / 32;
    if (SUM) {   // the block's lse, joined from its splits where nobody has done so before
      __syncthreads();
      const int col = block * WG_BLOCK + threadIdx.x;
      sh_lse[threadIdx.x] = P.joined ? P.lse[(size_t)g * P.cols_pad + col] : weigh_join(P, g, col, 0, 1);
      __syncthreads();
    }
    uint4 q[2][KK];
    int low[2];                 // last key of each tile's first column
    f32x16_t off[2];            // SUM: minus the lse of the rows
    int mine[2];                // else: last key of the lane's column
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int c = colw + 32 * t, col = min(c + (lane & 31), P.cols - 1), i = col / P.gs;
      mine[t] = first + i;
      low[t] = first + min(c, P.cols - 1) / P.gs;
      const uint16_t* at = P.q + b * P.qb + i * P.qt + (head * P.gs + col - i * P.gs) * P.qh + 8 * (lane >> 5);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) q[t][kk] = ri_ld16(at + 16 * kk);
      if (SUM) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float4 o = *reinterpret_cast<const float4*>(&sh_lse[wave * 64 + 32 * t + 8 * x + 4 * (lane >> 5)]);
          off[t][4 * x] = -o.x; off[t][4 * x + 1] = -o.y; off[t][4 * x + 2] = -o.z; off[t][4 * x + 3] = -o.w;
        }
      }
    }
    weigh_arrived(q);
    stage(0);
    if (tiles > 1) stage(1);
    if (tiles > 2) stage(2);
    if (tiles > 2) weigh_wait<2 * L>();
    else if (tiles > 1) weigh_wait<L>();
    else weigh_wait<0>();
    weigh_barrier();
    uint4 a[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) a[kk] = weigh_operand<D>(sh[0], 0, kk);
    const auto product = [&](int t, int kk, f32x16_t c) {
      return SUM ? weigh_mfma<HALF>(q[t][kk], a[kk], c) : weigh_mfma<HALF>(a[kk], q[t][kk], c);
    };
    const f32x16_t zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    f32x16_t s[2];
    s[0] = zero;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) s[0] = product(0, kk, s[0]);
    for (int u = 0; u < subs; ++u) {
      const int j = j0 + 32 * u;
      if ((u & 1) && u + 1 < subs) {   // the next sub-tile is the next tile's first; nobody reads this tile any more
        const int t = u >> 1;
        if (t + 2 < tiles) weigh_wait<L>();
        else weigh_wait<0>();
        weigh_barrier();
        if (t + 3 < tiles) stage(t + 3);
      }
      const int next = min(u + 1, subs - 1);
      const uint16_t* const tile = sh[(next >> 1) % WG_BUFFERS];
      float both = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float scale2 = P.scale2;
        if (j + 31 > low[t]) {   // some column does not see every key
          if (SUM) {
            const int key = j + (lane & 31), c = colw + 32 * t, i0 = c / P.gs, at = c - i0 * P.gs + 4 * (lane >> 5);
            const uint32_t inv = 65536 / P.gs + 1;   // (exact for what is divided here: less than 48 by up to 16)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int last = first + i0 + (int)(((uint32_t)(at + 8 * (i >> 2) + (i & 3)) * inv) >> 16);
              s[t][i] = key > last ? -INFINITY : s[t][i] * scale2;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = j + weigh_key_of(i, lane) > mine[t] ? -INFINITY : s[t][i] * scale2;
          }
          scale2 = 1.f;
        }
        // tile t's exponentials beside the product of the other tile (of the next sub-tile behind t = 1)
        f32x16_t p = zero;
        float sum = 0.f, x = 0.f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          p = product(1 - t, kk, p);
          if (t == 0) a[kk] = weigh_operand<D>(tile, (next & 1) * 32, kk);
        }
#pragma unroll
        for (int i = 0; i < 16; i += 2) {   // (two sums, so that an addition does not wait for the one before)
          sum += __builtin_amdgcn_exp2f(fmaf(s[t][i], scale2, SUM ? off[t][i] : -m[t]));
          x += __builtin_amdgcn_exp2f(fmaf(s[t][i + 1], scale2, SUM ? off[t][i + 1] : -m[t]));
        }
        sum += x;
        weigh_interleave<KK>();
        if (SUM) {
          both += sum;
        } else {
          if (__builtin_amdgcn_ballot_w64(!(sum < 0x1p100f))) {
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmaxf(most, s[t][i] * scale2);
            const float mn = fmaxf(m[t], most), ref = mn == -INFINITY ? 0.f : mn;
            l[t] *= __builtin_amdgcn_exp2f(m[t] - ref);
            m[t] = mn;
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f(fmaf(s[t][i], scale2, -ref));
          }
          l[t] += sum;
        }
        s[1 - t] = p;
      }
      if (SUM) {
        both = ri_xor_sum<32>(both);
        if (lane < 32) mine_sum[32 * u + lane] += both;
      }
    }
    if (SUM) weigh_barrier();   // (the tiles are loaded again)
  }

  if (SUM) {
    __syncthreads();
    float* const to = P.supers > 1 ? P.part + ((size_t)g * P.supers + blockIdx.y) * P.T : P.out + (size_t)g * P.T;
    for (int i = threadIdx.x; i < P.rows && j0 + i < P.T; i += 64 * WG_WAVES)
      to[j0 + i] = sh_sum[i] + sh_sum[P.rows + i] + sh_sum[2 * P.rows + i] + sh_sum[3 * P.rows + i];
    return;
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int col = block0 * WG_BLOCK + wave * 64 + 32 * t + (lane & 31);
    const float M = ri_xor_max<32>(m[t]);
    const float Z = ri_xor_sum<32>(m[t] == -INFINITY ? l[t] : l[t] * __builtin_amdgcn_exp2f(m[t] - M));
    if (lane < 32) {
      float* const at = P.stats + (((size_t)g * P.S + blockIdx.z) * P.cols_pad + col) * 2;
      at[0] = col < P.cols ? M : -INFINITY;
      at[1] = col < P.cols ? Z : 0.f;
    }
  }
}

// Grid (cols_pad / 32, B * heads), 256 threads: eight threads join the splits of a column.
__global__ __launch_bounds__(256) void weigh_join_kernel(WeighParams P) {
  const int g = blockIdx.y, col = blockIdx.x * 32 + (threadIdx.x >> 3);
  const float lse = weigh_join(P, g, col, threadIdx.x & 7, 8);
  if ((threadIdx.x & 7) == 0) P.lse[(size_t)g * P.cols_pad + col] = lse;
}

// Grid (ceil(T / 256), B * heads): a thread adds the columns' blocks of a key.
__global__ __launch_bounds__(256) void weigh_add_kernel(WeighParams P) {
  const int g = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  if (j >= P.T) return;
  float x = 0.f;
  for (int s = 0; s < P.supers; ++s) x += P.part[((size_t)g * P.supers + s) * P.T + j];
  P.out[(size_t)g * P.T + j] = x;
}

// ------------------------------------------------------------------------------------ host side
struct WeighPlan { int cols_pad, S, rows, per, supers; bool joined; };
static int weigh_up(int64_t n, int to) { return (int)((n + to - 1) / to * to); }
static WeighPlan weigh_plan(int64_t groups, int cols, int T) {
  WeighPlan p;
  p.cols_pad = weigh_up(cols, WG_BLOCK);
  const int64_t blocks = p.cols_pad / WG_BLOCK;
  // keys of a split: workgroups for the compute units, and no more keys than there is LDS for their sums
  const int64_t want = (T * groups * blocks + 767) / 768;
  p.rows = weigh_up(want < 128 ? 128 : want > WG_ROWS ? WG_ROWS : want, WG_TILE);
  p.S = (T + p.rows - 1) / p.rows;
  // blocks of columns whose sums a workgroup of the second kernel adds up
  p.per = (int)(groups * p.S * blocks / 2048);
  if (p.per > 8) p.per = 8;
  if (p.per < 1) p.per = 1;
  p.supers = (int)((blocks + p.per - 1) / p.per);
  p.joined = p.S > 8;
  return p;
}

extern "C" size_t ri_attention_weights_workspace_bytes(int B, int heads, int gs, int W, int T) {
  if (B <= 0 || heads <= 0 || gs <= 0 || gs > 16 || W <= 0 || T < W || T > 1 << 24 || (int64_t)B * heads > 65535) return 0;
  const WeighPlan p = weigh_plan((int64_t)B * heads, W * gs, T);
  return (size_t)B * heads * ((size_t)p.cols_pad * (2 * (size_t)p.S + (p.joined ? 1 : 0)) + (p.supers > 1 ? (size_t)p.supers * T : 0)) * sizeof(float);
}

template <int D, bool HALF>
static void launch_weigh(const WeighParams& P, int groups, hipStream_t s) {
  const int blocks = P.cols_pad / WG_BLOCK;
  weigh_kernel<D, HALF, false><<<dim3(groups, blocks, P.S), 64 * WG_WAVES, 0, s>>>(P);
  if (P.joined) weigh_join_kernel<<<dim3(P.cols_pad / 32, groups), 256, 0, s>>>(P);
  weigh_kernel<D, HALF, true><<<dim3(groups, P.supers, P.S), 64 * WG_WAVES, WG_WAVES * P.rows * sizeof(float), s>>>(P);
  if (P.supers > 1) weigh_add_kernel<<<dim3((P.T + 255) / 256, groups), 256, 0, s>>>(P);
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
  if (key_token_stride > 1 << 23) return RI_ERR_ARG;   // (a tile's rows are addressed by 32-bit offsets from its first)
  if (workspace_bytes < need) return RI_ERR_WORKSPACE;
  const int cols = W * gs, groups = B * heads;
  const WeighPlan p = weigh_plan(groups, cols, T);
  float* const stats = (float*)workspace;
  float* const lse = stats + (size_t)groups * p.cols_pad * 2 * p.S;
  const WeighParams P = {(const uint16_t*)q, (const uint16_t*)key, q_batch_stride, q_token_stride, q_head_stride, key_batch_stride,
                         key_token_stride, key_head_stride, seqlens, out, stats, lse,
                         lse + (p.joined ? (size_t)groups * p.cols_pad : 0), heads, gs, W, T, cols, p.cols_pad, p.S, p.rows, p.per,
                         p.supers, p.joined, scale * WG_LOG2E};
  hipStream_t s = (hipStream_t)stream;
  if (dim == 64) half ? launch_weigh<64, true>(P, groups, s) : launch_weigh<64, false>(P, groups, s);
  else half ? launch_weigh<128, true>(P, groups, s) : launch_weigh<128, false>(P, groups, s);
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
