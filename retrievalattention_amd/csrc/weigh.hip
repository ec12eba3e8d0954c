// The weights that a prompt's queries give its keys (gfx950).
//
// w[j] = sum over the query heads of a key-value head and over the last W tokens i of a prompt of exp(s_ij - lse_i), with
// s_ij = scale q_i.k_j for keys j up to the query's own token and lse_i = log sum_j exp(s_ij): column sums of the attention
// matrix, which is never stored.  The sums need every row's lse first, so the product is made twice: once for that of each
// (query, head), called a column here, and once for the sums.  A tile of it is 32 keys by 32 columns (MFMA 32x32x16), whose lane
// l holds one column of the product, l % 32, and of its rows 8 (i / 4) + 4 (l / 32) + i % 4 as accumulator i: with the columns as
// columns the sums over keys stay in the lane until all tiles are done, with the keys as columns those over columns do.
//
// A wave keeps 32 columns in registers, and a workgroup of eight streams the keys through LDS, 64 at a time straight from memory,
// two tiles ahead.  One tile's products are issued between the exponentials of the tile before: matrix instructions, exponentials
// and their products and sums in such turns take 400 cycles a tile of 128 dims (registers alone, two waves and more to a SIMD;
// one wave 570; the matrix instructions alone 300, the rest 275).
#include <math.h>

#include "ri_common.h"
#include "weigh_plan.h"

#define WG_BUFFERS 3
#define WG_LOG2E 1.4426950408889634f

typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct WeighParams {
  const uint16_t* q;      // [B, W, heads * gs, D]
  const uint16_t* key;    // [B, T, heads, D]
  int64_t qb, qt, qh, kb, kt, kh;
  const int32_t* lens;    // [B] or null: T each
  float* out;             // [B, heads, T]
  float* stats;           // [B * heads, S, cols_pad, 2] maximum (units of ln 2) and sum of the splits
  float2* norms;          // [B * heads, cols_pad]: a column's reference (units of ln 2) and the inverse of its sum
  float* part;            // [B * heads, supers, T] their sums
  int heads, gs, W, T, cols, cols_pad;
  int S;                  // splits of the keys in the first pass
  int rows;               // keys of a split of the pass
  int per, supers;        // blocks of columns to a workgroup of the second pass, workgroups to all
  int joined;             // whether norms is filled before the second pass
  float scale2;           // scale / ln 2
};

// A column's reference M and the inverse of its sum relative to M, of which a weight is exp(s - M) / sum, from its splits: this
// thread takes `part`, part + of, ...; `of` neighbouring lanes together.  (Not the log-sum-exp alone: rounded to 32 bits it shifts all
// weights of the column by up to half a unit of its size, 7e-7 of them, which is most of the error of a few queries' weights.)
// A column without keys: inf and 0, so that a score less inf weighs 0.  One whose sum is NaN: inf and NaN.
__device__ __forceinline__ float2 weigh_join(const WeighParams& P, int g, int col, int part, int of) {
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
  return L != L ? make_float2(INFINITY, L) : L != 0.f ? make_float2(M, 1.f / L) : make_float2(INFINITY, 0.f);
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
// a wave reads a piece of nor the loads, a row by a row's lanes, meet in a bank.  Load i of a wave: this lane's row
// of the tile and the byte offset of its piece in the row.
template <int D, int WAVES>
__device__ __forceinline__ int weigh_row(int wave, int i) {
  return (wave + i * WAVES) * (512 / D) + ((threadIdx.x & 63) / (D / 8));
}
template <int D, int WAVES>
__device__ __forceinline__ uint32_t weigh_piece(int wave, int i) {
  return (((threadIdx.x & 63) % (D / 8)) ^ (weigh_row<D, WAVES>(wave, i) % (D / 8))) << 4;
}

// The last key that the columns of part `super` of the second pass see.
__device__ __forceinline__ int weigh_last_key(const WeighParams& P, int n, int super, int block) {
  return n - P.W + min((super + 1) * P.per * block - 1, P.cols - 1) / P.gs;
}

// One pass over the keys [j0, j1) of a split of group blockIdx.x, of which the columns [32 wave, 32 wave + 32) of
// a block of 32 WAVES see some.
// SUM false: references and sums, of a block's columns as columns of the product;
// m and l of a lane: its reference and the sum of exponentials relative to it, over its own keys.  The reference is the maximum of
// the first tile that the column sees, and moves only where a tile's sum passes 2^100: until then neither the sums nor their
// precision suffer, and a score costs a product with its offset, an exponential and an addition.
// SUM true: the sums over the columns of `per` blocks, as rows of the product, so that the columns add
// up in the lane; the waves leave theirs in LDS, where one of them adds up a tile's behind the barrier that follows.
template <int D, bool HALF, bool SUM, int WAVES, int OCC>
__global__ __launch_bounds__(64 * WAVES, OCC) void weigh_kernel(WeighParams P) {
  constexpr int BLOCK = 32 * WAVES, LOADS = WG_TILE * D * 2 / (1024 * WAVES), KK = D / 16, EX = 16 / KK,   // EX: exponentials to a product
                RING = SUM && WAVES == 4 ? 2 : 4;   // operands read ahead (with 4 and the inverse sums 5 registers of the second pass spill: 334 us for 328)
  static_assert(KK % RING == 0, "a sub-tile's first operand is the ring's first");
  __shared__ __attribute__((aligned(16))) uint16_t sh[WG_BUFFERS][WG_TILE * D];
  __shared__ __attribute__((aligned(16))) float sh_ref[SUM ? BLOCK : 4], sh_inv[SUM ? BLOCK : 4];
  __shared__ float sh_part[SUM ? WG_BUFFERS : 1][SUM ? WAVES : 1][WG_TILE];
  // The last key that a column with a NaN for its sum sees, of the columns that a wave looks up.  The weights up to that key are made NaN
  // at the end; the column's own share is made 0, since the keys that it does not see have a share of every column, too.
  __shared__ int sh_nan[SUM ? WAVES / 2 : 1];
  extern __shared__ float sh_sum[];   // [rows], with several blocks
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x, b = g / P.heads, head = g - b * P.heads;
  const int n = weigh_len(P, b), first = n - P.W;                   // first: the first query's token
  const int blocks = (P.cols + BLOCK - 1) / BLOCK;
  const int super = gridDim.y - 1 - blockIdx.y;                     // (the columns that see most keys first)
  const int block0 = SUM ? super * P.per : super, block1 = SUM ? min(block0 + P.per, blocks) : block0 + 1;
  // (the second pass begins with the keys that the first ended with, which the memory-side cache may still hold)
  const int split = SUM ? gridDim.z - 1 - blockIdx.z : blockIdx.z;
  const int j0 = split * P.rows, jn = min(j0 + P.rows, n);
  const uint16_t* const keys = P.key + b * P.kb + head * P.kh;
  uint32_t at[LOADS];   // of this lane's piece of a tile's rows
#pragma unroll
  for (int i = 0; i < LOADS; ++i) at[i] = weigh_row<D, WAVES>(wave, i) * ((uint32_t)P.kt * 2) + weigh_piece<D, WAVES>(wave, i);
  const auto stage = [&](int t) {
    const int j = j0 + t * WG_TILE;
    const uint16_t* const from = keys + j * P.kt;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {   // (past the last key: that one)
      const uint32_t o = j + WG_TILE <= n ? at[i]
                                          : (uint32_t)min(weigh_row<D, WAVES>(wave, i), n - 1 - j) * ((uint32_t)P.kt * 2) + weigh_piece<D, WAVES>(wave, i);
      weigh_dma16(from, o, __builtin_amdgcn_readfirstlane(weigh_lds(sh[t % WG_BUFFERS]) + (wave + i * WAVES) * 1024));
    }
  };
  const uint16_t* operand_at[KK];   // operand kk of a tile's first 32 rows: row lane % 32, dims 16 kk + 8 (lane / 32) ..
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
    operand_at[kk] = &sh[0][(lane & 31) * D + (((2 * kk + (lane >> 5)) ^ (lane % (D / 8))) << 3)];
  float* const to = !SUM ? nullptr : P.supers > 1 ? P.part + ((size_t)g * P.supers + super) * P.T : P.out + (size_t)g * P.T;
  if (SUM && P.per > 1)
    for (int i = threadIdx.x; i < P.rows; i += 64 * WAVES) sh_sum[i] = 0.f;
  if (SUM && wave < WAVES / 2) sh_nan[SUM ? wave : 0] = -1;   // (a wave's own until the barrier behind its columns)
  float m = -INFINITY, l = 0.f;

  for (int block = block0; block < block1; ++block) {
    const int colw = block * BLOCK + wave * 32;
    const int j1 = min(jn, first + min(block * BLOCK + BLOCK - 1, P.cols - 1) / P.gs + 1);   // (the last key of the block)
    if (j0 >= j1) continue;
    const int tiles = (j1 - j0 + WG_TILE - 1) / WG_TILE, subs = (j1 - j0 + 31) / 32;
    // the first tile, the columns and what their sums were are requested together and waited for here, so that no wait for them
    // stands between those for the tiles
    stage(0);
    uint4 q[KK];
    f32x16_t off, inv;          // SUM: of the rows minus the reference, and the inverse sum
    const int col = min(colw + (lane & 31), P.cols - 1), qi = col / P.gs;
    const int low = first + min(colw, P.cols - 1) / P.gs, mine = first + qi;   // last keys of the tile's first and the lane's column
    const uint16_t* const from = P.q + b * P.qb + qi * P.qt + (head * P.gs + col - qi * P.gs) * P.qh + 8 * (lane >> 5);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) q[kk] = ri_ld16(from + 16 * kk);
    if (SUM) {   // the block's references and sums, joined from their splits where nobody has done so before
      if ((int)threadIdx.x < BLOCK) {
        const int col = block * BLOCK + threadIdx.x;
        const float2 x = P.joined ? P.norms[(size_t)g * P.cols_pad + col] : weigh_join(P, g, col, 0, 1);
        sh_ref[SUM ? threadIdx.x : 0] = x.x;
        sh_inv[SUM ? threadIdx.x : 0] = x.y != x.y ? 0.f : x.y;
        if (x.y != x.y) atomicMax(&sh_nan[SUM ? wave : 0], first + col / P.gs);
      }
      __syncthreads();
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float4 o = *reinterpret_cast<const float4*>(&sh_ref[wave * 32 + 8 * x + 4 * (lane >> 5)]);
        const float4 f = *reinterpret_cast<const float4*>(&sh_inv[wave * 32 + 8 * x + 4 * (lane >> 5)]);
        off[4 * x] = -o.x; off[4 * x + 1] = -o.y; off[4 * x + 2] = -o.z; off[4 * x + 3] = -o.w;
        inv[4 * x] = f.x; inv[4 * x + 1] = f.y; inv[4 * x + 2] = f.z; inv[4 * x + 3] = f.w;
      }
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) asm volatile("" : "+v"(q[kk].x), "+v"(q[kk].y), "+v"(q[kk].z), "+v"(q[kk].w));
    weigh_wait<0>();
    if (tiles > 1) stage(1);
    weigh_barrier();
    uint4 a[RING];
    const auto operand = [&](int buf, int sub, int kk) {
      return *reinterpret_cast<const uint4*>(operand_at[kk] + (buf * WG_TILE + sub * 32) * D);
    };
#pragma unroll
    for (int kk = 0; kk < RING; ++kk) a[kk] = operand(0, 0, kk);
    const f32x16_t zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    f32x16_t s;                 // the scores of the sub-tile before
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = -INFINITY;

    // keys from j on that a column does not see weigh nothing; the factor that the scores still want
    const auto mask = [&](int j) {
      if (j + 31 <= low) return P.scale2;
      int here = lane;
      asm volatile("" : "+v"(here));   // (what follows is rare: nothing of it is to be kept in registers for it)
      if (SUM) {
        const int key = j + (here & 31), i0 = colw / P.gs, o = colw - i0 * P.gs + 4 * (here >> 5);
        const uint32_t inv = 65536 / P.gs + 1;   // (exact for what is divided here: less than 48 by up to 16)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int last = first + i0 + (int)(((uint32_t)(o + 8 * (i >> 2) + (i & 3)) * inv) >> 16);
          s[i] = key > last ? -INFINITY : s[i] * P.scale2;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = j + weigh_key_of(i, here) > mine ? -INFINITY : s[i] * P.scale2;
      }
      return 1.f;
    };
    // the sum of a sub-tile's exponentials, to where it belongs
    const auto finish = [&](float sum, float scale2, int slot, int sub) {
      if (SUM) {
        sh_part[SUM ? slot : 0][SUM ? wave : 0][sub * 32 + (lane & 31)] = ri_xor_sum<32>(sum);
        return;
      }
      if (__builtin_amdgcn_ballot_w64(!(sum < 0x1p100f))) {
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, s[i] * scale2);
        const float mn = fmaxf(m, most), ref = mn == -INFINITY ? 0.f : mn;
        l *= __builtin_amdgcn_exp2f(m - ref);
        m = mn;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f(fmaf(s[i], scale2, -ref));
      }
      l += sum;
    };
    const auto add_tile = [&](int t) {   // (a tile is the same wave's in every block)
      if (wave == t % WAVES && t * WG_TILE + lane < subs * 32) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) x += sh_part[SUM ? t % WG_BUFFERS : 0][SUM ? w : 0][lane];
        if (P.per > 1) sh_sum[t * WG_TILE + lane] += x;
        else if (j0 + t * WG_TILE + lane < jn) to[j0 + t * WG_TILE + lane] = x;
      }
    };

    for (int t0 = 0; t0 < tiles; t0 += WG_BUFFERS) {
#pragma unroll
      for (int buf = 0; buf < WG_BUFFERS; ++buf) {   // (unrolled: the buffer is in the offset of every LDS access)
        const int t = t0 + buf;
        if (t >= tiles) break;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          const int u = 2 * t + sub;
          if (u >= subs) break;
          if (sub && t + 1 < tiles) {   // the operands read ahead are the next tile's; nobody reads the one before this any more
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (t + 2 < tiles) stage(t + 2);
            if (SUM && t) add_tile(t - 1);
          }
          // this sub-tile's product beside the exponentials of the one before
          const float scale2 = u ? mask(j0 + 32 * u - 32) : 1.f;
          f32x16_t p = zero;
          float sum = 0.f, x = 0.f, e[EX];
          const auto add = [&](int kk) {   // the products' kk; two sums, so that an addition does not wait for the one before
#pragma unroll
            for (int i = 0; i < EX; i += 2) {
              sum = SUM ? fmaf(e[i], inv[EX * kk + i], sum) : sum + e[i];
              x = SUM ? fmaf(e[i + 1], inv[EX * kk + i + 1], x) : x + e[i + 1];
            }
          };
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            uint4& from = a[kk % RING];
            p = SUM ? weigh_mfma<HALF>(q[kk], from, p) : weigh_mfma<HALF>(from, q[kk], p);
            from = kk + RING < KK ? operand(buf, sub, kk + RING)
                                  : sub ? operand((buf + 1) % WG_BUFFERS, 0, kk + RING - KK) : operand(buf, 1, kk + RING - KK);
            if (kk) add(kk - 1);
#pragma unroll
            for (int i = 0; i < EX; ++i)
              e[i] = __builtin_amdgcn_exp2f(fmaf(s[EX * kk + i], scale2, SUM ? off[EX * kk + i] : -m));
            // (the next product cannot move in front of these exponentials, nor they behind it)
#pragma unroll
            for (int i = 0; i < EX; i += 2) asm volatile("" : "+v"(e[i]), "+v"(e[i + 1]), "+v"(q[(kk + 1) % KK].x));
            __builtin_amdgcn_sched_barrier(0);
          }
          add(KK - 1);
          if (u) finish(sum + x, scale2, sub ? buf : (buf + WG_BUFFERS - 1) % WG_BUFFERS, sub ^ 1);
          s = p;
        }
      }
    }
    {
      const float scale2 = mask(j0 + 32 * subs - 32);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[i], scale2, SUM ? off[i] : -m));
        sum = SUM ? fmaf(e, inv[i], sum) : sum + e;
      }
      finish(sum, scale2, (tiles - 1) % WG_BUFFERS, (subs - 1) & 1);
    }
    if (SUM) {
      __syncthreads();
      if (tiles > 1) add_tile(tiles - 2);
      add_tile(tiles - 1);
      __syncthreads();
    }
  }

  if (SUM) {
    // (Where the part's columns see some of these keys a block was done, and a barrier stood behind it.)
    // Nobody reads what a part has of keys behind the last that its columns see; in the result those weigh nothing.
    const int seen = max(min(jn, weigh_last_key(P, n, super, BLOCK) + 1) - j0, 0), all = P.supers > 1 ? seen : min(P.rows, P.T - j0);
    for (int i = (P.per > 1 ? 0 : seen) + threadIdx.x; i < all; i += 64 * WAVES) to[j0 + i] = i < seen ? sh_sum[i] : 0.f;
    if (seen > 0) {
      int nan_key = -1;
#pragma unroll
      for (int w = 0; w < WAVES / 2; ++w) nan_key = max(nan_key, sh_nan[SUM ? w : 0]);
      for (int i = threadIdx.x; i < min(nan_key + 1, jn) - j0; i += 64 * WAVES) to[j0 + i] = NAN;
    }
    return;
  }
  const float M = ri_xor_max<32>(m);
  const float Z = ri_xor_sum<32>(m == -INFINITY ? l : l * __builtin_amdgcn_exp2f(m - M));
  if (lane < 32) {
    const int col = block0 * BLOCK + wave * 32 + lane;
    float* const to = P.stats + (((size_t)g * P.S + split) * P.cols_pad + col) * 2;
    to[0] = col < P.cols ? M : -INFINITY;
    to[1] = col < P.cols ? Z : 0.f;
  }
}

// Grid (cols_pad / 32, B * heads), 256 threads: eight threads join the splits of a column.
__global__ __launch_bounds__(256) void weigh_join_kernel(WeighParams P) {
  const int g = blockIdx.y, col = blockIdx.x * 32 + (threadIdx.x >> 3);
  const float2 x = weigh_join(P, g, col, threadIdx.x & 7, 8);
  if ((threadIdx.x & 7) == 0) P.norms[(size_t)g * P.cols_pad + col] = x;
}

// Grid (ceil(T / KEYS), B * heads): 256 / KEYS threads add the parts of a key, of those that have columns that see it, every
// so-many-th each.
template <int KEYS>
__global__ __launch_bounds__(256) void weigh_add_kernel(WeighParams P) {
  constexpr int OF = 256 / KEYS;
  __shared__ float sh[OF][KEYS];
  const int g = blockIdx.y, at = threadIdx.x % KEYS, mine = threadIdx.x / KEYS, j = blockIdx.x * KEYS + at, n = weigh_len(P, g / P.heads);
  float x = 0.f;
  if (j < n) {
    const float* const from = P.part + (size_t)g * P.supers * P.T + j;
    int s = max(j - (n - P.W), 0) * P.gs / (WG_SUM_COLS * P.per) + mine;
    for (; s + 7 * OF < P.supers; s += 8 * OF) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = from[(size_t)(s + i * OF) * P.T];
#pragma unroll
      for (int i = 0; i < 8; ++i) x += v[i];
    }
    for (; s < P.supers; s += OF) x += from[(size_t)s * P.T];
  }
  if (OF > 1) {
    sh[mine][at] = x;
    __syncthreads();
    if (mine) return;
#pragma unroll
    for (int i = 1; i < OF; ++i) x += sh[i][at];
  }
  if (j < P.T) P.out[(size_t)g * P.T + j] = x;
}

// ------------------------------------------------------------------------------------ host side
extern "C" size_t ri_attention_weights_workspace_bytes(int B, int heads, int gs, int W, int T) {
  if (B <= 0 || heads <= 0 || gs <= 0 || gs > 16 || W <= 0 || T < W || T > 1 << 24 || (int64_t)B * heads > 65535 ||
      (int64_t)W * gs > (int64_t)65535 * WG_SUM_COLS)   // (dimensions of grids)
    return 0;
  const WeighPlan p = weigh_plan((int64_t)B * heads, W * gs, T);
  return (size_t)B * heads * ((size_t)p.cols_pad * 2 * ((size_t)p.S + (p.joined ? 1 : 0)) + (p.supers > 1 ? (size_t)p.supers * T : 0)) * sizeof(float);
}

template <int D, bool HALF>
static void launch_weigh(WeighParams P, const WeighPlan& p, int groups, hipStream_t s) {
  // (Waves to a SIMD are what registers leave: four and three; two in either pass cost nothing, four in the second spill, 335 us for 328
  // of 8192 queries.  What bounds these passes is the clock that their power leaves.)
  weigh_kernel<D, HALF, false, WG_COLS / 32, 4><<<dim3(groups, P.cols_pad / WG_COLS, p.S), 2 * WG_COLS, 0, s>>>(P);
  if (P.joined) weigh_join_kernel<<<dim3(P.cols_pad / 32, groups), 256, 0, s>>>(P);
  P.rows = p.rows2;
  const dim3 grid(groups, p.supers, p.S2);
  if (p.wide) {
    weigh_kernel<D, HALF, true, WG_COLS / 32, 2><<<grid, 2 * WG_COLS, 0, s>>>(P);
  } else {
    weigh_kernel<D, HALF, true, WG_SUM_COLS / 32, 3><<<grid, 2 * WG_SUM_COLS, P.per > 1 ? P.rows * sizeof(float) : 0, s>>>(P);
    // (256 parts of 65536 sums: eight threads to one 9.8 us, one 16)
    if (P.supers >= 16) weigh_add_kernel<32><<<dim3((P.T + 31) / 32, groups), 256, 0, s>>>(P);
    else if (P.supers > 1) weigh_add_kernel<256><<<dim3((P.T + 255) / 256, groups), 256, 0, s>>>(P);
  }
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
  float* const norms = stats + (size_t)groups * p.cols_pad * 2 * p.S;
  const WeighParams P = {(const uint16_t*)q, (const uint16_t*)key, q_batch_stride, q_token_stride, q_head_stride, key_batch_stride,
                         key_token_stride, key_head_stride, seqlens, out, stats, (float2*)norms,
                         norms + (p.joined ? 2 * (size_t)groups * p.cols_pad : 0), heads, gs, W, T, cols, p.cols_pad, p.S, p.rows, p.per,
                         p.supers, p.joined, scale * WG_LOG2E};
  hipStream_t s = (hipStream_t)stream;
  if (dim == 64) half ? launch_weigh<64, true>(P, p, groups, s) : launch_weigh<64, false>(P, p, groups, s);
  else half ? launch_weigh<128, true>(P, p, groups, s) : launch_weigh<128, false>(P, p, groups, s);
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
