// The paged key-value cache (gfx950): a new token's attention over the pages, the append of a token, the write of a prompt.
//
// Row r of sequence b lies in page block_table[b, r / page_rows], at row r % page_rows of each of its heads' [page_rows, dim]
// pieces.  A table entry outside [0, pages) is a page that is not there: its rows are neither attended nor written.
#include <math.h>

#include "ri_common.h"

#define PG_WAVES 8             // waves of an attending workgroup
#define PG_ROWS_MIN 128        // rows of a workgroup at least: a chunk of 16 per wave
#define PG_LOG2E 1.4426950408889634f
#define PG_LN2 0.6931471805599453f

typedef short pg_s4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float pg_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

struct PagedView {
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* table;
  int64_t kp, kh, kr, vp, vh, vr, ts;   // strides in elements: page, head, row; of the table
  int pages, heads, shift, mask, table_pages;
};

struct PagedAttendParams {
  PagedView c;
  const uint16_t* q;      // [B, heads * gs, D]
  const int32_t* lens;    // [B]
  const int32_t* starts;  // [B] or null
  uint16_t* out;          // [B, heads * gs, D]
  float* lse;             // [B, heads * gs] or null
  float* scores;          // [B, heads, ..] or null
  int64_t sb, sh;         // its strides
  float* part_ml;         // [B * heads, S, GP, 2]: maximum (of scores in units of ln 2) and sum
  float* part_acc;        // [B * heads, S, GP, D]
  float* logits;          // [B * heads, gs, max_len], units of ln 2
  int gs, S, rows, max_len;   // rows: of a workgroup, a multiple of 16
  float scale2;           // scale / ln 2
};

// the attended rows [first, last) of sequence b
__device__ __forceinline__ void pg_range(const PagedAttendParams& P, int b, int* first, int* last) {
  *last = min(max(P.lens[b], 0), P.max_len);
  *first = P.starts ? min(max(P.starts[b], 0), *last) : 0;
}

template <bool HALF>
__device__ __forceinline__ f32x4_t pg_mfma32(uint4 a, uint4 b, f32x4_t c) {
  return HALF ? __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0)
              : __builtin_amdgcn_mfma_f32_16x16x32_bf16(ri_as_bf16x8(a), ri_as_bf16x8(b), c, 0, 0, 0);
}
template <bool HALF>
__device__ __forceinline__ f32x4_t pg_mfma16(pg_s4 a, pg_s4 b, f32x4_t c) {
  return HALF ? __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, a), __builtin_bit_cast(f16x4_t, b), c, 0, 0, 0)
              : __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
}

// maximum / sum over the 16 lanes of a row, in every lane
__device__ __forceinline__ float pg_row_max(float x) { return ri_xor_max<1>(ri_xor_max<2>(ri_xor_max<4>(ri_xor_max<8>(x)))); }
__device__ __forceinline__ float pg_row_sum(float x) { return ri_xor_sum<1>(ri_xor_sum<2>(ri_xor_sum<4>(ri_xor_sum<8>(x)))); }

// s = scale q.k, p = exp(s - m), out = sum p v / sum p over the rows of one (sequence, key-value head), one pass with the running
// maximum m.  Grid (B * heads, S): a workgroup has the `rows` rows from blockIdx.y * rows on, each of its waves a run of them in
// chunks of 16.  GP: query heads padded to 4, 8 or 16.  The products are MFMA 16x16x32 with the heads as rows of A (row m: head
// m % GP) and 16 cache rows as columns of B: lane (n, h) = (lane % 16, lane / 16) gets the scores of cache row n for the heads
// 4 h + i of A's rows, of which it keeps GP / 4, so that every (row, head) is some lane's once.
// UNI: a chunk lies in one page (pages of 16 rows and more), whose address is the same for the whole wave.
template <int D, int GP, bool HALF, bool UNI>
__global__ __launch_bounds__(64 * PG_WAVES, 4) void paged_attend_kernel(PagedAttendParams P) {
  constexpr int NH = GP / 4, DT = D / 16, KK = D / 32, VS = D + 16;
  constexpr int LPR = D / 8, RPI = 64 / LPR, NV = 16 / RPI;   // lanes to a value row, value rows to a load, loads to a chunk
  constexpr int TILE = (16 * VS * 2 > GP * D * 4) ? 16 * VS * 2 : GP * D * 4;
  __shared__ __attribute__((aligned(16))) char sh_tile[PG_WAVES][TILE];
  __shared__ __attribute__((aligned(16))) uint16_t sh_p[PG_WAVES][16 * 16];
  __shared__ __attribute__((aligned(16))) float sh_al[PG_WAVES][16];
  __shared__ float sh_m[PG_WAVES][GP], sh_l[PG_WAVES][GP];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, h = lane >> 4;
  const int g = blockIdx.x, split = blockIdx.y;
  const int b = g / P.c.heads, head = g - b * P.c.heads;
  int first, last;
  pg_range(P, b, &first, &last);
  const int w0 = max(split * P.rows, first & ~15), w1 = min((split + 1) * P.rows, last);
  if (P.S > 1 && w0 >= w1) return;   // (nothing of this workgroup is read)

  uint16_t* const vt = (uint16_t*)sh_tile[wave];
  uint16_t* const pb = sh_p[wave];
  float* const al_sh = sh_al[wave];
  reinterpret_cast<uint2*>(pb)[lane] = make_uint2(0u, 0u);
  if (lane < 16) al_sh[lane] = 1.f;

  const int hq = n % GP;
  uint4 q[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
    q[kk] = hq < P.gs ? ri_ld16(P.q + ((size_t)g * P.gs + hq) * D + kk * 32 + h * 8) : ri_zero16();

  float m[NH], l[NH];
  f32x4_t acc[DT];
#pragma unroll
  for (int i = 0; i < NH; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  const int rsel = GP == 4 ? h : (GP == 8 ? (h >> 1) * 2 : 0);   // first accumulator register that this lane keeps
  const auto head_of = [&](int i) { return (4 * h + rsel + i) % GP; };

  // this wave's chunks [c0, c1) of 16 rows
  const int chunks = (w1 - w0 + 15) >> 4, per = (max(chunks, 0) + PG_WAVES - 1) / PG_WAVES;
  const int c0 = (w0 >> 4) + min(chunks, wave * per), c1 = min(c0 + per, (w0 >> 4) + chunks);
  const int32_t* const table = P.c.table + b * P.c.ts;
  const uint16_t* const kb = P.c.k + head * P.c.kh;
  const uint16_t* const vb = P.c.v + head * P.c.vh;
  const int shift = P.c.shift, mask = P.c.mask;
  const int upc = UNI ? 1 : 16 >> shift;      // units, of which a lane holds the page, to a chunk
  const int ush = UNI ? 4 : shift;            // rows of a unit as a power of two
  const int cpb = 64 / upc;                   // chunks to a batch of 64 units

  for (int cb = c0; cb < c1; cb += cpb) {
    // lane's unit of this batch: its page, -1 where there is none
    int pid;
    {
      const int row = ((cb * upc) + lane) << ush;
      const int at = row >> shift;
      pid = row < w1 ? table[min(at, P.c.table_pages - 1)] : -1;
      if ((unsigned)pid >= (unsigned)P.c.pages) pid = -1;
    }
    const int ce = min(c1, cb + cpb);
    for (int c = cb; c < ce; ++c) {
      const int r0 = c << 4;
      uint4 k[KK], v[NV];
      int pk, pv[NV];
      if (UNI) {
        pk = __builtin_amdgcn_readlane(pid, c - cb);
#pragma unroll
        for (int i = 0; i < NV; ++i) pv[i] = pk;
      } else {
        pk = __shfl(pid, (c - cb) * upc + (n >> shift));
#pragma unroll
        for (int i = 0; i < NV; ++i) pv[i] = __shfl(pid, (c - cb) * upc + ((lane / LPR + RPI * i) >> shift));
      }
      const int rk = r0 + n;
      const bool valid = pk >= 0 && rk >= first && rk < last;
      const uint16_t* kp = kb + max(pk, 0) * P.c.kp + (rk & mask) * P.c.kr + h * 8;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) k[kk] = valid ? ri_ld16(kp + kk * 32) : ri_zero16();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int rv = r0 + lane / LPR + RPI * i;
        const bool ok = pv[i] >= 0 && rv >= first && rv < last;   // (rows that are not attended bring no NaN into the products)
        v[i] = ok ? ri_ld16(vb + max(pv[i], 0) * P.c.vp + (rv & mask) * P.c.vr + (lane % LPR) * 8) : ri_zero16();
      }
      f32x4_t s4 = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) s4 = pg_mfma32<HALF>(q[kk], k[kk], s4);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        *reinterpret_cast<uint4*>(vt + (lane / LPR + RPI * i) * VS + (lane % LPR) * 8) = v[i];
      float al[NH];
      bool rescale = false;
#pragma unroll
      for (int i = 0; i < NH; ++i) {
        const int r = GP == 16 ? i : rsel + i;
        const float x = r == 0 ? s4[0] : r == 1 ? s4[1] : r == 2 ? s4[2] : s4[3];
        const float s = valid ? x * P.scale2 : -INFINITY;
        if (P.logits && rk < w1 && head_of(i) < P.gs)
          P.logits[((size_t)g * P.gs + head_of(i)) * P.max_len + rk] = s;
        const float mn = fmaxf(m[i], pg_row_max(s));
        const bool none = mn == -INFINITY;   // relative to -inf they would weigh NaN
        al[i] = none ? 1.f : pg_exp2(m[i] - mn);
        const float p = pg_exp2(s - (none ? 0.f : mn));
        rescale |= al[i] != 1.f;
        l[i] = l[i] * al[i] + p;
        m[i] = mn;
        pb[head_of(i) * 16 + n] = ri_f32_to_e16<HALF>(p);
      }
      const bool any = __builtin_amdgcn_ballot_w64(rescale) != 0;
      if (any && n == 0) {
#pragma unroll
        for (int i = 0; i < NH; ++i) al_sh[head_of(i)] = al[i];
      }
      ri_wave_sync();
      if (any) {
        const float4 a4 = *reinterpret_cast<const float4*>(al_sh + 4 * h);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          acc[dt][0] *= a4.x; acc[dt][1] *= a4.y; acc[dt][2] *= a4.z; acc[dt][3] *= a4.w;
        }
      }
      // lane (n, h): P of head n and rows 4 h .., V of those rows and dim 16 dt + n by transpose reads
      const pg_s4 pa = *reinterpret_cast<const pg_s4*>(pb + n * 16 + 4 * h);
      const uint16_t* vsrc = vt + (4 * h + (n >> 2)) * VS + 4 * (n & 3);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const pg_s4 vv = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pg_s4 __attribute__((address_space(3)))*)(vsrc + 16 * dt));
        acc[dt] = pg_mfma16<HALF>(pa, vv, acc[dt]);
      }
      ri_wave_sync();
    }
  }

  // the waves merge in LDS
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const float s = pg_row_sum(l[i]);
    if (n == 0) {
      sh_m[wave][head_of(i)] = m[i];
      sh_l[wave][head_of(i)] = s;
    }
  }
  float* const mine = (float*)sh_tile[wave];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int hd = 4 * h + i;
    if (hd < GP) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) mine[hd * D + 16 * dt + n] = acc[dt][i];
    }
  }
  __syncthreads();
  for (int at = threadIdx.x; at < P.gs * D; at += 64 * PG_WAVES) {
    const int j = at / D, d = at % D;
    float M = -INFINITY, L = 0.f, A = 0.f;
#pragma unroll
    for (int w = 0; w < PG_WAVES; ++w) M = fmaxf(M, sh_m[w][j]);
#pragma unroll
    for (int w = 0; w < PG_WAVES; ++w) {
      const float f = sh_m[w][j] == -INFINITY ? 0.f : pg_exp2(sh_m[w][j] - M);
      L += sh_l[w][j] * f;
      A += ((const float*)sh_tile[w])[j * D + d] * f;
    }
    const size_t o = (size_t)g * P.gs + j, part = ((size_t)g * P.S + split) * GP + j;
    if (P.S == 1) {
      P.out[o * D + d] = ri_f32_to_e16<HALF>(L > 0.f ? A / L : 0.f);
      if (d == 0 && P.lse) P.lse[o] = L > 0.f ? (M + __log2f(L)) * PG_LN2 : -INFINITY;
    } else {
      P.part_acc[part * D + d] = A;
    }
    if (d == 0 && (P.S > 1 || P.logits)) {
      P.part_ml[2 * part] = M;
      P.part_ml[2 * part + 1] = L;
    }
  }
}

#define PG_JOIN_THREADS 256
#define PG_JOIN_ROWS 1024      // scores of a workgroup of the join

// Grid (B * heads, (S > 1 ? gs : 0) + ceil(max_len / PG_JOIN_ROWS) with scores): the first gs workgroups of a group join the
// parts of a head each; the others add the weights of PG_JOIN_ROWS rows, exp(s - lse) summed over the heads, to the scores.
template <int D, int GP, bool HALF>
__global__ __launch_bounds__(PG_JOIN_THREADS) void paged_join_kernel(PagedAttendParams P) {
  constexpr int PARTS = PG_JOIN_THREADS / D;
  __shared__ float sh_M[16], sh_L[16], sh_a[PARTS][D];
  const int g = blockIdx.x, b = g / P.c.heads, head = g - b * P.c.heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int first, last;
  pg_range(P, b, &first, &last);
  const int s0 = P.S > 1 ? first / P.rows : 0, s1 = P.S > 1 ? (last + P.rows - 1) / P.rows : 1;   // splits that have rows
  const int outs = P.S > 1 ? P.gs : 0;
  const bool joins = (int)blockIdx.y < outs;
  const float* const ml = P.part_ml + (size_t)g * P.S * GP * 2;
  for (int j = joins ? blockIdx.y + wave : wave; j < (joins ? (int)blockIdx.y + 1 : P.gs); j += PG_JOIN_THREADS / 64) {
    float M = -INFINITY, L = 0.f;
    if (first < last) {
      for (int s = s0 + lane; s < s1; s += 64) M = fmaxf(M, ml[((size_t)s * GP + j) * 2]);
      M = ri_wave_max(M);
      if (M != -INFINITY)
        for (int s = s0 + lane; s < s1; s += 64) L += ml[((size_t)s * GP + j) * 2 + 1] * pg_exp2(ml[((size_t)s * GP + j) * 2] - M);
      L = ri_wave_sum(L);
    }
    if (lane == 0) {
      sh_M[j] = M;
      sh_L[j] = L;
    }
  }
  __syncthreads();
  if (joins) {
    const int j = blockIdx.y, d = threadIdx.x % D, p = threadIdx.x / D;
    const float M = sh_M[j], L = sh_L[j];
    const float* const acc = P.part_acc + (size_t)g * P.S * GP * D;
    float A = 0.f;
    if (L > 0.f)
      for (int s = s0 + p; s < s1; s += PARTS) {
        const float ms = ml[((size_t)s * GP + j) * 2];
        A += acc[((size_t)s * GP + j) * D + d] * pg_exp2(ms - M);
      }
    sh_a[p][d] = A;
    __syncthreads();
    if (p == 0) {
      for (int i = 1; i < PARTS; ++i) A += sh_a[i][d];
      const size_t o = (size_t)g * P.gs + j;
      P.out[o * D + d] = ri_f32_to_e16<HALF>(L > 0.f ? A / L : 0.f);
      if (d == 0 && P.lse) P.lse[o] = L > 0.f ? (M + __log2f(L)) * PG_LN2 : -INFINITY;
    }
    return;
  }
  const int r0 = ((int)blockIdx.y - outs) * PG_JOIN_ROWS;
  float* const scores = P.scores + b * P.sb + head * P.sh;
  for (int r = r0 + threadIdx.x; r < min(r0 + PG_JOIN_ROWS, last); r += PG_JOIN_THREADS) {
    if (r < first) continue;
    float w = 0.f;
    for (int j = 0; j < P.gs; ++j) {
      const float x = P.logits[((size_t)g * P.gs + j) * P.max_len + r];
      w += sh_L[j] > 0.f ? pg_exp2(x - sh_M[j]) / sh_L[j] : 0.f;
    }
    scores[r] += w;
  }
}

// ------------------------------------------------------------------------------------ append
// A float's place in the order of the scores, -0 as 0, NaN behind everything else; 0xffffffff: a row that stays.
__device__ __forceinline__ uint32_t pg_order(float x) {
  if (x != x) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct PagedAppendParams {
  PagedView c;
  const uint16_t* key;    // [B, .., heads, D]
  const uint16_t* value;
  int64_t kb, kh, vb, vh;
  const int32_t* lens;
  int32_t* new_lens;
  float* scores;          // or null: then a full sequence takes no row
  int32_t* positions;
  int64_t sb, sh, pb, ph;
  const int32_t* token;   // [B] position of the token that comes
  int budget, sinks, recent, dim;
};

#define PG_APPEND_THREADS 512

// Grid (heads, B).
__global__ __launch_bounds__(PG_APPEND_THREADS) void paged_append_kernel(PagedAppendParams P) {
  __shared__ unsigned long long sh_best[PG_APPEND_THREADS / 64];
  const int head = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int held = min(max(P.lens[b], 0), P.budget);
  const int token = P.token ? P.token[b] : 0;
  int row = held;
  if (threadIdx.x == 0 && head == 0 && P.new_lens) P.new_lens[b] = min(held + 1, P.budget);
  float* const scores = P.scores ? P.scores + b * P.sb + head * P.sh : nullptr;
  int32_t* const positions = P.positions ? P.positions + b * P.pb + head * P.ph : nullptr;
  if (held == P.budget) {
    if (!scores) return;
    unsigned long long best = ~0ull;
    for (int r = threadIdx.x; r < held; r += PG_APPEND_THREADS) {
      const int at = positions[r];
      const bool stays = at < P.sinks || at > (int64_t)token - P.recent;
      const unsigned long long mine = (unsigned long long)(stays ? 0xffffffffu : pg_order(scores[r])) << 32 | (uint32_t)r;
      best = mine < best ? mine : best;
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      const unsigned long long other = __shfl_xor(best, d);
      best = other < best ? other : best;
    }
    if (lane == 0) sh_best[wave] = best;
    __syncthreads();
    best = sh_best[0];
    for (int w = 1; w < PG_APPEND_THREADS / 64; ++w) best = sh_best[w] < best ? sh_best[w] : best;
    row = (int)(uint32_t)best;
  }
  const int page = P.c.table[b * P.c.ts + (row >> P.c.shift)];
  if ((unsigned)page >= (unsigned)P.c.pages) return;
  const int pieces = P.dim / 8;
  if ((int)threadIdx.x < 2 * pieces) {
    const bool isv = (int)threadIdx.x >= pieces;
    const int piece = (threadIdx.x - (isv ? pieces : 0)) * 8, at = row & P.c.mask;
    const uint16_t* src = isv ? P.value + b * P.vb + head * P.vh : P.key + b * P.kb + head * P.kh;
    uint16_t* dst = const_cast<uint16_t*>(isv ? P.c.v + page * P.c.vp + head * P.c.vh + at * P.c.vr
                                              : P.c.k + page * P.c.kp + head * P.c.kh + at * P.c.kr);
    *reinterpret_cast<uint4*>(dst + piece) = ri_ld16(src + piece);
  }
  if (threadIdx.x == 0) {
    if (scores) scores[row] = 0.f;
    if (positions) positions[row] = token;
  }
}

// ------------------------------------------------------------------------------------ fill
struct PagedFillParams {
  PagedView c;
  const uint16_t* key;    // [B, T, heads, D]
  const uint16_t* value;
  int64_t kb, kt, kh, vb, vt, vh;
  const int32_t* lens;    // [B] or null: T each
  const float* weights;   // [B, heads, T] or null
  int64_t wb, wh;
  int32_t* new_lens;
  float* scores;
  int32_t* positions;
  int64_t sb, sh, pb, ph;
  int32_t* kept;          // [B * heads, budget]: the kept rows in order
  int T, budget, sinks, recent, dim;
};

__device__ __forceinline__ int pg_prompt(const PagedFillParams& P, int b) { return P.lens ? min(max(P.lens[b], 0), P.T) : P.T; }

#define PG_SEL_THREADS 1024

// The rows of a prompt that are kept, in order, with their weights and positions: the `sinks` first, the `recent` last and of the
// others those with the highest weights, at equal weights the first ones.  Grid (heads, B); a radix selection of the lowest kept
// weight (digits of 11, 11 and 10 bits), then one pass that lists.
__global__ __launch_bounds__(PG_SEL_THREADS) void paged_select_kernel(PagedFillParams P) {
  constexpr int NW = PG_SEL_THREADS / 64;
  __shared__ int hist[2048];
  __shared__ int sh_scan[NW], sh_pick[2], sh_tot[2][NW];
  const int head = blockIdx.x, b = blockIdx.y, n = pg_prompt(P, b);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* const w = P.weights ? P.weights + b * P.wb + head * P.wh : nullptr;
  float* const scores = P.scores ? P.scores + b * P.sb + head * P.sh : nullptr;
  int32_t* const positions = P.positions ? P.positions + b * P.pb + head * P.ph : nullptr;
  if (n <= P.budget) {
    for (int r = threadIdx.x; r < n; r += PG_SEL_THREADS) {
      if (scores) scores[r] = w[r];
      if (positions) positions[r] = r;
    }
    return;
  }
  const auto order_of = [&](int r) {
    return r < P.sinks || r >= n - P.recent ? 0xffffffffu : pg_order(w[r]);
  };
  uint32_t prefix = 0, known = 0;   // bits of the lowest kept order found so far
  int need = P.budget;              // of the rows whose bits agree, the highest `need` are kept
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    for (int i = threadIdx.x; i < 2048; i += PG_SEL_THREADS) hist[i] = 0;
    __syncthreads();
    for (int r = threadIdx.x; r < n; r += PG_SEL_THREADS) {
      const uint32_t o = order_of(r);
      if ((o & known) == prefix) atomicAdd(&hist[(o >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    // the bin from the top in which the count reaches `need`: thread t has bins 2 t and 2 t + 1 from the top
    const int top = bins - 1 - 2 * (int)threadIdx.x;
    const int a = top >= 0 ? hist[top] : 0, c = top >= 1 ? hist[top - 1] : 0;
    const int incl = (int)ri_wave_incl_scan((uint32_t)(a + c));
    if (lane == 63) sh_scan[wave] = incl;
    __syncthreads();
    int before = incl - a - c;
    for (int i = 0; i < wave; ++i) before += sh_scan[i];
    if (before < need && before + a + c >= need) {
      const bool second = before + a < need;
      sh_pick[0] = second ? top - 1 : top;
      sh_pick[1] = need - before - (second ? a : 0);
    }
    __syncthreads();
    prefix |= (uint32_t)sh_pick[0] << shift;
    known |= (uint32_t)(bins - 1) << shift;
    need = sh_pick[1];
    __syncthreads();
  }
  // rows above the found order are kept, and the first `need` of those at it
  int32_t* const kept = P.kept + ((size_t)b * P.c.heads + head) * P.budget;
  int base = 0, ties = 0;
  for (int r0 = 0; r0 < n; r0 += PG_SEL_THREADS) {
    const int r = r0 + threadIdx.x;
    const uint32_t o = r < n ? order_of(r) : 0u;
    const bool above = r < n && o > prefix, equal = r < n && o == prefix;
    const uint64_t ma = __ballot(above), me = __ballot(equal), below = (1ull << lane) - 1;
    if (lane == 0) {
      sh_tot[0][wave] = __popcll(ma);
      sh_tot[1][wave] = __popcll(me);
    }
    __syncthreads();
    int na = 0, ne = 0, ta = 0, te = 0;
    for (int i = 0; i < NW; ++i) {
      if (i < wave) { na += sh_tot[0][i]; ne += sh_tot[1][i]; }
      ta += sh_tot[0][i];
      te += sh_tot[1][i];
    }
    na += __popcll(ma & below);
    ne += __popcll(me & below) + ties;       // ties in front of this row
    const int at = base + na + min(ne, need) - min(ties, need);
    if (above || (equal && ne < need)) {
      kept[at] = r;
      if (scores) scores[at] = w[r];
      if (positions) positions[at] = r;
    }
    base += ta + min(ties + te, need) - min(ties, need);
    ties += te;
    __syncthreads();
  }
}

// Grid (ceil(rows / rows per workgroup), heads, B): the kept rows into their pages, a row by dim / 8 lanes.
__global__ __launch_bounds__(256) void paged_copy_kernel(PagedFillParams P) {
  const int head = blockIdx.y, b = blockIdx.z, n = pg_prompt(P, b), rows = min(n, P.budget);
  const int pieces = P.dim / 8, per = 256 / pieces;
  if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0 && P.new_lens) P.new_lens[b] = rows;
  const int row = blockIdx.x * per + threadIdx.x / pieces, piece = (threadIdx.x % pieces) * 8;
  if (row >= rows) return;
  const int src = n > P.budget ? P.kept[((size_t)b * P.c.heads + head) * P.budget + row] : row;
  const int page = P.c.table[b * P.c.ts + (row >> P.c.shift)], at = row & P.c.mask;
  if ((unsigned)page >= (unsigned)P.c.pages) return;
  *reinterpret_cast<uint4*>(const_cast<uint16_t*>(P.c.k) + page * P.c.kp + head * P.c.kh + at * P.c.kr + piece) =
      ri_ld16(P.key + b * P.kb + src * P.kt + head * P.kh + piece);
  *reinterpret_cast<uint4*>(const_cast<uint16_t*>(P.c.v) + page * P.c.vp + head * P.c.vh + at * P.c.vr + piece) =
      ri_ld16(P.value + b * P.vb + src * P.vt + head * P.vh + piece);
}

// ------------------------------------------------------------------------------------ host side
#define PG_MAX_ROWS (1 << 24)   // rows of a sequence
static bool strides_ok(int64_t a, int64_t b, int64_t c = 0) { return a >= 0 && b >= 0 && c >= 0 && (a | b | c) % 8 == 0; }

static int paged_view(const ri_paged_t* c, int B, PagedView* v) {
  if (!c || !c->k_pages || !c->v_pages || !c->block_table || ri_any_misaligned16(c->k_pages, c->v_pages)) return RI_ERR_ARG;
  if (c->pages <= 0 || c->heads <= 0 || c->table_pages <= 0 || B <= 0 || c->table_stride < 0) return RI_ERR_ARG;
  if (c->dim != 64 && c->dim != 128) return RI_ERR_ARG;
  if (c->page_rows <= 0 || (c->page_rows & (c->page_rows - 1)) || (int64_t)c->table_pages * c->page_rows > PG_MAX_ROWS)
    return RI_ERR_ARG;
  if (!strides_ok(c->k_page_stride, c->k_head_stride, c->k_row_stride) || !strides_ok(c->v_page_stride, c->v_head_stride, c->v_row_stride))
    return RI_ERR_ARG;
  if (c->heads > 65535 || B > 65535) return RI_ERR_ARG;   // (dimensions of grids)
  *v = {(const uint16_t*)c->k_pages, (const uint16_t*)c->v_pages, c->block_table, c->k_page_stride, c->k_head_stride, c->k_row_stride,
        c->v_page_stride, c->v_head_stride, c->v_row_stride, c->table_stride, c->pages, c->heads, __builtin_ctz(c->page_rows),
        c->page_rows - 1, c->table_pages};
  return RI_OK;
}

static int pg_pad(int gs) { return gs <= 4 ? 4 : gs <= 8 ? 8 : 16; }

// Rows of a workgroup: enough workgroups for the compute units, at least a chunk to a wave.
static int paged_rows(int64_t groups, int max_len) {
  const int64_t want = (groups * max_len + 1023) / 1024;
  const int64_t rows = (want + PG_ROWS_MIN - 1) / PG_ROWS_MIN * PG_ROWS_MIN;
  return (int)(rows < 512 ? 512 : rows);
}

extern "C" size_t ri_paged_attention_workspace_bytes(int B, int heads, int gs, int dim, int max_len, int scored) {
  if (B <= 0 || heads <= 0 || gs <= 0 || gs > 16 || max_len <= 0 || (dim != 64 && dim != 128)) return 0;
  const size_t groups = (size_t)B * heads, S = ((size_t)max_len + paged_rows(groups, max_len) - 1) / paged_rows(groups, max_len);
  return groups * S * pg_pad(gs) * (2 + dim) * sizeof(float) + (scored ? groups * gs * max_len * sizeof(float) : 0);
}

template <int D, int GP, bool HALF>
static void launch_paged(const PagedAttendParams& P, int groups, hipStream_t s) {
  auto* kernel = P.c.shift >= 4 ? paged_attend_kernel<D, GP, HALF, true> : paged_attend_kernel<D, GP, HALF, false>;
  kernel<<<dim3(groups, P.S), 64 * PG_WAVES, 0, s>>>(P);
  const int y = (P.S > 1 ? P.gs : 0) + (P.scores ? (P.max_len + PG_JOIN_ROWS - 1) / PG_JOIN_ROWS : 0);
  if (y) paged_join_kernel<D, GP, HALF><<<dim3(groups, y), PG_JOIN_THREADS, 0, s>>>(P);
}

template <int D, bool HALF>
static void launch_paged_gp(const PagedAttendParams& P, int groups, hipStream_t s) {
  switch (pg_pad(P.gs)) {
    case 4: return launch_paged<D, 4, HALF>(P, groups, s);
    case 8: return launch_paged<D, 8, HALF>(P, groups, s);
    default: return launch_paged<D, 16, HALF>(P, groups, s);
  }
}

extern "C" int ri_paged_attention(const ri_paged_t* cache, const void* q, const int32_t* lens, const int32_t* starts, float* scores,
                                  int64_t score_batch_stride, int64_t score_head_stride, void* out, float* lse_out, int B, int gs,
                                  int max_len, float scale, void* workspace, size_t workspace_bytes, ri_stream_t stream) {
  PagedAttendParams P = {};
  if (const int rc = paged_view(cache, B, &P.c)) return rc;
  if (!q || !lens || !out || !workspace || ri_any_misaligned16(q, out, workspace)) return RI_ERR_ARG;
  const int64_t groups = (int64_t)B * cache->heads;
  if (gs <= 0 || gs > 16 || max_len <= 0 || max_len > cache->table_pages * cache->page_rows || groups > INT32_MAX / 16) return RI_ERR_ARG;
  if (scores && (score_batch_stride < 0 || score_head_stride < max_len)) return RI_ERR_ARG;
  if (workspace_bytes < ri_paged_attention_workspace_bytes(B, cache->heads, gs, cache->dim, max_len, scores != nullptr))
    return RI_ERR_WORKSPACE;
  P.q = (const uint16_t*)q;
  P.lens = lens;
  P.starts = starts;
  P.out = (uint16_t*)out;
  P.lse = lse_out;
  P.scores = scores;
  P.sb = score_batch_stride;
  P.sh = score_head_stride;
  P.gs = gs;
  P.max_len = max_len;
  P.rows = paged_rows(groups, max_len);
  P.S = (max_len + P.rows - 1) / P.rows;
  P.scale2 = scale * PG_LOG2E;
  const size_t parts = (size_t)groups * P.S * pg_pad(gs);
  P.part_ml = (float*)workspace;
  P.part_acc = P.part_ml + 2 * parts;
  P.logits = scores ? P.part_acc + parts * cache->dim : nullptr;
  hipStream_t s = (hipStream_t)stream;
  if (cache->dim == 64) cache->half ? launch_paged_gp<64, true>(P, groups, s) : launch_paged_gp<64, false>(P, groups, s);
  else cache->half ? launch_paged_gp<128, true>(P, groups, s) : launch_paged_gp<128, false>(P, groups, s);
  RI_HIP_CHECK_LAUNCH();
  return RI_OK;
}

extern "C" int ri_paged_append(const ri_paged_t* cache, const void* key, const void* value, int64_t key_batch_stride,
                               int64_t key_head_stride, int64_t value_batch_stride, int64_t value_head_stride, const int32_t* lens,
                               int32_t* new_lens, float* scores, int64_t score_batch_stride, int64_t score_head_stride,
                               int32_t* positions, int64_t position_batch_stride, int64_t position_head_stride,
                               const int32_t* token_positions, int B, int budget, int sinks, int recent, ri_stream_t stream) {
  PagedAppendParams P = {};
  if (const int rc = paged_view(cache, B, &P.c)) return rc;
  if (!key || !value || !lens || lens == new_lens || ri_any_misaligned16(key, value)) return RI_ERR_ARG;
  if (!strides_ok(key_batch_stride, key_head_stride) || !strides_ok(value_batch_stride, value_head_stride)) return RI_ERR_ARG;
  if (budget <= 0 || budget > cache->table_pages * cache->page_rows || sinks < 0 || recent < 0 || (int64_t)sinks + recent >= budget)
    return RI_ERR_ARG;
  if (scores && (!positions || score_head_stride < budget || score_batch_stride < 0)) return RI_ERR_ARG;
  if (positions && (!token_positions || position_head_stride < budget || position_batch_stride < 0)) return RI_ERR_ARG;
  P.key = (const uint16_t*)key;
  P.value = (const uint16_t*)value;
  P.kb = key_batch_stride; P.kh = key_head_stride; P.vb = value_batch_stride; P.vh = value_head_stride;
  P.lens = lens;
  P.new_lens = new_lens;
  P.scores = scores;
  P.positions = positions;
  P.sb = score_batch_stride; P.sh = score_head_stride; P.pb = position_batch_stride; P.ph = position_head_stride;
  P.token = token_positions;
  P.budget = budget; P.sinks = sinks; P.recent = recent; P.dim = cache->dim;
  paged_append_kernel<<<dim3(cache->heads, B), PG_APPEND_THREADS, 0, (hipStream_t)stream>>>(P);
  RI_HIP_CHECK_LAUNCH();
  return RI_OK;
}

extern "C" size_t ri_paged_fill_workspace_bytes(int B, int heads, int T, int budget) {
  return B <= 0 || heads <= 0 || T <= budget || budget <= 0 ? 0 : (size_t)B * heads * budget * sizeof(int32_t);
}

extern "C" int ri_paged_fill(const ri_paged_t* cache, const void* key, const void* value, int64_t key_batch_stride,
                             int64_t key_token_stride, int64_t key_head_stride, int64_t value_batch_stride,
                             int64_t value_token_stride, int64_t value_head_stride, const int32_t* seqlens, const float* weights,
                             int64_t weight_batch_stride, int64_t weight_head_stride, int32_t* new_lens, float* scores,
                             int64_t score_batch_stride, int64_t score_head_stride, int32_t* positions,
                             int64_t position_batch_stride, int64_t position_head_stride, int B, int T, int budget, int sinks,
                             int recent, void* workspace, size_t workspace_bytes, ri_stream_t stream) {
  PagedFillParams P = {};
  if (const int rc = paged_view(cache, B, &P.c)) return rc;
  if (!key || !value || ri_any_misaligned16(key, value)) return RI_ERR_ARG;
  if (!strides_ok(key_batch_stride, key_token_stride, key_head_stride) || !strides_ok(value_batch_stride, value_token_stride, value_head_stride))
    return RI_ERR_ARG;
  if (T <= 0 || T > PG_MAX_ROWS || budget <= 0 || budget > cache->table_pages * cache->page_rows || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return RI_ERR_ARG;
  const int room = T < budget ? T : budget;
  if ((T > budget || scores) && !weights) return RI_ERR_ARG;
  if (weights && (weight_head_stride < T || weight_batch_stride < 0)) return RI_ERR_ARG;
  if (scores && (score_head_stride < room || score_batch_stride < 0)) return RI_ERR_ARG;
  if (positions && (position_head_stride < room || position_batch_stride < 0)) return RI_ERR_ARG;
  const size_t need = ri_paged_fill_workspace_bytes(B, cache->heads, T, budget);
  if (need && (!workspace || ri_misaligned16(workspace) || workspace_bytes < need)) return workspace ? RI_ERR_WORKSPACE : RI_ERR_ARG;
  P.key = (const uint16_t*)key;
  P.value = (const uint16_t*)value;
  P.kb = key_batch_stride; P.kt = key_token_stride; P.kh = key_head_stride;
  P.vb = value_batch_stride; P.vt = value_token_stride; P.vh = value_head_stride;
  P.lens = seqlens;
  P.weights = weights;
  P.wb = weight_batch_stride; P.wh = weight_head_stride;
  P.new_lens = new_lens;
  P.scores = scores;
  P.positions = positions;
  P.sb = score_batch_stride; P.sh = score_head_stride; P.pb = position_batch_stride; P.ph = position_head_stride;
  P.kept = (int32_t*)workspace;
  P.T = T; P.budget = budget; P.sinks = sinks; P.recent = recent; P.dim = cache->dim;
  hipStream_t s = (hipStream_t)stream;
  if (T > budget || scores || positions) paged_select_kernel<<<dim3(cache->heads, B), PG_SEL_THREADS, 0, s>>>(P);
  const int per = 256 / (cache->dim / 8);
  paged_copy_kernel<<<dim3((room + per - 1) / per, cache->heads, B), 256, 0, s>>>(P);
  RI_HIP_CHECK_LAUNCH();
  return RI_OK;
}
