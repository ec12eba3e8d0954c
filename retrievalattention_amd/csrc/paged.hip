// The paged key-value cache (gfx950): a new token's attention over the pages, the append of a token, the write of a prompt.
//
// Row r of sequence b lies in page block_table[b, r / page_rows], at row r % page_rows of each of its heads' [page_rows, dim]
// pieces.  A table entry outside [0, pages) is a page that is not there: its rows are neither attended nor written.
#include <math.h>

#include <type_traits>

#include "paged_plan.h"
#include "ri_common.h"

#define PG_LOG2E 1.4426950408889634f
#define PG_LN2 0.6931471805599453f

typedef short pg_s4 __attribute__((ext_vector_type(4)));
// four values, a row each, that need not be aligned to more than one
typedef float pg_f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef int pg_i4 __attribute__((ext_vector_type(4), aligned(4)));

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
  float* part_ml;         // [workgroups + B * heads, GP, 2]: maximum (of scores in units of ln 2) and sum of a part
  float* part_acc;        // [workgroups + B * heads, GP, D]
  int2* shares;           // [B * heads]: the workgroups that have a group's first and its last chunk
  float* logits;          // [B * heads, max_len, GP], units of ln 2, with scores
  int B, gs, max_len;
  int workgroups;         // that share the rows; 0: one to each group, which writes the output
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

// A probability p in [0, 1] as two elements, of which the first is below it and the second is what is left, rounded: their sum is within
// 2^-16 of p (bfloat16) or 2^-22 (half) relative to it, where one element is within 2^-8 or 2^-11: with one, 6 to 30 % of the outputs
// were not the exact result rounded, with two 0 to 0.3 % (fp32 throughout: 0 to 0.5 %).  It costs 0 to 2 %, since both parts fill
// one product of 32 where one filled a product of 16 (us, one part and two: four sequences of 131072 tokens, 8 heads of 4, 324 and 324; 32
// of 4096 with scores 98.7 and 98.9; one of 331 7.7 and 7.8; 256 of 400, 8 heads of 16, 88.7 and 90.4).
// Halves are of 2^15 p: their smallest normal number is 2^-14, and the weights of a long cache's rows are below it.  Both parts are
// above 0 as long as an element holds them, so that an infinite value stays one.
template <bool HALF>
__device__ __forceinline__ void pg_split(float p, uint16_t* first, uint16_t* left) {
  const float x = HALF ? p * 32768.f : p;
  const uint32_t below = max(__float_as_uint(x), 1u) - 1;   // (0 stays 0)
  if (HALF) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(__uint_as_float(below), 0.f);
    *first = __builtin_bit_cast(uint16_t, h[0]);
    *left = ri_f32_to_e16<HALF>(x - (float)h[0]);
  } else {
    *first = (uint16_t)(below >> 16);
    *left = ri_f32_to_e16<HALF>(x - __uint_as_float(below & 0xffff0000u));
  }
}

// What a part's sums weigh relative to the maximum M of all.  A part without rows and one whose scores are all NaN have no maximum: its
// own sum, 0 or NaN, stands in, so that a NaN arrives.
__device__ __forceinline__ float pg_weigh_part(float m, float l, float M) { return m == -INFINITY ? l : pg_exp2(m - M); }

// maximum / sum over the 16 lanes of a row, in every lane
__device__ __forceinline__ float pg_row_max(float x) { return ri_xor_max<1>(ri_xor_max<2>(ri_xor_max<4>(ri_xor_max<8>(x)))); }
__device__ __forceinline__ float pg_row_sum(float x) { return ri_xor_sum<1>(ri_xor_sum<2>(ri_xor_sum<4>(ri_xor_sum<8>(x)))); }

// places of a group of sequence b
__device__ __forceinline__ int pg_places(const PagedAttendParams& P, int b) {
  int first, last;
  pg_range(P, b, &first, &last);
  return first < last ? ((last + 15) >> 4) - (first >> 4) + PG_LEAD : 0;
}
struct PagedRun {
  int64_t each, total;   // places of a workgroup's share and of all groups
  int64_t from;          // those of one head in front of sequence b's
  int b;
};
// sixteen bytes that are read once: a load that leaves the caches to others
__device__ __forceinline__ uint4 pg_once16(const void* p) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load((const words*)p));
}
template <int N>
struct alignas(4 * N) pg_heads { float x[N]; };
// x, from which nothing that the compiler knows is to be kept in registers over what stands before
__device__ __forceinline__ int pg_anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ int64_t pg_uniform(int64_t x) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) | (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}
// Whole workgroup: the run, and the sequence that has this workgroup's first place (B where the run is shorter).
template <int THREADS>
__device__ __forceinline__ PagedRun pg_run(const PagedAttendParams& P) {
  constexpr int NW = THREADS / 64;
  __shared__ uint32_t sh_wave[NW];
  __shared__ int64_t sh_from;
  __shared__ int sh_b;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool one = P.B <= THREADS;
  const int64_t heads = P.c.heads;
  int64_t sum = 0, each = 0;
  if (threadIdx.x == 0) { sh_b = P.B; sh_from = 0; }
  for (int pass = one ? 1 : 0; pass < 2; ++pass) {   // the sum first; of few sequences everything at once
    int64_t in_front = 0;
    for (int b0 = 0; b0 < P.B; b0 += THREADS) {
      const int b = b0 + (int)threadIdx.x, n = b < P.B ? pg_places(P, b) : 0;
      const uint32_t incl = ri_wave_incl_scan((uint32_t)n);
      __syncthreads();
      if (lane == 63) sh_wave[wave] = incl;
      __syncthreads();
      uint32_t before = incl - n, all = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const uint32_t x = sh_wave[i];
        before += i < wave ? x : 0u;
        all += x;
      }
      if (one) sum = all;
      if (pass) {
        each = pg_each(sum * heads, P.workgroups);
        const int64_t from = in_front + before, place = blockIdx.x * each;
        if (from * heads <= place && place < (from + n) * heads) {
          sh_from = from;
          sh_b = b;
        }
      }
      in_front += all;
    }
    sum = in_front;
  }
  __syncthreads();
  return {pg_uniform(each), pg_uniform(sum * heads), pg_uniform(sh_from), __builtin_amdgcn_readfirstlane(sh_b)};
}

// s = scale q.k, p = exp(s - m), out = sum p v / sum p over the rows of one (sequence, key-value head), one pass with the running
// maximum m.  Each of a workgroup's waves takes a run of its chunks of 16 rows.  GP: query heads padded to 4, 8 or 16.  The products
// are MFMA 16x16x32 with the heads as rows of A (row m: head m % GP) and 16 cache rows as columns of B: lane (n, h) = (lane % 16,
// lane / 16) gets the scores of cache row n for the heads 4 h + i of A's rows, of which it keeps GP / 4, so that every (row, head) is
// some lane's once.
// UNI: a chunk lies in one page (pages of 16 rows and more), whose address is the same for the whole wave.  Four waves to a SIMD where
// that spills nothing: four sequences of 16384 tokens in pages of 8 rows 51 us with two, 57 with four, in pages of 16 50 and 47; 64 of 500
// 25.8 and 23.3.
template <int D, int GP, bool HALF, bool UNI>
__global__ __launch_bounds__(64 * PG_WAVES, UNI && GP < 16 ? 4 : 2) void paged_attend_kernel(PagedAttendParams P) {
  constexpr int NH = GP / 4, DT = D / 16, KK = D / 32, VS = D + 16;
  constexpr int LPR = D / 8, RPI = 64 / LPR, NV = 16 / RPI;   // lanes to a value row, value rows to a load, loads to a chunk
  constexpr int TILE = (16 * VS * 2 > GP * D * 4) ? 16 * VS * 2 : GP * D * 4;
  __shared__ __attribute__((aligned(16))) char sh_tile[PG_WAVES][TILE];
  __shared__ __attribute__((aligned(16))) uint16_t sh_p[PG_WAVES][16 * 32];   // a head's: of rows 4 h .. the first parts, then what is left
  __shared__ __attribute__((aligned(16))) float sh_al[PG_WAVES][16];
  __shared__ float sh_m[PG_WAVES][GP], sh_l[PG_WAVES][GP];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int b = blockIdx.x / P.c.heads, head = blockIdx.x - b * P.c.heads, skip = 0;   // skip: places of the group that are others'
  int64_t at = 0, end = 0;        // this workgroup's places of the run that are still to be done
  if (P.workgroups) {
    const int64_t heads = P.c.heads;
    const PagedRun run = pg_run<64 * PG_WAVES>(P);
    at = blockIdx.x * run.each;
    if (at >= run.total) return;
    end = min(at + run.each, run.total);
    b = run.b;
    if (b >= P.B) return;
    // (Here and below, what is read a second time may have been written meanwhile, by a caller who did not wait for it: the result is
    // undefined then, but no index leaves its buffer and every walk ends.)
    const int mine = (int)(at - run.from * heads), per_head = max(pg_places(P, b), 1);
    head = mine / per_head;
    if (head >= P.c.heads) return;
    skip = mine - head * per_head;
  }

  uint16_t* const vt = (uint16_t*)sh_tile[wave];
  uint16_t* const pb = sh_p[wave];
  float* const al_sh = sh_al[wave];
  reinterpret_cast<uint4*>(pb)[threadIdx.x & 63] = ri_zero16();
  if ((threadIdx.x & 63) < 16) al_sh[threadIdx.x & 63] = 1.f;
  const int shift = P.c.shift, mask = P.c.mask;
  const int upc = UNI ? 1 : 16 >> shift;      // units, of which a lane holds the page, to a chunk
  const int cpb = 64 / upc;                   // chunks to a batch of 64 units

  for (;;) {   // the groups that this workgroup has rows of
  const int lane = pg_anew(threadIdx.x & 63), n = lane & 15, h = lane >> 4;
  const int hq = n % GP, rsel = GP == 4 ? h : (GP == 8 ? (h >> 1) * 2 : 0);   // rsel: first accumulator register that this lane keeps
  const auto head_of = [&](int i) { return (4 * h + rsel + i) % GP; };
  const int g = b * P.c.heads + head;
  int first, last;
  pg_range(P, b, &first, &last);
  int w0 = first & ~15, w1 = last;
  if (P.workgroups) {
    const int places = pg_places(P, b), mine = (int)min((int64_t)(places - skip), end - at);
    if (mine <= 0) return;
    w1 = min(w0 + (max(skip + mine - PG_LEAD, 0) << 4), last);
    w0 += max(skip - PG_LEAD, 0) << 4;
    at += mine;
  }
  if (w0 < w1 || !P.workgroups) {
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

  // this wave's chunks of 16 rows: c0, c0 + PG_WAVES, ... below c1 (a run to each wave: 329 instead of 323 us of four sequences of
  // 131072 tokens, 51 instead of 49 of sixteen of unequal lengths)
  const int c0 = (w0 >> 4) + wave, c1 = (w1 + 15) >> 4;
  const int32_t* const table = P.c.table + b * P.c.ts;
  const uint16_t* const kb = P.c.k + head * P.c.kh;
  const uint16_t* const vb = P.c.v + head * P.c.vh;
  // the page of this lane's unit of the batch that begins with chunk c; -1 where there is none
  const auto units = [&](int c) {
    const int row = ((c + (UNI ? lane : lane / upc) * PG_WAVES) << 4) + (UNI ? 0 : (lane % upc) << shift);
    const int page = table[min(row >> shift, P.c.table_pages - 1)];
    return (unsigned)page < (unsigned)P.c.pages ? page : -1;
  };
  // A chunk's keys and values are requested as soon as the registers of the one before are free, whether their rows are attended
  // or not (rows of page 0 stand in for those of a page that is not there): no load is under a condition.  The values' lines are
  // read once and whole; told so, the memory gives 6.5 TB/s instead of 5.9 (four sequences of 131072 tokens, 8 heads: 365 -> 330 us;
  // 32 of 4096 104 -> 95).  The keys' are not: two loads share a line (with them too 332 and 96, sixteen query heads to a head 116
  // -> 126), nor are those of pages below sixteen rows (110 us either way).
  int ib = 0, pid = units(c0), pid_next = units(c0 + cpb * PG_WAVES);   // ib: the chunk's place in its batch
  int pk = -1, pv[NV];
  uint4 k[KK], v[NV];
  const uint32_t koff = (uint32_t)n * (uint32_t)P.c.kr + h * 8, voff = (uint32_t)(lane / LPR) * (uint32_t)P.c.vr + (lane % LPR) * 8;
  const auto pages = [&](int c) {
    if (ib == cpb) {
      ib = 0;
      pid = pid_next;
      pid_next = units(c + cpb * PG_WAVES);
    }
    if (UNI) {
      pk = __builtin_amdgcn_readlane(pid, ib);
    } else {
      pk = __shfl(pid, ib * upc + (n >> shift));
#pragma unroll
      for (int i = 0; i < NV; ++i) pv[i] = __shfl(pid, ib * upc + ((lane / LPR + RPI * i) >> shift));
    }
    ++ib;
  };
  const auto load_keys = [&](int c) {
    const uint16_t* from = UNI ? kb + max(pk, 0) * P.c.kp + ((c << 4) & mask) * P.c.kr + koff
                               : kb + max(pk, 0) * P.c.kp + (n & mask) * P.c.kr + h * 8;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) k[kk] = ri_ld16(from + kk * 32);
  };
  const auto load_values = [&](int c) {
    const uint16_t* from = vb + max(pk, 0) * P.c.vp + ((c << 4) & mask) * P.c.vr + voff;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      v[i] = UNI ? pg_once16(from + RPI * i * P.c.vr)
                 : ri_ld16(vb + max(pv[i], 0) * P.c.vp + ((lane / LPR + RPI * i) & mask) * P.c.vr + (lane % LPR) * 8);
  };
  if (c0 < c1) {
    pages(c0);
    load_keys(c0);
    load_values(c0);
  }
  for (int c = c0; c < c1; c += PG_WAVES) {
    const int r0 = c << 4, rk = r0 + n;
    const bool valid = pk >= 0 && rk >= first && rk < last;
    f32x4_t s4 = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) s4 = pg_mfma32<HALF>(q[kk], k[kk], s4);
    if (__builtin_amdgcn_ballot_w64(valid) != ~0ull) {   // values that are not attended bring no NaN into the products
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int rv = r0 + lane / LPR + RPI * i;
        if ((UNI ? pk : pv[i]) < 0 || rv < first || rv >= last) v[i] = ri_zero16();
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) *reinterpret_cast<uint4*>(vt + (lane / LPR + RPI * i) * VS + (lane % LPR) * 8) = v[i];
    pg_heads<NH> sv;
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      const int r = GP == 16 ? i : rsel + i;
      const float x = r == 0 ? s4[0] : r == 1 ? s4[1] : r == 2 ? s4[2] : s4[3];
      sv.x[i] = valid ? x * P.scale2 : -INFINITY;
    }
    // A lane's heads are neighbours, and a chunk's scores one piece of memory.  (In front of the next loads: whoever waits for these
    // waits for what was stored before, too.)
    if (P.logits && rk < w1) *reinterpret_cast<pg_heads<NH>*>(P.logits + ((size_t)g * P.max_len + rk) * GP + head_of(0)) = sv;
    if (c + PG_WAVES < c1) {
      pages(c + PG_WAVES);
      load_keys(c + PG_WAVES);
      load_values(c + PG_WAVES);
    }
    float al[NH];
    bool rescale = false;
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      const float s = sv.x[i], mn = fmaxf(m[i], pg_row_max(s));
      const bool none = mn == -INFINITY;   // relative to -inf they would weigh NaN
      al[i] = none ? 1.f : pg_exp2(m[i] - mn);
      const float p = pg_exp2(s - (none ? 0.f : mn));
      rescale |= al[i] != 1.f;
      l[i] = l[i] * al[i] + p;
      m[i] = mn;
      uint16_t* const to = pb + head_of(i) * 32 + (n >> 2) * 8 + (n & 3);   // (for the matrix cores; sums are of p itself)
      pg_split<HALF>(p, to, to + 4);
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
    // lane (n, h): both parts of P of head n and rows 4 h .., and twice V of those rows and dim 16 dt + n by transpose reads
    const uint4 pa = *reinterpret_cast<const uint4*>(pb + n * 32 + 8 * h);
    const uint16_t* vsrc = vt + (4 * h + (n >> 2)) * VS + 4 * (n & 3);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const pg_s4 vv = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pg_s4 __attribute__((address_space(3)))*)(vsrc + 16 * dt));
      const uint2 v2 = __builtin_bit_cast(uint2, vv);
      acc[dt] = pg_mfma32<HALF>(pa, make_uint4(v2.x, v2.y, v2.x, v2.y), acc[dt]);
    }
    ri_wave_sync();
  }

  // the waves merge in LDS
  const int tid = pg_anew(threadIdx.x), n2 = tid & 15, h2 = (tid & 63) >> 4;
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const float s = pg_row_sum(l[i]);
    if (n2 == 0) {
      sh_m[wave][head_of(i)] = m[i];
      sh_l[wave][head_of(i)] = s;
    }
  }
  float* const mine = (float*)sh_tile[wave];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int hd = 4 * h2 + i;
    if (hd < GP) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) mine[hd * D + 16 * dt + n2] = HALF ? acc[dt][i] * 0x1p-15f : acc[dt][i];
    }
  }
  if (P.workgroups && tid == 0) {
    if (w0 == (first & ~15)) P.shares[g].x = blockIdx.x;
    if (w1 == last) P.shares[g].y = blockIdx.x;
  }
  __syncthreads();
  for (int at = tid; at < P.gs * D; at += 64 * PG_WAVES) {
    const int j = at / D, d = at % D;
    float M = -INFINITY, L = 0.f, A = 0.f;
#pragma unroll
    for (int w = 0; w < PG_WAVES; ++w) M = fmaxf(M, sh_m[w][j]);
#pragma unroll
    for (int w = 0; w < PG_WAVES; ++w) {
      const float f = pg_weigh_part(sh_m[w][j], sh_l[w][j], M);
      L += sh_l[w][j] * f;
      A += ((const float*)sh_tile[w])[j * D + d] * f;
    }
    const size_t o = (size_t)g * P.gs + j, part = (g + (P.workgroups ? (size_t)blockIdx.x : 0)) * GP + j;
    if (P.workgroups) {
      P.part_acc[part * D + d] = A;
    } else {
      P.out[o * D + d] = ri_f32_to_e16<HALF>(L == 0.f ? 0.f : A / L);
      if (d == 0 && P.lse) P.lse[o] = L == 0.f ? -INFINITY : (M + __log2f(L)) * PG_LN2;
    }
    if (d == 0 && (P.workgroups || P.logits)) {
      P.part_ml[2 * part] = M;
      P.part_ml[2 * part + 1] = L;
    }
  }
  }
  if (at >= end) return;
  do {
    if (++head == P.c.heads) {
      head = 0;
      if (++b == P.B) return;
    }
  } while (pg_places(P, b) == 0);   // (there are places left, so there is such a group)
  skip = 0;
  __syncthreads();
  }
}

#define PG_JOIN_THREADS 256
#define PG_JOIN_ROWS (4 * PG_JOIN_THREADS)   // scores of a workgroup of the join

// Grid (B * heads, (workgroups ? gs : 0) + ceil(max_len / PG_JOIN_ROWS) with scores): the first gs workgroups of a group join the
// parts of a head each; the others add the weights of PG_JOIN_ROWS rows, exp(s - lse) summed over the heads, to the scores.
template <int D, int GP, bool HALF>
__global__ __launch_bounds__(PG_JOIN_THREADS) void paged_join_kernel(PagedAttendParams P) {
  constexpr int NW = PG_JOIN_THREADS / 64, DL = D / 64, MP = PG_WORKGROUPS / 64;   // DL: dims of a lane; MP: parts of a lane at most
  __shared__ float sh_M[16], sh_L[16], sh_f[PG_WORKGROUPS], sh_a[NW][D];
  const int g = blockIdx.x, b = g / P.c.heads, head = g - b * P.c.heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int first, last;
  pg_range(P, b, &first, &last);
  const int outs = P.workgroups ? P.gs : 0;
  const bool joins = (int)blockIdx.y < outs;
  const int r0 = ((int)blockIdx.y - outs) * PG_JOIN_ROWS;
  if (!joins && (r0 >= last || r0 + PG_JOIN_ROWS <= first)) return;
  // the group's parts: of each workgroup that has rows of it
  const int2 share = P.workgroups && first < last ? P.shares[g] : make_int2(0, first < last ? 0 : -1);
  const int share0 = min(max(share.x, 0), max(P.workgroups - 1, 0)), parts = max(min(share.y, max(P.workgroups - 1, 0)) - share0 + 1, 0);
  const size_t part0 = (size_t)g + share0;
  const float2* const ml = reinterpret_cast<const float2*>(P.part_ml) + part0 * GP;
  // maximum and sum of a head's parts, by a wave
  const auto join = [&](int j) {
    float M = -INFINITY, L = 0.f;
    float2 x[MP];
#pragma unroll
    for (int i = 0; i < MP; ++i)
      if (64 * i < parts) x[i] = ml[(size_t)min(64 * i + lane, parts - 1) * GP + j];
#pragma unroll
    for (int i = 0; i < MP; ++i)
      if (64 * i < parts) M = fmaxf(M, x[i].x);
    M = ri_wave_max(M);
#pragma unroll
    for (int i = 0; i < MP; ++i)
      if (64 * i + lane < parts) {
        const float f = pg_weigh_part(x[i].x, x[i].y, M);
        if (joins) sh_f[64 * i + lane] = f;
        L += x[i].y * f;
      }
    L = ri_wave_sum(L);
    if (lane == 0) {
      sh_M[j] = M;
      sh_L[j] = L;
    }
  };
  if (joins) {
    const int j = blockIdx.y;
    if (wave == 0) join(j);
    __syncthreads();
    const float M = sh_M[j], L = sh_L[j];
    float A[DL] = {};
    const float* const acc = P.part_acc + (part0 * GP + j) * D + DL * lane;
    const auto add = [&](auto ahead) {   // so many parts are requested at a time
      constexpr int U = decltype(ahead)::value;
      for (int s = wave; s < parts; s += U * NW) {
        float x[U][DL];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int d = 0; d < DL; ++d) x[u][d] = acc[(size_t)min(s + u * NW, parts - 1) * GP * D + d];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (s + u * NW < parts) {
#pragma unroll
            for (int d = 0; d < DL; ++d) A[d] += x[u][d] * sh_f[s + u * NW];
          }
      }
    };
    if (parts > 8 * NW) add(std::integral_constant<int, 16>());
    else add(std::integral_constant<int, 8>());
#pragma unroll
    for (int d = 0; d < DL; ++d) sh_a[wave][DL * lane + d] = A[d];
    __syncthreads();
    const size_t o = (size_t)g * P.gs + j;
    for (int d = threadIdx.x; d < D; d += PG_JOIN_THREADS) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) x += sh_a[w][d];
      P.out[o * D + d] = ri_f32_to_e16<HALF>(L == 0.f ? 0.f : x / L);
    }
    if (threadIdx.x == 0 && P.lse) P.lse[o] = L == 0.f ? -INFINITY : (M + __log2f(L)) * PG_LN2;
    return;
  }
  // rows r0 + threadIdx.x + 256 i
  float* const scores = P.scores + b * P.sb + head * P.sh;
  pg_heads<GP> x[4];
  float was[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = min(max(r0 + (int)threadIdx.x + PG_JOIN_THREADS * i, first), last - 1);
    x[i] = *reinterpret_cast<const pg_heads<GP>*>(P.logits + ((size_t)g * P.max_len + r) * GP);
    was[i] = scores[r];
  }
  for (int j = wave; j < P.gs; j += NW) join(j);
  __syncthreads();
  bool spoilt = false;
#pragma unroll
  for (int j = 0; j < GP; ++j) {
    const float M = sh_M[min(j, P.gs - 1)], L = sh_L[min(j, P.gs - 1)];
    if (j >= P.gs || L == 0.f) continue;   // (no rows: nothing to add)
    spoilt |= L != L;
    const float inv = 1.f / L;
#pragma unroll
    for (int i = 0; i < 4; ++i) was[i] += pg_exp2(x[i].x[j] - M) * inv;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + threadIdx.x + PG_JOIN_THREADS * i;
    if (r < first || r >= last) continue;
    if (spoilt) {   // the weights are NaN, and not those of rows that are not there
      const int page = P.c.table[b * P.c.ts + (r >> P.c.shift)];
      if ((unsigned)page >= (unsigned)P.c.pages) continue;
    }
    scores[r] = was[i];
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

// Grid (heads, B).  The search for the weakest row reads eight bytes to a row, four rows to a lane's load and U loads ahead.
template <int THREADS, int U>
__global__ __launch_bounds__(THREADS) void paged_append_kernel(PagedAppendParams P) {
  __shared__ unsigned long long sh_best[THREADS / 64];
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
    const int64_t old = (int64_t)token - P.recent;   // the last token that is not one of the recent ones
    uint32_t best = 0xffffffffu;
    int best_row = 0;
    const auto take = [&](int r, float score, int at) {   // (rows ascend: the first of equal ones stays)
      const uint32_t o = at < P.sinks || at > old ? 0xffffffffu : pg_order(score);
      if (o < best) { best = o; best_row = r; }
    };
    int r0 = threadIdx.x * 4;
    const int whole = held & ~3;
    for (; r0 + (U - 1) * THREADS * 4 < whole; r0 += U * THREADS * 4) {
      pg_f4 s[U];
      pg_i4 at[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = *reinterpret_cast<const pg_f4*>(scores + r0 + u * THREADS * 4);
        at[u] = *reinterpret_cast<const pg_i4*>(positions + r0 + u * THREADS * 4);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) take(r0 + u * THREADS * 4 + i, s[u][i], at[u][i]);
    }
    for (; r0 < whole; r0 += THREADS * 4) {
      const pg_f4 s = *reinterpret_cast<const pg_f4*>(scores + r0);
      const pg_i4 at = *reinterpret_cast<const pg_i4*>(positions + r0);
#pragma unroll
      for (int i = 0; i < 4; ++i) take(r0 + i, s[i], at[i]);
    }
    if ((int)threadIdx.x < (held & 3)) take(whole + threadIdx.x, scores[whole + threadIdx.x], positions[whole + threadIdx.x]);
    unsigned long long both = (unsigned long long)best << 32 | (uint32_t)best_row;
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      const unsigned long long other = __shfl_xor(both, d);
      both = other < both ? other : both;
    }
    if (lane == 0) sh_best[wave] = both;
    __syncthreads();
    both = sh_best[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) both = sh_best[w] < both ? sh_best[w] : both;
    row = (int)(uint32_t)both;
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
  // a selection over several chunks of a prompt
  uint16_t* hist;         // [B * heads, chunks, 2048] rows of a chunk by the first digit of their order, and [.., 64] by its bits 10 .. 5
  uint16_t* coarse;
  uint32_t* tied;         // [B * heads, chunks * PG_CHUNK]: the orders of a chunk's rows that share the digit in question
  int2* counts;           // [B * heads, chunks]: rows above that digit, rows of it; then where a chunk's rows go, ties in front
  int2* limit;            // [B * heads]: the digit and how many of its rows are kept; then the lowest kept order and its rows
  int T, budget, sinks, recent, dim, chunks;
};

__device__ __forceinline__ int pg_prompt(const PagedFillParams& P, int b) { return P.lens ? min(max(P.lens[b], 0), P.T) : P.T; }

#define PG_SEL_THREADS 1024
#define PG_SEL_WAVES (PG_SEL_THREADS / 64)
#define PG_CHUNK (4 * PG_SEL_THREADS)   // rows: four consecutive ones to a thread
#define PG_SEL_CHUNKS 4                 // that one workgroup selects from

// The rows of a prompt that are kept, in order, with their weights and positions: the `sinks` first, the `recent` last and of the
// others those with the highest weights, at equal weights the first ones.  A radix selection finds the lowest kept order, digits of
// 11, 11 and 10 bits, and how many of the rows of that order are kept, the first ones.
struct PagedRows {   // this thread's rows of a chunk
  int r0;
  uint32_t o[4];     // their orders; 0: no row
};
__device__ __forceinline__ PagedRows pg_rows(const PagedFillParams& P, const float* w, int n, int chunk) {
  PagedRows x;
  x.r0 = chunk * PG_CHUNK + 4 * threadIdx.x;
  pg_f4 v = {0.f, 0.f, 0.f, 0.f};
  if (x.r0 + 4 <= n) {
    v = *reinterpret_cast<const pg_f4*>(w + x.r0);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x.r0 + i < n ? w[x.r0 + i] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = x.r0 + i;
    x.o[i] = r >= n ? 0u : r < P.sinks || r >= n - P.recent ? 0xffffffffu : pg_order(v[i]);
  }
  return x;
}

// Whole workgroup: the bin from the top of hist[bins] (LDS, 2048 at most) in which the count reaches need; need becomes how many of
// that bin's are kept.
__device__ __forceinline__ int pg_pick(const int* hist, int bins, int& need) {
  __shared__ int sh_scan[PG_SEL_WAVES], sh_pick[2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  const int top = bins - 1 - 2 * (int)threadIdx.x;   // thread t: bins 2 t and 2 t + 1 from the top
  const int a = top >= 0 ? hist[top] : 0, c = top >= 1 ? hist[top - 1] : 0;
  const int incl = (int)ri_wave_incl_scan((uint32_t)(a + c));
  if (lane == 63) sh_scan[wave] = incl;
  __syncthreads();
  int before = incl - a - c;
#pragma unroll
  for (int i = 0; i < PG_SEL_WAVES; ++i) before += i < wave ? sh_scan[i] : 0;
  if (before < need && before + a + c >= need) {
    const bool second = before + a < need;
    sh_pick[0] = second ? top - 1 : top;
    sh_pick[1] = need - before - (second ? a : 0);
  }
  __syncthreads();
  need = sh_pick[1];
  return sh_pick[0] & (bins - 1);
}

// Whole workgroup: exclusive sums over the threads of a count below 2^16 in each half of x; the workgroup's in *all.
__device__ __forceinline__ uint32_t pg_scan(uint32_t x, uint32_t* all) {
  __shared__ uint32_t sh_wave[PG_SEL_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t incl = ri_wave_incl_scan(x);
  __syncthreads();
  if (lane == 63) sh_wave[wave] = incl;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < PG_SEL_WAVES; ++i) {
    const uint32_t v = sh_wave[i];
    before += i < wave ? v : 0;
    total += v;
  }
  *all = total;
  return before + incl - x;
}

// This thread's rows of order above `lowest`, and the first `need` of those of it, to their places: `base` rows and `ties` of that
// order are in front of the chunk's, and behind it when this returns.
__device__ __forceinline__ void pg_emit(const PagedFillParams& P, int g, int b, int head, const PagedRows& x, uint32_t lowest, int need,
                                        int& base, int& ties) {
  uint32_t mine = 0, all;
#pragma unroll
  for (int i = 0; i < 4; ++i) mine += (x.o[i] > lowest ? 1u : 0u) + (x.o[i] == lowest ? 0x10000u : 0u);
  const uint32_t before = pg_scan(mine, &all);
  int above = before & 0xffffu, tie = ties + (int)(before >> 16);
  int32_t* const kept = P.kept + (size_t)g * P.budget;
  float* const scores = P.scores ? P.scores + b * P.sb + head * P.sh : nullptr;
  int32_t* const positions = P.positions ? P.positions + b * P.pb + head * P.ph : nullptr;
  const float* const w = P.weights + b * P.wb + head * P.wh;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool is_above = x.o[i] > lowest, is_tie = x.o[i] == lowest;
    if (is_above || (is_tie && tie < need)) {
      const int at = base + above + min(tie, need) - min(ties, need);
      if ((unsigned)at < (unsigned)P.budget) {   // (always, of lengths that stay as they are)
        kept[at] = x.r0 + i;
        if (scores) scores[at] = w[x.r0 + i];
        if (positions) positions[at] = x.r0 + i;
      }
    }
    above += is_above;
    tie += is_tie;
  }
  const int more = (int)(all >> 16);
  base += (int)(all & 0xffffu) + min(ties + more, need) - min(ties, need);
  ties += more;
}

// Scores and positions of the rows [r0, r1) of a prompt that is kept whole.
__device__ __forceinline__ void pg_whole(const PagedFillParams& P, int b, int head, int r0, int r1) {
  const float* const w = P.weights ? P.weights + b * P.wb + head * P.wh : nullptr;
  float* const scores = P.scores ? P.scores + b * P.sb + head * P.sh : nullptr;
  int32_t* const positions = P.positions ? P.positions + b * P.pb + head * P.ph : nullptr;
  for (int r = r0 + threadIdx.x; r < r1; r += PG_SEL_THREADS) {
    if (scores) scores[r] = w[r];
    if (positions) positions[r] = r;
  }
}

// Grid (heads, B): a workgroup has a prompt of up to CHUNKS chunks, whose orders stay in registers (0: prompts that are kept whole).
// A prompt of 6000 tokens, 16 (sequence, head) pairs, with the copy: 11.9 us against 20 in launches over chunks, 12000: 15.7 and 20.1;
// with eight chunks it loses, 30011: 30.7 and 21.7.
template <int CHUNKS>
__global__ __launch_bounds__(PG_SEL_THREADS) void paged_select_kernel(PagedFillParams P) {
  __shared__ int hist[2048];
  const int head = blockIdx.x, b = blockIdx.y, n = pg_prompt(P, b), g = b * P.c.heads + head;
  if (n <= P.budget) return pg_whole(P, b, head, 0, n);
  if constexpr (CHUNKS > 0) {
    PagedRows x[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) x[c] = pg_rows(P, P.weights + b * P.wb + head * P.wh, n, c);
    uint32_t lowest = 0, known = 0;   // bits of the lowest kept order found so far
    int need = P.budget;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
      hist[threadIdx.x] = hist[threadIdx.x + PG_SEL_THREADS] = 0;
      __syncthreads();
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (x[c].o[i] && (x[c].o[i] & known) == lowest) atomicAdd(&hist[(x[c].o[i] >> shift) & (bins - 1)], 1);
      lowest |= (uint32_t)pg_pick(hist, bins, need) << shift;
      known |= (uint32_t)(bins - 1) << shift;
      __syncthreads();
    }
    int base = 0, ties = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      if (c * PG_CHUNK < n) pg_emit(P, g, b, head, x[c], lowest, need, base, ties);
  }
}

// Longer prompts: launches over all chunks.  1: the chunks' rows by the first
// digit.  Grid (chunks, heads, B).
__global__ __launch_bounds__(PG_SEL_THREADS) void paged_digit_kernel(PagedFillParams P) {
  __shared__ int hist[2048];
  const int chunk = blockIdx.x, head = blockIdx.y, b = blockIdx.z, n = pg_prompt(P, b);
  if (n <= P.budget || chunk * PG_CHUNK >= n) return;
  const PagedRows x = pg_rows(P, P.weights + b * P.wb + head * P.wh, n, chunk);
  hist[threadIdx.x] = hist[threadIdx.x + PG_SEL_THREADS] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (x.o[i]) atomicAdd(&hist[x.o[i] >> 21], 1);
  __syncthreads();
  const size_t at = (size_t)(b * P.c.heads + head) * P.chunks + chunk;
  const int lo = hist[2 * threadIdx.x], hi = hist[2 * threadIdx.x + 1];
  reinterpret_cast<uint32_t*>(P.hist + at * 2048)[threadIdx.x] = (uint32_t)lo | (uint32_t)hi << 16;   // (4096 at most)
  float sum = (float)(lo + hi);   // of 32 bins, sixteen lanes
  sum = ri_xor_sum<1>(ri_xor_sum<2>(ri_xor_sum<4>(ri_xor_sum<8>(sum))));
  if (threadIdx.x % 16 == 0) P.coarse[at * 64 + threadIdx.x / 16] = (uint16_t)sum;
}

// 2: the digit in which the count of kept rows ends, and of a chunk how many rows are above it and the orders of those that have it.
// Grid (chunks, heads, B).
__global__ __launch_bounds__(PG_SEL_THREADS) void paged_tied_kernel(PagedFillParams P) {
  __shared__ int hist[64];
  const int chunk = blockIdx.x, head = blockIdx.y, b = blockIdx.z, n = pg_prompt(P, b), g = b * P.c.heads + head;
  if (n <= P.budget || chunk * PG_CHUNK >= n) return;
  const PagedRows x = pg_rows(P, P.weights + b * P.wb + head * P.wh, n, chunk);
  const int chunks = (n + PG_CHUNK - 1) / PG_CHUNK, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int need = P.budget, digit = 0;
#pragma unroll
  for (int fine = 0; fine < 2; ++fine) {   // 64 groups of 32 digits, then the digits of one
    if (threadIdx.x < 64) hist[threadIdx.x] = 0;
    __syncthreads();
    int sum = 0;
    if (!fine || lane < 32) {
#pragma unroll 4
      for (int c = wave; c < chunks; c += PG_SEL_WAVES) {
        const size_t at = (size_t)g * P.chunks + c;
        sum += fine ? P.hist[at * 2048 + digit * 32 + lane] : P.coarse[at * 64 + lane];
      }
      if (sum) atomicAdd(&hist[lane], sum);
    }
    digit = digit * 32 + pg_pick(hist, fine ? 32 : 64, need);
    __syncthreads();
  }
  uint32_t mine = 0, all;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    mine += (x.o[i] && (int)(x.o[i] >> 21) > digit ? 1u : 0u) + (x.o[i] && (int)(x.o[i] >> 21) == digit ? 0x10000u : 0u);
  uint32_t* to = P.tied + ((size_t)g * P.chunks + chunk) * PG_CHUNK + (pg_scan(mine, &all) >> 16);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (x.o[i] && (int)(x.o[i] >> 21) == digit) *to++ = x.o[i];
  if (threadIdx.x == 0) {
    P.counts[(size_t)g * P.chunks + chunk] = make_int2(all & 0xffffu, all >> 16);
    if (chunk == 0) P.limit[g] = make_int2(digit, need);
  }
}

// Whole workgroup, a wave to a chunk's tied rows at a time: the lowest kept order, and in `need` how many of its rows are kept.
__device__ __forceinline__ uint32_t pg_lowest(const PagedFillParams& P, int g, int chunks, int& need) {
  __shared__ int hist[2048];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int2* const counts = P.counts + (size_t)g * P.chunks;
  const uint32_t* const tied = P.tied + (size_t)g * P.chunks * PG_CHUNK;
  need = P.limit[g].y;
  uint32_t lowest = (uint32_t)P.limit[g].x << 21, known = 0x7ffu << 21;
#pragma unroll
  for (int pass = 1; pass < 3; ++pass) {
    const int shift = pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    hist[threadIdx.x] = hist[threadIdx.x + PG_SEL_THREADS] = 0;
    __syncthreads();
    for (int c = wave; c < chunks; c += PG_SEL_WAVES) {
      const int m = min(counts[c].y, PG_CHUNK);
      for (int i = lane; i < m; i += 64) {
        const uint32_t o = tied[(size_t)c * PG_CHUNK + i];
        if ((o & known) == lowest) atomicAdd(&hist[(o >> shift) & (bins - 1)], 1);
      }
    }
    lowest |= (uint32_t)pg_pick(hist, bins, need) << shift;
    known |= (uint32_t)(bins - 1) << shift;
    __syncthreads();
  }
  return lowest;
}
// By a wave: of a chunk's tied rows those above `lowest`, and in the upper half those of it.
__device__ __forceinline__ uint32_t pg_kept_of(const uint32_t* tied, int m, uint32_t lowest) {
  uint32_t x = 0;
  for (int i = threadIdx.x & 63; i < min(m, PG_CHUNK); i += 64) {
    const uint32_t o = tied[i];
    x += (o > lowest ? 1u : 0u) + (o == lowest ? 0x10000u : 0u);
  }
  return __shfl(ri_wave_incl_scan(x), 63);
}

// 3: the lowest kept order and where each chunk's rows go.  Grid (heads, B).
__global__ __launch_bounds__(PG_SEL_THREADS) void paged_limit_kernel(PagedFillParams P) {
  __shared__ uint32_t sh_chunk[PG_SEL_THREADS];
  const int head = blockIdx.x, b = blockIdx.y, n = pg_prompt(P, b), g = b * P.c.heads + head;
  if (n <= P.budget) return;
  const int chunks = (n + PG_CHUNK - 1) / PG_CHUNK, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int2* const counts = P.counts + (size_t)g * P.chunks;
  const uint32_t* const tied = P.tied + (size_t)g * P.chunks * PG_CHUNK;
  int need;
  const uint32_t lowest = pg_lowest(P, g, chunks, need);
  int base = 0, ties = 0;
  for (int c0 = 0; c0 < chunks; c0 += PG_SEL_THREADS) {
    const int c1 = min(chunks, c0 + PG_SEL_THREADS);
    for (int c = c0 + wave; c < c1; c += PG_SEL_WAVES) {
      const uint32_t sum = pg_kept_of(tied + (size_t)c * PG_CHUNK, counts[c].y, lowest);
      if (lane == 0) sh_chunk[c - c0] = sum;
    }
    __syncthreads();
    const int c = c0 + threadIdx.x;
    const int above = c < c1 ? counts[c].x + (int)(sh_chunk[threadIdx.x] & 0xffffu) : 0;
    const int equal = c < c1 ? (int)(sh_chunk[threadIdx.x] >> 16) : 0;
    // (a chunk has 4096 rows and a part of 1024 chunks 2^22: sums of their own)
    uint32_t all_above, all_equal;
    const int b0 = base + (int)pg_scan((uint32_t)above, &all_above);
    const int t0 = ties + (int)pg_scan((uint32_t)equal, &all_equal);
    if (c < c1) counts[c] = make_int2(b0 + min(t0, need), t0);
    base += (int)all_above;
    ties += (int)all_equal;
    __syncthreads();
  }
  if (threadIdx.x == 0) P.limit[g] = make_int2((int)lowest, need);
}

// 4: the list.  Grid (chunks, heads, B).  OWN: without launch 3, each workgroup finds out for itself: up to PG_OWN_CHUNKS chunks to a
// prompt, whose tied rows are few for one to go over (of more the work grows with their square), and as many workgroups as run at a
// time (131072 tokens, 8 heads, with the copy 30.8 us against 33.8; 16 prompts of 20000, 8 heads 76 against 73).
#define PG_OWN_CHUNKS 64
#define PG_OWN_WORKGROUPS 512
template <bool OWN>
__global__ __launch_bounds__(PG_SEL_THREADS) void paged_list_kernel(PagedFillParams P) {
  __shared__ int sh_sum[2];
  const int chunk = blockIdx.x, head = blockIdx.y, b = blockIdx.z, n = pg_prompt(P, b), g = b * P.c.heads + head;
  if (chunk * PG_CHUNK >= n) return;
  if (n <= P.budget) return pg_whole(P, b, head, chunk * PG_CHUNK, min(n, (chunk + 1) * PG_CHUNK));
  const PagedRows x = pg_rows(P, P.weights + b * P.wb + head * P.wh, n, chunk);
  int base, ties, need;
  uint32_t lowest;
  if (OWN) {
    const int2* const counts = P.counts + (size_t)g * P.chunks;
    lowest = pg_lowest(P, g, (n + PG_CHUNK - 1) / PG_CHUNK, need);
    if (threadIdx.x < 2) sh_sum[threadIdx.x] = 0;
    __syncthreads();
    for (int c = threadIdx.x >> 6; c < chunk; c += PG_SEL_WAVES) {   // what is in front of this chunk
      const int2 count = counts[c];
      const uint32_t sum = pg_kept_of(P.tied + ((size_t)g * P.chunks + c) * PG_CHUNK, count.y, lowest);
      if (threadIdx.x % 64 == 0) {
        atomicAdd(&sh_sum[0], count.x + (int)(sum & 0xffffu));
        atomicAdd(&sh_sum[1], (int)(sum >> 16));
      }
    }
    __syncthreads();
    ties = sh_sum[1];
    base = sh_sum[0] + min(ties, need);
  } else {
    const int2 limit = P.limit[g], at = P.counts[(size_t)g * P.chunks + chunk];
    lowest = (uint32_t)limit.x;
    need = limit.y;
    base = at.x;
    ties = at.y;
  }
  pg_emit(P, g, b, head, x, lowest, need, base, ties);
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
  if ((unsigned)page >= (unsigned)P.c.pages || (unsigned)src >= (unsigned)P.T) return;
  *reinterpret_cast<uint4*>(const_cast<uint16_t*>(P.c.k) + page * P.c.kp + head * P.c.kh + at * P.c.kr + piece) =
      ri_ld16(P.key + b * P.kb + src * P.kt + head * P.kh + piece);
  *reinterpret_cast<uint4*>(const_cast<uint16_t*>(P.c.v) + page * P.c.vp + head * P.c.vh + at * P.c.vr + piece) =
      ri_ld16(P.value + b * P.vb + src * P.vt + head * P.vh + piece);
}

// ------------------------------------------------------------------------------------ host side
#define PG_MAX_ROWS (1 << 24)   // rows of a sequence
static bool strides_ok(int64_t a, int64_t b, int64_t c = 0) { return a >= 0 && b >= 0 && c >= 0 && (a | b | c) % 8 == 0; }

// two tables of n, one of which is written while others may still read the other
static bool pg_meet(const int32_t* a, const int32_t* b, int n) {
  return a && b && (uintptr_t)a < (uintptr_t)(b + n) && (uintptr_t)b < (uintptr_t)(a + n);
}

static int paged_view(const ri_paged_t* c, int B, PagedView* v) {
  if (!c || !c->k_pages || !c->v_pages || !c->block_table || ri_any_misaligned16(c->k_pages, c->v_pages)) return RI_ERR_ARG;
  if (c->pages <= 0 || c->heads <= 0 || c->table_pages <= 0 || B <= 0 || c->table_stride < 0) return RI_ERR_ARG;
  if (c->dim != 64 && c->dim != 128) return RI_ERR_ARG;
  if (c->page_rows <= 0 || (c->page_rows & (c->page_rows - 1)) || (int64_t)c->table_pages * c->page_rows > PG_MAX_ROWS)
    return RI_ERR_ARG;
  if (!strides_ok(c->k_page_stride, c->k_head_stride, c->k_row_stride) || !strides_ok(c->v_page_stride, c->v_head_stride, c->v_row_stride))
    return RI_ERR_ARG;
  if (c->k_row_stride > 1 << 24 || c->v_row_stride > 1 << 24) return RI_ERR_ARG;   // (sixteen rows are addressed by 32 bits)
  if (c->heads > 65535 || B > 65535) return RI_ERR_ARG;   // (dimensions of grids)
  *v = {(const uint16_t*)c->k_pages, (const uint16_t*)c->v_pages, c->block_table, c->k_page_stride, c->k_head_stride, c->k_row_stride,
        c->v_page_stride, c->v_head_stride, c->v_row_stride, c->table_stride, c->pages, c->heads, __builtin_ctz(c->page_rows),
        c->page_rows - 1, c->table_pages};
  return RI_OK;
}

static int pg_pad(int gs) { return gs <= 4 ? 4 : gs <= 8 ? 8 : 16; }

extern "C" size_t ri_paged_attention_workspace_bytes(int B, int heads, int gs, int dim, int max_len, int scored) {
  if (B <= 0 || heads <= 0 || gs <= 0 || gs > 16 || max_len <= 0 || max_len > PG_MAX_ROWS || (dim != 64 && dim != 128)) return 0;
  const int64_t groups = (int64_t)B * heads;
  const size_t parts = groups + paged_workgroups(groups, max_len);
  return parts * pg_pad(gs) * (2 + dim) * sizeof(float) + (scored ? (size_t)groups * pg_pad(gs) * max_len * sizeof(float) : 0) +
         groups * sizeof(int2);
}

template <int D, int GP, bool HALF>
static void launch_paged(const PagedAttendParams& P, int groups, hipStream_t s) {
  auto* kernel = P.c.shift >= 4 ? paged_attend_kernel<D, GP, HALF, true> : paged_attend_kernel<D, GP, HALF, false>;
  kernel<<<P.workgroups ? P.workgroups : groups, 64 * PG_WAVES, 0, s>>>(P);
  const int y = (P.workgroups ? P.gs : 0) + (P.scores ? (P.max_len + PG_JOIN_ROWS - 1) / PG_JOIN_ROWS : 0);
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
  const int64_t places = max_len / 16 + 2 + PG_LEAD;   // of a group; those of a head's sequences and of a sequence's heads are counted in 32 bits
  if (B * places > INT32_MAX || cache->heads * places > INT32_MAX) return RI_ERR_ARG;
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
  P.B = B;
  P.workgroups = paged_workgroups(groups, max_len);
  P.scale2 = scale * PG_LOG2E;
  const size_t parts = (size_t)(groups + P.workgroups) * pg_pad(gs);
  P.part_ml = (float*)workspace;
  P.part_acc = P.part_ml + 2 * parts;
  P.logits = scores ? P.part_acc + parts * cache->dim : nullptr;
  P.shares = (int2*)(P.part_acc + parts * cache->dim + (scores ? (size_t)groups * pg_pad(gs) * max_len : 0));
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
  if (!key || !value || !lens || ri_any_misaligned16(key, value) || cache->k_pages == cache->v_pages) return RI_ERR_ARG;
  if (pg_meet(lens, new_lens, B) || pg_meet(token_positions, new_lens, B)) return RI_ERR_ARG;
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
  const dim3 grid(cache->heads, B);
  // (8 heads, 1024 rows 3.2 us, with 1024 threads 3.6; 4096 3.9 and 4.0; 8192 5.0 and 4.4; 32768 11.6 and 7.1; 256 heads, 4096 rows 4.1
  // and 4.4, 8192 7.0 and 6.7: round trips and a launch, the rows' 8 bytes at most 4.7 TB/s)
  if (!scores || budget <= 4096) paged_append_kernel<256, 2><<<grid, 256, 0, (hipStream_t)stream>>>(P);
  else paged_append_kernel<1024, 2><<<grid, 1024, 0, (hipStream_t)stream>>>(P);
  RI_HIP_CHECK_LAUNCH();
  return RI_OK;
}

// 16-byte aligned parts of the workspace of a fill: kept, hist, coarse, tied, counts, limit
static size_t paged_fill_carve(PagedFillParams* P, size_t groups, int T, int budget, char* at) {
  const size_t chunks = T > PG_CHUNK * PG_SEL_CHUNKS ? ((size_t)T + PG_CHUNK - 1) / PG_CHUNK : 0;
  size_t used = 0;
  const auto part = [&](size_t bytes) {
    char* const p = at + used;
    used += (bytes + 15) / 16 * 16;
    return p;
  };
  char* const kept = part(groups * budget * 4);
  char* const hist = part(groups * chunks * 2048 * 2);
  char* const coarse = part(groups * chunks * 64 * 2);
  char* const tied = part(groups * chunks * PG_CHUNK * 4);
  char* const counts = part(groups * chunks * sizeof(int2));
  char* const limit = part(groups * sizeof(int2));
  if (P) {
    P->kept = (int32_t*)kept;
    P->hist = (uint16_t*)hist;
    P->coarse = (uint16_t*)coarse;
    P->tied = (uint32_t*)tied;
    P->counts = (int2*)counts;
    P->limit = (int2*)limit;
    P->chunks = (int)chunks;
  }
  return used;
}

extern "C" size_t ri_paged_fill_workspace_bytes(int B, int heads, int T, int budget) {
  return B <= 0 || heads <= 0 || T <= budget || budget <= 0 ? 0 : paged_fill_carve(nullptr, (size_t)B * heads, T, budget, nullptr);
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
  if (!key || !value || ri_any_misaligned16(key, value) || cache->k_pages == cache->v_pages || pg_meet(seqlens, new_lens, B)) return RI_ERR_ARG;
  if (!strides_ok(key_batch_stride, key_token_stride, key_head_stride) || !strides_ok(value_batch_stride, value_token_stride, value_head_stride))
    return RI_ERR_ARG;
  if (T <= 0 || T > PG_MAX_ROWS || budget <= 0 || budget > cache->table_pages * cache->page_rows || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return RI_ERR_ARG;
  const int room = T < budget ? T : budget;
  if ((T > budget || scores) && !weights) return RI_ERR_ARG;
  if (scores && scores == weights) return RI_ERR_ARG;   // (written while others still read)
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
  if (need) paged_fill_carve(&P, (size_t)B * cache->heads, T, budget, (char*)workspace);
  P.T = T; P.budget = budget; P.sinks = sinks; P.recent = recent; P.dim = cache->dim;
  hipStream_t s = (hipStream_t)stream;
  const dim3 each(cache->heads, B), chunks(P.chunks, cache->heads, B);
  if (T <= budget) {
    if (scores || positions) paged_select_kernel<0><<<each, PG_SEL_THREADS, 0, s>>>(P);
  } else if (T <= PG_CHUNK) {
    paged_select_kernel<1><<<each, PG_SEL_THREADS, 0, s>>>(P);
  } else if (T <= 2 * PG_CHUNK) {
    paged_select_kernel<2><<<each, PG_SEL_THREADS, 0, s>>>(P);
  } else if (P.chunks == 0) {
    paged_select_kernel<PG_SEL_CHUNKS><<<each, PG_SEL_THREADS, 0, s>>>(P);
  } else {
    paged_digit_kernel<<<chunks, PG_SEL_THREADS, 0, s>>>(P);
    paged_tied_kernel<<<chunks, PG_SEL_THREADS, 0, s>>>(P);
    if (P.chunks <= PG_OWN_CHUNKS && (int64_t)P.chunks * cache->heads * B <= PG_OWN_WORKGROUPS) {
      paged_list_kernel<true><<<chunks, PG_SEL_THREADS, 0, s>>>(P);
    } else {
      paged_limit_kernel<<<each, PG_SEL_THREADS, 0, s>>>(P);
      paged_list_kernel<false><<<chunks, PG_SEL_THREADS, 0, s>>>(P);
    }
  }
  const int per = 256 / (cache->dim / 8);
  paged_copy_kernel<<<dim3((room + per - 1) / per, cache->heads, B), 256, 0, s>>>(P);
  RI_HIP_CHECK_LAUNCH();
  return RI_OK;
}
