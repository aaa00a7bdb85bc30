// th_paged_attention: attention of one query per token over a paged KV cache
// (no counterpart in the reference, which has no cache; the math is that of
// optimizer/evaluate.py:139-146 for one query row, with a window, capped scores
// and a bias by distance).
//
// HBM bound: 2 G operations per byte of a bf16 cache (G = query heads per kv
// head), so what counts is that every visible K and V byte is read once, that
// enough of them are in flight, and that all CUs have the same amount to read.
//
// Work: a tile is 8 KiB of K and 8 KiB of V (KT keys of one kv head), whatever
// the head size and type. Two forms deal the tiles out:
//   line     the key tiles of all tokens form one line; the waves (eight a CU)
//            form groups with one wave for each kv head, and each group takes an
//            equal stretch of the line, so ragged batches, one long sequence and
//            many short ones are dealt out alike, with nothing about the lengths
//            known on the host (a captured graph serves any lengths). The parts
//            of a token that was cut go through the workspace (m, l, o in fp32)
//            to the join kernel; a token inside one stretch is finished by its
//            group. The waves of a CU keep step (keep_step): left alone, the
//            older half of them is served first and ends at 108 us where the
//            younger ends at 134 (64 sequences of 2048-4096 keys); and the heads of
//            a key, neighbours in memory, are read together.
//   pair     a workgroup for each (token, kv head) pair, its tiles dealt out to
//            the waves in turn and the waves merged in LDS: where a pair can have
//            only a few tiles by its table and window, one launch and no line to
//            lay out.
//
// One tile (figures of alternatives were taken with p as one bf16 half, 0.6 us less):
//   V        loaded by whole rows (16-byte pieces, consecutive lanes next to each
//            other) and staged in 16 bits in the wave's own LDS slice, swizzled.
//   S^T      = K Q^T, v_mfma_f32_16x16x32_bf16: lane l supplies row l % 16 and 8
//            dims from 8 (l / 16). A bf16 K goes through the slice too, before V:
//            loaded in its operand layout, half a 128-byte line of 16 rows at a
//            time, 64 sequences of 2048-4096 keys took 139.7 us for 134.4. An e4m3
//            K is loaded in that layout, the dims of a row permuted (16 consecutive
//            ones serve two k steps, q alike): 100.3 us, through the slice 101.6.
//   O^T      += V^T P^T: V is read transposed (ds_read_b64_tr_b16); P^T is the S^T
//            accumulators as they are, sums and maxima stay fp32. With a bf16 V each
//            p goes in as two bf16 halves, h + (p - h): off by 2^-15 of it. h is less
//            than p, so that p - h is above zero and an infinite value stays one (0 inf
//            and inf - inf are NaN). One half (2^-8) took the error against 64 bits
//            from 0.0017, the output's own rounding, to 0.0020-0.0022, for 132.5 us
//            instead of 133.3 (64 sequences of 2048-4096 keys), 17.2 instead of 18.0
//            (23 windows of 1000, 12 heads of 64). An e4m3 V is staged as fp16, which
//            holds it exactly, and p is one fp16 (2^-11: error 0.0017): 95.9 us, as with
//            one bf16 half (0.0021); two halves 100.3.
// The next tile's loads are issued as soon as this one has left its registers, and
// land during the softmax and the second product. Buffer loads return zero past
// their range: unseen slots of a page and pages outside the cache cost no branch, and
// whatever they hold (NaN) never meets a zero probability.
#include "common.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace th {

struct PAttnK {
  const uint16_t* q; int64_t ldq;
  const char* k; int64_t kp, kt, kh;  // byte strides: page, token, head
  const char* v; int64_t vp, vt, vh;
  uint16_t* o; int64_t ldo;
  const int32_t* positions;
  const int32_t* rows;
  const int32_t* table; int64_t ldt;
  int64_t pages;
  int n_rows, row_pages, pshift;
  int tokens, Hkv, G, nqb, gq;  // nqb blocks of gq <= 16 query heads per kv head
  int window;
  int o8;           // o in whole 8-byte pieces
  int turn;         // pair: workgroups that give each XCD one token (0: no order)
  float scale, softcap;
  const float* slopes;
  const float* ks;
  const float* vs;
  int64_t* prefix;  // line: [tokens + 1], tiles of the tokens before
  float* ml;        // line: [2 waves][gq][2]
  float* part;      // line: [2 waves][gq][D], unnormalised
};

constexpr float kLog2e = 1.4426950408889634f;

typedef unsigned pa_u32x4 __attribute__((ext_vector_type(4)));
typedef short pa_s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void pa_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A token's keys: [lo, hi) of its row; units start at lo rounded down to 16.
struct Span { int row, lo, hi, base, units; };  // units of KU keys

template <int KU>
__device__ __forceinline__ Span span_from(const PAttnK& p, int pos, int row) {
  Span s;
  s.row = row;
  const bool in = row >= 0 && row < p.n_rows && pos >= 0;
  s.hi = in ? (int)min((int64_t)pos + 1, (int64_t)p.row_pages << p.pshift) : 0;
  s.lo = p.window ? (int)max((int64_t)0, (int64_t)pos + 1 - p.window) : 0;
  s.base = s.lo & ~15;
  s.units = s.hi > s.lo ? (s.hi - s.base + KU - 1) / KU : 0;
  return s;
}

template <int KU>
__device__ __forceinline__ Span span_of(const PAttnK& p, int t) {
  return span_from<KU>(p, p.positions[t], p.rows ? p.rows[t] : t);
}

// Equal stretches of n tiles over w groups: the first n % w get one more.
struct Share {
  int64_t each, more;
  __device__ __forceinline__ Share(int64_t n, int w) {
    if (n >> 31) {
      each = n / w;
      more = n - each * w;
    } else {
      each = (uint32_t)n / (uint32_t)w;
      more = (uint32_t)n - (uint32_t)each * (uint32_t)w;
    }
  }
  __device__ __forceinline__ int64_t begin(int i) const { return i * each + min((int64_t)i, more); }
  __device__ __forceinline__ int owner(int64_t u) const {
    const int64_t big = more * (each + 1);
    if ((u | big) >> 31) return (int)(u < big ? u / (each + 1) : more + (u - big) / each);
    return (int)((uint32_t)u < (uint32_t)big ? (uint32_t)u / (uint32_t)(each + 1)
                                             : (uint32_t)more + (uint32_t)(u - big) / (uint32_t)each);
  }
};

// 8 e4m3 values (two dwords) as 8 bf16: exact.
__device__ __forceinline__ bf16x8_t e4m3x8_to_bf16(unsigned lo, unsigned hi) {
  typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
  union { b2_t h[4]; bf16x8_t v; } u;
  u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return u.v;
}

// The same as 8 fp16: exact too.
__device__ __forceinline__ f16x8_t e4m3x8_to_f16(unsigned lo, unsigned hi) {
  typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
  union { h2_t h[4]; f16x8_t v; } u;
  u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
  u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
  u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return u.v;
}

// LDS slot of 16-byte chunk c of K row r is c ^ ksw(r): the 16 rows of an operand
// read then hit distinct banks.
template <int CPR>
__device__ __forceinline__ int pa_ksw(int r) { return CPR == 16 ? r & 15 : CPR == 8 ? (r >> 1) & 7 : (r >> 2) & 3; }

// The same of V in 16 bits: a transposing read (16 rows, 32 bytes each) hits every
// bank twice. The lowest bit lets neighbouring rows of e4m3, whose 16-byte pieces
// become two chunks each, write to even and odd slots at once.
template <int D>
__device__ __forceinline__ int pa_sw(int r) {
  return D == 128 ? 2 * (r & 7) + (r & 1) : 2 * ((r >> 1) & 3) + ((r >> 1) & 1);
}

template <int D, bool E4>
struct PaTile {
  static constexpr int RB = D * (E4 ? 1 : 2);   // bytes of a cached row
  static constexpr int KT = 8192 / RB;          // keys per tile
  static constexpr int NB = KT / 16;            // 16-key blocks
  static constexpr int CPR = RB / 16;           // 16-byte chunks per row
  static constexpr int RPI = 64 / CPR;          // V rows per load instruction
  static constexpr int LDS = KT * D * 2;        // one wave's slice: V in 16 bits, K (as it is) before it
  typedef std::conditional_t<E4, f16x8_t, bf16x8_t> V8;  // the second product's operands
  // What the exponents of a softmax with maximum m are taken from, and its parts joined by.
  // For fp16 14 less, so that its smallest step is 2^-38 of the largest p and many keys of
  // little weight are not lost (2^-24 with m itself). From 2^24 on a float's own steps are
  // 2 and more, and m - 14 could round to m - 16, of which a p overflows: there it is m.
  // (A product with 2^14 after the exponential: 97.3 us for 95.5, 64 rows of 1-8191 keys.)
  static __device__ __forceinline__ float from(float m) { return E4 && fabsf(m) < 0x1p24f ? m - 14.f : m; }
};

constexpr int kLineWaves = 8;

// The waves of a line's workgroup meet at every other tile: with a barrier at each
// one 64 sequences of 2048-4096 keys took 134.4 us for 131.3 (an 8-bit cache 100.5
// for 96.7), at every fourth 130.6 (99.0).
__device__ __forceinline__ void keep_step(int64_t step) {
  if ((step & 1) == 0) barrier_keep_loads();
}

// NW: waves of a workgroup. NT: what is loaded past the caches (non-temporal): 1 V,
// 2 a bf16 K too. In a graph, us, with neither, V, both: 64 sequences of 2048-4096
// keys 149.7, 136.9, 132.9, two of 100-131k 171.5, 155.4, 152.2; an 8-bit cache, 64
// of 1-8191, 100.5, 92.3, 93.6. Where what is read stays in the 256 MB last-level
// cache it costs: 288 windows of 1000 (pair form) 17.6, 19.7, 19.9, 64 short lines
// (82 MB) 25.2, 26.3, 27.6; caches of that size that are not there yet, 16 sequences
// of 500-4000 keys: 40.2, 37.2, 37.9.
template <int D, bool E4, bool PAIR, int NW, int NT>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2))) paged_attn_kernel(PAttnK p) {
  using T = PaTile<D, E4>;
  constexpr int KU = PAIR ? NW * T::KT : T::KT;  // keys of a step: of the workgroup's, or of one wave's
  constexpr int RB = T::RB, KT = T::KT, NB = T::NB, CPR = T::CPR, RPI = T::RPI;
  constexpr int NKS = D / 32, NDB = D / 16, JPR = RB / 64;  // JPR: loads per 16-key block
  constexpr int OW = PAIR ? NW * 16 * D * 4 : 0;  // the merge's o rows share the V tiles' LDS
  __shared__ __attribute__((aligned(16))) char smem[NW * T::LDS > OW ? NW * T::LDS : OW];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qc = lane & 15, g = lane >> 4;  // query column, lane group
  const int HB = p.Hkv * p.nqb;
  int me;          // pair: the pair; line: the wave's number, group by group
  int64_t u0, u1;  // the stretch; where it begins:
  int t, hb, k;    // token, kv head block, unit of the token
  int64_t steps = 0, step = 0;  // line: the barriers that the waves keep step with
  Span sp;
  if constexpr (PAIR) {
    me = blockIdx.x;
    if (p.turn) {  // the heads of a token on one XCD (workgroups go to the eight in turn)
      const int at = me / p.turn * p.turn, i = me - at;
      if (at + p.turn <= (int)gridDim.x) me = at + (i & 7) * HB + (i >> 3);
    }
    t = me / HB;
    hb = me - t * HB;
    k = 0;
    sp = span_of<KU>(p, t);
    u0 = 0;
    u1 = sp.units;
    if (u1 == 0) {
      const int kvh = hb / p.nqb, qb = hb - kvh * p.nqb, gn = min(p.gq, p.G - qb * 16);
      for (int e = tid; e < gn * D; e += 64 * NW) p.o[(int64_t)t * p.ldo + (int64_t)(kvh * p.G + qb * 16) * D + e] = 0;
      return;
    }
  } else {
    const int groups = (int)gridDim.x * NW / HB;
    int64_t at;  // tiles before token t
    // no step to keep (a tile a wave at most): neighbours on different CUs, so
    // that few tiles spread out
    auto deal = [&](int64_t total) {
      const Share share(total, groups);
      if (share.each) steps = share.each + (share.more != 0);
      me = steps ? (int)blockIdx.x * NW + wave : wave * (int)gridDim.x + (int)blockIdx.x;
      const int group = me / HB;
      hb = me - group * HB;
      u0 = share.begin(group);
      u1 = group < groups ? share.begin(group + 1) : u0;
    };
    if (p.tokens <= 64) {  // a token a lane: every wave counts for itself
      const int i = min(lane, p.tokens - 1);
      const int pos = p.positions[i], row = p.rows ? p.rows[i] : i;
      const uint32_t n = lane < p.tokens ? span_from<KU>(p, pos, row).units : 0;
      uint32_t inc = n;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t up = __shfl_up(inc, d);
        if (lane >= d) inc += up;
      }
      const uint32_t total = __builtin_amdgcn_readlane(inc, 63);
      if (blockIdx.x == 0 && wave == 0) {  // for the join kernel
        if (lane < p.tokens) p.prefix[lane] = inc - n;
        if (lane == 0) p.prefix[p.tokens] = total;
      }
      deal(total);
      t = __popcll(__ballot(lane < p.tokens && inc - n <= u0)) - 1;  // the last that begins at or before u0
      at = (uint32_t)__builtin_amdgcn_readlane(inc - n, t);
      sp = span_from<KU>(p, __builtin_amdgcn_readlane(pos, t), __builtin_amdgcn_readlane(row, t));
    } else {
      __shared__ int64_t pre[64 * NW + 1];  // tiles before each of 64 NW runs of tokens
      __shared__ int64_t wsum[NW];
      const int per = (p.tokens + 64 * NW - 1) / (64 * NW);
      int64_t n = 0;
      const int t0 = min(p.tokens, tid * per), t1 = min(p.tokens, t0 + per);
      for (int i = t0; i < t1; ++i) n += span_of<KU>(p, i).units;
      int64_t inc = n;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int64_t up = __shfl_up(inc, d);
        if (lane >= d) inc += up;
      }
      if (lane == 63) wsum[wave] = inc;
      __syncthreads();
      int64_t before = inc - n;
      for (int w = 0; w < wave; ++w) before += wsum[w];
      pre[tid] = before;
      if (tid == 64 * NW - 1) pre[64 * NW] = before + n;
      if (blockIdx.x == 0) {
        int64_t sum = before;
        for (int i = t0; i < t1; ++i) {
          p.prefix[i] = sum;
          sum += span_of<KU>(p, i).units;
        }
        if (tid == 64 * NW - 1) p.prefix[p.tokens] = before + n;
      }
      __syncthreads();
      deal(pre[64 * NW]);
      int run = -1;  // the last run that begins at or before u0
      for (int i = 0; i < NW; ++i) run += __popcll(__ballot(pre[64 * i + lane] <= u0));
      t = run * per;
      at = pre[run];
      if (u0 < u1) {
        sp = span_of<KU>(p, t);
        while (at + sp.units <= u0 && t < p.tokens - 1) {
          at += sp.units;
          sp = span_of<KU>(p, ++t);
        }
      }
    }
    if (u0 >= u1) {
      for (; step < steps; ++step) keep_step(step);
      return;
    }
    k = (int)(u0 - at);
  }
  int64_t u = u0;
  t = __builtin_amdgcn_readfirstlane(t);
  hb = __builtin_amdgcn_readfirstlane(hb);
  k = __builtin_amdgcn_readfirstlane(k);

  char* sv = smem + wave * T::LDS;
  // V: lane's row and chunk within one load instruction
  const int lr = lane / CPR, lc = lane % CPR;
  // V^T operand reads: this lane is source lane 4 e + j of group g, reading row
  // 4 g + e (and 16 + 4 g + e) of a 32-key block, columns 16 db + 4 j .. +3
  const int e4 = (lane & 15) >> 2, j4 = lane & 3;
  const int vr0 = 4 * g + e4;
  const int vxo = pa_sw<D>(vr0) >> 1;
  const char* rv = sv + vr0 * D * 2 + ((j4 >> 1) ^ (pa_sw<D>(vr0) & 1)) * 16 + (j4 & 1) * 8;

  // ---- the load cursor (t, k; sp): one tile ahead of the computation, also over the
  // ends of tokens
  // (the next token's position and row wait in vector registers: a scalar copy
  // would make the compiler wait for them where they are loaded)
  const int last_t = p.tokens - 1;
  int vzero = 0;
  asm volatile("" : "+v"(vzero));
  int npos, nrow = 0;
  auto load_next = [&]() {
    const int at_ = min(t + 1, last_t) + vzero;
    npos = p.positions[at_];
    if (p.rows) nrow = p.rows[at_];
  };
  load_next();
  // page numbers p0 .. p0 + 63 of the row, one a lane (-1: not in the cache)
  int p0 = 1 << 30, ids = -1;
  unsigned okbits = 0;  // bit b: block b of the loaded tile is in the cache
  pa_u32x4 kr[8], vr[8];
  auto load = [&]() {
    const int kvh = hb / p.nqb;
    const char* kb = p.k + (int64_t)kvh * p.kh;
    const char* vb = p.v + (int64_t)kvh * p.vh;
    const int j0 = sp.base + (PAIR ? NW * k + wave : k) * KT;
    okbits = 0;
    if (j0 >= sp.hi) return;  // past the pair's end: this wave sits the unit out
    const int first = j0 >> p.pshift, last = (min(j0 + KT, sp.hi) - 1) >> p.pshift;
    if (first < p0 || last - p0 >= 64) {
      p0 = first;
      const int at_ = p0 + lane;
      ids = at_ < p.row_pages ? p.table[(int64_t)sp.row * p.ldt + at_] : -1;
      if (ids >= p.pages) ids = -1;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int jb = j0 + 16 * b;
      const int id = __builtin_amdgcn_readlane(ids, ((jb >> p.pshift) - p0) & 63);
      const int in = jb & ((1 << p.pshift) - 1);
      const int rows = min(16, sp.hi - jb);       // rows of this block below hi
      const bool ok = id >= 0 && rows > 0;
      okbits |= (ok ? 1u : 0u) << b;
      const char* kpage = kb + (int64_t)(ok ? id : 0) * p.kp + (int64_t)in * p.kt;
      const char* vpage = vb + (int64_t)(ok ? id : 0) * p.vp + (int64_t)in * p.vt;
      const auto kres = __builtin_amdgcn_make_buffer_rsrc((void*)kpage, 0, ok ? (int)((rows - 1) * p.kt) + RB : 0, 0x00020000);
      const auto vres = __builtin_amdgcn_make_buffer_rsrc((void*)vpage, 0, ok ? (int)((rows - 1) * p.vt) + RB : 0, 0x00020000);
#pragma unroll
      for (int i = 0; i < JPR; ++i) {
        const int r = i * RPI + lr;
        const int off = jb + r >= sp.lo ? r * (int)p.vt + 16 * lc : 0x7ffffff0;
        const int koff = E4 ? qc * (int)p.kt + 64 * i + 16 * g : r * (int)p.kt + 16 * lc;
        kr[b * JPR + i] =
            __builtin_bit_cast(pa_u32x4, __builtin_amdgcn_raw_buffer_load_b128(kres, koff, 0, NT > 1 ? 2 : 0));
        vr[b * JPR + i] = __builtin_bit_cast(pa_u32x4, __builtin_amdgcn_raw_buffer_load_b128(vres, off, 0, NT ? 2 : 0));
      }
    }
  };
  // the pair's queries and scalars; a column past its heads repeats the last one
  // (no lane depends on another's column, and none of them is stored)
  bf16x8_t qn[NKS];
  float kscale_n = 1.f, slope_n = 0.f;
  auto load_pair = [&]() {
    const int kvh = hb / p.nqb, qb = hb - kvh * p.nqb;
    const int head = kvh * p.G + qb * 16 + min(qc, min(p.gq, p.G - qb * 16) - 1);
    const uint16_t* qrow = p.q + (int64_t)t * p.ldq + (int64_t)head * D;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
      qn[ks] = *(const bf16x8_t*)(qrow + (E4 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g));
    if (p.ks) kscale_n = p.ks[kvh];
    if (p.slopes) slope_n = p.slopes[head];
  };

  bf16x8_t qf[NKS];
  f32x4_t oacc[NDB];
  float m_run = 0.f, r_run = 0.f, l_run = 0.f, mul = 0.f, slope = 0.f;
  // capped: softcap log2(e) tanh(mul s / (2 log2(e))), else mul s
  const bool cap = p.softcap > 0.f;
  const float mul0 = p.scale * (cap ? 2.f * kLog2e / p.softcap : kLog2e);
  const float capl = p.softcap * kLog2e;
  int k_begin = 0;
  int64_t u_begin = u0;
  bool fresh = true;
  load();
  load_pair();
  for (;;) {
    // ---- one unit of pair (ct, hb)
    const int ct = t, ck = k;
    const Span cs = sp;
    const unsigned ok = okbits;
    const int j0 = cs.base + (PAIR ? NW * ck + wave : ck) * KT;
    const bool busy = j0 < cs.hi;
    if (fresh) {
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) qf[ks] = qn[ks];
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) oacc[d][r] = 0.f;
      m_run = r_run = -INFINITY;
      l_run = 0.f;
      mul = mul0 * kscale_n;
      slope = slope_n * kLog2e;
      k_begin = ck;
      u_begin = u;
    }
    f32x4_t s[NB];
    auto stage_k = [&]() {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * RPI + lr;
        *(pa_u32x4*)(sv + r * RB + ((lc ^ pa_ksw<CPR>(r)) << 4)) = kr[i];
      }
    };
    auto stage_v = [&]() {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * RPI + lr;
        if constexpr (E4) {
          const int at_ = ((2 * lc) ^ pa_sw<D>(r)) << 4;
          *(f16x8_t*)(sv + r * D * 2 + at_) = e4m3x8_to_f16(vr[i][0], vr[i][1]);
          *(f16x8_t*)(sv + r * D * 2 + (at_ ^ 16)) = e4m3x8_to_f16(vr[i][2], vr[i][3]);
        } else {
          *(pa_u32x4*)(sv + r * D * 2 + ((lc ^ pa_sw<D>(r)) << 4)) = vr[i];
        }
      }
    };
    if (busy) {
      pa_lds_order();  // the tile before has been read
      if constexpr (E4) stage_v();
      else stage_k();
      pa_lds_order();
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[b][r] = 0.f;
#pragma unroll
        for (int j = 0; j < JPR; ++j) {
          const int row = 16 * b + qc;
          const pa_u32x4 x = E4 ? kr[b * JPR + j] : *(const pa_u32x4*)(sv + row * RB + (((4 * j + g) ^ pa_ksw<CPR>(row)) << 4));
          if constexpr (E4) {
            s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3x8_to_bf16(x[0], x[1]), qf[2 * j], s[b], 0, 0, 0);
            s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3x8_to_bf16(x[2], x[3]), qf[2 * j + 1], s[b], 0, 0, 0);
          } else {
            s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x), qf[j], s[b], 0, 0, 0);
          }
        }
      }
      if constexpr (!E4) {
        pa_lds_order();  // a wave's LDS accesses complete in order: V may replace K
        stage_v();
      }
    }
    ++u;
    const bool more = u < u1, ends = !more || ck + 1 == cs.units;
    if (more) {
      if (++k == sp.units) {
        k = 0;
        ++t;
        sp = span_from<KU>(p, __builtin_amdgcn_readfirstlane(npos), p.rows ? __builtin_amdgcn_readfirstlane(nrow) : t);
        while (sp.units == 0 && t < last_t) sp = span_of<KU>(p, ++t);
        load_next();
        p0 = 1 << 30;
      }
      load();
      if (ends) load_pair();
    }
    if (busy) {
      pa_lds_order();

      // scores in log2 units; this lane holds keys 16 b + 4 g + r of column qc
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = s[b][r] * mul;
          if (cap) x = capl - 2.f * capl * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x));
          s[b][r] = x;
        }
      if (p.slopes) {  // from the last key: what lies between it and pos is the same for all
        const float far = slope * (float)(cs.hi - 1 - j0 - 4 * g);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[b][r] = fmaf(slope, (float)(16 * b + r), s[b][r] - far);
      }
      if (j0 < cs.lo || j0 + KT > cs.hi || ok != (1u << NB) - 1) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = j0 + 16 * b + 4 * g + r;
            if (j < cs.lo || j >= cs.hi || !(ok >> b & 1)) s[b][r] = -INFINITY;
          }
      }
      float mloc = -INFINITY;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) mloc = fmaxf(mloc, s[b][r]);
      mloc = fmaxf(mloc, __shfl_xor(mloc, 16));
      mloc = fmaxf(mloc, __shfl_xor(mloc, 32));
      const float m_new = fmaxf(m_run, mloc);
      const float r_new = T::from(m_new), r_use = m_new == -INFINITY ? 0.f : r_new;
      const float alpha = __builtin_amdgcn_exp2f(r_run - r_use);
      m_run = m_new;
      r_run = r_new;
      float lsum = 0.f;
      typename T::V8 pf[NB / 2];
      bf16x8_t pl[NB / 2];  // bf16: the halves that pf leaves over
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 4 * (b & 1) + r;
          const float e = __builtin_amdgcn_exp2f(s[b][r] - r_use);
          lsum += e;
          if constexpr (E4) {
            pf[b / 2][i] = (_Float16)e;
          } else {
            const __bf16 h = (__bf16)(e * 0.99609375f);  // 1 - 2^-8: less than e when rounded
            pf[b / 2][i] = h;
            pl[b / 2][i] = (__bf16)(e - (float)h);
          }
        }
      l_run = l_run * alpha + lsum;
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) oacc[d][r] *= alpha;
#pragma unroll
      for (int b = 0; b < NB / 2; ++b)
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const char* x = rv + b * 32 * D * 2 + ((db ^ vxo) << 5);
          const pa_s16x4 vlo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s16x4*)x);
          const pa_s16x4 vhi =
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s16x4*)(x + 16 * D * 2));
          const auto vf =
              __builtin_bit_cast(typename T::V8, __builtin_shufflevector(vlo, vhi, 0, 1, 2, 3, 4, 5, 6, 7));
          if constexpr (E4) {
            oacc[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[b], oacc[db], 0, 0, 0);
          } else {
            oacc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[b], oacc[db], 0, 0, 0);
            oacc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl[b], oacc[db], 0, 0, 0);
          }
        }
    }
    if (step < steps) {
      keep_step(step);
      ++step;
    }
    fresh = ends;
    if (!ends) continue;

    // ---- the pair's result here: the output, or a part for the join
    float l = l_run + __shfl_xor(l_run, 16);
    l += __shfl_xor(l, 32);
    const int kvh = hb / p.nqb, qb = hb - kvh * p.nqb;
    const int gn = min(p.gq, p.G - qb * 16);
    const float vscale = p.vs ? p.vs[kvh] : 1.f;
    uint16_t* o = p.o + (int64_t)ct * p.ldo + (int64_t)(kvh * p.G + qb * 16) * D;
    auto put4 = [&](uint16_t* at, const f32x4_t x, float f) {
      if (p.o8) {
        *(uint2*)at = make_uint2(pk_bf16x2(x[0] * f, x[1] * f), pk_bf16x2(x[2] * f, x[3] * f));
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) at[r] = f32_to_bf16(x[r] * f);
      }
    };
    if constexpr (PAIR) {  // one pair, one result: the waves are merged
      __shared__ float mw[NW][16], lw[NW][16];
      float(*ow)[16][D] = (float(*)[16][D])smem;
      lds_barrier();  // every wave is done with its V tile
      if (qc < gn) {
        if (g == 0) {
          mw[wave][qc] = r_run;
          lw[wave][qc] = l;
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) *(f32x4_t*)&ow[wave][qc][16 * db + 4 * g] = oacc[db];
      }
      lds_barrier();
      for (int e = tid; e < gn * (D / 4); e += 64 * NW) {
        const int c = e / (D / 4), d4 = e % (D / 4) * 4;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) mx = fmaxf(mx, mw[w][c]);
        const float mu = mx == -INFINITY ? 0.f : mx;
        float lt = 0.f;
        f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float f = __builtin_amdgcn_exp2f(mw[w][c] - mu);
          const f32x4_t y = *(const f32x4_t*)&ow[w][c][d4];
          lt += lw[w][c] * f;
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] += y[r] * f;
        }
        put4(o + c * D + d4, x, lt == 0.f ? 0.f : vscale / lt);
      }
    } else if (qc < gn) {
      if (k_begin == 0 && ck + 1 == cs.units) {
#pragma unroll
        for (int db = 0; db < NDB; ++db) put4(o + qc * D + 16 * db + 4 * g, oacc[db], l == 0.f ? 0.f : vscale / l);
      } else {
        const int64_t slot = (int64_t)(2 * me + (u_begin != u0)) * p.gq + qc;
        if (g == 0) {
          p.ml[2 * slot] = r_run;
          p.ml[2 * slot + 1] = l;
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) *(f32x4_t*)(p.part + slot * D + 16 * db + 4 * g) = oacc[db];
      }
    }
    if (!more) break;
  }
  for (; step < steps; ++step) keep_step(step);
}

// Joins the parts of hw heads of one (token, kv head) pair: o = sum_i o_i
// 2^(m_i - m) / sum_i l_i 2^(m_i - m). Tokens without keys get zeros; pairs that
// one wave finished are left alone.
// A workgroup takes DS of the dims: rows in 256 / (DS / 4) slices.
template <int D, int DS>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(PAttnK p, int waves, int hw) {
  constexpr int LPR = DS / 4, NG = 256 / LPR;  // lanes per row, rows at a time
  __shared__ f32x4_t os[NG][LPR];
  __shared__ float ms[NG], ls[NG];
  const int HB = p.Hkv * p.nqb, per = (p.gq + hw - 1) / hw;  // workgroups per pair
  const int d0 = blockIdx.x % (D / DS) * DS, bx = blockIdx.x / (D / DS);
  const int hb = bx / per, c0 = (bx - hb * per) * hw, t = blockIdx.y, tid = threadIdx.x;
  const int kvh = hb / p.nqb, qb = hb - kvh * p.nqb, gn = min(p.gq, p.G - qb * 16);
  const int64_t a = p.prefix[t], tiles = p.prefix[t + 1] - a, all = p.prefix[p.tokens];
  uint16_t* o = p.o + (int64_t)t * p.ldo + (int64_t)(kvh * p.G + qb * 16) * D;
  if (tiles == 0) {
    for (int e = tid; e < (min(gn, c0 + hw) - c0) * DS; e += 256) o[(c0 + e / DS) * D + d0 + e % DS] = 0;
    return;
  }
  const Share share(all, waves / HB);
  const int g0 = share.owner(a), n = share.owner(a + tiles - 1) - g0 + 1;
  if (n == 1) return;
  const bool late = a != share.begin(g0);  // part 0 is its wave's last segment, not its first
  const float vscale = p.vs ? p.vs[kvh] : 1.f;
  // rows at a time: hw heads, and as many slices of the parts as that leaves
  const int grp = tid / LPR, ln = tid - grp * LPR;
  const int slices = NG / hw, slice = grp / hw, c = c0 + grp - slice * hw;
  float m = -INFINITY, l = 0.f;
  f32x4_t x = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float mi, float li, const f32x4_t y) {
    const float mn = fmaxf(m, mi), mu = mn == -INFINITY ? 0.f : mn;
    const float fo = __builtin_amdgcn_exp2f(m - mu), fi = __builtin_amdgcn_exp2f(mi - mu);
    m = mn;
    l = l * fo + li * fi;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = x[r] * fo + y[r] * fi;
  };
  if (c < gn && slice < slices) {
#pragma unroll 8
    for (int i = slice; i < n; i += slices) {
      const int64_t s = (int64_t)(2 * ((g0 + i) * HB + hb) + (i == 0 && late)) * p.gq + c;
      add(p.ml[2 * s], p.ml[2 * s + 1], *(const f32x4_t*)(p.part + s * D + d0 + 4 * ln));
    }
  }
  if (hw == 1) {  // every row is a slice of one head: those of a wave by shuffles
#pragma unroll
    for (int d = LPR; d < 64; d <<= 1) {
      f32x4_t y;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = __shfl_xor(x[r], d);
      add(__shfl_xor(m, d), __shfl_xor(l, d), y);
    }
  }
  os[grp][ln] = x;
  if (ln == 0) {
    ms[grp] = m;
    ls[grp] = l;
  }
  __syncthreads();
  if (slice != 0 || c >= gn) return;
  const int next = hw == 1 ? 64 / LPR : hw;  // rows apart: one a wave, or one a slice
  for (int i = next; i + grp < (hw == 1 ? NG : slices * hw); i += next) add(ms[i + grp], ls[i + grp], os[i + grp][ln]);
  const float f = l == 0.f ? 0.f : vscale / l;
#pragma unroll
  for (int r = 0; r < 4; ++r) o[c * D + d0 + 4 * ln + r] = f32_to_bf16(x[r] * f);
}

// pair: 0, the line form, or the waves of a pair's workgroup. nt: past the caches.
template <int D, bool E4>
static void launch_paged_as(const PAttnK& k, int pair, bool nt, unsigned grid, hipStream_t s) {
  constexpr int kPast = E4 ? 1 : 2;
  const dim3 g(grid), b(64 * (pair ? pair : kLineWaves));
  if (pair == 0 && nt) hipLaunchKernelGGL((paged_attn_kernel<D, E4, false, kLineWaves, kPast>), g, b, 0, s, k);
  else if (pair == 0) hipLaunchKernelGGL((paged_attn_kernel<D, E4, false, kLineWaves, 1>), g, b, 0, s, k);
  else if (pair == 8) hipLaunchKernelGGL((paged_attn_kernel<D, E4, true, 8, 0>), g, b, 0, s, k);
  else if (pair == 4 && nt) hipLaunchKernelGGL((paged_attn_kernel<D, E4, true, 4, kPast>), g, b, 0, s, k);
  else if (pair == 4) hipLaunchKernelGGL((paged_attn_kernel<D, E4, true, 4, 0>), g, b, 0, s, k);
  else if (pair == 2) hipLaunchKernelGGL((paged_attn_kernel<D, E4, true, 2, 0>), g, b, 0, s, k);
  else if (nt) hipLaunchKernelGGL((paged_attn_kernel<D, E4, true, 1, kPast>), g, b, 0, s, k);
  else hipLaunchKernelGGL((paged_attn_kernel<D, E4, true, 1, 0>), g, b, 0, s, k);
}

static void launch_paged(const PAttnK& k, int head_dim, bool e4, int pair, bool nt, unsigned grid, hipStream_t s) {
  if (head_dim == 128) {
    if (e4) launch_paged_as<128, true>(k, pair, nt, grid, s);
    else launch_paged_as<128, false>(k, pair, nt, grid, s);
  } else {
    if (e4) launch_paged_as<64, true>(k, pair, nt, grid, s);
    else launch_paged_as<64, false>(k, pair, nt, grid, s);
  }
}

// One workgroup of eight waves per CU.
static int line_grid() { return device_cus() > 0 ? device_cus() : 256; }

}  // namespace th

using namespace th;

// The most tiles that a pair can have, by its table and window.
static int64_t most_tiles(int64_t max_keys, int window, int row_bytes) {
  const int64_t keys = window ? std::min<int64_t>(max_keys, (int64_t)window + 15) : max_keys;
  return cdiv(keys * row_bytes, 8192);
}

// Whether pairs take the pair form. In a graph, us, pair against line form, lengths
// of half to all of the room, one token all of it (bf16, 128 dims, 8 kv heads, 4
// query heads each):
//   tiles of room      16            32            64
//     8 pairs       8.3 /  9.2   11.5 /  9.4   19.1 / 10.3
//   128 pairs      10.1 / 14.3   15.2 / 20.8   24.0 / 28.3
//   512 pairs      20.8 / 28.7   38.2 / 44.0   73.3 / 74.9
//  2048 pairs      69.8 / 81.2    130 /  141    255 /  259
// and with an e4m3 cache at 32 tiles 16.4 / 9.8 for 8 pairs, 18.5 / 22.0 for 128.
// 64 tiles and more stay with the line: lengths are not known here, and one full
// row among short ones would cost the pair form 20 us where the line takes 9.
static bool pair_form(int64_t tiles, int64_t pairs) { return tiles <= 16 || (tiles <= 32 && pairs >= 128); }

// Waves of a pair's workgroup: as many as the pair can have tiles, while the CUs
// (eight waves each) hold all pairs at once. us with 4, 2, 1 waves, bf16, 128 dims:
//   tiles of room          1                  2                   4                   8
//   512 pairs       6.0  5.5  5.2      6.4  5.9  6.6      9.1  9.1 10.9     12.7 13.8 17.5
//   768 pairs       9.2  5.8  5.4     10.0  7.4  8.0     13.0 11.2 12.6     18.3 16.7 19.6
//  2048 pairs      18.9 12.9  9.2     20.3 15.5 13.5     24.5 22.6 21.4     41.6 44.9 37.1
// Past 8 tiles 8 waves where there is a CU for each pair (256 pairs, 16 tiles of
// e4m3: 15.9 against 17.0 with 4, 32 tiles 24.6 against 26.8), else 4.
static int pair_waves(int64_t tiles, int64_t pairs) {
  const int64_t cus = line_grid();
  if (tiles > 8) return pairs <= cus ? 8 : 4;
  int w = tiles > 2 ? 4 : (int)tiles;
  while (w > 1 && pairs * w > 8 * cus) w >>= 1;
  return w;
}

extern "C" int64_t th_paged_attention_workspace_bytes(int32_t tokens, int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                                                       int32_t cache_dtype, int64_t max_keys, int32_t window) {
  if (tokens < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv || (head_dim != 64 && head_dim != 128) ||
      (cache_dtype != TH_BF16 && cache_dtype != TH_F8E4M3) || max_keys <= 0 || max_keys >= (int64_t)1 << 30 || window < 0)
    return -1;
  const int g = heads_q / heads_kv, row_bytes = head_dim * (cache_dtype == TH_BF16 ? 2 : 1);
  if (tokens == 0 || pair_form(most_tiles(max_keys, window, row_bytes), (int64_t)tokens * heads_kv * cdiv(g, 16))) return 0;
  const int64_t gq = std::min(g, 16), slots = (int64_t)line_grid() * kLineWaves * 2;
  return cdiv((int64_t)(tokens + 1) * 8, 16) * 16 + cdiv(slots * gq * 2 * 4, 16) * 16 + slots * gq * head_dim * 4;
}

extern "C" int th_paged_attention(const th_paged_attn_desc* d, void* stream) {
  TH_CHECK_ARG(d != nullptr, "th_paged_attention: null descriptor");
  TH_CHECK_ARG(d->tokens >= 0 && d->tokens <= 65535, "th_paged_attention: tokens %d out of range", d->tokens);
  TH_CHECK_ARG(d->heads_q > 0 && d->heads_kv > 0 && d->heads_q % d->heads_kv == 0,
               "th_paged_attention: heads_q=%d must be a multiple of heads_kv=%d", d->heads_q, d->heads_kv);
  TH_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128, "th_paged_attention: head_dim %d unsupported", d->head_dim);
  TH_CHECK_ARG(d->cache_dtype == TH_BF16 || d->cache_dtype == TH_F8E4M3, "th_paged_attention: cache_dtype %d unsupported",
               d->cache_dtype);
  TH_CHECK_ARG(d->page_size >= 16 && (d->page_size & (d->page_size - 1)) == 0,
               "th_paged_attention: page_size %d must be a power of two of at least 16", d->page_size);
  TH_CHECK_ARG(d->n_rows > 0 && d->row_pages > 0 && d->pages > 0 && d->ld_page_table >= d->row_pages,
               "th_paged_attention: bad page table sizes");
  TH_CHECK_ARG((int64_t)d->row_pages * d->page_size < (int64_t)1 << 30, "th_paged_attention: row of 2^30 keys or more");
  // The capped score's error is 1e-7 of the cap (its tanh is 1 - 2 / (1 + e^2x)): up
  // to here 1e-4, a fortieth of what rounding p to bf16 does.
  TH_CHECK_ARG(d->window >= 0 && (d->softcap == 0.f || (d->softcap >= 0x1p-20f && d->softcap <= 1024.f)),
               "th_paged_attention: window %d must not be negative, softcap %g 0 or in 2^-20..1024", d->window,
               (double)d->softcap);
  const int64_t row = (int64_t)d->heads_q * d->head_dim;
  TH_CHECK_ARG(d->ld_q >= row && d->ld_o >= row, "th_paged_attention: q/o row strides smaller than heads_q*head_dim");
  TH_CHECK_ARG(d->q != d->o || d->ld_q == d->ld_o || d->tokens <= 1, "th_paged_attention: in place needs one row stride");
  const int per = d->cache_dtype == TH_BF16 ? 8 : 16;  // elements in 16 bytes
  TH_CHECK_ARG(d->k_stride_h >= d->head_dim && d->v_stride_h >= d->head_dim && d->k_stride_t >= d->head_dim &&
                   d->v_stride_t >= d->head_dim && d->k_stride_page >= d->head_dim && d->v_stride_page >= d->head_dim,
               "th_paged_attention: cache stride < head_dim");
  TH_CHECK_ARG(d->ld_q % 8 == 0 && d->k_stride_h % per == 0 && d->v_stride_h % per == 0 && d->k_stride_t % per == 0 &&
                   d->v_stride_t % per == 0 && d->k_stride_page % per == 0 && d->v_stride_page % per == 0,
               "th_paged_attention: q and cache strides must be multiples of 16 bytes");
  TH_CHECK_ARG(d->k_stride_t < (1 << 22) && d->v_stride_t < (1 << 22) &&
                   d->k_stride_t * d->page_size < (int64_t)1 << 30 && d->v_stride_t * d->page_size < (int64_t)1 << 30,
               "th_paged_attention: token strides must be under 2^22 elements and 2^30 per page");
  TH_CHECK_ARG((((uintptr_t)d->q | (uintptr_t)d->k_cache | (uintptr_t)d->v_cache) & 15) == 0,
               "th_paged_attention: q and caches must be 16-byte aligned");
  TH_CHECK_ARG((!d->k_scale && !d->v_scale) || d->cache_dtype == TH_F8E4M3,
               "th_paged_attention: scales need an e4m3 cache");
  if (d->tokens == 0) return TH_OK;
  TH_CHECK_ARG(d->heads_kv * cdiv(d->heads_q / d->heads_kv, 16) <= std::min(256, line_grid() * kLineWaves),
               "th_paged_attention: more than 256 kv heads (each block of 16 query heads counts)");
  TH_CHECK_ARG(d->rows || d->tokens <= d->n_rows, "th_paged_attention: %d tokens without rows exceed the table's %d",
               d->tokens, d->n_rows);
  TH_CHECK_ARG(d->q && d->k_cache && d->v_cache && d->o && d->positions && d->page_table,
               "th_paged_attention: null tensor pointer");
  const int64_t need = th_paged_attention_workspace_bytes(
      d->tokens, d->heads_q, d->heads_kv, d->head_dim, d->cache_dtype, (int64_t)d->row_pages * d->page_size, d->window);
  TH_CHECK_ARG(need == 0 || (d->workspace && ((uintptr_t)d->workspace & 15) == 0 && d->workspace_bytes >= need),
               "th_paged_attention: workspace %lld < %lld bytes, or not 16-byte aligned", (long long)d->workspace_bytes,
               (long long)need);
  if (!device_ready()) {
    set_error("th_paged_attention: th_init was not called for the current device");
    return TH_ERR_NOT_INIT;
  }
  PAttnK k{};
  k.q = (const uint16_t*)d->q; k.ldq = d->ld_q;
  const int64_t es = d->cache_dtype == TH_BF16 ? 2 : 1;
  k.k = (const char*)d->k_cache; k.kp = d->k_stride_page * es; k.kt = d->k_stride_t * es; k.kh = d->k_stride_h * es;
  k.v = (const char*)d->v_cache; k.vp = d->v_stride_page * es; k.vt = d->v_stride_t * es; k.vh = d->v_stride_h * es;
  k.o = (uint16_t*)d->o; k.ldo = d->ld_o;
  k.positions = d->positions; k.rows = d->rows; k.table = d->page_table; k.ldt = d->ld_page_table; k.pages = d->pages;
  k.n_rows = d->n_rows; k.row_pages = d->row_pages; k.pshift = __builtin_ctz((unsigned)d->page_size);
  k.tokens = d->tokens; k.Hkv = d->heads_kv; k.G = d->heads_q / d->heads_kv;
  k.gq = std::min(k.G, 16); k.nqb = (int)cdiv(k.G, 16);
  k.o8 = d->ld_o % 4 == 0 && ((uintptr_t)d->o & 7) == 0;
  k.window = d->window; k.scale = d->scale; k.softcap = d->softcap;
  k.slopes = d->slopes; k.ks = d->k_scale; k.vs = d->v_scale;
  const int grid = line_grid(), waves = grid * kLineWaves;
  char* ws = (char*)d->workspace;
  k.prefix = (int64_t*)ws;
  ws += cdiv((int64_t)(d->tokens + 1) * 8, 16) * 16;
  k.ml = (float*)ws;
  ws += cdiv((int64_t)waves * 2 * k.gq * 8, 16) * 16;
  k.part = (float*)ws;
  hipStream_t s = (hipStream_t)stream;
  const bool e4 = d->cache_dtype == TH_F8E4M3;
  const int64_t pairs = (int64_t)d->tokens * d->heads_kv * k.nqb;  // below 2^24
  const int64_t tiles = most_tiles((int64_t)d->row_pages * d->page_size, d->window, (int)(d->head_dim * es));
  if (pair_form(tiles, pairs)) {
    // Heads of a token side by side on one XCD, whose L2 they share: where a row is half
    // a 128-byte line (the other half is the next head's), and from 512 MB on, where
    // neighbours are read together. us, in order and so: 64-byte rows of 512 pairs, 16
    // tiles 36.8 / 27.0, of 5600 pairs, 32 tiles 679 / 477; 128-byte rows of 2048 pairs,
    // 32 tiles 152 / 143, of 5600 pairs 388 / 341; 256-byte rows 134 / 135, 351 / 346;
    // smaller calls lose up to 5 percent: 512 pairs, 16 tiles 21.1 / 21.4.
    k.turn = d->head_dim * es < 128 || pairs * tiles >= (512 << 20) / 16384 ? 8 * d->heads_kv * k.nqb : 0;
    launch_paged(k, d->head_dim, e4, pair_waves(tiles, pairs), pairs * tiles > (128 << 20) / 16384, (unsigned)pairs, s);
    TH_CHECK_LAUNCH();
    return TH_OK;
  }
  // the most that the call can read: K goes past the caches where that does not fit them
  const int64_t room = std::min(d->pages * d->page_size * d->heads_kv * 2 * d->head_dim * es, pairs * tiles * 16384);
  launch_paged(k, d->head_dim, e4, 0, room > (256 << 20), (unsigned)grid, s);
  TH_CHECK_LAUNCH();
  // Few pairs can be cut into many parts: a workgroup for each head, and for very
  // few one for each 32 dims of it, reads more of them at once.
  const int hw = pairs < 256 ? 1 : std::min(k.gq, 1024 / d->head_dim);
  const bool few = pairs * k.gq <= 128;
  const int split = few ? d->head_dim / 32 : 1;
  const dim3 join((unsigned)(d->heads_kv * k.nqb * cdiv(k.gq, hw) * split), (unsigned)d->tokens);
  if (d->head_dim == 128) {
    if (few) hipLaunchKernelGGL((paged_attn_join_kernel<128, 32>), join, dim3(256), 0, s, k, waves, hw);
    else hipLaunchKernelGGL((paged_attn_join_kernel<128, 128>), join, dim3(256), 0, s, k, waves, hw);
  } else {
    if (few) hipLaunchKernelGGL((paged_attn_join_kernel<64, 32>), join, dim3(256), 0, s, k, waves, hw);
    else hipLaunchKernelGGL((paged_attn_join_kernel<64, 64>), join, dim3(256), 0, s, k, waves, hw);
  }
  TH_CHECK_LAUNCH();
  return TH_OK;
}
