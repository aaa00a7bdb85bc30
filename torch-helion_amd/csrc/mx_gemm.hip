// th_mx_gemm: microscaled activations (e4m3 or e2m1) times e2m1 weights, both in
// blocks of 32 along k (no counterpart in the reference).
//
// out[m, n] = sum_b 2^(sa[m, b] + sw[n, b] - 254) sum_{i < 32} a[m, 32 b + i] w[n, 32 b + i]:
// gfx950's scaled MFMAs take the elements as they are stored and both scale
// bytes, so nothing is converted on the way. Weights are the first operand: a
// lane then holds four consecutive columns n of one row m.
//
// The matrix cores add the products of 16 consecutive k at the largest sum E of their operands' exponents (of subnormal
// values the least exponent; found with pairs of products, all of 8 million as this says) and cut what lies below
// 2^(E - 13). Of e2m1 activations nothing does. Of e4m3 ones E <= 8 + 2 and bits reach down to 2^-10, so that the values of 2
// and more and those below are multiplied apart, two products for one: of the former E <= 10 and the last bit is 2^-3, of
// the latter E <= 2 and 2^-10, and nothing is cut. The sums are fp32. (With one product 16384 x 4096 x 14336 took 690 us
// for 1100, 64 rows 15.2 for 15.9, and of the SwiGLU's e4m3 codes one in 18000 fell on the other side of a rounding. bf16
// products have a quarter of the rate, and both operands to convert.)
// (The 32x32x64 form has the same rate on zeros, and 3.98 against 4.73 PFLOP/s on random values.)
//
// What bounds it: with few rows the weights (64 x 4096 x 14336: 31 MB, 6 us at the 5.2 TB/s of a copy; 15.9 us, since each
// CU takes in 40 to 50 GB/s of activations and weights), with many the matrix cores and what feeds them:
// 16384 x 4096 x 14336 1100 us (1.75 PFLOP/s, of two products each 3.5), SwiGLU of 8192 x 14336 x 4096 1110 (1.73); 6001 x
// 14336 x 4096 of e2m1 235 us (3.0). Of the first the matrix cores are busy for 79 % of the cycles, at 2.15 GHz.
//
// Operand layout of v_mfma_scale_f32_16x16x128_f8f6f4: lane l supplies row l % 16;
// of e2m1 the 32 values (16 bytes) of k block g = l / 16; of e4m3 the 16 bytes from
// 16 g and the 16 bytes from 64 + 16 g; and the scale of k block g. Which block of
// the tensor stands for k block g is free as long as both operands agree: the kernels
// choose it so that a lane's pieces and scale bytes over several MFMAs lie together.
#include "mx.h"

#include <algorithm>
#include <type_traits>

namespace th {

typedef int mx_v8i __attribute__((ext_vector_type(8)));

struct MxGemmK {
  int64_t M;
  int N, nb;             // output columns (of y with swiglu), blocks along k
  const uint8_t* a; int64_t lda;
  const uint8_t* as; int64_t ldas;
  const uint8_t* w; int64_t ldw;
  const uint8_t* ws; int64_t ldws;
  const void* res; int64_t ldr;
  void* o; int64_t ldo;
  uint8_t* os; int64_t ldos;
  bool out32, e2m1;      // out in fp32; swiglu: out in e2m1
};

__device__ __forceinline__ mx_v8i mx_wide(uint4 x) { return mx_v8i{(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0}; }
__device__ __forceinline__ mx_v8i mx_wide(mx_v8i x) { return x; }
__device__ __forceinline__ mx_v8i mx_wide(uint4 x, uint4 y) {
  return mx_v8i{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, (int)y.z, (int)y.w};
}

// e4m3 values of 2 and more (exponent fields from 8 on, NaN among them) and those below, in each half zeros of their sign
// in the others' places.
__device__ __forceinline__ void mx_split(mx_v8i x, mx_v8i& large, mx_v8i& small) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t v = (uint32_t)x[i], f = v & 0x40404040u;
    const uint32_t s = v & ~(f | (f - (f >> 6)));  // (0x40 and 0x3f of a large byte)
    large[i] = (int)(v ^ (s & 0x7f7f7f7fu));
    small[i] = (int)s;
  }
}

// The sums of WAVES waves, [WAVES][ROWS][LDR] in LDS (with SWIGLU the gate's OUTS columns, then the up
// projection's), added in their order and stored: out[m0 ..][n0 ..].
template <bool SWIGLU, int ROWS, int OUTS, int LDR, int WAVES>
__device__ __forceinline__ void mx_finish(const MxGemmK& p, const float* red, int64_t m0, int n0) {
  for (int e = threadIdx.x; e < ROWS * (OUTS / 4); e += 64 * WAVES) {
    const int m = e / (OUTS / 4), n4 = e % (OUTS / 4) * 4;
    const int64_t row = m0 + m;
    f32x4_t x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      x += *(const f32x4_t*)(red + (w * ROWS + m) * LDR + n4);
      if constexpr (SWIGLU) y += *(const f32x4_t*)(red + (w * ROWS + m) * LDR + OUTS + n4);
    }
    const int left = p.N - (n0 + n4);  // columns from here on
    if constexpr (SWIGLU) {
      // eight lanes hold a block (whole blocks: N is a multiple of 32)
      float v[4];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = x[i] * sigmoidf_(x[i]) * y[i];
        top = max(top, mx_bits(v[i]));
      }
      top = mx_quad_max(top);
      top = max(top, (uint32_t)__shfl_xor((int)top, 4));
      const int s = mx_scale(top, p.e2m1);
      const int fine = s == 255 ? 127 : s;
      if (s == 255) v[0] = v[1] = v[2] = v[3] = 0.f;
      if (row >= p.M || left <= 0) continue;
      uint8_t* o = (uint8_t*)p.o + row * p.ldo;
      const int n = n0 + n4;
      if ((n & 31) == 0) p.os[row * p.ldos + (n >> 5)] = (uint8_t)s;
      if (p.e2m1) {
        const float z[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
        *(uint16_t*)(o + n / 2) = (uint16_t)mx_e2m1x8(z, mx_scale_operand(fine));
      } else {
        *(uint32_t*)(o + n) = mx_e4m3x4(v, mx_scale_operand(fine), mx_limit(fine));
      }
    } else {
      if (row >= p.M) continue;
      const int64_t at = row * p.ldo + n0 + n4, from = row * p.ldr + n0 + n4;
      if (left >= 4) {
        if (p.out32) {
          if (p.res) x += __builtin_bit_cast(f32x4_t, mx_load16((const float*)p.res + from));
          mx_store16((float*)p.o + at, __builtin_bit_cast(mx_u4, x));
        } else {
          if (p.res) {
            const uint2 u = mx_load8b((const uint16_t*)p.res + from);
            x += f32x4_t{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
          }
          mx_store8b((uint16_t*)p.o + at, make_uint2(pk_bf16x2(x[0], x[1]), pk_bf16x2(x[2], x[3])));
        }
        continue;
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        if (i >= left) break;
        float f = x[i];
        if (p.out32) {
          if (p.res) f += ((const float*)p.res)[from + i];
          ((float*)p.o)[at + i] = f;
        } else {
          if (p.res) f += bf16_to_f32(((const uint16_t*)p.res)[from + i]);
          ((uint16_t*)p.o)[at + i] = f32_to_bf16(f);
        }
      }
    }
  }
}

// Rows of whole stages of four blocks, their scales whole dwords. (Else the scales are loaded byte by byte.)
static bool mx_whole_stages(const MxGemmK& k) {
  return k.nb % 4 == 0 && (((uintptr_t)k.as | (uintptr_t)k.ws | (uint64_t)k.ldas | (uint64_t)k.ldws) & 3) == 0;
}

// Which form takes least time: what a workgroup loads over what a CU takes in (bytes a microsecond), in as many rounds as
// the workgroups need. us by form, in a graph:
//                             e4m3 activations                         e2m1
//                           ring   64x64  64x128  128x256  256x256     ring   64x64  64x128  128x256  256x256
//     1 x 6144 x 4096        5.9    15.2    19.7     40.8     71.8
//    64 x 4096 x 4096        7.1    15.4    20.5     43.2     75.7      5.5    11.3    13.2     21.8     32.1
//   128 x 4096 x 4096       12.3    15.7    20.7     44.9     76.4      9.2    11.5    14.3     26.7     34.4
//    64 x 14336 x 4096      23.4    16.6    21.0     43.8     76.5     18.6    12.4    15.3     24.3     34.1
//   256 x 4096 x 4096       23.3    16.6    21.0     45.0     78.9     17.2    12.2    14.7     26.9     38.5
//   512 x 4096 x 4096       43.2    22.8    22.1     45.3     79.7     32.2    19.6    16.0     26.9     38.4
//  1024 x 4096 x 14336     226     129     100      134      238      185     108      79.6     76.1    101
//  2048 x 4096 x 4096      156      79.4    61.5     52.2     80.9    119      64.5    48.4     32.7     40.1
//  2048 x 14336 x 4096     584     282     226      214      189      468     239     192      141      110
//   333 x 2050 x 1376       11.8     8.8    12.3     23.9   (43 blocks)
//  2048 x 4096 x 4064      180     103      81.6     59.1   (127)     133      85.4    72.7     44.4
//  8192 x 4096 x 14304            1347    1070      733     (447)
//  SwiGLU (weights 2 x)
//     1 x 14336 x 4096      15.9            20.0     40.4     71.6
//    64 x 14336 x 4096      34.0            20.5     41.4     72.2     30.9            15.7     23.0     30.1
//   256 x 14336 x 4096     113              57.0     45.0     73.8    103              44.3     27.9     34.8
//  1024 x 14336 x 4096     444             198      183      157      405             158      108       80.2
//  8192 x 14336 x 4064                    2058     1484     (127)
// Of 55 such calls the choice was the best or within 6 % of it in 50, within 14 % in the others (1000 x 4096 x 4096: 37.4, in
// tiles of 64 x 128 32.8).
static int mx_form(const MxGemmK& k, bool a4, bool swiglu) {
  const double cus = device_cus() > 0 ? device_cus() : 256, nk = (double)cdiv(k.nb, 4);
  const bool odd = !mx_whole_stages(k);
  const double ka = a4 ? 64 : 128;
  auto rounds = [&](double groups, double at_once) { return (double)cdiv((int64_t)groups, (int64_t)at_once); };
  double best = 1e30;
  int form = TH_MX_TILE_256X256;
  auto offer = [&](int f, double us) {
    if (us < best) best = us, form = f;
  };
  const int sides = swiglu ? 2 : 1;
  const double rows = (double)std::min<int64_t>(k.M, k.M <= 8 ? 8 : k.M <= 16 ? 16 : 32);
  if (k.M <= 4096) offer(TH_MX_RING, 3.0 + rounds(cdiv(k.N, 32) * cdiv(k.M, 32), cus) * nk * (rows * ka + 2200.0 * sides) / (odd ? 35e3 : 50e3));
  auto tile = [&](int f, int bm, int bn, double per_cu, double rate, double fixed) {
    const double n = (double)(cdiv(k.M, bm) * cdiv(k.N, bn / sides)), load = nk * (bm * ka + bn * 64.0 + 4.0 * (bm + bn));
    offer(f, fixed + (n <= cus ? load / rate : rounds(n, per_cu * cus) * per_cu * load / rate));
  };
  if (!swiglu) tile(TH_MX_TILE_64X64, 64, 64, 2, odd ? 33e3 : 40e3, 3);
  tile(TH_MX_TILE_64X128, 64, 128, 2, odd ? 29e3 : 40e3, 3);
  tile(TH_MX_TILE_128X256, 128, 256, 1, odd ? 25e3 : 34e3, 4);
  if (odd) return form;
  tile(TH_MX_TILE_256X256, 256, 256, 1, 33e3, 6);
  return form;
}

// ------------------------------------------------------------- tiles of many rows
// dma_load16 with 4 bytes a lane.
__device__ __forceinline__ void dma_load4(const void* base, uint32_t voff, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(base), "{m0}"(lds) : "memory");
}

// With one byte a lane, which becomes a dword.
__device__ __forceinline__ void dma_load1(const void* base, uint32_t voff, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_ubyte %0, %1" ::"v"(voff), "s"(base), "{m0}"(lds) : "memory");
}

// The same two with an address a lane.
__device__ __forceinline__ void dma_load4_at(const void* at, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(at), "{m0}"(lds) : "memory");
}

__device__ __forceinline__ void dma_load1_at(const void* at, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_ubyte %0, off" ::"v"(at), "{m0}"(lds) : "memory");
}

// The compiler moves no memory access across this point.
__device__ __forceinline__ void mx_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Output tile of a workgroup: XCD x (workgroups x, x + 8, ...) takes one contiguous range of
// tiles, four tile rows at a time: of the lines that its 32 workgroups load a stage, those of a
// count twice those of w (e4m3), so that 4 x 8 tiles load fewest (16384 x 4096 x 14336 with one product for all of an
// e4m3 value: 720 us, with eight tile rows 733, with two 729).
__device__ __forceinline__ void mx_tile_of(int L, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int all = tiles_m * tiles_n, q = all >> 3, r = all & 7, x = L & 7;
  const int id = x * q + min(x, r) + (L >> 3);
  constexpr int G = 4;
  const int group = id / (G * tiles_n), first = group * G;
  const int gm = min(tiles_m - first, G), in = id - group * G * tiles_n;
  tm = first + in % gm;
  tn = in / gm;
}

// LDS rows: of e4m3 128 bytes of k, chunk c of row R in slot c ^ mx_sw8(R); of e2m1 64 bytes, two rows a
// line of 128 bytes, chunk 4 (R & 1) + c of line P = R / 2 in slot ^ mx_sw4(P) (activations) or ^ mx_sww(P) (weights,
// whose rows an operand takes as 8 (i / 4) + i % 4). A read of 16 bytes a lane goes 16 lanes at a time, lanes 0 .. 3, 12 .. 15
// and 20 .. 27 first, then 4 .. 11, 16 .. 19 and 28 .. 31 (found from the conflicts counted): each such sixteen hits
// every one of 64 banks once, in tiles and rings. (Swizzles made for sixteen lanes in a row cost four cycles a read more:
// of 16384 x 4096 x 14336, then in waves of 4 x 8 subtiles, 155 million LDS cycles for 96 in the same time. In waves of 2 x 16
// it takes 136 million, 29 of them conflicts.)
__device__ __forceinline__ int mx_sw8(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int mx_sw4(int p) { return (p & 2) ^ (((p >> 2) & 1) * 3); }
__device__ __forceinline__ int mx_sww(int p) { return (p >> 1) & 2; }

// WM x WN waves over the tile, each with TM x TN subtiles of 16 x 16; stages of 128 along k. ODD: rows of any number of
// blocks and scales at any address.
template <bool A4, bool SWIGLU, bool ODD, int TM, int TN, int WM, int WN, int STAGES>
struct MxTile {
  static constexpr int WAVES = WM * WN;
  static constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN;   // rows of a, rows of w
  static constexpr int OUTS = SWIGLU ? BN / 2 : BN;
  static constexpr int ABYTES = BM * (A4 ? 64 : 128), WBYTES = BN * 64;
  // ODD: a stage's scales lie behind it, a dword each. Else:
  static constexpr int STAGE = ABYTES + WBYTES + (ODD ? 16 * (BM + BN) : 0);
  // scales: sets of 8 bytes a row, those of two stages; half a set is loaded with each stage, the set after the stage's
  // own, over one whose last stage has been read then. (16384 x 4096 x 14336 with one product for all of an e4m3 value: a
  // dword a row and stage 902 us instead of 833, since each row is a line of its own; none at all, in a copy, 798. Sets of
  // 16 and 32 bytes were slower, 750 against 716, for the addresses that they take.)
  static constexpr int SETS = ODD ? 0 : (STAGES + 4) / 2, SET = 8 * (BM + BN), SCALES = STAGES * STAGE;
  static constexpr int LDS = SCALES + SETS * SET;
  static constexpr int PA = ABYTES / 1024, PW = WBYTES / 1024, SP = (BM + BN) / (ODD ? 16 : 64);  // loads: 1 KiB, 32 rows of scales (ODD: 16)
  static constexpr int GROUP = TN > 8 ? TN / 4 : TN / 2;  // column subtiles multiplied while the next are read
  static constexpr int share(int n) { return (n + WAVES - 1) / WAVES; }  // of them a wave issues
  static constexpr int LA = share(PA), LW = share(PW), LS = share(SP), LOADS = LA + LW + LS;
  static_assert(BM % 64 == 0 && OUTS % 64 == 0 && TN % 4 == 0, "tile shape");
  static_assert(STAGES >= 3 && (STAGES - 1) * LOADS < 64, "stages, vmcnt");
  static_assert(LDS <= 160 * 1024, "LDS");
};

// The order of what stands between two points that nothing moves across: N times a product, then READS reads of LDS and
// VALU vector instructions.
template <int N, int READS, int VALU>
__device__ __forceinline__ void mx_interleave() {
  if constexpr (N > 0) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if constexpr (READS > 0) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    if constexpr (VALU > 0) __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
    mx_interleave<N - 1, READS, VALU>();
  }
}

template <bool A4, bool SWIGLU, bool ODD, int TM, int TN, int WM, int WN, int STAGES>
__global__ void __launch_bounds__(64 * WM * WN) mx_gemm_tile_kernel(MxGemmK p, int tiles_m, int tiles_n) {
#if defined(__HIP_DEVICE_COMPILE__)
  using T = MxTile<A4, SWIGLU, ODD, TM, TN, WM, WN, STAGES>;
  __shared__ __attribute__((aligned(16))) char smem[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int tm, tn;
  mx_tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * T::BM;
  const int n0 = tn * T::OUTS;
  const int mrows = (int)min((int64_t)T::BM, p.M - m0);  // rows past the last repeat it and are not stored
  const int nouts = min(T::OUTS, p.N - n0);
  const int nk = (p.nb + 3) >> 2;  // stages (ODD: the last may be short)

  // ---- loads: per-lane offsets of this wave's pieces. ODD: chunks past a row's end come from its last one, and are
  // cleared in LDS (see mend).
  const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
  const uint8_t* ga = p.a + m0 * p.lda;
  const uint8_t* gw = p.w + (int64_t)n0 * p.ldw;
  auto wrow = [&](int r) {  // row of w, from n0 (of the up projection: from p.N + n0), of LDS row r
    return min(SWIGLU && r >= T::OUTS ? r - T::OUTS : r, nouts - 1);
  };
  // (where the waves do not divide the pieces some are loaded twice, the same bytes to the same place, so that
  // every wave has the same number in flight)
  auto apiece = [&](int i) { return (wave * T::LA + i) % T::PA; };
  auto wpiece = [&](int i) { return (wave * T::LW + i) % T::PW; };
  uint32_t va[T::LA], vw[T::LW];  // rows
  uint32_t xa[T::LA], xw[T::LW];  // bytes of k within the stage
#pragma unroll
  for (int i = 0; i < T::LA; ++i) {
    const int line = 8 * apiece(i) + (lane >> 3), slot = lane & 7;
    const int c = slot ^ (A4 ? mx_sw4(line) : mx_sw8(line));
    va[i] = (uint32_t)(min(A4 ? 2 * line + (c >> 2) : line, mrows - 1) * p.lda);
    xa[i] = 16 * (A4 ? c & 3 : c);
  }
  // (the up projection's rows may lie 2^32 bytes and more behind the gate's: a piece has rows of one of them)
  const uint8_t* gws[T::LW];
#pragma unroll
  for (int i = 0; i < T::LW; ++i) {
    const int piece = wpiece(i);  // 16 rows
    const int line = 8 * piece + (lane >> 3), c = (lane & 7) ^ mx_sww(line);
    gws[i] = gw + (SWIGLU && 16 * piece >= T::OUTS ? (int64_t)p.N * p.ldw : 0);
    vw[i] = (uint32_t)(wrow(2 * line + (c >> 2)) * p.ldw);
    xw[i] = 16 * (c & 3);
  }
  if constexpr (!ODD) {
#pragma unroll
    for (int i = 0; i < T::LA; ++i) va[i] += xa[i];
#pragma unroll
    for (int i = 0; i < T::LW; ++i) vw[i] += xw[i];
  }
  // scales: a piece is 64 of the rows of a and then w, 32 of them a stage, two lanes a row; ODD: 16 rows, four lanes a row
  constexpr int RS = ODD ? 16 : 64;
  auto spiece = [&](int i) { return (wave * T::LS + i) % T::SP; };
  const uint8_t* gs[T::LS];
  uint32_t vs[T::LS], vs32[T::LS];
#pragma unroll
  for (int i = 0; i < T::LS; ++i) {
    const int r0 = RS * spiece(i);
    const bool sa = r0 < T::BM;
    const int sr = (sa ? r0 : r0 - T::BM) + (lane >> (ODD ? 2 : 1));
    auto srow = [&](int r) { return sa ? (uint32_t)(min(r, mrows - 1) * p.ldas) : (uint32_t)(wrow(r) * p.ldws); };
    gs[i] = sa ? p.as + m0 * p.ldas : p.ws + (int64_t)(n0 + (SWIGLU && r0 - T::BM >= T::OUTS ? p.N : 0)) * p.ldws;
    vs[i] = srow(sr);
    vs32[i] = ODD ? 0 : srow(sr + 32) - vs[i];
  }
  auto load_scales = [&](int i, int set, int half) __attribute__((always_inline)) {
    // (a row's last set may be half a set, and one past it is that again)
    const int b = min(8 * set + 4 * (lane & 1), p.nb - 4);
    dma_load4(gs[i], vs[i] + half * vs32[i] + b, lds0 + T::SCALES + set % (ODD ? 1 : T::SETS) * T::SET + spiece(i) * 512 + half * 256);
  };
  auto load = [&](int i, int kt, int st) __attribute__((always_inline)) {  // load i of stage kt
    const uint32_t d = lds0 + st * T::STAGE;
    constexpr int KA = A4 ? 64 : 128;
    if (i < T::LA) {
      const int j = i < T::LA ? i : 0;
      if constexpr (ODD) dma_load16(ga, va[j] + min(kt * KA + (int)xa[j], p.nb * (KA / 4) - 16), d + apiece(j) * 1024);
      else dma_load16(ga + (int64_t)kt * KA, va[j], d + apiece(j) * 1024);
    } else if (i < T::LA + T::LW) {
      const int j = i < T::LA + T::LW ? i - T::LA : 0;
      if constexpr (ODD) dma_load16(gws[j], vw[j] + min(kt * 64 + (int)xw[j], p.nb * 16 - 16), d + T::ABYTES + wpiece(j) * 1024);
      else dma_load16(gws[j] + (int64_t)kt * 64, vw[j], d + T::ABYTES + wpiece(j) * 1024);
    } else {
      const int j = i < T::LA + T::LW ? 0 : i - T::LA - T::LW;
      if constexpr (ODD) dma_load1(gs[j], vs[j] + min(4 * kt + (lane & 3), p.nb - 1), d + T::ABYTES + T::WBYTES + spiece(j) * 256);
      else load_scales(j, (kt >> 1) + 1, kt & 1);
    }
  };
  // ODD: the last stage has arrived; what lies past its last block adds nothing
  auto mend = [&](int kt, int st) __attribute__((always_inline)) {
    if constexpr (ODD) {
      if (kt != nk - 1 || (p.nb & 3) == 0) return;
      const int blocks = p.nb & 3;
      char* b = smem + st * T::STAGE;
      const uint4 none = make_uint4(0, 0, 0, 0);
      for (int e = tid; e < T::ABYTES / 16; e += 64 * T::WAVES) {
        const int line = e >> 3, c = (e & 7) ^ (A4 ? mx_sw4(line) : mx_sw8(line));
        if ((A4 ? c & 3 : c >> 1) >= blocks) *(uint4*)(b + 16 * e) = none;
      }
      for (int e = tid; e < T::WBYTES / 16; e += 64 * T::WAVES)
        if ((((e & 7) ^ mx_sww(e >> 3)) & 3) >= blocks) *(uint4*)(b + T::ABYTES + 16 * e) = none;
      lds_barrier();
    }
  };

  // ---- operands: a lane's k block is g. Column subtiles go in pairs: row 4 g + e of the first is column 8 g + e,
  // of the second 8 g + 4 + e, so that a lane's eight sums of a pair are consecutive columns.
  const int r = lane & 15, g = lane >> 4;
  const int rw = 8 * (r >> 2) + (r & 3);
  auto wfirst = [&](int i) {  // first LDS row of w of column subtile i, pairs apart by 32 (with SWIGLU the second half are the up projection's)
    constexpr int H = TN / 2;
    if constexpr (SWIGLU) return (i < H ? 0 : T::OUTS) + wn * H * 16 + (i % H) / 2 * 32 + 4 * (i & 1);
    return wn * TN * 16 + i / 2 * 32 + 4 * (i & 1);
  };
  int oa[2], ow[2];  // offsets of this lane's chunks from a subtile's first row: the two of e4m3, of weights in even and odd subtiles
  if constexpr (A4) {
    oa[0] = oa[1] = (r >> 1) * 128 + ((((r & 1) * 4 + g) ^ mx_sw4(r >> 1)) * 16);
  } else {
    oa[0] = r * 128 + (g ^ mx_sw8(r)) * 16;
    oa[1] = r * 128 + ((4 + g) ^ mx_sw8(r)) * 16;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = rw + 4 * i, line = row >> 1;
    ow[i] = line * 128 + ((((row & 1) * 4 + g) ^ mx_sww(line)) * 16);
  }
  f32x4_t acc[TN][TM] = {};
  uint4 fw[TN];
  std::conditional_t<A4, uint4, mx_v8i> fa[TM];
  mx_v8i large[TM], small[TM];  // of e4m3
  int cw[TN], ca[TM], cn[TM];  // scales; of fa
  auto scale_of = [&](int row, int kt, int st) {
    if constexpr (ODD) return (int)*(const uint8_t*)(smem + st * T::STAGE + T::ABYTES + T::WBYTES + row * 16 + 4 * g);
    else return (int)*(const uint8_t*)(smem + T::SCALES + (kt >> 1) % T::SETS * T::SET + 4 * (kt & 1) + row * 8 + g);
  };
  auto read_a = [&](int j, int kt, int st) __attribute__((always_inline)) {
    const char* b = smem + st * T::STAGE + (wm * TM + j) * 16 * (A4 ? 64 : 128);
    if constexpr (A4) fa[j] = *(const uint4*)(b + oa[0]);
    else fa[j] = mx_wide(*(const uint4*)(b + oa[0]), *(const uint4*)(b + oa[1]));
    cn[j] = scale_of((wm * TM + j) * 16 + r, kt, st);
    if constexpr (A4) ca[j] = cn[j];
  };
  auto read_w = [&](int i, int kt, int st) __attribute__((always_inline)) {
    fw[i] = *(const uint4*)(smem + st * T::STAGE + T::ABYTES + (wfirst(i) - 4 * (i & 1)) * 64 + ow[i & 1]);
    cw[i] = scale_of(T::BM + wfirst(i) + rw, kt, st);
  };
  auto product = [&](int i0, int j, mx_v8i a) __attribute__((always_inline)) {
#pragma unroll
    for (int i = i0; i < i0 + T::GROUP; ++i)
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_wide(fw[i]), a, acc[i][j], 4, A4 ? 4 : 0, 0, cw[i], 0, ca[j]);
  };
  auto multiply = [&](int i0, int j) __attribute__((always_inline)) {
    if constexpr (A4) {
      product(i0, j, mx_wide(fa[j]));
    } else {
      product(i0, j, small[j]);
      product(i0, j, large[j]);
    }
  };
  auto split = [&](int j) __attribute__((always_inline)) {
    if constexpr (!A4) mx_split(fa[j], large[j], small[j]);
    ca[j] = cn[j];
  };
  // (Touching lines ahead into L2, starting the workgroups at different stages, and four waves of 128 x 128 gained
  // nothing.)
  // A stage: a group of its weights' subtiles is multiplied while the next is read. Once the last group is read every wave
  // has the stage in registers, and while that group is multiplied the stage's place is refilled, the next stage's first
  // group is read, and its activations. All of that goes between the products: the two waves of a SIMD meet at the
  // barrier, and what stands before their next products leaves the matrix cores idle. e4m3 activations are split there too,
  // once a stage for all columns: so a wave has few row subtiles and many column subtiles (256 x 256: 2 and 16;
  // with 4 and 8, split for every group, 1196 us for 1132 when the split was two instructions longer).
  constexpr int H = T::GROUP;
  int st = 0;
  auto stage = [&](int kt) __attribute__((always_inline)) {
    if constexpr (A4) {
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        multiply(0, j);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = j * H / TM; i < (j + 1) * H / TM; ++i) read_w(H + i, kt, st);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int p = 0; p < TN - H; p += H) {
#pragma unroll
        for (int i = 0; i < H; ++i) read_w(p + H + i, kt, st);
        if (p == 0) split(TM - 1);
#pragma unroll
        for (int j = 0; j < TM; ++j) multiply(p, j);
        if (p == 0) mx_interleave<2 * H, 1, (TM > 1 ? 40 / (2 * H) : 0)>();
        else mx_interleave<2 * H, 1, 0>();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // the next stage's loads of this wave have landed, those of later ones stay in flight; after the barrier
    // every wave's have
    wait_vmcnt<(STAGES - 2) * T::LOADS>();
    lds_barrier();
    const int now = st;
    st = st == STAGES - 1 ? 0 : st + 1;
    mend(kt + 1, st);
    // (behind the last stage what is read is not used)
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      if constexpr (!A4) {
        if (j == 0) {
#pragma unroll
          for (int i = 0; i < TM; ++i) read_a(i, kt + 1, st);
#pragma unroll
          for (int i = 0; i < H; ++i) read_w(i, kt + 1, st);
        } else {
          split(j - 1);
        }
      }
      multiply(TN - H, j);
      if constexpr (!A4) {
        if (j == 0) mx_interleave<2 * H, (3 * TM + 2 * H + 2 * H - 1) / (2 * H), 0>();
        else mx_interleave<2 * H, 0, 40 / (2 * H)>();
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (A4) {
#pragma unroll
        for (int i = j * H / TM; i < (j + 1) * H / TM; ++i) read_w(i, kt + 1, st);
        read_a(j, kt + 1, st);
        __builtin_amdgcn_sched_barrier(0);
      }
      // (near the end the last stage again, which nobody reads: the number in flight stays the same)
#pragma unroll
      for (int i = j * T::LOADS / TM; i < (j + 1) * T::LOADS / TM; ++i) load(i, min(kt + STAGES, nk - 1), now);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if constexpr (!ODD) {
#pragma unroll
    for (int i = 0; i < T::LS; ++i) {
      load_scales(i, 0, 0);
      load_scales(i, 0, 1);
    }
  }
#pragma unroll
  for (int i = 0; i < STAGES; ++i)
#pragma unroll
    for (int e = 0; e < T::LOADS; ++e) load(e, min(i, nk - 1), i);
  wait_vmcnt<(STAGES - 1) * T::LOADS>();
  lds_barrier();
  mend(0, 0);
#pragma unroll
  for (int i = 0; i < H; ++i) read_w(i, 0, 0);
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    read_a(j, 0, 0);
    if (j < TM - 1) split(j);
  }
#pragma unroll 1
  for (int kt = 0; kt < nk; ++kt) stage(kt);
  wait_vmcnt<0>();

  // ---- epilogue: lane l has row l % 16 of a subtile and columns 8 (l / 16) .. + 8 of a pair of them
  constexpr int NP = SWIGLU ? TN / 4 : TN / 2;  // pairs of columns to store
  auto column = [&](int i) { return (wn * NP + i) * 32 + 8 * g; };
  if constexpr (SWIGLU) {
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int mrow = (wm * TM + j) * 16 + r;
      const int64_t row = m0 + mrow;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int c = column(i), n = n0 + c;
        float v[8];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = acc[2 * i + (e >> 2)][j][e & 3], y = acc[TN / 2 + 2 * i + (e >> 2)][j][e & 3];
          v[e] = x * sigmoidf_(x) * y;
          top = max(top, mx_bits(v[e]));
        }
        top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        const int s = mx_scale(top, p.e2m1), fine = s == 255 ? 127 : s;
        if (s == 255) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = 0.f;
        }
        if (mrow >= mrows || c >= nouts) continue;
        const float scale = mx_scale_operand(fine);
        if (g == 0) p.os[row * p.ldos + (n >> 5)] = (uint8_t)s;
        uint8_t* o = (uint8_t*)p.o + row * p.ldo;
        if (p.e2m1) {
          *(uint32_t*)(o + n / 2) = mx_e2m1x8(v, scale);
        } else {
          const float limit = mx_limit(fine);
          *(uint2*)(o + n) = make_uint2(mx_e4m3x4(v, scale, limit), mx_e4m3x4(v + 4, scale, limit));
        }
      }
    }
  } else {
    // the residual of four pairs of a row subtile is loaded ahead of the stores of the four before: one round trip, not one a
    // store (it may be out itself, so the compiler keeps the order as it is written)
    constexpr int NR = NP < 4 ? NP : 4, PARTS = NP / NR;
    float to[NR][8];
    auto load_residual = [&](int part) __attribute__((always_inline)) {
      const int mrow = (wm * TM + part / PARTS) * 16 + r;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int c = column(part % PARTS * NR + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) to[i][e] = 0.f;
        if (!p.res || mrow >= mrows || c >= nouts) continue;
        const int64_t from = (m0 + mrow) * p.ldr + n0 + c;
        if (c + 8 <= nouts) {
          if (p.out32) {
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
              const f32x4_t y = __builtin_bit_cast(f32x4_t, mx_load16((const float*)p.res + from + e));
#pragma unroll
              for (int k = 0; k < 4; ++k) to[i][e + k] = y[k];
            }
          } else {
            const mx_u4 u = mx_load16((const uint16_t*)p.res + from);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              to[i][2 * k] = __uint_as_float(u[k] << 16);
              to[i][2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < nouts) to[i][e] = p.out32 ? ((const float*)p.res)[from + e] : bf16_to_f32(((const uint16_t*)p.res)[from + e]);
        }
      }
    };
    load_residual(0);
#pragma unroll
    for (int part = 0; part < TM * PARTS; ++part) {
      const int j = part / PARTS, i0 = part % PARTS * NR;
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[2 * (i0 + i) + (e >> 2)][j][e & 3] += to[i][e];
      if (part + 1 < TM * PARTS) load_residual(part + 1);
      const int mrow = (wm * TM + j) * 16 + r;
      if (mrow >= mrows) continue;
#pragma unroll
      for (int i = i0; i < i0 + NR; ++i) {
        const int c = column(i);
        if (c >= nouts) continue;
        const int64_t at = (m0 + mrow) * p.ldo + n0 + c;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[2 * i + (e >> 2)][j][e & 3];
        if (c + 8 <= nouts) {
          if (p.out32) {
            mx_store16((float*)p.o + at, __builtin_bit_cast(mx_u4, f32x4_t{v[0], v[1], v[2], v[3]}));
            mx_store16((float*)p.o + at + 4, __builtin_bit_cast(mx_u4, f32x4_t{v[4], v[5], v[6], v[7]}));
          } else {
            mx_store16((uint16_t*)p.o + at, mx_u4{pk_bf16x2(v[0], v[1]), pk_bf16x2(v[2], v[3]), pk_bf16x2(v[4], v[5]), pk_bf16x2(v[6], v[7])});
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < nouts) {
              if (p.out32) ((float*)p.o)[at + e] = v[e];
              else ((uint16_t*)p.o)[at + e] = f32_to_bf16(v[e]);
            }
        }
      }
    }
  }
#endif
}

template <bool A4, bool SWIGLU, bool ODD, int TM, int TN, int WM, int WN, int STAGES>
static void launch_tile(const MxGemmK& k, hipStream_t s) {
  using T = MxTile<A4, SWIGLU, ODD, TM, TN, WM, WN, STAGES>;
  const int tm = (int)cdiv(k.M, T::BM), tn = (int)cdiv(k.N, T::OUTS);
  hipLaunchKernelGGL((mx_gemm_tile_kernel<A4, SWIGLU, ODD, TM, TN, WM, WN, STAGES>), dim3((unsigned)(tm * tn)), dim3(64 * T::WAVES), 0, s, k,
                     tm, tn);
}

// ------------------------------------------------------------- few rows, many bytes of weights
// 32 columns (with SWIGLU of the gate and of the up projection) of up to 32 rows a workgroup; the stages
// of k (128 values) are dealt out to its eight waves, each with a ring of STAGES stages of its own in LDS:
// no wave waits for another before the sums are added, and all of a ring's loads are in flight (1 x 6144 x 4096
// 5.9 us, 2.3 TB/s of weights; 64 x 4096 x 14336 15.9 us, where operands held in registers took 42).
// AP: pieces of a stage's activations (8 rows of e4m3, 16 of e2m1). ODD: as above.
template <bool A4, bool SWIGLU, bool ODD, int AP, int STAGES>
__global__ void __launch_bounds__(512) mx_gemm_ring_kernel(MxGemmK p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int WAVES = 8, TN = SWIGLU ? 2 : 1, AROWS = (A4 ? 16 : 8) * AP;
  static_assert(AROWS <= 32, "rows");
  constexpr int ABYTES = 1024 * AP, WBYTES = 2048 * TN;
  // scales: of 32 rows of a, then of w, four bytes a row (ODD: four dwords)
  constexpr int LS = ODD ? 2 + 2 * TN : (32 + 32 * TN + 63) / 64, STAGE = ABYTES + WBYTES + 256 * LS;
  constexpr int LOADS = AP + 2 * TN + LS, LDR = 32 * TN + 4;
  constexpr int RING = WAVES * STAGES * STAGE, RED = WAVES * AROWS * LDR * 4;
  static_assert(RING <= 160 * 1024 && RED <= 160 * 1024 && STAGES * LOADS < 64, "LDS, vmcnt");
  __shared__ __attribute__((aligned(16))) char smem[RING > RED ? RING : RED];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t m0 = (int64_t)blockIdx.y * AROWS;
  const int n0 = blockIdx.x * 32;
  const int mrows = (int)min((int64_t)AROWS, p.M - m0), nouts = min(32, p.N - n0);
  const int nk = (p.nb + 3) >> 2;
  const uint32_t ring0 = (uint32_t)(uintptr_t)smem + wave * STAGES * STAGE;
  const uint8_t* ga = p.a + m0 * p.lda;
  const uint8_t* gs = p.as + m0 * p.ldas;
  const uint8_t *gw[TN], *gws[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) {
    gw[t] = p.w + (int64_t)(n0 + t * p.N) * p.ldw;
    gws[t] = p.ws + (int64_t)(n0 + t * p.N) * p.ldws;
  }
  uint32_t va[AP], vw[2], xa[AP], xw[2];  // rows, bytes of k within the stage
#pragma unroll
  for (int i = 0; i < AP; ++i) {
    const int line = 8 * i + (lane >> 3), c = (lane & 7) ^ (A4 ? mx_sw4(line) : mx_sw8(line));
    va[i] = (uint32_t)(min(A4 ? 2 * line + (c >> 2) : line, mrows - 1) * p.lda);
    xa[i] = 16 * (A4 ? c & 3 : c);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int line = 8 * i + (lane >> 3), c = (lane & 7) ^ mx_sw4(line);
    vw[i] = (uint32_t)(min(2 * line + (c >> 2), nouts - 1) * p.ldw);
    xw[i] = 16 * (c & 3);
  }
  // scales, a lane's address in load i: rows 64 i .. of the 32 of a and the 32 TN of w (ODD: 16 i ..)
  const uint8_t* ps[LS];
#pragma unroll
  for (int i = 0; i < LS; ++i) {
    const int row = ODD ? 16 * i + (lane >> 2) : 64 * i + lane, t = min((row >> 5) - 1, TN - 1);
    ps[i] = row < 32 ? gs + min(row, mrows - 1) * p.ldas : gws[TN == 2 ? max(t, 0) : 0] + min(row & 31, nouts - 1) * p.ldws;
  }
  auto issue = [&](int kt, int st) __attribute__((always_inline)) {
    const uint32_t d = ring0 + st * STAGE;
    constexpr int KA = A4 ? 64 : 128;
#pragma unroll
    for (int i = 0; i < AP; ++i) {
      if constexpr (ODD) dma_load16(ga, va[i] + min(kt * KA + (int)xa[i], p.nb * (KA / 4) - 16), d + i * 1024);
      else dma_load16(ga + (int64_t)kt * KA, va[i] + xa[i], d + i * 1024);
    }
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (ODD) dma_load16(gw[t], vw[i] + min(kt * 64 + (int)xw[i], p.nb * 16 - 16), d + ABYTES + (2 * t + i) * 1024);
        else dma_load16(gw[t] + (int64_t)kt * 64, vw[i] + xw[i], d + ABYTES + (2 * t + i) * 1024);
      }
#pragma unroll
    for (int i = 0; i < LS; ++i) {
      if constexpr (ODD) dma_load1_at(ps[i] + min(4 * kt + (lane & 3), p.nb - 1), d + ABYTES + WBYTES + 256 * i);
      else dma_load4_at(ps[i] + (int64_t)kt * 4, d + ABYTES + WBYTES + 256 * i);
    }
  };
  const int r = lane & 31, h = lane >> 5, ra = r & (AROWS - 1);
  auto at4 = [&](int row, int c) {
    const int line = row >> 1;
    return line * 128 + (((row & 1) * 4 + c) ^ mx_sw4(line)) * 16;
  };
  f32x16_t acc[TN] = {};
  const int mine = nk > wave ? (nk - wave + WAVES - 1) / WAVES : 0;  // stages wave, wave + 8, ...
#pragma unroll
  for (int i = 0; i < STAGES; ++i)
    if (i < mine) issue(wave + WAVES * i, i);
  int st = 0;
  for (int it = 0; it < mine; ++it) {
    if (it + STAGES <= mine) wait_vmcnt<(STAGES - 1) * LOADS>();
    else wait_vmcnt<0>();
    mx_lds_order();
    char* base = smem + (wave * STAGES + st) * STAGE;
    const char* wb = base + ABYTES;
    const char* sb = wb + WBYTES;
    if (ODD && wave + WAVES * it == nk - 1 && (p.nb & 3)) {  // what lies past the last block adds nothing
      const int blocks = p.nb & 3;
      const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int e = lane; e < ABYTES / 16; e += 64) {
        const int line = e >> 3, c = (e & 7) ^ (A4 ? mx_sw4(line) : mx_sw8(line));
        if ((A4 ? c & 3 : c >> 1) >= blocks) *(uint4*)(base + 16 * e) = none;
      }
#pragma unroll
      for (int e = lane; e < WBYTES / 16; e += 64)
        if ((((e & 7) ^ mx_sw4((e >> 3) & 15)) & 3) >= blocks) *(uint4*)(base + ABYTES + 16 * e) = none;
      wait_lgkmcnt0();
      mx_lds_order();
    }
    auto scale_of = [&](int row) {  // blocks 2 h and 2 h + 1 of the stage, as bytes 0 and 1
      if constexpr (ODD) {
        const uint2 x = *(const uint2*)(sb + row * 16 + 8 * h);
        return (int)(x.x | x.y << 8);
      } else {
        return (int)*(const uint16_t*)(sb + row * 4 + 2 * h);
      }
    };
    const int sa = scale_of(ra);
    int sw[TN];
    uint4 a[2][2], w[TN][2];
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      sw[t] = scale_of(32 + t * 32 + r);
#pragma unroll
      for (int s = 0; s < 2; ++s) w[t][s] = *(const uint4*)(wb + t * 2048 + at4(r, 2 * h + s));
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if constexpr (A4) {
        a[s][0] = *(const uint4*)(base + at4(ra, 2 * h + s));
      } else {
        a[s][0] = *(const uint4*)(base + ra * 128 + ((2 * s + h) ^ mx_sw8(ra)) * 16);
        a[s][1] = *(const uint4*)(base + ra * 128 + ((4 + 2 * s + h) ^ mx_sw8(ra)) * 16);
      }
    }
    wait_lgkmcnt0();  // the stage is in registers: its place may be filled again
    mx_lds_order();
    if (it + STAGES < mine) issue(wave + WAVES * (it + STAGES), st);
    auto product = [&](auto half, mx_v8i x) __attribute__((always_inline)) {
      constexpr int s = decltype(half)::value;
#pragma unroll
      for (int t = 0; t < TN; ++t)
        acc[t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_wide(w[t][s]), x, acc[t], 4, A4 ? 4 : 0, s, sw[t], s, sa);
    };
    auto multiply = [&](auto half) __attribute__((always_inline)) {
      constexpr int s = decltype(half)::value;
      if constexpr (A4) {
        product(half, mx_wide(a[s][0]));
      } else {
        mx_v8i large, small;
        mx_split(mx_wide(a[s][0], a[s][1]), large, small);
        product(half, small);
        product(half, large);
      }
    };
    multiply(std::integral_constant<int, 0>());
    multiply(std::integral_constant<int, 1>());
    st = st == STAGES - 1 ? 0 : st + 1;
  }
  __syncthreads();  // the rings are done with
  float* red = (float*)smem;
  if (r < AROWS) {
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4_t x = {acc[t][4 * q], acc[t][4 * q + 1], acc[t][4 * q + 2], acc[t][4 * q + 3]};
        *(f32x4_t*)(red + (wave * AROWS + r) * LDR + 32 * t + 8 * q + 4 * h) = x;
      }
  }
  __syncthreads();
  mx_finish<SWIGLU, AROWS, 32, LDR, WAVES>(p, red, m0, n0);
#endif
}

template <bool A4, bool SWIGLU, bool ODD>
static void launch_ring(const MxGemmK& k, hipStream_t s) {
  const unsigned gx = (unsigned)cdiv(k.N, 32);
#define TH_MX_RING(AP, STAGES, ROWS)                                                                                          \
  hipLaunchKernelGGL((mx_gemm_ring_kernel<A4, SWIGLU, ODD, AP, STAGES>), dim3(gx, (unsigned)cdiv(k.M, ROWS)), dim3(512), 0, s, k)
  if constexpr (A4) {
    if (k.M <= 16) TH_MX_RING(1, SWIGLU ? 3 : 4, 16);
    else TH_MX_RING(2, SWIGLU ? 2 : 3, 32);
  } else {
    if (k.M <= 8) TH_MX_RING(1, SWIGLU ? 3 : 4, 8);
    else if (k.M <= 16) TH_MX_RING(2, SWIGLU ? 2 : 3, 16);
    else TH_MX_RING(4, SWIGLU || ODD ? 2 : 3, 32);
  }
#undef TH_MX_RING
}

template <bool A4, bool SWIGLU>
static void launch_gemm(const MxGemmK& k, int form, hipStream_t s) {
  const bool odd = !mx_whole_stages(k);
  if (form == TH_MX_RING) {
    if (odd) launch_ring<A4, SWIGLU, true>(k, s);
    else launch_ring<A4, SWIGLU, false>(k, s);
  } else if (form == TH_MX_TILE_64X64) {
    if constexpr (!SWIGLU) {
      if (odd) launch_tile<A4, false, true, 1, 4, 4, 1, 4>(k, s);
      else launch_tile<A4, false, false, 1, 4, 4, 1, 4>(k, s);
    }
  } else if (form == TH_MX_TILE_64X128) {
    if (odd) launch_tile<A4, SWIGLU, true, A4 ? 2 : 1, A4 ? 4 : 8, A4 ? 2 : 4, A4 ? 2 : 1, 4>(k, s);
    else launch_tile<A4, SWIGLU, false, A4 ? 2 : 1, A4 ? 4 : 8, A4 ? 2 : 4, A4 ? 2 : 1, 4>(k, s);
  } else if (form == TH_MX_TILE_128X256) {
    if (odd) launch_tile<A4, SWIGLU, true, A4 ? 4 : 2, A4 ? 4 : 8, A4 ? 2 : 4, A4 ? 4 : 2, 4>(k, s);
    else launch_tile<A4, SWIGLU, false, A4 ? 4 : 2, A4 ? 4 : 8, A4 ? 2 : 4, A4 ? 4 : 2, 4>(k, s);
  } else {
    launch_tile<A4, SWIGLU, false, A4 ? 4 : 2, A4 ? 8 : 16, A4 ? 4 : 8, A4 ? 2 : 1, A4 ? 4 : 3>(k, s);
  }
}

}  // namespace th

using namespace th;

static int check(const th_mx_gemm_desc* d) {
  TH_CHECK_ARG(d != nullptr, "th_mx_gemm: null descriptor");
  TH_CHECK_ARG(d->rows >= 0 && d->rows <= 1 << 21 && d->outs > 0 && d->outs <= 1 << 24 && d->blocks > 0 && d->blocks <= 1 << 18,
               "th_mx_gemm: rows=%lld (at most 2^21) outs=%d (2^24) blocks=%d (2^18) out of range", (long long)d->rows,
               d->outs, d->blocks);
  TH_CHECK_ARG(d->rows * d->outs <= (int64_t)1 << 35, "th_mx_gemm: more than 2^35 outputs");
  TH_CHECK_ARG(d->a_dtype == TH_F8E4M3 || d->a_dtype == TH_F4E2M1, "th_mx_gemm: a_dtype %d is neither e4m3 nor e2m1", d->a_dtype);
  const bool a4 = d->a_dtype == TH_F4E2M1;
  TH_CHECK_ARG(d->ld_a >= (int64_t)d->blocks * (a4 ? 16 : 32) && d->ld_w >= (int64_t)d->blocks * 16 && d->ld_a % 16 == 0 &&
                   d->ld_w % 16 == 0 && (((uintptr_t)d->a | (uintptr_t)d->w) & 15) == 0,
               "th_mx_gemm: codes must be 16-byte aligned, their rows whole blocks in whole 16 bytes apart");
  TH_CHECK_ARG(d->ld_a_scales >= d->blocks && d->ld_w_scales >= d->blocks, "th_mx_gemm: scale rows of fewer than %d bytes",
               d->blocks);
  // (the offsets within a tile of 256 rows are kept in 32 bits)
  TH_CHECK_ARG(d->ld_a < 1 << 23 && d->ld_w < 1 << 23 && d->ld_a_scales < 1 << 23 && d->ld_w_scales < 1 << 23,
               "th_mx_gemm: row strides of codes and scales must be under 2^23 bytes");
  if (d->swiglu) {
    TH_CHECK_ARG(d->out_dtype == TH_F8E4M3 || d->out_dtype == TH_F4E2M1,
                 "th_mx_gemm: out_dtype %d with swiglu, which gives e4m3 or e2m1", d->out_dtype);
    TH_CHECK_ARG(d->outs % 32 == 0, "th_mx_gemm: swiglu needs outs=%d in whole blocks of 32", d->outs);
    TH_CHECK_ARG(d->ld_out >= (int64_t)d->outs / (d->out_dtype == TH_F4E2M1 ? 2 : 1) && d->ld_out % 16 == 0 &&
                     ((uintptr_t)d->out & 15) == 0,
                 "th_mx_gemm: codes must be 16-byte aligned, their rows whole blocks in whole 16 bytes apart");
    TH_CHECK_ARG(d->ld_out_scales >= d->outs / 32, "th_mx_gemm: scale rows of fewer than %d bytes", d->outs / 32);
    TH_CHECK_ARG(!d->residual, "th_mx_gemm: no residual with swiglu");
  } else {
    TH_CHECK_ARG(d->out_dtype == TH_BF16 || d->out_dtype == TH_F32, "th_mx_gemm: out_dtype %d unsupported", d->out_dtype);
    TH_CHECK_ARG(d->ld_out >= d->outs && (!d->residual || d->ld_residual >= d->outs),
                 "th_mx_gemm: out or residual row stride smaller than outs");
    TH_CHECK_ARG(!d->residual || d->residual != d->out || d->ld_residual == d->ld_out || d->rows <= 1,
                 "th_mx_gemm: in place needs one row stride");
  }
  return TH_OK;
}

static MxGemmK operands(const th_mx_gemm_desc* d) {
  MxGemmK k{};
  k.M = d->rows; k.N = d->outs; k.nb = d->blocks;
  k.a = (const uint8_t*)d->a; k.lda = d->ld_a; k.as = d->a_scales; k.ldas = d->ld_a_scales;
  k.w = (const uint8_t*)d->w; k.ldw = d->ld_w; k.ws = d->w_scales; k.ldws = d->ld_w_scales;
  k.res = d->residual; k.ldr = d->ld_residual; k.o = d->out; k.ldo = d->ld_out; k.os = d->out_scales; k.ldos = d->ld_out_scales;
  k.out32 = d->out_dtype == TH_F32; k.e2m1 = d->out_dtype == TH_F4E2M1;
  return k;
}

// What is written shares no byte with what is read; the residual may be out.
static int check_memory(const th_mx_gemm_desc* d) {
  const int64_t size = d->swiglu ? 1 : d->out_dtype == TH_F32 ? 4 : 2, sides = d->swiglu ? 2 : 1;
  const MxSpan read[] = {{d->a, d->rows, d->ld_a, (int64_t)d->blocks * (d->a_dtype == TH_F4E2M1 ? 16 : 32)},
                         {d->a_scales, d->rows, d->ld_a_scales, d->blocks},
                         {d->w, sides * d->outs, d->ld_w, (int64_t)d->blocks * 16},
                         {d->w_scales, sides * d->outs, d->ld_w_scales, d->blocks}};
  const MxSpan out{d->out, d->rows, d->ld_out * size, d->swiglu && d->out_dtype == TH_F4E2M1 ? d->outs / 2 : d->outs * size};
  const MxSpan scales{d->swiglu ? d->out_scales : nullptr, d->rows, d->ld_out_scales, d->outs / 32};
  const MxSpan residual{d->residual, d->rows, d->ld_residual * size, d->outs * size};
  for (const MxSpan& r : read)
    TH_CHECK_ARG(!mx_meet(out, r) && !mx_meet(scales, r), "th_mx_gemm: the result needs memory of its own");
  TH_CHECK_ARG(!mx_meet(out, scales) && mx_same_or_apart(out, residual),
               "th_mx_gemm: the result needs memory of its own; a residual may be out, row for row");
  return TH_OK;
}

extern "C" int th_mx_gemm_form(const th_mx_gemm_desc* d, int32_t* form) {
  int status = check(d);
  if (status == TH_OK) status = check_memory(d);
  if (status != TH_OK) return status;
  TH_CHECK_ARG(form != nullptr, "th_mx_gemm_form: null pointer");
  const MxGemmK k = operands(d);
  form[0] = mx_form(k, d->a_dtype == TH_F4E2M1, d->swiglu);
  form[1] = !mx_whole_stages(k);
  return TH_OK;
}

extern "C" int th_mx_gemm(const th_mx_gemm_desc* d, void* stream) {
  int status = check(d);
  if (status != TH_OK || d->rows == 0) return status;
  TH_CHECK_ARG(d->a && d->a_scales && d->w && d->w_scales && d->out && (!d->swiglu || d->out_scales),
               "th_mx_gemm: null tensor pointer");
  TH_CHECK_ARG(d->out != d->a && d->out != d->w && (!d->swiglu || d->out != (const void*)d->out_scales),
               "th_mx_gemm: the result needs memory of its own");
  if (!device_ready()) {
    set_error("th_mx_gemm: th_init was not called for the current device");
    return TH_ERR_NOT_INIT;
  }
  status = check_memory(d);
  if (status != TH_OK) return status;
  const MxGemmK k = operands(d);
  const bool a4 = d->a_dtype == TH_F4E2M1;
  hipStream_t s = (hipStream_t)stream;
  const int form = mx_form(k, a4, d->swiglu);
  if (d->swiglu) {
    if (a4) launch_gemm<true, true>(k, form, s);
    else launch_gemm<false, true>(k, form, s);
  } else {
    if (a4) launch_gemm<true, false>(k, form, s);
    else launch_gemm<false, false>(k, form, s);
  }
  TH_CHECK_LAUNCH();
  return TH_OK;
}
