// The tiled matrix product of the dense layers: fp32 operands on the bf16 matrix cores, split three ways.
#pragma once
#include <type_traits>

#include "flm_common.h"

namespace flm {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// ---- tiled matrix product ---------------------------------------------------------------------------
// C[M,N] (+)= A[M,K] * B[K,N].  A is addressed A[m*lda + k] when A_KC (k contiguous) else A[k*lda + m];
// B is B[n*ldb + k] when B_KC else B[k*ldb + n].  Workgroup tile 128x128.  The z index of the grid selects a
// batch / K-slice through the z strides.
enum { EPI_PLAIN = 0, EPI_CONV = 1, EPI_MASK = 2 };

struct GemmArgs {
  const float* A;
  const float* B;
  float* C;
  const float* bias;   // per n, or nullptr
  const float* mask;   // EPI_MASK: same indexing as C; output kept where mask > 0
  int M, N, K;
  long lda, ldb, ldc;
  long a_zs, b_zs, c_zs;
  int relu, accumulate;
  int H3;              // EPI_CONV: rows are (b,h) with h < H3; C index = b*N*H3 + n*H3 + h
  int ksplit;          // > 0: blockIdx.z = group*nks + slice; the slice selects the K range
                       // [slice*ksplit, min(K, (slice+1)*ksplit)) and C += slice*c_zs; the group (groups > 1)
                       // selects an independent product: A += group*a_zs, B += group*b_zs, C += group*c_gs
  int groups;
  long c_gs;
  int x_slowest;       // order in which workgroups are dealt to the XCDs (split-operand kernel): see there
  int b_break_k;       // > 0 (B not k-contiguous only): rows k >= b_break_k of B start b_break_off floats further on
  long b_break_off;    // (two [K/2, N] blocks that are not adjacent in memory multiplied as one [K, N] matrix)
  // Segment mapping (kernels with SEG != 0): an index i of the product stands for element
  // seg(i) = (i / b_seg_len) * b_seg_stride + i % b_seg_len of a wider row in memory (b_seg_len a multiple of 4, the
  // index range below 65536; b_seg_magic = ceil(2^32 / b_seg_len) turns the division into a multiply).  SEG 1: the k of
  // a k-contiguous B, B[n*ldb + seg(k)]; SEG 2: the n of a row-contiguous B, B[k*ldb + seg(n)]; SEG 3: the n of C,
  // C[m*ldc + seg(n)] (plain epilogue).
  int b_seg_len, b_seg_stride;
  unsigned b_seg_magic;
};

#define GBM 128
#define GBN 128

// ---- the product on the bf16 matrix cores, fp32 operands split three ways -----------------------------------
// An fp32 number is the exact sum of three bf16 numbers (8 + 8 + 8 significant bits, taken by truncation:
// hi = top half of the word, mid = top half of x - hi, lo = x - hi - mid).  Of the nine partial products of
// (a_hi + a_mid + a_lo) * (b_hi + b_mid + b_lo) the six of order 2^-16 and above are accumulated in fp32 by
// v_mfma_f32_32x32x16_bf16; every partial product is exact, and what is left out (a_mid*b_lo, a_lo*b_mid,
// a_lo*b_lo) is below 2^-21 of the product, 2^-23 on average: the rounding of an fp32 multiply-add.  Six bf16
// instructions of 32 cycles cover the sixteen k of eight fp32 instructions of 64 cycles.  Infinities and NaNs
// in the operands give NaN.
// Workgroup tile 128x128, 8 waves as 2x4, each wave 2x1 tiles of 32x32 (at most 128 registers: four waves per
// SIMD with two workgroups on a CU).  Memory is read 32 k at a time into
// registers (two fetches in flight), LDS is filled 16 k at a time: a stage holds [split][row][16 k] for both
// operands, a lane's operand of one instruction is one 16-byte read, rows are 48 bytes apart (an odd number of
// 16-byte slots: the reads of a 16-lane group fall into 16 different slots).  There are two stages: while the
// matrix cores work on one, the same wave splits the next 16 k into the other, so its vector instructions run
// in the shadow of its matrix instructions; one barrier per stage.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
#define XBK 32                          // k per fetch
#define XROW 12                         // 32-bit words per LDS row
#define XSTAGE (3 * 128 * XROW)         // words per operand and stage
#define X3_LDS_BYTES (2 * 2 * XSTAGE * 4)

// bytes 2,3 of a below bytes 2,3 of b
__device__ __forceinline__ unsigned pack_hi16(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

__device__ __forceinline__ void split3(float x, unsigned& h, unsigned& m, unsigned& l) {
  h = __float_as_uint(x) & 0xffff0000u;
  const float r1 = x - __uint_as_float(h);
  m = __float_as_uint(r1) & 0xffff0000u;
  l = __float_as_uint(r1 - __uint_as_float(m));        // at most 8 significant bits are left
}

// One thread's share of a 128-row x 32-k operand slice: 8 floats, v[half] the four of one stage.  512 threads.
// KC (k contiguous): thread (row = tid >> 2, kq = tid & 3); v[half][i] = row, k 16*half + 4*kq + i.
// otherwise (rows contiguous): thread (rq = tid >> 4, k16 = tid & 15); v[half][i] = k 16*half + k16, row 4*rq + i.
// FAST: the slice lies inside the matrix and its rows are 16-byte aligned: no test around any load.
// SEG: the operand's contiguous axis (k when KC, the rows otherwise) is mapped through segments (GemmArgs::b_seg_*);
// the 16-byte loads are then only 4-byte aligned, which global memory allows.
// EDGE (with FAST): rows at any float, and the slice may pass the last row, whose place the rows behind are then read from
// (their results are not stored); without KC the number of rows is a multiple of four.
struct __attribute__((aligned(4))) F4U { float v[4]; };
template <bool KC, bool FAST, bool SEG = false, bool EDGE = false>
__device__ __forceinline__ void fetch_x3(const float* __restrict__ P, long ld, int r0, int rmax, int k0, int kmax, bool vec,
                                         int tid, float (&v)[2][4], int break_k = 0, long break_off = 0, int seg_len = 0,
                                         int seg_stride = 0, unsigned seg_magic = 0) {
#pragma unroll
  for (int half = 0; half < 2; half++) {
    int r, k;
    const float* p;
    bool ok;
    if (KC) {
      r = r0 + (tid >> 2);
      if (EDGE && FAST) r = min(r, rmax - 1);
      k = k0 + 16 * half + 4 * (tid & 3);
      if (SEG) {
        const unsigned sg = __umulhi((unsigned)k, seg_magic);
        p = P + (long)r * ld + (long)sg * seg_stride + ((unsigned)k - sg * (unsigned)seg_len);
      } else {
        p = P + (long)r * ld + k;
      }
      ok = r < rmax && k + 3 < kmax;
    } else {
      r = r0 + 4 * (tid >> 4);
      if (EDGE && FAST) r = min(r, rmax - 4);
      k = k0 + 16 * half + (tid & 15);
      long rr = r;
      if (SEG) {                      // the rows of this operand are the mapped axis (four consecutive ones stay together)
        const unsigned sg = __umulhi((unsigned)r, seg_magic);
        rr = (long)sg * seg_stride + ((unsigned)r - sg * (unsigned)seg_len);
      }
      p = P + (long)k * ld + rr + ((break_k > 0 && k >= break_k) ? break_off : 0);
      ok = k < kmax && r + 3 < rmax;
    }
    if ((SEG && (FAST || (vec && ok))) || (EDGE && FAST)) {
      const F4U t = *reinterpret_cast<const F4U*>(p);
      v[half][0] = t.v[0]; v[half][1] = t.v[1]; v[half][2] = t.v[2]; v[half][3] = t.v[3];
    } else if (FAST || (vec && ok)) {
      const float4 t = *reinterpret_cast<const float4*>(p);
      v[half][0] = t.x; v[half][1] = t.y; v[half][2] = t.z; v[half][3] = t.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) v[half][i] = (KC ? (r < rmax && k + i < kmax) : (k < kmax && r + i < rmax)) ? p[i] : 0.f;
    }
  }
}

// value of the neighbouring lane (lane ^ 1)
__device__ __forceinline__ float from_pair_lane(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xF, 0xF, true));   // quad_perm [1,0,3,2]
}

// the thread's four floats of one half, split, into a stage S = [3][128][XROW] words
template <bool KC>
__device__ __forceinline__ void place_x3(unsigned* __restrict__ S, int tid, const float (&x)[4]) {
  if (KC) {
    unsigned h[4], m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) split3(x[i], h[i], m[i], l[i]);
    unsigned* d = S + (tid >> 2) * XROW + (tid & 3) * 2;
    *reinterpret_cast<uint2*>(d) = make_uint2(pack_hi16(h[0], h[1]), pack_hi16(h[2], h[3]));
    *reinterpret_cast<uint2*>(d + 128 * XROW) = make_uint2(pack_hi16(m[0], m[1]), pack_hi16(m[2], m[3]));
    *reinterpret_cast<uint2*>(d + 2 * 128 * XROW) = make_uint2(pack_hi16(l[0], l[1]), pack_hi16(l[2], l[3]));
  } else {
    // Two neighbouring lanes hold the same four rows at an even and an odd k.  They swap halves: the even lane
    // ends up with both k of rows 0 and 1, the odd lane with both k of rows 2 and 3, and each writes whole words.
    const bool even = (tid & 1) == 0;
    const float g0 = from_pair_lane(even ? x[2] : x[0]), g1 = from_pair_lane(even ? x[3] : x[1]);
    const float ke[2] = {even ? x[0] : g0, even ? x[1] : g1};      // the even k of this lane's two rows
    const float ko[2] = {even ? g0 : x[2], even ? g1 : x[3]};      // the odd k
    unsigned* d = S + (4 * (tid >> 4) + (even ? 0 : 2)) * XROW + ((tid & 15) >> 1);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      unsigned h0, m0, l0, h1, m1, l1;
      split3(ke[i], h0, m0, l0);
      split3(ko[i], h1, m1, l1);
      d[i * XROW] = pack_hi16(h0, h1);
      d[i * XROW + 128 * XROW] = pack_hi16(m0, m1);
      d[i * XROW + 2 * 128 * XROW] = pack_hi16(l0, l1);
    }
  }
}

// end of a stage: the workgroup's barrier, and nothing of the next stage is moved in front of it (its split
// would otherwise be hoisted to where its loads have not arrived yet)
__device__ __forceinline__ void stage_end() {
  __builtin_amdgcn_sched_barrier(0);
  __syncthreads();
  __builtin_amdgcn_sched_barrier(0);
}

// Order of the instructions of one stage, given to the compiler's scheduler: the operand reads first, then per
// matrix instruction a few of the vector instructions of the split, its LDS writes and (WITH_FETCH) the loads of
// a later slice in between.
template <bool WITH_FETCH>
__device__ __forceinline__ void stage_schedule() {
  __builtin_amdgcn_sched_group_barrier(0x100, 9, 0);        // LDS reads
#pragma unroll
  for (int i = 0; i < 12; i++) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);      // one matrix instruction
    __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);      // vector instructions
    __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);      // an LDS write
    if (WITH_FETCH && i >= 4 && i < 8) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);   // a load
  }
}

// One workgroup (512 threads) of the product; li: its launch index among gx * gy * gz, x3_lds: X3_LDS_BYTES of LDS,
// [stage][A, B][split][row][XROW].  EDGE: operands at any float and matrices that end inside a tile keep the loads without
// tests (fetch_x3).
template <bool A_KC, bool B_KC, int EPI, int SEG = 0, bool EDGE = false>
__device__ __forceinline__ void gemm_x3_body(const GemmArgs& g, unsigned li, unsigned gx, unsigned gy, unsigned gz,
                                             unsigned* x3_lds) {
  constexpr bool B_SEG = SEG == 1 || SEG == 2;
  static_assert(SEG == 0 || (SEG == 1 && B_KC) || (SEG == 2 && !B_KC) || (SEG == 3 && EPI == EPI_PLAIN), "segment mapping");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave >> 2, wn = wave & 3;                 // 8 waves as 2 x 4, each 2 x 1 tiles of 32 x 32
  // Workgroups go round-robin to the 8 XCDs, each with an L2 of its own.  The launch index is turned into a
  // logical one that is consecutive within an XCD, and logical neighbours are the workgroups that read the same
  // operand tiles: with x_slowest the column tile changes last (few row tiles share a wide B), otherwise the
  // z index (the K slice) does.
  const unsigned nwg = gx * gy * gz;
  if ((nwg & 7) == 0) li = (li & 7) * (nwg >> 3) + (li >> 3);
  unsigned bx, by, bz;
  if (g.x_slowest) {
    by = li % gy; li /= gy;
    bz = li % gz; bx = li / gz;
  } else {
    bx = li % gx; li /= gx;
    by = li % gy; bz = li / gy;
  }
  const int m0 = by * GBM, n0 = bx * GBN;
  const int nks = g.ksplit ? (int)gz / (g.groups > 1 ? g.groups : 1) : 1;
  const int grp = g.ksplit ? (int)bz / nks : (int)bz;
  const int slice = g.ksplit ? (int)bz - grp * nks : 0;
  const float* A = g.A + (long)grp * g.a_zs;
  const float* B = g.B + (long)grp * g.b_zs;
  float* C = g.C + (g.ksplit ? (long)slice * g.c_zs + (long)grp * g.c_gs : (long)grp * g.c_zs);
  const int k_begin = slice * g.ksplit;
  const int k_end = g.ksplit ? min(g.K, k_begin + g.ksplit) : g.K;
  const bool a_vec = (g.lda & 3) == 0 && (reinterpret_cast<size_t>(A) & 15) == 0;
  const bool b_vec = B_SEG || ((g.ldb & 3) == 0 && (reinterpret_cast<size_t>(B) & 15) == 0 && (g.b_break_off & 3) == 0);
  f32x16 acc[2];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) acc[i][r] = 0.f;

  const int r32 = lane & 31, h4 = (lane >> 5) * 4;
  // the 16 k of one stage: 9 operand reads, 12 matrix instructions.  The reads stand in front of the split of
  // the next stage in program order (the compiler cannot tell that the two stages do not overlap), so that
  // the matrix instructions depend on nothing behind them and can be spread over the split.
  bf16x8 fa[2][3], fb[3];
  auto operands = [&](int stage) {
    const unsigned* As = x3_lds + stage * 2 * XSTAGE;
    const unsigned* Bs = As + XSTAGE;
#pragma unroll
    for (int s = 0; s < 3; s++) {
      fb[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(Bs + (s * 128 + wn * 32 + r32) * XROW + h4));
#pragma unroll
      for (int i = 0; i < 2; i++)
        fa[i][s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(As + (s * 128 + wm * 64 + i * 32 + r32) * XROW + h4));
    }
  };
  auto products = [&]() {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      f32x16 c = acc[i];
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i][2], fb[0], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i][0], fb[2], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i][1], fb[1], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i][1], fb[0], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i][0], fb[1], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i][0], fb[0], c, 0, 0, 0);
      acc[i] = c;
    }
  };
  auto run = [&](auto fast_tag, int k_begin, int k_end) {
    constexpr bool FAST = decltype(fast_tag)::value;
    const int nf = (k_end - k_begin + XBK - 1) / XBK;          // fetches of 32 k; stages 2f and 2f+1 hold fetch f
    float a0[2][4], b0[2][4], a1[2][4], b1[2][4];
    auto fetch = [&](int f, float (&ra)[2][4], float (&rb)[2][4]) {
      // past the end the last slice is fetched again (FAST has no tests) and never placed
      const int k0 = k_begin + (FAST ? min(f, nf - 1) : f) * XBK;
      fetch_x3<A_KC, FAST, false, EDGE>(A, g.lda, m0, g.M, k0, k_end, a_vec, tid, ra);
      fetch_x3<B_KC, FAST, B_SEG, EDGE>(B, g.ldb, n0, g.N, k0, k_end, b_vec, tid, rb, g.b_break_k, g.b_break_off, g.b_seg_len,
                                  g.b_seg_stride, g.b_seg_magic);
    };
    auto place = [&](int stage, int half, const float (&ra)[2][4], const float (&rb)[2][4]) {
      unsigned* As = x3_lds + stage * 2 * XSTAGE;
      place_x3<A_KC>(As, tid, ra[half]);
      place_x3<B_KC>(As + XSTAGE, tid, rb[half]);
    };
    if (nf <= 0) return;
    fetch(0, a0, b0);
    fetch(1, a1, b1);
    place(0, 0, a0, b0);
    __syncthreads();
    // Four stages per trip.  At its top a0/b0 hold fetch f, a1/b1 fetch f+1, and stage 0 holds the first half of
    // fetch f.  A fetch past the end is never multiplied: the trip that would place it is not run.
    int f = 0;
    for (; f + 1 < nf; f += 2) {
      operands(0);
      place(1, 1, a0, b0);
      fetch(f + 2, a0, b0);
      products();
      stage_schedule<true>();
      stage_end();
      operands(1);
      place(0, 0, a1, b1);
      products();
      stage_schedule<false>();
      stage_end();
      operands(0);
      place(1, 1, a1, b1);
      fetch(f + 3, a1, b1);
      products();
      stage_schedule<true>();
      stage_end();
      operands(1);
      place(0, 0, a0, b0);
      products();
      stage_schedule<false>();
      stage_end();
    }
    if (f < nf) {      // an odd number of fetches: the last one is in a0/b0, its first half already in stage 0
      operands(0);
      place(1, 1, a0, b0);
      products();
      __syncthreads();
      operands(1);
      products();
    }
  };
  if constexpr (EDGE) {
    static_assert(A_KC && !B_SEG, "");
    // whole fetches without tests, what is left of k with them
    const int whole = B_KC || (g.N & 3) == 0 ? k_begin + (k_end - k_begin) / XBK * XBK : k_begin;
    if (whole > k_begin) run(std::true_type{}, k_begin, whole);
    if (whole < k_end) {
      __syncthreads();
      run(std::false_type{}, whole, k_end);
    }
  } else {
    const bool full = a_vec && b_vec && m0 + GBM <= g.M && n0 + GBN <= g.N && ((k_end - k_begin) & (XBK - 1)) == 0;
    if (full) run(std::true_type{}, k_begin, k_end);
    else run(std::false_type{}, k_begin, k_end);
  }
  {
    const int n = n0 + wn * 32 + (lane & 31);
    if (n < g.N) {
      const float bv = g.bias ? g.bias[n] : 0.f;
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int m = m0 + wm * 64 + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5);
          if (m >= g.M) continue;
          float v = acc[i][r] + bv;
          long idx;
          if (EPI == EPI_CONV) {
            const int b = m / g.H3, h = m - b * g.H3;
            idx = ((long)b * g.N + n) * g.H3 + h;
          } else if (SEG == 3) {
            const unsigned sg = __umulhi((unsigned)n, g.b_seg_magic);
            idx = (long)m * g.ldc + (long)sg * g.b_seg_stride + ((unsigned)n - sg * (unsigned)g.b_seg_len);
          } else {
            idx = (long)m * g.ldc + n;
          }
          if (g.accumulate) v += C[idx];
          if (g.relu) v = v > 0.f ? v : 0.f;
          if (EPI == EPI_MASK) v = g.mask[idx] > 0.f ? v : 0.f;
          C[idx] = v;
        }
    }
  }
}

template <bool A_KC, bool B_KC, int EPI, int SEG = 0>
__global__ __launch_bounds__(512, 4) void gemm_x3_kernel(GemmArgs g) {
  extern __shared__ __attribute__((aligned(16))) unsigned x3_lds[];
  gemm_x3_body<A_KC, B_KC, EPI, SEG>(g, blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z), gridDim.x, gridDim.y,
                                     gridDim.z, x3_lds);
}

}  // namespace flm
