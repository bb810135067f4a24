// A shared projection with low-rank adapters of many requests at once, and its backward pass, on gfx950.
//
//   low_i = A_e x_i                       e = the adapter of row i, A [E,r,K], B [E,N,r]
//   y_i   = W x_i + bias + s_e B_e low_i  (rows without an adapter: the projection alone)
//   u_i   = s_e B_e^T dy_i,   dx_i = W^T dy_i + A_e^T u_i
//   dA_e  = sum_{i of e} u_i x_i^T,   dB_e = s_e sum_{i of e} dy_i low_i^T
//
// Rows are taken in the order of a grouping (flm_group_rows): tiles of rows that share an adapter.  Types: fp32, bf16,
// fp16 for all tensors of a call; every sum is kept in fp32 and rounded once, at the end.  fp32 operands enter the matrix
// cores as three bf16 terms each, of whose nine products six are kept.  In the few-row projection, the narrow products and the
// adapters' gradients the first term is cut off and the others are rounded: what is left out is below 2^-22 of the product.
// The projection of more than 64 rows and the inputs' gradient run through the dense layers' product, which cuts every term
// off: below 2^-21 (flm_gemm_x3.h).  The narrow products low and u stay fp32 in memory and enter the next product as two bf16
// terms beside bf16 or fp16 operands (2^-17 of the value, far below the rounding of the result).
#include <initializer_list>

#include "flm_adapters.h"
#include "flm_gemm_x3.h"

namespace flm {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// ---- eight consecutive elements, at any alignment the type allows ------------------------------------------------
template <typename T> struct Vec8 { T v[8]; };
// (as words: an array of 16-bit elements at 2-byte alignment may be loaded one by one, words at that alignment are not)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Packed8 { unsigned w[2 * sizeof(T)]; };
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Packed4 { unsigned w[sizeof(T)]; };
template <typename T> struct Vec4 { T v[4]; };

// avail: elements that exist from p on (may be <= 0: zeros, nothing is read)
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p, long avail) {
  Vec8<T> o;
  if (avail >= 8) {
    o = __builtin_bit_cast(Vec8<T>, *reinterpret_cast<const Packed8<T>*>(p));
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) o.v[j] = j < avail ? p[j] : (T)0.f;
  }
  return o;
}

template <typename T>
__device__ __forceinline__ Vec8<T> load8_strided(const T* p, long stride, long avail) {
  Vec8<T> o;
#pragma unroll
  for (int j = 0; j < 8; j++) o.v[j] = j < avail ? p[j * stride] : (T)0.f;
  return o;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4], long avail) {
  if (avail >= 4) {
    Vec4<T> t;
#pragma unroll
    for (int j = 0; j < 4; j++) t.v[j] = (T)v[j];
    *reinterpret_cast<Packed4<T>*>(p) = __builtin_bit_cast(Packed4<T>, t);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j < avail) p[j] = (T)v[j];
  }
}

// ---- operands as bf16 terms ---------------------------------------------------------------------------------------
// x = t[0] + t[1] + ..., every term behind the first rounded to nearest.  The first:
//   ROUND  to nearest, for types whose range ends below bf16's: the most exact.
//   CLAMP  to nearest, but no further than to the largest bf16, whose difference from a finite x the other terms hold: rounded
//          to infinity, a finite fp32 x above 3.396e38 would become NaN.  Two instructions a pair of values more.
//   CUT    towards zero, for the same reason, at no cost: the second term then holds up to 2^-7 of x instead of 2^-8.
// KEEP_INF: an infinite value is an infinity and zeros from that term on (its difference from itself would be NaN; its difference
// from the largest bf16 still is one); without, it becomes NaN, which saves two instructions a term.
enum First { ROUND, CLAMP, CUT };
template <int N, bool KEEP_INF, First FIRST>
__device__ __forceinline__ void split_terms(const float (&x)[8], bf16x8 (&t)[N]) {
  static_assert(FIRST != CUT || !KEEP_INF, "");
  constexpr float TOP = 0x1.fep127f;                       // the largest bf16
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f32x2 r;
    r[0] = x[2 * i];
    r[1] = x[2 * i + 1];
#pragma unroll
    for (int s = 0; s < N; s++) {
      bf16x2 h;
      f32x2 f;
      if (FIRST == CUT && s == 0) {
        h = __builtin_bit_cast(bf16x2, pack_hi16(__float_as_uint(r[0]), __float_as_uint(r[1])));
        f[0] = __uint_as_float(__float_as_uint(r[0]) & 0xffff0000u);
        f[1] = __uint_as_float(__float_as_uint(r[1]) & 0xffff0000u);
      } else {
        f32x2 near = r;
        if (FIRST == CLAMP && s == 0) {
          near[0] = __builtin_amdgcn_fmed3f(r[0], -TOP, TOP);
          near[1] = __builtin_amdgcn_fmed3f(r[1], -TOP, TOP);
        }
        h = __builtin_convertvector(near, bf16x2);
        f = __builtin_convertvector(h, f32x2);
      }
      t[s][2 * i] = h[0];
      t[s][2 * i + 1] = h[1];
      if (s + 1 < N) {
        const bool finite = !KEEP_INF || (FIRST == CLAMP && s == 0);
        r[0] = finite || __builtin_fabsf(f[0]) < __builtin_inff() ? r[0] - f[0] : 0.f;
        r[1] = finite || __builtin_fabsf(f[1]) < __builtin_inff() ? r[1] - f[1] : 0.f;
      }
    }
  }
}

// Terms of a tensor's own values (exact for bf16: one; fp16: two; fp32: three) and number of terms of the fp32 values
// they are multiplied with in the narrow products.
template <typename T> struct Terms;
template <> struct Terms<float> { static constexpr int own = 3, low = 3; };
template <> struct Terms<__bf16> { static constexpr int own = 1, low = 2; };
template <> struct Terms<_Float16> { static constexpr int own = 2, low = 2; };

template <typename T>
__device__ __forceinline__ void own_terms(const Vec8<T>& v, bf16x8 (&t)[Terms<T>::own]) {
  if constexpr (Terms<T>::own == 1) {
    t[0] = __builtin_bit_cast(bf16x8, v);
  } else {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = (float)v.v[j];
    split_terms<Terms<T>::own, sizeof(T) != 4, sizeof(T) == 4 ? CUT : ROUND>(f, t);
  }
}

// c += a * b over the products of order up to LOW - 1, the smallest first
template <int OWN, int LOW>
__device__ __forceinline__ f32x16 mul_terms32(const bf16x8 (&a)[OWN], const bf16x8 (&b)[LOW], f32x16 c) {
#pragma unroll
  for (int order = LOW - 1; order >= 0; order--)
#pragma unroll
    for (int i = 0; i < OWN; i++)
      if (order - i >= 0 && order - i < LOW) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[order - i], c, 0, 0, 0);
  return c;
}

template <int OWN, int LOW, int A, int B>
__device__ __forceinline__ f32x4 mul_terms16(const bf16x8 (&a)[A], const bf16x8 (&b)[B], f32x4 c) {
#pragma unroll
  for (int order = LOW - 1; order >= 0; order--)
#pragma unroll
    for (int i = 0; i < A; i++)
      if (order - i >= 0 && order - i < B) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[order - i], c, 0, 0, 0);
  return c;
}

// operands of the wide products: 16-bit types as they are, fp32 as three bf16 terms
template <typename T> struct Operand { typedef bf16x8 V; };
template <> struct Operand<_Float16> { typedef f16x8 V; };
template <typename T> struct Wide { typename Operand<T>::V t[1]; };
template <> struct Wide<float> { bf16x8 t[3]; };

__device__ __forceinline__ Wide<__bf16> wide(const Vec8<__bf16>& v) {
  Wide<__bf16> w;
  w.t[0] = __builtin_bit_cast(bf16x8, v);
  return w;
}
__device__ __forceinline__ Wide<_Float16> wide(const Vec8<_Float16>& v) {
  Wide<_Float16> w;
  w.t[0] = __builtin_bit_cast(f16x8, v);
  return w;
}
__device__ __forceinline__ Wide<float> wide(const Vec8<float>& v) {
  Wide<float> w;
  split_terms<3, false, CUT>(v.v, w.t);
  return w;
}
__device__ __forceinline__ f32x4 mul16(const Wide<__bf16>& a, const Wide<__bf16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t[0], b.t[0], c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mul16(const Wide<_Float16>& a, const Wide<_Float16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.t[0], b.t[0], c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mul16(const Wide<float>& a, const Wide<float>& b, f32x4 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t[2], b.t[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t[0], b.t[2], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t[1], b.t[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t[1], b.t[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t[0], b.t[1], c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t[0], b.t[0], c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mul32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mul32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// ---- few rows times few columns over a long K ------------------------------------------------------------------------
// Waves form 16*MR rows of X times 16*NR rows of V over k_begin..k_end, `parts` of them taking 32*S k in turn (part: which),
// both operands straight from memory in the matrix instruction's layout (a lane reads 16 consecutive elements of one row;
// which k a lane holds is the same for both operands, so their order does not matter), and meet in LDS.  Nothing is reused
// between workgroups but through the L2, so this form is for operands that are read once: few rows, or few columns.
// result: lane (c = lane & 15, q = lane >> 4) holds D[v = 16*ni + 4q .. +3][x = 16*mi + c]
// The loads of a wave's next step are in flight while the matrix cores work on the one before.
// S: steps of 32 k taken together (a lane then holds 8*S consecutive elements of a row).
// Every row pointer must be readable: a lane without a row of its own is given another's, its results are not used.  The
// loop then has no test around a load: launches of a few microseconds run cold, and straight code costs what it is long.
template <typename T, int MR, int NR, int S, bool V_STRIDED>
__device__ __forceinline__ void mini_product(const T* const (&xr)[MR], const T* const (&vr)[NR], long v_stride, int k_begin,
                                             int k_end, f32x4 (&acc)[MR][NR], int part, int parts) {
  const int q = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int mi = 0; mi < MR; mi++)
#pragma unroll
    for (int ni = 0; ni < NR; ni++) acc[mi][ni] = f32x4{0.f, 0.f, 0.f, 0.f};
  Vec8<T> rx[S][MR], rv[S][NR];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int s = 0; s < S; s++) {
      const int k = k0 + q * (8 * S) + s * 8;
#pragma unroll
      for (int ni = 0; ni < NR; ni++)
        rv[s][ni] = V_STRIDED ? load8_strided(vr[ni] + (long)k * v_stride, v_stride, 8) : load8(vr[ni] + k, 8);
#pragma unroll
      for (int mi = 0; mi < MR; mi++) rx[s][mi] = load8(xr[mi] + k, 8);
    }
  };
  auto products = [&](const Wide<T> (&x)[S][MR], const Wide<T> (&v)[S][NR]) {
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
      for (int ni = 0; ni < NR; ni++)
#pragma unroll
        for (int mi = 0; mi < MR; mi++) acc[mi][ni] = mul16(v[s][ni], x[s][mi], acc[mi][ni]);
  };
  auto convert = [&](Wide<T> (&x)[S][MR], Wide<T> (&v)[S][NR]) {
#pragma unroll
    for (int s = 0; s < S; s++) {
#pragma unroll
      for (int mi = 0; mi < MR; mi++) x[s][mi] = wide(rx[s][mi]);
#pragma unroll
      for (int ni = 0; ni < NR; ni++) v[s][ni] = wide(rv[s][ni]);
    }
  };
  constexpr int STEP = 32 * S;
  const int whole = k_begin + (k_end - k_begin) / STEP * STEP;       // steps that lie inside; one more may not
  int k0 = k_begin + part * STEP;
  if (k0 < whole) fetch(k0);
  for (; k0 < whole; k0 += parts * STEP) {
    Wide<T> x[S][MR], v[S][NR];
    convert(x, v);
    if (k0 + parts * STEP < whole) fetch(k0 + parts * STEP);
    products(x, v);
  }
  if (k0 == whole && k0 < k_end) {                                   // this wave's turn is the last, ragged step
#pragma unroll
    for (int s = 0; s < S; s++) {
      const int k = k0 + q * (8 * S) + s * 8, avail = k_end - k;
#pragma unroll
      for (int ni = 0; ni < NR; ni++)
        rv[s][ni] = V_STRIDED ? load8_strided(vr[ni] + (long)k * v_stride, v_stride, avail) : load8(vr[ni] + k, avail);
#pragma unroll
      for (int mi = 0; mi < MR; mi++) rx[s][mi] = load8(xr[mi] + k, avail);
    }
    Wide<T> x[S][MR], v[S][NR];
    convert(x, v);
    products(x, v);
  }
}

// sums the PARTS waves' results; f(mi, ni, values) is called by one wave per pair.  red: PARTS * MR * NR * 64 of LDS
template <int MR, int NR, int PARTS, typename F>
__device__ __forceinline__ void mini_meet(const f32x4 (&acc)[MR][NR], f32x4* red, F&& f) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int mi = 0; mi < MR; mi++)
#pragma unroll
    for (int ni = 0; ni < NR; ni++) red[(w * MR * NR + mi * NR + ni) * 64 + lane] = acc[mi][ni];
  __syncthreads();
  for (int s = w; s < MR * NR; s += PARTS) {
    f32x4 v = red[s * 64 + lane];
#pragma unroll
    for (int k = 1; k < PARTS; k++) v += red[(k * MR * NR + s) * 64 + lane];
    f(s / NR, s - s / NR * NR, v);
  }
}

struct ShrinkArgs {
  const void *x, *v;
  long ldx, v_group, v_row, v_k;         // V_e(j, k) = v[e*v_group + j*v_row + k*v_k]
  int K, r, rp, n, kslice;
  float* out;                            // [slice][sorted position][rp]; what lies behind r is not meant to be read
};

// low (or u) of row tile t, read once from memory, the adapter's vectors from the L2 (16384 rows of 4096 bf16, 64 ranks: 55-60
// us, 134 MB of rows; 4099 rows, 32 ranks: 13 us, 2.5 TB/s): its 16*MR rows times ranks rank .. rank + 16*NR - 1 of their adapter, over one K slice.
// A workgroup of PARTS waves; red: PARTS * MR * NR * 64 of LDS
template <typename T, int MR, int NR, int S, int PARTS, bool V_STRIDED>
__device__ __forceinline__ void shrink_tile(const ShrinkArgs& a, const RowGroups& g, int t, int slice, int rank, f32x4* red) {
  const int2 tile = g.tiles[t];
  const int rows = tile.y >> 16, e = tile.y & 0xffff;
  if (rows == 0) return;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int k_begin = slice * a.kslice, k_end = min(a.K, k_begin + a.kslice);
  const T *xr[MR], *vr[NR];
#pragma unroll
  for (int mi = 0; mi < MR; mi++) {
    const int m = min(mi * 16 + c, rows - 1);
    xr[mi] = (const T*)a.x + (long)g.order[tile.x + m] * a.ldx;
  }
#pragma unroll
  for (int ni = 0; ni < NR; ni++) {
    const int j = min(rank + ni * 16 + c, a.r - 1);
    vr[ni] = (const T*)a.v + (long)e * a.v_group + (long)j * a.v_row;
  }
  f32x4 acc[MR][NR];
  mini_product<T, MR, NR, S, V_STRIDED>(xr, vr, a.v_k, k_begin, k_end, acc, threadIdx.x >> 6, PARTS);
  mini_meet<MR, NR, PARTS>(acc, red, [&](int mi, int ni, const f32x4& v) {
    const int m = mi * 16 + c, j = rank + ni * 16 + 4 * q;
    if (m < rows && j < a.rp) *reinterpret_cast<f32x4*>(a.out + ((long)slice * a.n + tile.x + m) * a.rp + j) = v;
  });
}

// Two neighbouring tiles of one adapter at a time (tiles of two adapters one after the other): half the way of the vectors
// through the L2, which is longer than the rows' from 32 ranks on.  Eight waves; grid (tiles / 2, K slices)
template <typename T, int NR>
__global__ __launch_bounds__(512) void shrink_pair_kernel(ShrinkArgs a, RowGroups g) {
  __shared__ f32x4 red[8 * 2 * NR * 64];
  const int t = 2 * blockIdx.x;
  const int2 one = g.tiles[t], two = t + 1 < g.cap ? g.tiles[t + 1] : make_int2(0, 0);
  if ((one.y >> 16) == 0) return;
  const int slice = blockIdx.y;
  if ((two.y >> 16) == 0 || (one.y & 0xffff) != (two.y & 0xffff)) {
#pragma unroll 1
    for (int i = 0; i < 2; i++) {
      if (t + i < g.cap) shrink_tile<T, 2, NR, 1, 8, false>(a, g, t + i, slice, 0, red);
      __syncthreads();
    }
    return;
  }
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4, e = one.y & 0xffff, rows = 32 + (two.y >> 16);
  const int k_begin = slice * a.kslice, k_end = min(a.K, k_begin + a.kslice);
  const T *xr[4], *vr[NR];
#pragma unroll
  for (int mi = 0; mi < 4; mi++) xr[mi] = (const T*)a.x + (long)g.order[one.x + min(mi * 16 + c, rows - 1)] * a.ldx;
#pragma unroll
  for (int ni = 0; ni < NR; ni++) vr[ni] = (const T*)a.v + (long)e * a.v_group + (long)min(ni * 16 + c, a.r - 1) * a.v_row;
  f32x4 acc[4][NR];
  mini_product<T, 4, NR, 1, false>(xr, vr, 1, k_begin, k_end, acc, threadIdx.x >> 6, 8);
  // the waves meet in two halves of the rows
#pragma unroll
  for (int half = 0; half < 2; half++) {
    f32x4 part[2][NR];
#pragma unroll
    for (int mi = 0; mi < 2; mi++)
#pragma unroll
      for (int ni = 0; ni < NR; ni++) part[mi][ni] = acc[2 * half + mi][ni];
    if (half) __syncthreads();
    mini_meet<2, NR, 8>(part, red, [&](int mi, int ni, const f32x4& v) {
      const int m = 32 * half + mi * 16 + c, j = ni * 16 + 4 * q;
      if (m < rows && j < a.rp) *reinterpret_cast<f32x4*>(a.out + ((long)slice * a.n + one.x + m) * a.rp + j) = v;
    });
  }
}

// grid (tiles, K slices)
template <typename T, int NR, bool V_STRIDED>
__global__ __launch_bounds__(256) void shrink_kernel(ShrinkArgs a, RowGroups g) {
  __shared__ f32x4 red[4 * 2 * NR * 64];
  shrink_tile<T, 2, NR, (NR <= 2 ? 2 : 1), 4, V_STRIDED>(a, g, blockIdx.x, blockIdx.y, 0, red);
}

struct BaseArgs {
  const void *x, *w;
  long ldx, ldw;
  int n, K, N, kslice;
  float* part;                           // [slice][n][N]
};

// Up to 64 rows: the projection (16*MR rows x 16*NR outputs a workgroup) and the narrow products (32 rows x 16 ranks) in one
// launch.  The first base_groups workgroups are (output block, K slice) pairs of the projection, the others (tile, K slice,
// rank block) of the narrow product: at these sizes both are streams of weights with little else to do.  One row of 13440 x 512
// fp32: 8.3 us, 29 MB at 3.4 TB/s; 37 rows of 4096 x 4096 bf16, 24 adapters: 13.5 us, 37 MB at 2.7 TB/s: the loads' latency
// twice over and the way through the CUs (48 rows of X pass every workgroup) rather than the memory.
template <typename T, int MRS, int MR, int NR>
__global__ __launch_bounds__(256) void few_rows_kernel(BaseArgs a, ShrinkArgs s, RowGroups g, int base_groups, int low_slices) {
  __shared__ f32x4 red[4 * (MR * NR > MRS ? MR * NR : MRS) * 64];
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  if ((int)blockIdx.x < base_groups) {
    const int cols = (a.N + 16 * NR - 1) / (16 * NR), slice = blockIdx.x / cols;
    const int n0 = (blockIdx.x - slice * cols) * (16 * NR);
    const int k_begin = slice * a.kslice, k_end = min(a.K, k_begin + a.kslice);
    const T *xr[MR], *vr[NR];
#pragma unroll
    for (int mi = 0; mi < MR; mi++) xr[mi] = (const T*)a.x + (long)min(mi * 16 + c, a.n - 1) * a.ldx;
#pragma unroll
    for (int ni = 0; ni < NR; ni++) vr[ni] = (const T*)a.w + (long)min(n0 + ni * 16 + c, a.N - 1) * a.ldw;
    f32x4 acc[MR][NR];
    mini_product<T, MR, NR, 2, false>(xr, vr, 1, k_begin, k_end, acc, threadIdx.x >> 6, 4);
    mini_meet<MR, NR, 4>(acc, red, [&](int mi, int ni, const f32x4& v) {
      const int m = mi * 16 + c, n = n0 + ni * 16 + 4 * q;
      if (m < a.n) {
        const float f[4] = {v[0], v[1], v[2], v[3]};
        store4(a.part + ((long)slice * a.n + m) * a.N + n, f, a.N - n);
      }
    });
  } else {
    const int i = blockIdx.x - base_groups, rest = i / g.cap;
    shrink_tile<T, MRS, 1, 2, 4, false>(s, g, i - rest * g.cap, rest % low_slices, rest / low_slices * 16, red);
  }
}

// ---- the adapters' part and the result ---------------------------------------------------------------------------------
struct FinishArgs {
  const float* part;                     // [slices][n][N]
  int slices, part_sorted;               // rows of part: in their own order, or (part_sorted) by position
  const void* bias;
  const float* low;                      // [low_slices][sorted position][rp], low_step floats a slice
  long low_step;
  int low_slices, r, rp;
  const void* v;                         // V_e(n, j) = v[e*v_group + n*v_row + j*v_j]; without V_STRIDED v_j = 1, r >= 8
  long v_group, v_row, v_j;
  const float* scale;                    // per adapter, or nullptr: scale_all
  float scale_all;
  int n, N, E;
  void* y;
  long ldy;
};

__device__ __forceinline__ float adapter_scale(const float* scale, float all, int e) { return scale ? scale[e] : all; }
// Where s_e is applied: a factor of at most one to the narrow product, a larger one to the sums behind it.  Neither can then
// pass fp32's range where the narrow product and the result do not.
__device__ __forceinline__ float scale_before(float s) { return __builtin_fabsf(s) > 1.f ? 1.f : s; }
__device__ __forceinline__ float scale_after(float s) { return __builtin_fabsf(s) > 1.f ? s : 1.f; }

// The scaled narrow products of `rows` sorted positions from pos on, as bf16 terms in LDS: lt[(term*rows + row)*stride + j],
// stride = low_stride(rp).  threads of the workgroup share the work; a barrier follows at the caller.
// Without V_STRIDED the last piece of eight ranks ends at the last rank, as AddAdapters reads it of V, and holds zeros where
// it repeats those of the piece before.  Behind the terms: scale_after of every row.
__device__ __forceinline__ int low_stride(int rp) { return rp + 8; }          // (16 bytes more: rows fall into different banks)
static size_t staged_low_bytes(int low_terms, int rows, int rp) { return ((size_t)low_terms * (rp + 8) * 2 + 4) * rows; }
template <int LOW, bool V_STRIDED>
__device__ __forceinline__ void stage_low(const FinishArgs& a, const RowGroups& g, long pos, int rows, __bf16* lt) {
  const int per = a.rp >> 3, stride = low_stride(a.rp);
#pragma unroll 1
  for (int i = threadIdx.x; i < rows * per; i += blockDim.x) {
    const int row = i / per, j = (i - row * per) * 8, jr = V_STRIDED ? j : min(j, a.r - 8);
    float f[8];
#pragma unroll
    for (int u = 0; u < 8; u++) f[u] = 0.f;
    const int e = pos + row < a.n ? g.key[pos + row] : a.E;
    float after = 1.f;
    if (e < a.E) {
      const float* p = a.low + (pos + row) * a.rp + jr;
      const long step = a.low_step;
#pragma unroll 1
      for (int z = 0; z < a.low_slices; z += 8) {                    // eight slices in flight, the last one again behind the end
        Packed8<float> v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = *reinterpret_cast<const Packed8<float>*>(p + min(z + k, a.low_slices - 1) * step);
#pragma unroll
        for (int k = 0; k < 8; k++)
#pragma unroll
          for (int u = 0; u < 8; u++) f[u] += z + k < a.low_slices ? __uint_as_float(v[k].w[u]) : 0.f;
      }
      const float scale = adapter_scale(a.scale, a.scale_all, e), s = scale_before(scale);
      after = scale_after(scale);
#pragma unroll
      for (int u = 0; u < 8; u++) f[u] = u >= j - jr && jr + u < a.r ? f[u] * s : 0.f;
    }
    bf16x8 t[LOW];
    split_terms<LOW, true, CLAMP>(f, t);
#pragma unroll
    for (int k = 0; k < LOW; k++) *reinterpret_cast<bf16x8*>(lt + (k * rows + row) * stride + j) = t[k];
    if (j == 0) reinterpret_cast<float*>(lt + LOW * rows * stride)[row] = after;
  }
}

// Adds s_e * low_i . V_e(n, .) to acc[mi] (low is staged with scale_before, scale_after is applied here): lane (c, h) holds
// row lds_row0 + 32*mi + c of the staged tile of lds_rows rows, outputs n0 + 8*(r >> 2) + 4*h + (r & 3).  The rows may use
// several adapters: each adapter's product is formed apart and added to its own rows only, so that no value of one adapter (an
// infinity, a NaN) can reach the rows of another.
// key[mi]: the lane's adapter (E: none), ascending over the rows.  V comes straight from memory (the L2): NB adapters and
// 16*JB ranks at a time, so that NB*JB loads are in flight; start() fetches the first of them, before the narrow products are
// staged if the caller likes.  Waves that hold the same tile may share its adapters.  All lanes of the wave take part.
template <typename T, bool V_STRIDED, int MI, int JB, int NB>
struct AddAdapters {
  int es[NB], j0, seen;
  unsigned todo[MI];
  Vec8<T> v[NB][JB];
  int turn = 0, share = 1;                 // this wave takes the adapters whose number in the tile is turn modulo share

  __device__ __forceinline__ void restart(const FinishArgs& a, const int (&key)[MI]) {
    seen = 0;
#pragma unroll
    for (int mi = 0; mi < MI; mi++) todo[mi] = (unsigned)__ballot(key[mi] < a.E);   // (both halves of the wave: the same rows)
  }
  // the next adapters of the rows and their vectors; es[0] < 0: none left
  __device__ __forceinline__ void fetch(const FinishArgs& a, const int (&key)[MI], int n0) {
    const int lane = threadIdx.x & 63, n = min(n0 + (lane & 31), a.N - 1), h = lane >> 5;
#pragma unroll
    for (int b = 0; b < NB; b++) {
      do {
        es[b] = -1;
#pragma unroll
        for (int mi = 0; mi < MI; mi++)
          if (es[b] < 0 && todo[mi]) es[b] = __builtin_amdgcn_readlane(key[mi], __builtin_ctz(todo[mi]));
#pragma unroll
        for (int mi = 0; mi < MI; mi++) todo[mi] &= ~(unsigned)__ballot(key[mi] == es[b]);
        seen++;
      } while (es[b] >= 0 && share > 1 && (seen & (share - 1)) != turn);
    }
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int jj = 0; jj < JB; jj++) {
        if (jj > 0 && j0 + 16 * jj >= a.r) break;              // (the same for all lanes)
        const int j = j0 + 16 * jj + 8 * h;
        const T* p = (const T*)a.v + (long)max(es[b], 0) * a.v_group + (long)n * a.v_row;
        // (no lane's test around a load: ranks behind the last are read from the last, or the last eight, and cleared)
        if (V_STRIDED) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const T x = p[(long)min(j + i, a.r - 1) * a.v_j];
            v[b][jj].v[i] = j + i < a.r ? x : (T)0.f;
          }
        } else {
          const int jr = min(j, a.r - 8);
          v[b][jj] = load8(p + jr, 8);
#pragma unroll
          for (int i = 0; i < 8; i++) v[b][jj].v[i] = i < j - jr ? (T)0.f : v[b][jj].v[i];
        }
      }
  }
  __device__ __forceinline__ void start(const FinishArgs& a, const int (&key)[MI], int n0) {
    j0 = 0;
    restart(a, key);
    fetch(a, key, n0);
  }
  __device__ __forceinline__ void run(const FinishArgs& a, const __bf16* lt, int lds_rows, int lds_row0, const int (&key)[MI],
                                      int n0, f32x16 (&acc)[MI]) {
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5, stride = low_stride(a.rp);
    const float* afters = reinterpret_cast<const float*>(lt + Terms<T>::low * lds_rows * stride);
    while (true) {
      if (es[0] < 0) {                     // the rows are through: the next ranks
        j0 += 16 * JB;
        if (j0 >= a.r) break;
        restart(a, key);
        fetch(a, key, n0);
        if (es[0] < 0) break;
      }
#pragma unroll
      for (int b = 0; b < NB; b++) {
        if (es[b] >= 0) {
          bf16x8 vt[JB][Terms<T>::own];
#pragma unroll
          for (int jj = 0; jj < JB; jj++)
            if (jj == 0 || j0 + 16 * jj < a.r) own_terms<T>(v[b][jj], vt[jj]);
#pragma unroll
          for (int mi = 0; mi < MI; mi++) {
            const bool mine = key[mi] == es[b];
            if (__ballot(mine) != 0) {
              const float after = afters[lds_row0 + 32 * mi + c];
              f32x16 t;
#pragma unroll
              for (int r = 0; r < 16; r++) t[r] = 0.f;
#pragma unroll
              for (int jj = 0; jj < JB; jj++)
                if (j0 + 16 * jj < a.r) {
                  bf16x8 l[Terms<T>::low];
#pragma unroll
                  for (int k = 0; k < Terms<T>::low; k++)
                    l[k] = *reinterpret_cast<const bf16x8*>(lt + (k * lds_rows + lds_row0 + 32 * mi + c) * stride + j0 + 16 * jj + 8 * h);
                  t = mul_terms32<Terms<T>::own, Terms<T>::low>(vt[jj], l, t);
                }
#pragma unroll
              for (int r = 0; r < 16; r++) acc[mi][r] = mine ? __builtin_fmaf(after, t[r], acc[mi][r]) : acc[mi][r];
            }
          }
        }
      }
      fetch(a, key, n0);
    }
  }
};

// y = sum of the K slices + bias + adapters: 32 sorted rows and 32 outputs a wave, or (SHARED) a workgroup of four waves
// that take the K slices and the adapters in turn and meet in LDS.  Bound by its chain of dependent loads where tiles are few, by
// the slices' way from the caches where they are many (512 x 512 outputs, 16 slices, fp32: 9.5 us; 1001 x 515: 8.4).
template <typename T, bool V_STRIDED, bool SHARED>
__global__ __launch_bounds__(256) void finish_kernel(FinishArgs a, RowGroups g) {
  extern __shared__ __attribute__((aligned(16))) __bf16 lt[];
  __shared__ float meet[SHARED ? 3 : 1][16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int n0 = (SHARED ? blockIdx.x : blockIdx.x * (blockDim.x >> 6) + w) * 32;
  const long pos = (long)blockIdx.y * 32;
  const bool in = pos + c < a.n;
  const int key[1] = {in ? g.key[pos + c] : a.E};
  // Where fewer than 17 rows are left, the lanes of the missing rows take K slices of the others: lane c sums every
  // (32 / span)-th slice of row c mod span.
  int span = 32;
  while (span > 1 && pos + span / 2 >= a.n) span >>= 1;
  const int mine = c & (span - 1);
  const int row = pos + mine < a.n ? g.order[pos + mine] : -1;
  f32x16 acc[1];
#pragma unroll
  for (int r = 0; r < 16; r++) acc[0][r] = 0.f;
  const float* p = a.part + (a.part_sorted ? pos + mine : (long)row) * a.N;
  const long step = (long)a.n * a.N;
  const int first = SHARED ? c / span * 4 + w : c / span, stride = SHARED ? 128 / span : 32 / span;
  const bool some = row >= 0 && n0 < a.N, whole = some && n0 + 32 <= a.N;
  auto slice = [&](int z) {
    Vec4<float> f[4];
#pragma unroll
    for (int r4 = 0; r4 < 4; r4++)
      f[r4] = __builtin_bit_cast(Vec4<float>, *reinterpret_cast<const Packed4<float>*>(p + z * step + n0 + 8 * r4 + 4 * h));
#pragma unroll
    for (int r = 0; r < 16; r++) acc[0][r] += f[r >> 2].v[r & 3];
  };
  AddAdapters<T, V_STRIDED, 1, 2, 2> add;
  if (SHARED) {
    add.turn = w;
    add.share = 4;
  }
  add.start(a, key, n0);
  if (whole) {
    int z = first;
    for (; z + 3 * stride < a.slices; z += 4 * stride) {
#pragma unroll
      for (int k = 0; k < 4; k++) slice(z + k * stride);
    }
#pragma unroll 1
    for (; z < a.slices; z += stride) slice(z);
  } else if (some) {
    // (columns behind the last are read from the last, not stored; two slices in flight: 83 rows of 8821 x 6361 91 -> 60 us)
#pragma unroll 1
    for (int z = first; z < a.slices; z += 2 * stride) {
      float f[2][16];
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int r = 0; r < 16; r++)
          f[k][r] = p[min(z + k * stride, a.slices - 1) * step + min(n0 + 8 * (r >> 2) + 4 * h + (r & 3), a.N - 1)];
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[0][r] += z + k * stride < a.slices ? f[k][r] : 0.f;
    }
  }
  stage_low<Terms<T>::low, V_STRIDED>(a, g, pos, 32, lt);
  for (int o = span; o < 32; o <<= 1)
#pragma unroll
    for (int r = 0; r < 16; r++) acc[0][r] += __shfl_xor(acc[0][r], o);
  __syncthreads();
  if (n0 < a.N) add.run(a, lt, 32, 0, key, n0, acc);
  if (SHARED) {
    if (w > 0)
#pragma unroll
      for (int r = 0; r < 16; r++) meet[w - 1][r][lane] = acc[0][r];
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int k = 0; k < 3; k++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[0][r] += meet[k][r][lane];
  }
  if (n0 >= a.N) return;
  if (a.bias) {
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int n = n0 + 8 * (r >> 2) + 4 * h + (r & 3);
      if (n < a.N) acc[0][r] += (float)((const T*)a.bias)[n];
    }
  }
  if (in) {
    T* y = (T*)a.y + (long)row * a.ldy;
#pragma unroll
    for (int r4 = 0; r4 < 4; r4++) {
      const int n = n0 + 8 * r4 + 4 * h;
      const float v[4] = {acc[0][4 * r4], acc[0][4 * r4 + 1], acc[0][4 * r4 + 2], acc[0][4 * r4 + 3]};
      store4(y + n, v, a.N - n);
    }
  }
}

// The same for few rows, one output a thread and one row a workgroup, in fp32 without the matrix cores: a fifth of the code
// and three loads that wait for each other, which is what a launch of this size takes its time for (one row of 512 outputs 3.3
// us, finish_kernel 7.9; 37 of 4096 4.2, 7.5).  V_e(n, .) contiguous.
template <typename T>
__global__ __launch_bounds__(256) void finish_rows_kernel(FinishArgs a, RowGroups g) {
  __shared__ float low[FLM_ADAPTER_MAX_RANK + 8];
  const int pos = blockIdx.y, n = blockIdx.x * blockDim.x + threadIdx.x, at = min(n, a.N - 1);
  const int e = g.key[pos], row = g.order[pos];
  float y = 0.f;
  const float* p = a.part + (long)row * a.N + at;
  const long step = (long)a.n * a.N;
#pragma unroll 1
  for (int z = 0; z < a.slices; z += 8) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = p[min(z + k, a.slices - 1) * step];
#pragma unroll
    for (int k = 0; k < 8; k++) y += z + k < a.slices ? v[k] : 0.f;
  }
  if (a.bias) y += (float)((const T*)a.bias)[at];
  if (e < a.E) {                                             // (the same for the whole workgroup)
    const float s = adapter_scale(a.scale, a.scale_all, e);
    for (int j = threadIdx.x; j < a.rp; j += blockDim.x) {
      const float* q = a.low + (long)pos * a.rp + j;
      float f = 0.f;
#pragma unroll 1
      for (int z = 0; z < a.low_slices; z += 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = q[min(z + k, a.low_slices - 1) * a.low_step];
#pragma unroll
        for (int k = 0; k < 8; k++) f += z + k < a.low_slices ? v[k] : 0.f;
      }
      low[j] = j < a.r ? f * scale_before(s) : 0.f;
    }
    const T* v = (const T*)a.v + (long)e * a.v_group + (long)at * a.v_row;
    Vec8<T> b = load8(v, a.r);
    __syncthreads();
    float t = 0.f;
#pragma unroll 1
    for (int j = 0; j < a.r; j += 8) {
      const Vec8<T> c = b;
      if (j + 8 < a.r) b = load8(v + j + 8, a.r - j - 8);
#pragma unroll
      for (int u = 0; u < 8; u++) t = __builtin_fmaf((float)c.v[u], low[j + u], t);
    }
    y = __builtin_fmaf(scale_after(s), t, y);
  }
  if (n < a.N) ((T*)a.y)[(long)row * a.ldy + n] = (T)y;
}

// ---- the projection of many rows, 16-bit types -------------------------------------------------------------------------
// Tiles of BM sorted rows x BN outputs, waves as WM x WN of them, 64 k a stage, two stages in LDS.  A thread fetches its
// share of the stage after next into registers while the matrix cores work on one stage; it goes to LDS one stage later.
// A stage's row is 128 bytes; the 16-byte piece p of row r lies at slot p ^ (r & 7), so that the eight rows a group of lanes
// reads at once fall into different banks.  The weight is the instruction's first operand: a lane then holds one row's
// outputs, four consecutive ones at a time.
// FUSED: with bias and adapters, straight to y.  Otherwise one K slice to part[slice][position][N].
// 16384 rows of 4096 x 4096 bf16, 48 adapters of 64 ranks: 560-610 us, 1.0 PFLOP/s; 1.17 in the loop (LDS and the matrix cores
// are both busy nine tenths of it), 12 us a round of tiles for the adapters and the stores.  Four waves of 128 x 128 with half
// the LDS reads: a fifth slower (nothing hides a wave's own fetches).  W_KN, 4096 rows of 4096 x 4096: 155 us.
// li: the workgroup's index among the tiles; lds: two stages, then the terms of low, then the result
#define WIDE_K 64
// W_KN: W is [K,N] with contiguous outputs (the gradient of the inputs).  A thread then fetches eight outputs of four
// consecutive k and turns them in registers; lanes of a wave take the sixteen groups of k first, so that they write whole
// LDS rows.
template <typename T, int BM, int BN, int WM, int WN, bool FUSED, bool W_KN, bool V_STRIDED>
__device__ __forceinline__ void wide_tile(const BaseArgs& b, const FinishArgs& a, const RowGroups& g, unsigned li, int slice, char* lds) {
  constexpr int NT = 64 * WM * WN, MI = BM / (32 * WM), NI = BN / (32 * WN), RX = BM * 8 / NT, RW = BN * 8 / NT;
  constexpr int STAGE = (BM + BN) * 128;                  // bytes
  typedef typename Operand<T>::V V;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = lane & 31, h = lane >> 5;
  const int wm = w / WN, wn = w % WN;
  // workgroups go round-robin to the 8 XCDs: consecutive tiles of one XCD share eight row tiles' and a few column tiles' data
  const unsigned tm = (b.n + BM - 1) / BM, tn = (b.N + BN - 1) / BN, nwg = tm * tn;
  if ((nwg & 7) == 0) li = (li & 7) * (nwg >> 3) + (li >> 3);
  const unsigned band = li / (8 * tn), rows_in_band = min(8u, tm - band * 8), in_band = li - band * 8 * tn;
  const int m0 = (band * 8 + in_band % rows_in_band) * BM, n0 = (in_band / rows_in_band) * BN;
  const int k_begin = slice * b.kslice, k_end = min(b.K, k_begin + b.kslice);
  // (rows behind the last are fetched from the last: their results are not stored)
  static_assert(!W_KN || RW % 4 == 0, "four rows of W a thread");
  const T *xp[RX], *wp[RW];
  const int piece = tid & 7;
#pragma unroll
  for (int i = 0; i < RX; i++) xp[i] = (const T*)b.x + (long)g.order[min(m0 + (tid >> 3) + i * (NT / 8), b.n - 1)] * b.ldx + piece * 8;
#pragma unroll
  for (int i = 0; i < RW; i++) {
    if (W_KN) wp[i] = (const T*)b.w + (long)(4 * (tid & 15) + (i & 3)) * b.ldw + n0 + 8 * ((tid >> 4) + (NT / 16) * (i >> 2));
    else wp[i] = (const T*)b.w + (long)min(n0 + (tid >> 3) + i * (NT / 8), b.N - 1) * b.ldw + piece * 8;
  }
  f32x16 acc[NI][MI];
#pragma unroll
  for (int ni = 0; ni < NI; ni++)
#pragma unroll
    for (int mi = 0; mi < MI; mi++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[ni][mi][r] = 0.f;
  Vec8<T> fx[RX], fw[RW];
  auto fetch_whole = [&](int k0) {
#pragma unroll
    for (int i = 0; i < RX; i++) fx[i] = load8(xp[i] + k0, 8);
#pragma unroll
    for (int i = 0; i < RW; i++) fw[i] = load8(W_KN ? wp[i] + (long)k0 * b.ldw : wp[i] + k0, 8);
  };
  auto fetch = [&](int k0) {
    const int avail = k_end - k0 - piece * 8;
#pragma unroll
    for (int i = 0; i < RX; i++) fx[i] = load8(xp[i] + k0, avail);
#pragma unroll
    for (int i = 0; i < RW; i++) {
      if (W_KN) {
        const bool in = k0 + 4 * (tid & 15) + (i & 3) < k_end;
        fw[i] = load8(wp[i] + (long)k0 * b.ldw, in ? b.N - (n0 + 8 * ((tid >> 4) + (NT / 16) * (i >> 2))) : 0);
      } else {
        fw[i] = load8(wp[i] + k0, avail);
      }
    }
  };
  const int slot = ((piece ^ ((tid >> 3) & 7)) << 4) + (tid >> 3) * 128;
  auto place = [&](char* st) {
#pragma unroll
    for (int i = 0; i < RX; i++) *reinterpret_cast<uint4*>(st + slot + i * (NT / 8) * 128) = __builtin_bit_cast(uint4, fx[i]);
    if constexpr (W_KN) {
#pragma unroll
      for (int i = 0; i < RW; i += 4) {
        uint4 d[4];
#pragma unroll
        for (int k = 0; k < 4; k++) d[k] = __builtin_bit_cast(uint4, fw[i + k]);
        const int row = 8 * ((tid >> 4) + (NT / 16) * (i >> 2)), kg = tid & 15;
        auto put = [&](int j, unsigned w0, unsigned w1, unsigned w2, unsigned w3) {       // outputs 2j, 2j+1 of the four k
#pragma unroll
          for (int o = 0; o < 2; o++) {
            // (lanes of one instruction write even and odd rows alike, so both halves of the banks)
            const int odd = o ^ ((tid >> 4) & 1);
            const unsigned sel = odd ? 0x07060302u : 0x05040100u;
            const int r = row + 2 * j + odd;
            *reinterpret_cast<uint2*>(st + BM * 128 + r * 128 + (((kg >> 1) ^ (r & 7)) << 4) + (kg & 1) * 8) =
                make_uint2(__builtin_amdgcn_perm(w1, w0, sel), __builtin_amdgcn_perm(w3, w2, sel));
          }
        };
        put(0, d[0].x, d[1].x, d[2].x, d[3].x);
        put(1, d[0].y, d[1].y, d[2].y, d[3].y);
        put(2, d[0].z, d[1].z, d[2].z, d[3].z);
        put(3, d[0].w, d[1].w, d[2].w, d[3].w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < RW; i++)
        *reinterpret_cast<uint4*>(st + BM * 128 + slot + i * (NT / 8) * 128) = __builtin_bit_cast(uint4, fw[i]);
    }
  };
  auto products = [&](const char* st) {
    const char* sx = st + (wm * (BM / WM) + c) * 128;
    const char* sw = st + BM * 128 + (wn * (BN / WN) + c) * 128;
    V x[2][MI], v[2][NI];
    auto operands = [&](int s) {
      const int at = ((2 * s + h) ^ (c & 7)) << 4;
#pragma unroll
      for (int ni = 0; ni < NI; ni++) v[s & 1][ni] = __builtin_bit_cast(V, *reinterpret_cast<const uint4*>(sw + ni * 32 * 128 + at));
#pragma unroll
      for (int mi = 0; mi < MI; mi++) x[s & 1][mi] = __builtin_bit_cast(V, *reinterpret_cast<const uint4*>(sx + mi * 32 * 128 + at));
    };
    operands(0);
#pragma unroll
    for (int s = 0; s < 4; s++) {
      if (s < 3) operands(s + 1);
#pragma unroll
      for (int mi = 0; mi < MI; mi++)
#pragma unroll
        for (int ni = 0; ni < NI; ni++) acc[ni][mi] = mul32(v[s & 1][ni], x[s & 1][mi], acc[ni][mi]);
    }
    // order: the first operands, then a matrix instruction at a time with a read of the next operands in its shadow
    constexpr int READS = MI + NI, MULS = MI * NI;
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
      for (int j = 0; j < MULS; j++) {
        if (s < 3 && j < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
  };
  // (W_KN: outputs behind the last must not be fetched either)
  const int whole = W_KN && n0 + BN > b.N ? 0 : (k_end - k_begin) / WIDE_K, stages = (k_end - k_begin + WIDE_K - 1) / WIDE_K;
  if (stages > 0) {
    fetch(k_begin);
    place(lds);
    fetch(k_begin + WIDE_K);                                // (behind the end: zeros)
    __syncthreads();
    int i = 0;
    for (; i + 2 < whole; i++) {
      char* st = lds + (i & 1) * STAGE;
      place(lds + ((i & 1) ^ 1) * STAGE);
      fetch_whole(k_begin + (i + 2) * WIDE_K);
      __builtin_amdgcn_sched_barrier(0);                    // (the loads are not moved behind the products: a stage's time ahead)
      products(st);
      __syncthreads();
    }
    for (; i < stages; i++) {
      char* st = lds + (i & 1) * STAGE;
      if (i + 1 < stages) place(lds + ((i & 1) ^ 1) * STAGE);
      if (i + 2 < stages) fetch(k_begin + (i + 2) * WIDE_K);
      products(st);
      __syncthreads();
    }
  }
  const int nw = n0 + wn * (BN / WN);
  if constexpr (FUSED) {
    int key[MI];
#pragma unroll
    for (int mi = 0; mi < MI; mi++) {
      const long pos = m0 + wm * (BM / WM) + 32 * mi + c;
      key[mi] = pos < b.n ? g.key[pos] : a.E;
    }
    __bf16* lt = reinterpret_cast<__bf16*>(lds);
    stage_low<Terms<T>::low, V_STRIDED>(a, g, m0, BM, lt);
    __syncthreads();
#pragma unroll
    for (int ni = 0; ni < NI; ni++)
      if (nw + 32 * ni < b.N) {
        AddAdapters<T, V_STRIDED, MI, V_STRIDED ? 2 : 4, 1> add;
        add.start(a, key, nw + 32 * ni);
        add.run(a, lt, BM, wm * (BM / WM), key, nw + 32 * ni, acc[ni]);
      }
  }
  // The tile goes through LDS and out in whole rows, 16 bytes a lane: as the matrix cores leave it, a row's line would be
  // written sixteen bytes at a time by eight instructions, and the L2 takes one such piece a cycle and channel (measured:
  // 28 us per 33 MB of a round of tiles, 8 in whole rows).
  auto store_tile = [&](auto* out, long ld, auto zero) {
    typedef decltype(zero) O;
    constexpr int ROW = BN * sizeof(O) + 16, PER = BN * sizeof(O) / 16;        // bytes and 16-byte pieces of a row
    __syncthreads();
#pragma unroll
    for (int ni = 0; ni < NI; ni++)
#pragma unroll
      for (int r4 = 0; r4 < 4; r4++) {
        const int n = wn * (BN / WN) + 32 * ni + 8 * r4 + 4 * h;
        float bias[4] = {0.f, 0.f, 0.f, 0.f};
        if (FUSED && a.bias) {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (n0 + n + i < b.N) bias[i] = (float)((const T*)a.bias)[n0 + n + i];
        }
#pragma unroll
        for (int mi = 0; mi < MI; mi++) {
          Vec4<O> v;
#pragma unroll
          for (int i = 0; i < 4; i++) v.v[i] = (O)(acc[ni][mi][4 * r4 + i] + bias[i]);
          *reinterpret_cast<Vec4<O>*>(lds + (wm * (BM / WM) + 32 * mi + c) * ROW + n * sizeof(O)) = v;
        }
      }
    __syncthreads();
    for (int i = tid; i < BM * PER; i += NT) {
      const int m = i / PER, n = n0 + (i - m * PER) * (16 / (int)sizeof(O));
      if (m0 + m >= b.n || n >= b.N) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(lds + m * ROW + (i - m * PER) * 16);
      O* p = out + (long)(FUSED ? g.order[m0 + m] : m0 + m) * ld + n;
      struct __attribute__((packed, aligned(sizeof(O)))) Piece { unsigned w[4]; };
      if (n + 16 / (int)sizeof(O) <= b.N) {
        *reinterpret_cast<Piece*>(p) = Piece{{v.x, v.y, v.z, v.w}};
      } else {
        struct { O v[16 / sizeof(O)]; } e = __builtin_bit_cast(decltype(e), v);
#pragma unroll
        for (int u = 0; u < 16 / (int)sizeof(O); u++)
          if (n + u < b.N) p[u] = e.v[u];
      }
    }
  };
  if constexpr (FUSED) store_tile((T*)a.y, a.ldy, (T)0.f);
  else store_tile(b.part + (long)slice * b.n * b.N, (long)b.N, 0.f);
}

template <typename T, int BM, int BN, int WM, int WN, bool W_KN, bool V_STRIDED>
__global__ __launch_bounds__(64 * WM * WN, 2) void base_wide_kernel(BaseArgs b, FinishArgs a, RowGroups g) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  wide_tile<T, BM, BN, WM, WN, true, W_KN, V_STRIDED>(b, a, g, blockIdx.x, 0, lds);
}

// K slices of the projection, and beside them the narrow products (ranks in blocks of 16*NR), in one launch: the products of
// the first `tiles` * slices workgroups keep the matrix cores busy, the others mostly wait for memory (1001 rows of 1003 x 515
// fp16: 14 us, rows at odd addresses).
template <typename T, int NR, bool W_KN>
__global__ __launch_bounds__(256, 2) void parts_kernel(BaseArgs b, ShrinkArgs s, RowGroups g, int tiles, int slices, int low_slices) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int i = (int)blockIdx.x - tiles * slices;
  if (i < 0) {
    const int slice = blockIdx.x / tiles;
    wide_tile<T, 128, 128, 2, 2, false, W_KN, false>(b, FinishArgs{}, g, blockIdx.x - slice * tiles, slice, lds);
  } else {
    const int rest = i / g.cap;
    shrink_tile<T, 2, NR, (NR <= 2 ? 2 : 1), 4, false>(s, g, i - rest * g.cap, rest % low_slices, rest / low_slices * 16 * NR,
                                                       reinterpret_cast<f32x4*>(lds));
  }
}

// the same for fp32: the first gx * gy * gz workgroups are the dense layers' product over K slices (512 rows of 13440 x 512: 48
// us, 42 GFLOP of bf16 products at 0.88 PFLOP/s)
template <int NR, bool W_KN>
__global__ __launch_bounds__(512, 4) void x3_parts_kernel(GemmArgs p, unsigned gx, unsigned gy, unsigned gz, ShrinkArgs s, RowGroups g,
                                                          int low_slices) {
  extern __shared__ __attribute__((aligned(16))) unsigned x3_lds[];
  const int i = (int)blockIdx.x - (int)(gx * gy * gz);
  if (i < 0) {
    gemm_x3_body<true, !W_KN, EPI_PLAIN, 0, true>(p, blockIdx.x, gx, gy, gz, x3_lds);
  } else {
    const int rest = i / g.cap;
    shrink_tile<float, 2, NR, 1, 8, false>(s, g, i - rest * g.cap, rest % low_slices, rest / low_slices * 16 * NR,
                                           reinterpret_cast<f32x4*>(x3_lds));
  }
}

// part[0] = sum of the K slices part[z], n4 float4 each
__global__ __launch_bounds__(256) void sum_slices_kernel(float* part, int slices, long n4) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n4) return;
  f32x4* p = reinterpret_cast<f32x4*>(part) + i;
  f32x4 s = p[0];
#pragma unroll 4
  for (int z = 1; z < slices; z++) s += p[z * n4];
  p[0] = s;
}

// low[row][r] of every row, in the rows' own order, from the K slices; rows without an adapter get zeros
__global__ __launch_bounds__(256) void low_rows_kernel(const float* __restrict__ part, int slices, int n, int r, int rp, int E,
                                                       RowGroups g, float* __restrict__ low) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long pos = i / rp;
  const int j = (int)(i - pos * rp);
  if (pos >= n || j >= r) return;
  float s = 0.f;
  if (g.key[pos] < E)
    for (int z = 0; z < slices; z++) s += part[((long)z * n + pos) * rp + j];
  low[(long)g.order[pos] * r + j] = s;
}

// ---- gradients of the adapters -----------------------------------------------------------------------------------------
// G_e(j, q) = sum over the rows i of e of s_e * P(i, j) * Q(i, q), with P fp32 and narrow (u or low), Q wide (x or dy).
// The row tiles of the grouping are cut into chunks of `chunk` tiles whatever the groups' sizes; a workgroup walks a chunk
// for 4 waves of 16*CPL columns of Q.  A tile's 32 rows are one matrix instruction deep: a lane fetches CPL neighbouring
// columns of eight rows, which are the operands of CPL instructions whose outputs interleave (a lane ends up with 4*CPL
// neighbouring columns of one rank); P goes through LDS as bf16 terms, rows contiguous.  Row numbers run two tiles ahead, Q
// and P one.
// A group that lies inside one chunk is written at once; a longer one leaves a partial sum per chunk (at most two a chunk: the
// group it begins in and the one it ends in), added up in order by a second launch, which also clears the groups without
// rows.  512 rows of 13440 and 512 columns, 20 adapters of 16 ranks, fp32: 18 us and 5 for the join, 46 MB at 2.6 TB/s; 4099 rows
// of twice 4096, 24 adapters of 32 ranks, bf16: 33 and 9 us: P's terms are turned through LDS for 512 columns at a time.
struct OuterArgs {
  const float* p;                        // [.][pld]: by sorted position, or (p_gather) by row
  int pld, p_gather;
  const void* q;
  long ldq;
  int KQ, r, E, n, chunk;
  const float* scale;
  float scale_all;
  float* part;                           // [chunks][2][r*KQ], laid out as out
  void* out;                             // out[e*r*KQ + j*o_j + q*o_q]
  long o_j, o_q;
  int cols, across;                      // workgroups over the columns, and over columns and blocks of ranks
};

// CPL neighbouring elements as words
template <typename T, int CPL> struct __attribute__((packed, aligned(sizeof(T)))) ColWords { unsigned w[CPL * sizeof(T) / 4]; };

// Column u of eight rows' words, as eight elements.
template <typename T, int CPL>
__device__ __forceinline__ Vec8<T> column(const ColWords<T, CPL> (&q)[8], int u) {
  if constexpr (sizeof(T) == 4) {
    Vec8<T> v;
#pragma unroll
    for (int i = 0; i < 8; i++) v.v[i] = __uint_as_float(q[i].w[u]);
    return v;
  } else {
    uint4 o;
    const unsigned sel = u & 1 ? 0x07060302u : 0x05040100u;
    o.x = __builtin_amdgcn_perm(q[1].w[u >> 1], q[0].w[u >> 1], sel);
    o.y = __builtin_amdgcn_perm(q[3].w[u >> 1], q[2].w[u >> 1], sel);
    o.z = __builtin_amdgcn_perm(q[5].w[u >> 1], q[4].w[u >> 1], sel);
    o.w = __builtin_amdgcn_perm(q[7].w[u >> 1], q[6].w[u >> 1], sel);
    return __builtin_bit_cast(Vec8<T>, o);
  }
}

#define OUTER_ROW 40                     // bf16 per LDS row of 32 rows of P
template <typename T, int NRJ, int CPL>
__global__ __launch_bounds__(256, 2) void outer_kernel(OuterArgs first, OuterArgs second, int groups, RowGroups g) {
  constexpr int LOW = Terms<T>::low, PER = 2 * NRJ, PI = (32 * PER + 255) / 256;     // pieces of eight P values: a row, a thread
  __shared__ __attribute__((aligned(16))) __bf16 pt[LOW * NRJ * 16 * OUTER_ROW];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = lane & 15, h = lane >> 4;
  // the first `groups` workgroups form one gradient, the others the other
  const bool one = (int)blockIdx.x < groups;
  const OuterArgs a = one ? first : second;
  const int block = one ? blockIdx.x : blockIdx.x - groups, chunk = block / a.across;
  const int t0 = chunk * a.chunk, t1 = min(t0 + a.chunk, g.first_tile[a.E]);
  const int part_of = block - chunk * a.across, rank0 = part_of / a.cols * (16 * NRJ);
  const int q0 = (part_of % a.cols * 4 + w) * (16 * CPL), q = q0 + c * CPL;
  if (t0 >= t1) return;
  // whichever axis is contiguous in the result ends up four neighbouring elements a lane: the ranks' (by_rank: a lane holds
  // one rank and 4*CPL neighbouring columns) or the columns' (one column and four neighbouring ranks)
  const bool by_rank = a.o_q == 1;
  f32x4 acc[NRJ][CPL];
  int rows_of[8];                          // row numbers of the lane's rows of a tile, -1 behind its last
  ColWords<T, CPL> qv[8];
  float pv[PI][8];
  auto fetch_rows = [&](int2 tile) {
    const int rows = tile.y >> 16;
#pragma unroll
    for (int i = 0; i < 8; i++) rows_of[i] = 8 * h + i < rows ? g.order[tile.x + 8 * h + i] : -1;
  };
  // A lane whose columns pass the last one reads the last CPL instead and stores those that are its own: no load is tested
  // (12638 rows, 274 and 1036 columns, 113 ranks: 150 -> 83 us; 9115 rows, 6345 and 54, 10: 116 -> 47).
  const bool inside = q0 + 16 * CPL <= a.KQ;
  const int qc = min(q, a.KQ - CPL);
  auto fetch_q = [&]() {
    if (a.KQ >= CPL) {
#pragma unroll
      for (int i = 0; i < 8; i++)
        qv[i] = *reinterpret_cast<const ColWords<T, CPL>*>((const T*)a.q + (long)max(rows_of[i], 0) * a.ldq + qc);
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int u = 0; u < CPL * (int)sizeof(T) / 4; u++) qv[i].w[u] = rows_of[i] >= 0 ? qv[i].w[u] : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const T* p = (const T*)a.q + (long)rows_of[i] * a.ldq + q;
#pragma unroll
        for (int u = 0; u < CPL * (int)sizeof(T) / 4; u++) qv[i].w[u] = 0;
#pragma unroll
        for (int u = 0; u < CPL; u++)
          if (rows_of[i] >= 0 && q + u < a.KQ) {
            if constexpr (sizeof(T) == 4) qv[i].w[u] = __float_as_uint((float)p[u]);
            else qv[i].w[u >> 1] |= (unsigned)__builtin_bit_cast(unsigned short, p[u]) << (16 * (u & 1));
          }
      }
    }
  };
  // Piece i of the tile's P: row i / PER, values 8*(i % PER) ..  Values behind the last rank belong to outputs that are not
  // stored; rows behind the last are cleared.
  int p_row[PI];
  auto fetch_p_rows = [&](int2 tile) {
#pragma unroll
    for (int k = 0; k < PI; k++) {
      const int at = tile.x + max(min((tid + 256 * k) / PER, (tile.y >> 16) - 1), 0);
      p_row[k] = a.p_gather ? g.order[at] : at;
    }
  };
  auto fetch_p = [&](int2 tile) {
#pragma unroll
    for (int k = 0; k < PI; k++) {
      const int i = tid + 256 * k, m = i / PER, j = rank0 + (i - m * PER) * 8;
      const float* p = a.p + (long)p_row[k] * a.pld + (j < a.r ? j : 0);
      Vec8<float> f;
      if (j + 8 <= a.pld || j >= a.r) f = load8(p, min(8, a.pld));
      else f = load8(p, a.r - j);
#pragma unroll
      for (int u = 0; u < 8; u++) pv[k][u] = f.v[u];
    }
  };
  auto place_p = [&](float s, int rows) {
#pragma unroll
    for (int k = 0; k < PI; k++) {
      const int i = tid + 256 * k, m = i / PER, j = (i - m * PER) * 8;
      if (PI * 256 > 32 * PER && i >= 32 * PER) continue;
#pragma unroll
      for (int u = 0; u < 8; u++) pv[k][u] = m < rows ? pv[k][u] * s : 0.f;
      bf16x8 t[LOW];
      split_terms<LOW, true, CLAMP>(pv[k], t);
#pragma unroll
      for (int o = 0; o < LOW; o++)
#pragma unroll
        for (int u = 0; u < 8; u++) pt[(o * NRJ * 16 + j + u) * OUTER_ROW + m] = t[o][u];
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int jj = 0; jj < NRJ; jj++)
#pragma unroll
      for (int u = 0; u < CPL; u++) acc[jj][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  auto flush = [&](int e, float after) {
    if (after != 1.f) {
#pragma unroll
      for (int jj = 0; jj < NRJ; jj++)
#pragma unroll
        for (int u = 0; u < CPL; u++)
#pragma unroll
          for (int x = 0; x < 4; x++) acc[jj][u][x] *= after;
    }
    const int head = g.first_tile[e], last = g.first_tile[e + 1] - 1;
    const bool whole = head >= t0 && last < t0 + a.chunk;
    float* part = a.part + ((long)chunk * 2 + (head < t0 ? 0 : 1)) * a.r * a.KQ;
    T* out = (T*)a.out + (long)e * a.r * a.KQ;
    // (the places are worked out here, not kept in registers over the whole walk: hundreds of them)
    int at = c;
    asm volatile("" : "+v"(at));
    const int shift = a.KQ >= CPL ? a.KQ - CPL : q0 + 16 * CPL;          // columns of a lane begin here at the latest
    if (by_rank && !inside) {
#pragma unroll
      for (int jj = 0; jj < NRJ; jj++) {
        const int j = rank0 + jj * 16 + at;
        if (j >= a.r) continue;
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const int own = q0 + (4 * h + x) * CPL, from = min(own, shift);
#pragma unroll
          for (int u = 0; u < CPL; u++) {
            const int col = from + u;
            if (col < own || col >= a.KQ) continue;
            if (whole) out[(long)j * a.o_j + col] = (T)acc[jj][u][x];
            else part[(long)j * a.o_j + col] = acc[jj][u][x];
          }
        }
      }
    } else if (by_rank) {
      const int col = q0 + 4 * h * CPL;
#pragma unroll
      for (int jj = 0; jj < NRJ; jj++) {
        const int j = rank0 + jj * 16 + at;
        if (j >= a.r) continue;
#pragma unroll
        for (int i = 0; i < CPL; i++) {
          float v[4];
#pragma unroll
          for (int u = 0; u < 4; u++) v[u] = acc[jj][(4 * i + u) % CPL][(4 * i + u) / CPL];
          if (whole) store4(out + (long)j * a.o_j + col + 4 * i, v, a.KQ - col - 4 * i);
          else store4(part + (long)j * a.o_j + col + 4 * i, v, a.KQ - col - 4 * i);
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < CPL; u++) {
        const int own = q0 + at * CPL, col = min(own, shift) + u;
        if (col < own || col >= a.KQ) continue;
#pragma unroll
        for (int jj = 0; jj < NRJ; jj++) {
          const int j = rank0 + jj * 16 + 4 * h;
          const float v[4] = {acc[jj][u][0], acc[jj][u][1], acc[jj][u][2], acc[jj][u][3]};
          if (whole) store4(out + (long)col * a.o_q + j, v, a.r - j);
          else store4(part + (long)col * a.o_q + j, v, a.r - j);
        }
      }
    }
  };
  clear();
  int2 tile = g.tiles[t0];
  int2 next = t0 + 1 < t1 ? g.tiles[t0 + 1] : make_int2(0, 0);
  fetch_rows(tile);
  fetch_p_rows(tile);
  for (int t = t0 - 1; t < t1; t++) {
    // (the step before the first only fetches)
    const int e = tile.y & 0xffff;
    bf16x8 qt[CPL][Terms<T>::own];
    const float scale = adapter_scale(a.scale, a.scale_all, e);
    if (t >= t0) {
      __syncthreads();                     // (the products of the tile before have read pt)
      place_p(scale_before(scale), tile.y >> 16);
      __syncthreads();
#pragma unroll
      for (int u = 0; u < CPL; u++) own_terms<T>(column<T, CPL>(qv, u), qt[u]);
    }
    const int2 ahead = t < t0 ? tile : next, after = t < t0 ? next : (t + 2 < t1 ? g.tiles[t + 2] : make_int2(0, 0));
    if (t + 1 < t1) {
      fetch_p(ahead);
      fetch_q();
      fetch_rows(after);
      fetch_p_rows(after);
    }
    if (t < t0) continue;
#pragma unroll
    for (int jj = 0; jj < NRJ; jj++) {
      bf16x8 l[LOW];
#pragma unroll
      for (int o = 0; o < LOW; o++) l[o] = *reinterpret_cast<const bf16x8*>(pt + (o * NRJ * 16 + jj * 16 + c) * OUTER_ROW + 8 * h);
#pragma unroll
      for (int u = 0; u < CPL; u++)
        acc[jj][u] = by_rank ? mul_terms16<Terms<T>::own, LOW>(qt[u], l, acc[jj][u]) : mul_terms16<Terms<T>::own, LOW>(l, qt[u], acc[jj][u]);
    }
    if (t + 1 == t1 || (next.y & 0xffff) != e) {
      flush(e, scale_after(scale));
      clear();
    }
    tile = next;
    next = after;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void outer_join_kernel(OuterArgs one, OuterArgs other, RowGroups g) {
  const OuterArgs a = blockIdx.z == 0 ? one : other;
  const int e = blockIdx.y;
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  const long total = (long)a.r * a.KQ;
  if (i >= total) return;
  const int begin = g.first_tile[e], end = g.first_tile[e + 1];
  const int first = begin / a.chunk, last = (end - 1) / a.chunk;
  if (begin < end && first == last) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (begin < end)
    for (int k = first; k <= last; k++) {
      const float* p = a.part + ((long)k * 2 + (begin < k * a.chunk ? 0 : 1)) * total + i;
      if (i + 4 <= total) {
        const Vec4<float> f = __builtin_bit_cast(Vec4<float>, *reinterpret_cast<const Packed4<float>*>(p));
#pragma unroll
        for (int u = 0; u < 4; u++) s[u] += f.v[u];
      } else {
#pragma unroll
        for (int u = 0; u < 4; u++)
          if (i + u < total) s[u] += p[u];
      }
    }
  store4((T*)a.out + (long)e * total + i, s, total - i);
}

// ---- sizes and launches ------------------------------------------------------------------------------------------------
static int ranks_padded(int r) { return (r + 15) & ~15; }

// K slices: enough that `tiles` workgroups per slice come to about `want`, none shorter than min_k; a multiple of 64 each
static int k_slices(long tiles, long want, int K, int min_k, int max_slices, int* kslice) {
  long s = (want + tiles - 1) / tiles;
  const long most = K / min_k;
  if (s > most) s = most;
  if (s > max_slices) s = max_slices;
  if (s < 1) s = 1;
  *kslice = (int)(((K + s - 1) / s + 63) / 64 * 64);
  return (K + *kslice - 1) / *kslice;
}

// Up to this many rows the projection's weight is streamed past all rows at once (few_rows_kernel).
#define BASE_ROWS_MAX 64

// How the projection [n,K] x [N,K]^T is formed.  16-bit types with more than 64 rows: whole tiles of 256 x 256 for the first
// `rows` rows (sorted positions), tiles of 128 x 128, in K slices if need be, for the others.
enum { BASE_ROWS, BASE_X3, BASE_TILES };
struct BasePlan {
  int form, slices, kslice;              // of the rows behind the first `rows`
  int rows;
  bool straight;                         // these rows' tiles go straight to the result (one slice); otherwise finish_kernel ends them
};

// What the adapters cost at the end of tiles of 64 rows a wave and 64 outputs / in finish_kernel, ns: an adapter is 300 ns and
// 15 (10) per rank, one after the other (204 rows of 50 adapters, 120 ranks: 84 us in the tiles, 22 in finish_kernel).
static double adapters_64_time(int n, int N, int r, int E) {
  const long tiles = (long)((n + 127) / 128) * ((N + 127) / 128);
  const double each = 1.0 + 64.0 * E / n;
  return (double)((tiles + 511) / 512) * 2 * (each < 64 ? each : 64) * (300 + 15 * r);
}
static double adapters_finish_time(int n, int N, int r, int E) {
  const double tiles = (double)((n + 31) / 32) * ((N + 31) / 32), each = 1.0 + 32.0 * E / n;
  return (tiles > 1024 ? tiles / 1024 : 1.0) * (each < 32 ? each : 32) * (tiles <= 256 ? 0.25 : 1.0) * (300 + 10 * r);
}

// The time of 128 x 128 tiles for n rows, in units of one round of 256 x 256 tiles (one a CU), and the K slices to take.
// Measured: a round of 512 tiles of 128 x 128 (two a CU) takes 0.62 of one of 256 tiles of 256 x 256 that do twice its work,
// half a round 0.4.  Slices are added up at 4 bytes per slice and output and 5 TB/s, against 28.7 ns per k for a round, and
// by a launch of its own: join ns, 5000, or 0 where whole tiles would have to wait for the narrow products' launch and slices
// do not (250 rows of 512 x 1000 24 -> 14.6 us, 2000 of 2048 x 1024 41 -> 38).
static double tiles_128_time(int n, int K, int N, int r, int E, double join, int* slices, int* kslice, bool* straight) {
  const double t = (double)((n + 127) / 128) * ((N + 127) / 128), rest = t - 512.0 * (long)(t / 512);
  *slices = 1;
  *kslice = K;
  *straight = true;
  const double round = 28.7 * K, last = rest == 0 ? 0 : (rest <= 256 ? 0.4 : 0.62);
  const double whole = 0.62 * (long)(t / 512) + last + adapters_64_time(n, N, r, E) / round;
  int ks;
  const int s = k_slices((long)t, 512, K, 256, 16, &ks);
  const double cut = (s > 1 ? 0.62 * t / 512 : 0.62 * (long)(t / 512) + last) +
                     (join + (4.0 * (2 * s) + 2) * n * N / 5000 + adapters_finish_time(n, N, r, E)) / round;
  if (cut >= whole) return whole;
  *slices = s;
  *kslice = ks;
  *straight = false;
  return cut;
}

// w_kn: W is [K,N]: the few-row form is for [N,K] only.
static BasePlan base_plan(int n, int K, int N, int r, int E, bool f32, bool w_kn = false) {
  BasePlan b;
  b.rows = 0;
  b.straight = false;
  b.slices = 1;
  b.kslice = K;
  const int tn = (N + 255) / 256, tm = (n + 255) / 256;
  if (n <= BASE_ROWS_MAX && !w_kn) {
    b.form = BASE_ROWS;
    const int cols = n <= 16 ? 16 : 32;
    // (workgroups measured: one row of 13440 x 512 fp32, 256 / 512 / 768: 10.3 / 9.2 / 10.5 us; 37 rows of 4096 x 4096 bf16:
    // 13.8 / 15.0 / 14.9)
    b.slices = k_slices((N + cols - 1) / cols, n <= 16 ? 512 : 256, K, 512, 32, &b.kslice);
    return b;
  }
  if (f32) {
    b.form = BASE_X3;
    // (slices of at least 512 / 256 / 128 k: 100 rows of 512 x 256 39 / 26 / 19 us, 1001 of 700 x 515 51 / 35 / 31)
    b.slices = k_slices((long)((n + 127) / 128) * ((N + 127) / 128), 512, K, 128, 16, &b.kslice);
    return b;
  }
  b.form = BASE_TILES;
  double best = tiles_128_time(n, K, N, r, E, w_kn ? 5000.0 : 0.0, &b.slices, &b.kslice, &b.straight);
  // all rows in large tiles, or as many row tiles as fill whole rounds and the rest in small ones
  const int rounds = (int)(((long)tm * tn + 255) / 256);
  const double each = 1.0 + 128.0 * E / n, walk = 2 * (each < 128 ? each : 128) * (300 + 15 * r) / (28.7 * K);
  if (rounds * (1 + walk) < best) {
    best = rounds * (1 + walk);
    b.rows = n;
    b.slices = 1;
    b.kslice = K;
    b.straight = true;
  }
  const int full = (int)((rounds - 1) * 256L / tn);
  if (full > 0 && full * 256 < n) {
    int s, ks;
    bool straight;
    // (the rows behind use as many adapters a row as all do)
    const int behind = n - full * 256, e = 1 + (int)((long)E * behind / n);
    const double t = (rounds - 1) * (1 + walk) + tiles_128_time(behind, K, N, r, e, 5000.0, &s, &ks, &straight) + 3000.0 / (28.7 * K);
    if (t < best) {
      b.straight = straight;
      b.rows = full * 256;
      b.slices = s;
      b.kslice = ks;
    }
  }
  return b;
}
// bytes of the projection's partial sums (0: it goes straight to the result)
static long base_part_bytes(const BasePlan& b, int n, int N) {
  return b.form == BASE_TILES && b.straight ? 0 : 4L * b.slices * (n - b.rows) * N;
}
struct ShrinkPlan { int slices, kslice; };
static ShrinkPlan shrink_plan(int n, int K, int E) {
  ShrinkPlan b;
  b.slices = k_slices(row_tiles_cap(n, E), 512, K, 512, 16, &b.kslice);
  return b;
}

template <typename T, bool V_STRIDED>
static int launch_shrink(const ShrinkArgs& a, const RowGroups& g, int slices, hipStream_t st) {
  if constexpr (!V_STRIDED) {
    // pairs where they still leave a workgroup a CU, from 32 ranks (16384 rows of 4096, 64 ranks: 70 -> 60 us)
    if (g.cap >= 512 && a.rp > 16 && a.rp <= 64) {
      const dim3 pairs((g.cap + 1) / 2, slices);
      if (a.rp <= 32) hipLaunchKernelGGL((shrink_pair_kernel<T, 2>), pairs, dim3(512), 0, st, a, g);
      else hipLaunchKernelGGL((shrink_pair_kernel<T, 4>), pairs, dim3(512), 0, st, a, g);
      FLM_CHECK_LAUNCH();
      return FLM_OK;
    }
  }
  const dim3 grid(g.cap, slices);
  if (a.rp <= 16) hipLaunchKernelGGL((shrink_kernel<T, 1, V_STRIDED>), grid, dim3(256), 0, st, a, g);
  else if (a.rp <= 32) hipLaunchKernelGGL((shrink_kernel<T, 2, V_STRIDED>), grid, dim3(256), 0, st, a, g);
  else if (a.rp <= 64) hipLaunchKernelGGL((shrink_kernel<T, 4, V_STRIDED>), grid, dim3(256), 0, st, a, g);
  else hipLaunchKernelGGL((shrink_kernel<T, 8, V_STRIDED>), grid, dim3(256), 0, st, a, g);
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}

// the projection's K slices and (low_slices > 0) the narrow product's of up to 64 rows
template <typename T>
static int launch_few_rows(const BaseArgs& a, int base_slices, const ShrinkArgs& s, int low_slices, const RowGroups& g, hipStream_t st) {
  const int cols = a.n <= 16 ? 16 : 32, base_groups = (a.N + cols - 1) / cols * base_slices;
  const dim3 grid(base_groups + g.cap * low_slices * (s.rp / 16));
  if (a.n <= 16) hipLaunchKernelGGL((few_rows_kernel<T, 1, 1, 1>), grid, dim3(256), 0, st, a, s, g, base_groups, low_slices);
  else if (a.n <= 32) hipLaunchKernelGGL((few_rows_kernel<T, 2, 2, 2>), grid, dim3(256), 0, st, a, s, g, base_groups, low_slices);
  else if (a.n <= 48) hipLaunchKernelGGL((few_rows_kernel<T, 2, 3, 2>), grid, dim3(256), 0, st, a, s, g, base_groups, low_slices);
  else hipLaunchKernelGGL((few_rows_kernel<T, 2, 4, 2>), grid, dim3(256), 0, st, a, s, g, base_groups, low_slices);
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}

template <typename T, int BM, int BN, int WM, int WN, bool W_KN, bool V_STRIDED>
static int launch_wide(const BaseArgs& b, const FinishArgs& f, const RowGroups& g, hipStream_t st) {
  FLM_RAISE_LDS_ONCE((base_wide_kernel<T, BM, BN, WM, WN, W_KN, V_STRIDED>));
  size_t lds = 2 * (BM + BN) * 128;                                  // two stages; the narrow products' terms; the result
  const size_t tail = staged_low_bytes(Terms<T>::low, BM, f.rp), out = (size_t)BM * (BN * sizeof(T) + 16);
  if (tail > lds) lds = tail;
  if (out > lds) lds = out;
  hipLaunchKernelGGL((base_wide_kernel<T, BM, BN, WM, WN, W_KN, V_STRIDED>), dim3(((b.n + BM - 1) / BM) * ((b.N + BN - 1) / BN)),
                     dim3(64 * WM * WN), lds, st, b, f, g);
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}

template <typename T, int NR, bool W_KN>
static int launch_parts_ranks(const BaseArgs& b, int slices, const RowGroups& g, const ShrinkArgs& s, int low_slices, hipStream_t st) {
  const int low = g.cap * low_slices * ((s.rp + 16 * NR - 1) / (16 * NR));
  if constexpr (sizeof(T) == 4) {
    GemmArgs p{};
    p.A = (const float*)b.x; p.B = (const float*)b.w; p.C = b.part;
    p.M = b.n; p.N = b.N; p.K = b.K; p.lda = b.ldx; p.ldb = b.ldw; p.ldc = b.N;
    p.ksplit = slices > 1 ? b.kslice : 0; p.c_zs = (long)b.n * b.N;
    const unsigned gx = (b.N + GBN - 1) / GBN, gy = (b.n + GBM - 1) / GBM;
    FLM_RAISE_LDS_ONCE((x3_parts_kernel<NR, W_KN>));
    hipLaunchKernelGGL((x3_parts_kernel<NR, W_KN>), dim3(gx * gy * slices + low), dim3(512), X3_LDS_BYTES, st, p, gx, gy, (unsigned)slices,
                       s, g, low_slices);
  } else {
    const int tiles = ((b.n + 127) / 128) * ((b.N + 127) / 128);
    const size_t lds = 128 * (128 * 4 + 16);                         // (the stages take 64 KiB, the result a little more)
    FLM_RAISE_LDS_ONCE((parts_kernel<T, NR, W_KN>));
    hipLaunchKernelGGL((parts_kernel<T, NR, W_KN>), dim3(tiles * slices + low), dim3(256), lds, st, b, s, g, tiles, slices, low_slices);
  }
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}

// K slices of the projection into b.part and, with low_slices > 0, the narrow products beside them
template <typename T, bool W_KN>
static int launch_parts(const BaseArgs& b, int slices, const RowGroups& g, const ShrinkArgs& s, int low_slices, hipStream_t st) {
  return W_KN || s.rp <= 16 ? launch_parts_ranks<T, 1, W_KN>(b, slices, g, s, low_slices, st)
                            : launch_parts_ranks<T, 2, false>(b, slices, g, s, low_slices, st);
}

template <typename T, bool V_STRIDED>
static int launch_finish(const FinishArgs& a, const RowGroups& g, hipStream_t st) {
  const long tiles = (long)((a.N + 31) / 32) * ((a.n + 31) / 32);
  const size_t lds = staged_low_bytes(Terms<T>::low, 32, a.rp);
  const unsigned down = (a.n + 31) / 32;
  // Up to a tile a CU, four waves share each (64 rows of 64 adapters, 128 ranks: 83 -> 55 us a call); up to 1024 a wave each,
  // spread over the CUs (1001 rows, 515 outputs: 8.7 us, shared 11.9); beyond that four a workgroup
  if (tiles <= 256) {
    hipLaunchKernelGGL((finish_kernel<T, V_STRIDED, true>), dim3((a.N + 31) / 32, down), dim3(256), lds, st, a, g);
  } else {
    const int per = tiles <= 1024 ? 1 : 4;
    hipLaunchKernelGGL((finish_kernel<T, V_STRIDED, false>), dim3((a.N + 32 * per - 1) / (32 * per), down), dim3(64 * per), lds, st, a,
                       g);
  }
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}

// Whether finish_rows_kernel ends a few-row projection: its vectors' way through the caches grows with the product, the
// matrix cores' form takes a fixed time (replayed, with / without, all kernels of the call, bf16: one row of 13440 x 512, 16
// ranks 8.2 / 12.3 us, 37 rows of 4096 x 4096 17.0 / 21.4, 16 rows of 128 ranks 24.7 / 30.7, 64 rows of 64 ranks 40.8 / 35.7;
// fp32: 64 rows of 64 ranks 74 / 80, of 128 ranks, two adapters 58 / 48).
template <typename T>
static bool finish_by_rows(const FinishArgs& f) {
  return (long)f.n * f.N * f.r <= (sizeof(T) == 4 ? 1L << 24 : 1L << 23);
}

// The narrow product (low_slices = 0: it is there already, as always with W_KN) and y = X * W^T + bias + adapters, any type
// and size.  W is [N,K], or (W_KN) [K,N].  f.part / b.part: base_part_bytes() of workspace
template <typename T, bool W_KN, bool V_STRIDED>
static int launch_projection(BaseArgs b, const BasePlan& plan, const ShrinkArgs& s, int low_slices, FinishArgs f, const RowGroups& g,
                             hipStream_t st) {
  int rc;
  if constexpr (!W_KN) {
    if (plan.form == BASE_ROWS) {
      if ((rc = launch_few_rows<T>(b, plan.slices, s, low_slices, g, st))) return rc;
      if (finish_by_rows<T>(f)) {
        const int threads = (long)f.n * f.N <= 32768 ? 64 : 256;
        hipLaunchKernelGGL(finish_rows_kernel<T>, dim3((f.N + threads - 1) / threads, f.n), dim3(threads), 0, st, f, g);
        FLM_CHECK_LAUNCH();
        return FLM_OK;
      }
      return launch_finish<T, V_STRIDED>(f, g, st);
    }
  }
  if constexpr (sizeof(T) == 4) {
    if ((rc = launch_parts<float, W_KN>(b, plan.slices, g, s, low_slices, st))) return rc;
  } else {
    const bool beside = plan.rows == 0 && !plan.straight;            // nothing needs low before it is through
    if (!W_KN && low_slices && !beside && (rc = launch_shrink<T, false>(s, g, low_slices, st))) return rc;
    if (plan.rows) {
      BaseArgs large = b;
      FinishArgs fl = f;
      large.n = fl.n = plan.rows;
      large.kslice = b.K;
      if ((rc = launch_wide<T, 256, 256, 2, 4, W_KN, V_STRIDED>(large, fl, g, st))) return rc;
      if (plan.rows == b.n) return FLM_OK;
    }
    // the rows behind: the same with the sorted positions from plan.rows on
    RowGroups rest = g;
    rest.order += plan.rows;
    rest.key += plan.rows;
    b.n = f.n = b.n - plan.rows;
    f.low += (long)plan.rows * f.rp;
    f.part_sorted = 1;
    if (plan.straight) return launch_wide<T, 128, 128, 2, 2, W_KN, V_STRIDED>(b, f, rest, st);
    if ((rc = launch_parts<T, W_KN>(b, plan.slices, rest, s, beside ? low_slices : 0, st))) return rc;
    return launch_finish<T, V_STRIDED>(f, rest, st);
  }
  return launch_finish<T, V_STRIDED>(f, g, st);
}

// Columns a lane of outer_kernel holds: 16 bytes' worth, half of 16-bit types where more ranks leave no registers (bf16 33, fp16
// with its two terms 17); ranks go in blocks of 64 (16282 rows, 79 ranks, fp32: 88 us, all ranks in one workgroup 144).
// terms: Terms<T>::own
static int outer_cols(int r, int terms) { return terms == 3 || r > (terms == 1 ? 32 : 16) ? 4 : 8; }
static int outer_across(int KQ, int r, int terms) {
  const int cols = 64 * outer_cols(r, terms);
  return (KQ + cols - 1) / cols * ((r + 63) / 64);
}

// both gradients
template <typename T>
static int launch_outer(OuterArgs a, OuterArgs b, const RowGroups& g, hipStream_t st) {
  constexpr int CPL = sizeof(T) == 4 ? 4 : 8;
  const int ranks = (a.r + 63) / 64;
  a.across = outer_across(a.KQ, a.r, Terms<T>::own);
  b.across = outer_across(b.KQ, b.r, Terms<T>::own);
  a.cols = a.across / ranks;
  b.cols = b.across / ranks;
  const int groups = a.across * ((g.cap + a.chunk - 1) / a.chunk);
  const dim3 grid(groups + b.across * ((g.cap + b.chunk - 1) / b.chunk));
  if (a.r <= 16) hipLaunchKernelGGL((outer_kernel<T, 1, CPL>), grid, dim3(256), 0, st, a, b, groups, g);
  else if (a.r <= 32) hipLaunchKernelGGL((outer_kernel<T, 2, Terms<T>::own == 2 ? 4 : CPL>), grid, dim3(256), 0, st, a, b, groups, g);
  else hipLaunchKernelGGL((outer_kernel<T, 4, 4>), grid, dim3(256), 0, st, a, b, groups, g);
  FLM_CHECK_LAUNCH();
  const long most = (long)a.r * (a.KQ > b.KQ ? a.KQ : b.KQ);
  hipLaunchKernelGGL(outer_join_kernel<T>, dim3((unsigned)((most + 1023) / 1024), a.E, 2), dim3(256), 0, st, a, b, g);
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}

static long round16(long bytes) { return (bytes + 255) & ~255L; }

// Tiles a workgroup of outer_kernel takes.  Both gradients' workgroups in one round of 512 (4099 rows of 24 adapters, chunks of
// 4 / 5 / 6 / 8 tiles: 259 / 251 / 253 / 251 us for the whole pass; 512 rows of 20, 3 / 7: 23 / 34 for product and join); where
// groups are long, each chunk that one spans costs a partial sum, and half as many workgroups are better (4099 rows, 2 / 4: 65 / 54).
static int outer_chunk(long tiles, int n, int E, int K, int N, int r, int terms) {
  const long work = tiles * (outer_across(K, r, terms) + outer_across(N, r, terms)), group = n / (32L * E);
  const long least = work < 512 ? 1 : work / 512, most = work / 256;
  const long wish = group < most ? group : most;
  return (int)(least > wish ? least : wish);
}

// partial sums of outer_kernel: two a chunk
static long outer_part(long tiles, int chunk) { return 2 * ((tiles + chunk - 1) / chunk); }

template <typename T>
static int forward(const void* x, long ldx, const void* w, long ldw, const void* bias, const void* a, const void* b,
                   const RowGroups& g, const float* scale, float scale_all, int n, int K, int N, int r, int E, char* ws, void* y,
                   long ldy, float* low, hipStream_t st) {
  const int rp = ranks_padded(r);
  const ShrinkPlan ss = shrink_plan(n, K, E);
  const BasePlan bs = base_plan(n, K, N, r, E, sizeof(T) == 4);
  float* low_part = (float*)ws;
  float* part = (float*)(ws + round16(4L * ss.slices * n * rp));
  const ShrinkArgs s{x, a, ldx, (long)r * K, K, 1, K, r, rp, n, ss.kslice, low_part};
  const FinishArgs f{part, bs.slices, 0, bias, low_part, (long)n * rp, ss.slices, r, rp, b, (long)N * r, r, 1, scale, scale_all, n, N, E, y, ldy};
  const BaseArgs base{x, w, ldx, ldw, n, K, N, bs.kslice, part};
  const int rc = r >= 8 ? launch_projection<T, false, false>(base, bs, s, ss.slices, f, g, st)
                            : launch_projection<T, false, true>(base, bs, s, ss.slices, f, g, st);
  if (rc) return rc;
  if (low) {
    hipLaunchKernelGGL(low_rows_kernel, dim3((unsigned)(((long)n * rp + 255) / 256)), dim3(256), 0, st, low_part, ss.slices, n, r,
                       rp, E, g, low);
    FLM_CHECK_LAUNCH();
  }
  return FLM_OK;
}

template <typename T>
static int backward(const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw, const void* a, const void* b,
                    const RowGroups& g, const float* scale, float scale_all, const float* low, int n, int K, int N, int r, int E,
                    char* ws, void* dx, long lddx, void* da, void* db, hipStream_t st) {
  const int rp = ranks_padded(r);
  const ShrinkPlan ss = shrink_plan(n, N, E);
  float* u = (float*)ws;                                             // s_e is applied where u is used (scale_before, scale_after)
  ws += round16(4L * ss.slices * n * rp);
  const ShrinkArgs s{dy, b, lddy, (long)N * r, 1, r, N, r, rp, n, ss.kslice, u};
  int rc = launch_shrink<T, true>(s, g, ss.slices, st);
  if (rc) return rc;
  if (ss.slices > 1) {                                               // read many times below: added up once
    hipLaunchKernelGGL(sum_slices_kernel, dim3((unsigned)(((long)n * rp / 4 + 255) / 256)), dim3(256), 0, st, u, ss.slices, (long)n * rp / 4);
    FLM_CHECK_LAUNCH();
  }
  const int chunk = outer_chunk(g.cap, n, E, K, N, r, Terms<T>::own);
  float *part_a = (float*)ws, *part_b = part_a + outer_part(g.cap, chunk) * r * K;
  if ((rc = launch_outer<T>(OuterArgs{u, rp, 0, x, ldx, K, r, E, n, chunk, scale, scale_all, part_a, da, K, 1, 0},
                            OuterArgs{low, r, 1, dy, lddy, N, r, E, n, chunk, scale, scale_all, part_b, db, 1, r, 0}, g, st)))
    return rc;
  if (!dx) return FLM_OK;
  const BasePlan bs = base_plan(n, N, K, r, E, sizeof(T) == 4, true);
  float* dx_part = (float*)ws;
  const FinishArgs f{dx_part, bs.slices, 0, nullptr, u, (long)n * rp, 1, r, rp, a, (long)r * K, 1, K, scale, scale_all, n, K, E, dx, lddx};
  return launch_projection<T, true, true>(BaseArgs{dy, w, lddy, ldw, n, N, K, bs.kslice, dx_part}, bs, s, 0, f, g, st);
}

}  // namespace flm

using namespace flm;

// Whether two operands may share an element: rows of `width` elements, ld apart (ld is no less than width, or 0 and more
// where rows may coincide).  Columns of one matrix that do not meet do not overlap.
struct Span { const void* p; long ld, rows, width; };
static bool spans_meet(const Span& a, const Span& b, int size) {
  if (!a.p || !b.p) return false;
  const long pa = (long)(uintptr_t)a.p, pb = (long)(uintptr_t)b.p;
  const long ea = pa + ((a.rows - 1) * a.ld + a.width) * size, eb = pb + ((b.rows - 1) * b.ld + b.width) * size;
  if (pa >= eb || pb >= ea) return false;
  const long ld = a.ld * size;
  if (a.ld != b.ld || a.rows < 2 || b.rows < 2 || a.width + b.width > a.ld) return true;
  const long d = ((pb - pa) % ld + ld) % ld;               // where b's rows begin within a's
  return d < a.width * size || d + b.width * size > ld;
}

static bool misplaced(int bytes, std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if ((uintptr_t)p & (bytes - 1)) return true;
  return false;
}

static bool adapter_sizes(int n, int K, int N, int r, int E, int dtype) {
  return n > 0 && n <= (1 << 20) && K > 0 && N > 0 && K <= (1 << 20) && N <= (1 << 20) && r > 0 && r <= FLM_ADAPTER_MAX_RANK && E > 0 &&
         E <= FLM_GROUPS_MAX && dtype >= FLM_F32 && dtype <= FLM_F16;
}

extern "C" long flm_adapter_workspace(int n, int K, int N, int r, int E, int dtype) {
  if (!adapter_sizes(n, K, N, r, E, dtype)) return 0;
  return round16(4L * shrink_plan(n, K, E).slices * n * ranks_padded(r)) + base_part_bytes(base_plan(n, K, N, r, E, dtype == FLM_F32), n, N) +
         256;
}

extern "C" long flm_adapter_backward_workspace(int n, int K, int N, int r, int E, int dtype, int need_dx) {
  if (!adapter_sizes(n, K, N, r, E, dtype)) return 0;
  const long tiles = row_tiles_cap(n, E);
  long rest = 4L * r * outer_part(tiles, outer_chunk(tiles, n, E, K, N, r, dtype == FLM_F32 ? 3 : (dtype == FLM_BF16 ? 1 : 2))) * ((long)K + N);
  if (need_dx) {
    const long base = base_part_bytes(base_plan(n, N, K, r, E, dtype == FLM_F32, true), n, K);
    if (base > rest) rest = base;
  }
  return round16(4L * shrink_plan(n, N, E).slices * n * ranks_padded(r)) + rest + 256;
}

extern "C" int flm_adapter_linear(const void* x, long ldx, const void* w, long ldw, const void* bias, const void* a, const void* b,
                                  const int32_t* groups, const float* scale, float scale_all, int n, int K, int N, int r, int E,
                                  int dtype, void* workspace, void* y, long ldy, float* low, void* stream) {
  if (!x || !w || !a || !b || !groups || !workspace || !y || !adapter_sizes(n, K, N, r, E, dtype) || ldx < 0 || ldw < 0 || ldy < N ||
      ((uintptr_t)workspace & 15))
    return FLM_E_ARG;
  const int size = dtype == FLM_F32 ? 4 : 2;
  if (misplaced(size, {x, w, bias, a, b, y}) || misplaced(4, {scale, low}) || misplaced(16, {groups})) return FLM_E_ARG;
  const long words = 4 / size;                             // elements of the call's type in a float or an int
  const Span in[] = {{x, ldx, n, K}, {w, ldw, N, K}, {bias, 0, 1, N}, {a, 0, 1, (long)E * r * K}, {b, 0, 1, (long)E * N * r},
                     {scale, 0, 1, E * words}, {groups, 0, 1, row_groups_ints(n, E) * words}};
  const Span out[] = {{y, ldy, n, N}, {low, 0, 1, (long)n * r * words}};
  if (spans_meet(out[0], out[1], size)) return FLM_E_OVERLAP;
  for (const Span& o : out)
    for (const Span& i : in)
      if (spans_meet(o, i, size)) return FLM_E_OVERLAP;
  const RowGroups g = row_groups(groups, n, E);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == FLM_F32) return forward<float>(x, ldx, w, ldw, bias, a, b, g, scale, scale_all, n, K, N, r, E, (char*)workspace, y, ldy, low, st);
  if (dtype == FLM_BF16) return forward<__bf16>(x, ldx, w, ldw, bias, a, b, g, scale, scale_all, n, K, N, r, E, (char*)workspace, y, ldy, low, st);
  return forward<_Float16>(x, ldx, w, ldw, bias, a, b, g, scale, scale_all, n, K, N, r, E, (char*)workspace, y, ldy, low, st);
}

extern "C" int flm_adapter_linear_backward(const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw, const void* a,
                                           const void* b, const int32_t* groups, const float* scale, float scale_all,
                                           const float* low, int n, int K, int N, int r, int E, int dtype, void* workspace, void* dx,
                                           long lddx, void* da, void* db, void* stream) {
  if (!dy || !x || !b || !groups || !low || !workspace || !da || !db || !adapter_sizes(n, K, N, r, E, dtype) || lddy < 0 ||
      ldx < 0 || (dx && (!w || !a || ldw < 0 || lddx < K)) || ((uintptr_t)workspace & 15))
    return FLM_E_ARG;
  const int size = dtype == FLM_F32 ? 4 : 2;
  if (misplaced(size, {dy, x, w, a, b, dx, da, db}) || misplaced(4, {scale, low}) || misplaced(16, {groups})) return FLM_E_ARG;
  const long na = (long)E * r * K, nb = (long)E * N * r, words = 4 / size;
  const Span in[] = {{dy, lddy, n, N}, {x, ldx, n, K}, {dx ? w : nullptr, ldw, N, K}, {dx ? a : nullptr, 0, 1, na}, {b, 0, 1, nb},
                     {low, 0, 1, (long)n * r * words}, {scale, 0, 1, E * words}, {groups, 0, 1, row_groups_ints(n, E) * words}};
  const Span out[] = {{da, 0, 1, na}, {db, 0, 1, nb}, {dx, lddx, n, K}};
  for (int i = 0; i < 3; i++) {
    for (const Span& s : in)
      if (spans_meet(out[i], s, size)) return FLM_E_OVERLAP;
    for (int j = 0; j < i; j++)
      if (spans_meet(out[i], out[j], size)) return FLM_E_OVERLAP;
  }
  const RowGroups g = row_groups(groups, n, E);
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  if (dtype == FLM_F32) return backward<float>(dy, lddy, x, ldx, w, ldw, a, b, g, scale, scale_all, low, n, K, N, r, E, ws, dx, lddx, da, db, st);
  if (dtype == FLM_BF16) return backward<__bf16>(dy, lddy, x, ldx, w, ldw, a, b, g, scale, scale_all, low, n, K, N, r, E, ws, dx, lddx, da, db, st);
  return backward<_Float16>(dy, lddy, x, ldx, w, ldw, a, b, g, scale, scale_all, low, n, K, N, r, E, ws, dx, lddx, da, db, st);
}
