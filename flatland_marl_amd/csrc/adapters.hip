// A shared projection with low-rank adapters of many requests at once, and its backward pass, on gfx950.
//
//   low_i = A_e x_i                       e = the adapter of row i, A [E,r,K], B [E,N,r]
//   y_i   = W x_i + bias + s_e B_e low_i  (rows without an adapter: the projection alone)
//   u_i   = s_e B_e^T dy_i,   dx_i = W^T dy_i + A_e^T u_i
//   dA_e  = sum_{i of e} u_i x_i^T,   dB_e = s_e sum_{i of e} dy_i low_i^T
//
// Rows are taken in the order of a grouping (flm_group_rows): tiles of rows that share an adapter.  Types: fp32, bf16,
// fp16 for all tensors of a call; every sum is kept in fp32 and rounded once, at the end.  fp32 operands enter the matrix
// cores as three bf16 terms each (rounded to nearest: the six products that are kept leave out less than 2^-25 of the
// largest); the narrow products low and u stay fp32 in memory and enter the next product as two bf16 terms beside bf16 or
// fp16 operands (2^-17 of the value, far below the rounding of the result).
#include "flm_adapters.h"

namespace flm {

// the split-operand fp32 product of the dense layers (dqn.hip): C[slice][M,N] = A[M,K] * B over the K slices;
// B is [N,K] (b_kc) or [K,N]
int gemm_x3_slices(const float* A, long lda, const float* B, long ldb, bool b_kc, float* C, int M, int N, int K, int slices,
                   int kslice, hipStream_t stream);

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// ---- eight consecutive elements, at any alignment the type allows ------------------------------------------------
template <typename T> struct Vec8 { T v[8]; };
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Packed8 { T v[8]; };
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Packed4 { T v[4]; };

// avail: elements that exist from p on (may be <= 0: zeros, nothing is read)
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p, long avail) {
  Vec8<T> o;
  if (avail >= 8) {
    const Packed8<T> t = *reinterpret_cast<const Packed8<T>*>(p);
#pragma unroll
    for (int j = 0; j < 8; j++) o.v[j] = t.v[j];
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
    Packed4<T> t;
#pragma unroll
    for (int j = 0; j < 4; j++) t.v[j] = (T)v[j];
    *reinterpret_cast<Packed4<T>*>(p) = t;
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j < avail) p[j] = (T)v[j];
  }
}

// ---- operands as bf16 terms ---------------------------------------------------------------------------------------
// x = t[0] + t[1] + ... with every term rounded to nearest.  A value that is infinite in bf16 keeps zero in its further
// terms (its difference from itself would be NaN).
template <int N>
__device__ __forceinline__ void split_terms(const float (&x)[8], bf16x8 (&t)[N]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f32x2 r;
    r[0] = x[2 * i];
    r[1] = x[2 * i + 1];
#pragma unroll
    for (int s = 0; s < N; s++) {
      const bf16x2 h = __builtin_convertvector(r, bf16x2);
      t[s][2 * i] = h[0];
      t[s][2 * i + 1] = h[1];
      if (s + 1 < N) {
        const f32x2 f = __builtin_convertvector(h, f32x2);
        r[0] = __builtin_fabsf(f[0]) < __builtin_inff() ? r[0] - f[0] : 0.f;
        r[1] = __builtin_fabsf(f[1]) < __builtin_inff() ? r[1] - f[1] : 0.f;
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
#pragma unroll
    for (int j = 0; j < 8; j++) t[0][j] = v.v[j];
  } else {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = (float)v.v[j];
    split_terms<Terms<T>::own>(f, t);
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

// operands of the wide products: 16-bit types as they are, fp32 as three bf16 terms
template <typename T> struct Operand { typedef bf16x8 V; };
template <> struct Operand<_Float16> { typedef f16x8 V; };
template <typename T> struct Wide { typename Operand<T>::V t[1]; };
template <> struct Wide<float> { bf16x8 t[3]; };

__device__ __forceinline__ Wide<__bf16> wide(const Vec8<__bf16>& v) {
  Wide<__bf16> w;
#pragma unroll
  for (int j = 0; j < 8; j++) w.t[0][j] = v.v[j];
  return w;
}
__device__ __forceinline__ Wide<_Float16> wide(const Vec8<_Float16>& v) {
  Wide<_Float16> w;
#pragma unroll
  for (int j = 0; j < 8; j++) w.t[0][j] = v.v[j];
  return w;
}
__device__ __forceinline__ Wide<float> wide(const Vec8<float>& v) {
  Wide<float> w;
  split_terms<3>(v.v, w.t);
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
// A workgroup of four waves forms 16*MR rows of X times 16*NR rows of V over k_begin..k_end: the waves take 64 k in turn,
// both operands straight from memory in the matrix instruction's layout (a lane reads 16 consecutive elements of one row;
// which k a lane holds is the same for both operands, so their order does not matter), and meet in LDS.  Nothing is reused
// between workgroups but through the L2, so this form is for operands that are read once: few rows, or few columns.
// result: lane (c = lane & 15, q = lane >> 4) holds D[v = 16*ni + 4q .. +3][x = 16*mi + c]
#define MINI_K 64
template <typename T, int MR, int NR, bool V_STRIDED>
__device__ __forceinline__ void mini_product(const T* const (&xr)[MR], const T* const (&vr)[NR], long v_stride, int k_begin,
                                             int k_end, f32x4 (&acc)[MR][NR]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, q = lane >> 4;
#pragma unroll
  for (int mi = 0; mi < MR; mi++)
#pragma unroll
    for (int ni = 0; ni < NR; ni++) acc[mi][ni] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k0 = k_begin + w * MINI_K; k0 < k_end; k0 += 4 * MINI_K) {
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int k = k0 + q * 16 + s * 8;
      const int avail = k_end - k;
      Wide<T> x[MR];
#pragma unroll
      for (int mi = 0; mi < MR; mi++) x[mi] = wide(load8(xr[mi] + k, xr[mi] ? avail : 0));
#pragma unroll
      for (int ni = 0; ni < NR; ni++) {
        const int have = vr[ni] ? avail : 0;
        const Wide<T> v = wide(V_STRIDED ? load8_strided(vr[ni] + (long)k * v_stride, v_stride, have) : load8(vr[ni] + k, have));
#pragma unroll
        for (int mi = 0; mi < MR; mi++) acc[mi][ni] = mul16(v, x[mi], acc[mi][ni]);
      }
    }
  }
}

// sums the four waves' results; f(mi, ni, values) is called by one wave per pair
template <int MR, int NR, typename F>
__device__ __forceinline__ void mini_meet(const f32x4 (&acc)[MR][NR], f32x4* red, F&& f) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int mi = 0; mi < MR; mi++)
#pragma unroll
    for (int ni = 0; ni < NR; ni++) red[(w * MR * NR + mi * NR + ni) * 64 + lane] = acc[mi][ni];
  __syncthreads();
  for (int s = w; s < MR * NR; s += 4) {
    f32x4 v = red[s * 64 + lane];
#pragma unroll
    for (int k = 1; k < 4; k++) v += red[(k * MR * NR + s) * 64 + lane];
    f(s / NR, s - s / NR * NR, v);
  }
}

struct ShrinkArgs {
  const void *x, *v;
  long ldx, v_group, v_row, v_k;         // V_e(j, k) = v[e*v_group + j*v_row + k*v_k]
  int K, r, rp, n, kslice;
  float* out;                            // [slice][sorted position][rp]
};

// low (or u): tiles of rows of one adapter times its r vectors; grid (tiles, K slices)
template <typename T, int MR, int NR, bool V_STRIDED>
__global__ __launch_bounds__(256) void shrink_kernel(ShrinkArgs a, RowGroups g) {
  __shared__ f32x4 red[4 * MR * NR * 64];
  const int2 tile = g.tiles[blockIdx.x];
  const int rows = tile.y >> 16, e = tile.y & 0xffff;
  if (rows == 0) return;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int k_begin = blockIdx.y * a.kslice, k_end = min(a.K, k_begin + a.kslice);
  // (a tile holds up to 32 rows; MR = 1 is only launched for calls of up to 16 rows)
  const T *xr[MR], *vr[NR];
#pragma unroll
  for (int mi = 0; mi < MR; mi++) {
    const int m = mi * 16 + c;
    xr[mi] = m < rows ? (const T*)a.x + (long)g.order[tile.x + m] * a.ldx : nullptr;
  }
#pragma unroll
  for (int ni = 0; ni < NR; ni++) {
    const int j = ni * 16 + c;
    vr[ni] = j < a.r ? (const T*)a.v + (long)e * a.v_group + (long)j * a.v_row : nullptr;
  }
  f32x4 acc[MR][NR];
  mini_product<T, MR, NR, V_STRIDED>(xr, vr, a.v_k, k_begin, k_end, acc);
  mini_meet<MR, NR>(acc, red, [&](int mi, int ni, const f32x4& v) {
    const int m = mi * 16 + c, j = ni * 16 + 4 * q;
    if (m < rows && j < a.rp)
      *reinterpret_cast<f32x4*>(a.out + ((long)blockIdx.y * a.n + tile.x + m) * a.rp + j) = v;
  });
}

struct BaseArgs {
  const void *x, *w;
  long ldx, ldw;
  int n, K, N, kslice;
  float* part;                           // [slice][n][N]
};

// the projection of up to 16*MR rows: 16 outputs a workgroup, grid (outputs / 16, K slices)
template <typename T, int MR>
__global__ __launch_bounds__(256) void base_rows_kernel(BaseArgs a) {
  __shared__ f32x4 red[4 * MR * 64];
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int k_begin = blockIdx.y * a.kslice, k_end = min(a.K, k_begin + a.kslice);
  const T *xr[MR], *vr[1];
#pragma unroll
  for (int mi = 0; mi < MR; mi++) xr[mi] = mi * 16 + c < a.n ? (const T*)a.x + (long)(mi * 16 + c) * a.ldx : nullptr;
  vr[0] = n0 + c < a.N ? (const T*)a.w + (long)(n0 + c) * a.ldw : nullptr;
  f32x4 acc[MR][1];
  mini_product<T, MR, 1, false>(xr, vr, 1, k_begin, k_end, acc);
  mini_meet<MR, 1>(acc, red, [&](int mi, int, const f32x4& v) {
    const int m = mi * 16 + c, n = n0 + 4 * q;
    if (m < a.n) {
      const float f[4] = {v[0], v[1], v[2], v[3]};
      store4(a.part + ((long)blockIdx.y * a.n + m) * a.N + n, f, a.N - n);
    }
  });
}

// ---- the projection of many rows, 16-bit types -------------------------------------------------------------------------
// part[slice][n][N] = X[n,K] * W[N,K]^T: tiles of 128 x 128, four waves of 64 x 64, 32 k a stage, the next stage fetched
// into registers while the matrix cores work on the one in LDS.  Any sizes and strides.
#define BT_ROW 40                        // elements per LDS row of 32 k
template <typename T>
__global__ __launch_bounds__(256) void base_tile_kernel(BaseArgs a) {
  __shared__ __attribute__((aligned(16))) T lx[128 * BT_ROW], lw[128 * BT_ROW];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = lane & 31, h = lane >> 5;
  const int m0 = blockIdx.y * 128, n0 = blockIdx.x * 128, wm = (w >> 1) * 64, wn = (w & 1) * 64;
  const int k_begin = blockIdx.z * a.kslice, k_end = min(a.K, k_begin + a.kslice);
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
  Vec8<T> fx[2], fw[2];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int row = (tid >> 2) + 64 * s, k = k0 + (tid & 3) * 8;
      fx[s] = load8((const T*)a.x + (long)(m0 + row) * a.ldx + k, m0 + row < a.n ? k_end - k : 0);
      fw[s] = load8((const T*)a.w + (long)(n0 + row) * a.ldw + k, n0 + row < a.N ? k_end - k : 0);
    }
  };
  fetch(k_begin);
  for (int k0 = k_begin; k0 < k_end; k0 += 32) {
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int at = ((tid >> 2) + 64 * s) * BT_ROW + (tid & 3) * 8;
      *reinterpret_cast<uint4*>(lx + at) = __builtin_bit_cast(uint4, fx[s]);
      *reinterpret_cast<uint4*>(lw + at) = __builtin_bit_cast(uint4, fw[s]);
    }
    __syncthreads();
    if (k0 + 32 < k_end) fetch(k0 + 32);
#pragma unroll
    for (int s = 0; s < 2; s++) {
      typedef typename Operand<T>::V V;
      V x[2], v[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        x[i] = __builtin_bit_cast(V, *reinterpret_cast<const uint4*>(lx + (wm + i * 32 + c) * BT_ROW + s * 16 + h * 8));
        v[i] = __builtin_bit_cast(V, *reinterpret_cast<const uint4*>(lw + (wn + i * 32 + c) * BT_ROW + s * 16 + h * 8));
      }
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = mul32(v[j], x[i], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int m = m0 + wm + i * 32 + c;
    if (m >= a.n) continue;
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int r4 = 0; r4 < 4; r4++) {
        const int n = n0 + wn + j * 32 + 8 * r4 + 4 * h;
        const float f[4] = {acc[i][j][4 * r4], acc[i][j][4 * r4 + 1], acc[i][j][4 * r4 + 2], acc[i][j][4 * r4 + 3]};
        store4(a.part + ((long)blockIdx.z * a.n + m) * a.N + n, f, a.N - n);
      }
  }
}

// out[C][R] = in[R][C] (the weight with its contraction axis last, for the gradient of the inputs)
template <typename T>
__global__ __launch_bounds__(256) void transpose_kernel(const T* __restrict__ in, long ld, int R, int C, T* __restrict__ out) {
  __shared__ T t[64][66];
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int r = i >> 6, c = i & 63;
    if (r0 + r < R && c0 + c < C) t[r][c] = in[(long)(r0 + r) * ld + c0 + c];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int c = i >> 6, r = i & 63;
    if (r0 + r < R && c0 + c < C) out[(long)(c0 + c) * R + r0 + r] = t[r][c];
  }
}

// ---- the adapters' part and the result ---------------------------------------------------------------------------------
struct FinishArgs {
  const float* part;                     // [slices][n][N], rows in their own order
  int slices;
  const void* bias;
  const float* low;                      // [low_slices][sorted position][rp]
  int low_slices, r, rp;
  const void* v;                         // V_e(n, j) = v[e*v_group + n*v_row + j*v_j]
  long v_group, v_row, v_j;
  const float* scale;                    // per adapter, or nullptr: scale_all
  float scale_all;
  int n, N, E;
  void* y;
  long ldy;
};

__device__ __forceinline__ float adapter_scale(const float* scale, float all, int e) { return scale ? scale[e] : all; }

// Adds s_e * low_i . V_e(n, .) to acc: lane (c, h) of the wave holds row (sorted position) pos + c of a tile of 32, outputs
// n0 + 8*(r >> 2) + 4*h + (r & 3).  The rows of a tile may use several adapters: each adapter's product is formed apart and
// added to its own rows only, so that no value of one adapter (an infinity, a NaN) can reach the rows of another.
// key: the lane's adapter (E or more: none).  All lanes of the wave take part.
template <typename T, bool V_STRIDED>
__device__ __forceinline__ void add_adapters(const FinishArgs& a, long pos, int key, int n0, f32x16& acc) {
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  unsigned todo = (unsigned)__ballot(key < a.E);                  // (both halves of the wave hold the same 32 rows)
  while (todo) {
    const int first = __builtin_ctz(todo);
    const int e = __builtin_amdgcn_readlane(key, first);
    todo &= ~(unsigned)__ballot(key == e);
    const float s = adapter_scale(a.scale, a.scale_all, e);
    f32x16 t;
#pragma unroll
    for (int r = 0; r < 16; r++) t[r] = 0.f;
    const bool mine = key == e;
    for (int j0 = 0; j0 < a.r; j0 += 16) {
      const int j = j0 + 8 * h;
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = 0.f;
      if (mine)
        for (int z = 0; z < a.low_slices; z++) {
          const float* p = a.low + ((long)z * a.n + pos + c) * a.rp + j;
          const f32x4 p0 = reinterpret_cast<const f32x4*>(p)[0], p1 = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            f[i] += p0[i];
            f[4 + i] += p1[i];
          }
        }
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = j + i < a.r ? f[i] * s : 0.f;
      bf16x8 lt[Terms<T>::low], vt[Terms<T>::own];
      split_terms<Terms<T>::low>(f, lt);
      const int n = n0 + c;
      const T* vp = (const T*)a.v + (long)e * a.v_group + (long)n * a.v_row + (long)j * a.v_j;
      const int have = n < a.N ? a.r - j : 0;
      own_terms<T>(V_STRIDED ? load8_strided(vp, a.v_j, have) : load8(vp, have), vt);
      t = mul_terms32<Terms<T>::own, Terms<T>::low>(vt, lt, t);
    }
#pragma unroll
    for (int r = 0; r < 16; r++) acc[r] = mine ? acc[r] + t[r] : acc[r];
  }
}

// y = sum of the K slices + bias + adapters, for 32 sorted rows and 128 outputs a workgroup
template <typename T, bool V_STRIDED>
__global__ __launch_bounds__(256) void finish_kernel(FinishArgs a, RowGroups g) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int n0 = blockIdx.x * 128 + w * 32;
  const long pos = (long)blockIdx.y * 32;
  const bool in = pos + c < a.n;
  const int row = in ? g.order[pos + c] : 0;
  const int key = in ? g.key[pos + c] : a.E;
  if (n0 >= a.N) return;
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; r++) acc[r] = 0.f;
  if (in) {
    for (int z = 0; z < a.slices; z++) {
      const float* p = a.part + ((long)z * a.n + row) * a.N;
#pragma unroll
      for (int r4 = 0; r4 < 4; r4++) {
        const int n = n0 + 8 * r4 + 4 * h;
        if (n + 4 <= a.N) {
          const Packed4<float> f = *reinterpret_cast<const Packed4<float>*>(p + n);
#pragma unroll
          for (int i = 0; i < 4; i++) acc[4 * r4 + i] += f.v[i];
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (n + i < a.N) acc[4 * r4 + i] += p[n + i];
        }
      }
    }
    if (a.bias) {
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int n = n0 + 8 * (r >> 2) + 4 * h + (r & 3);
        if (n < a.N) acc[r] += (float)((const T*)a.bias)[n];
      }
    }
  }
  add_adapters<T, V_STRIDED>(a, pos, key, n0, acc);
  if (in) {
    T* y = (T*)a.y + (long)row * a.ldy;
#pragma unroll
    for (int r4 = 0; r4 < 4; r4++) {
      const int n = n0 + 8 * r4 + 4 * h;
      const float f[4] = {acc[4 * r4], acc[4 * r4 + 1], acc[4 * r4 + 2], acc[4 * r4 + 3]};
      store4(y + n, f, a.N - n);
    }
  }
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
// The sorted rows are cut into chunks of equal length whatever the groups' sizes; a workgroup walks the groups inside its
// chunk for 256 columns of Q.  A group that lies inside one chunk is written at once; a longer one leaves a partial sum
// per chunk (at most two a chunk: the group it begins in and the one it ends in), added up in order by a second launch,
// which also clears the groups without rows.
struct OuterArgs {
  const float* p;                        // [p_slices][.][pld]: by sorted position, or (p_gather) by row
  int p_slices, pld, p_gather;
  long p_slice;                          // floats per slice
  const void* q;
  long ldq;
  int KQ, r, E, n, chunk;
  const float* scale;
  float scale_all;
  float* part;                           // [chunks][2][r][KQ]
  void* out;                             // out[e*r*KQ + j*o_j + q*o_q]
  long o_j, o_q;
};

template <typename T, int NRJ>
__global__ __launch_bounds__(256) void outer_kernel(OuterArgs a, RowGroups g) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
  const int q0 = blockIdx.x * 256 + w * 64;
  if (q0 >= a.KQ) return;
  const int c0 = blockIdx.y * a.chunk;
  const int c1 = min(c0 + a.chunk, g.offsets[a.E]);
  int pos = c0;
  while (pos < c1) {
    const int e = g.key[pos];
    const int begin = g.offsets[e], finish = g.offsets[e + 1];
    const int end = min(finish, c1);
    const float s = adapter_scale(a.scale, a.scale_all, e);
    f32x16 acc[2][NRJ];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < NRJ; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
    for (int p = pos; p < end; p += 16) {
      int row[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int at = p + 8 * h + i;
        row[i] = at < end ? g.order[at] : -1;
      }
      bf16x8 qt[2][Terms<T>::own];
#pragma unroll
      for (int sub = 0; sub < 2; sub++) {
        const int q = q0 + sub * 32 + c;
        Vec8<T> v;
#pragma unroll
        for (int i = 0; i < 8; i++) v.v[i] = row[i] >= 0 && q < a.KQ ? ((const T*)a.q)[(long)row[i] * a.ldq + q] : (T)0.f;
        own_terms<T>(v, qt[sub]);
      }
#pragma unroll
      for (int jj = 0; jj < NRJ; jj++) {
        const int j = jj * 32 + c;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          f[i] = 0.f;
          if (row[i] >= 0 && j < a.r) {
            const long at = (long)(a.p_gather ? row[i] : p + 8 * h + i) * a.pld + j;
            for (int z = 0; z < a.p_slices; z++) f[i] += a.p[z * a.p_slice + at];
            f[i] *= s;
          }
        }
        bf16x8 pt[Terms<T>::low];
        split_terms<Terms<T>::low>(f, pt);
#pragma unroll
        for (int sub = 0; sub < 2; sub++) acc[sub][jj] = mul_terms32<Terms<T>::own, Terms<T>::low>(qt[sub], pt, acc[sub][jj]);
      }
    }
    const bool whole = begin >= c0 && finish <= c0 + a.chunk;
    float* part = a.part + ((long)blockIdx.y * 2 + (begin < c0 ? 0 : 1)) * a.r * a.KQ;
    T* out = (T*)a.out + (long)e * a.r * a.KQ;
#pragma unroll
    for (int sub = 0; sub < 2; sub++)
#pragma unroll
      for (int jj = 0; jj < NRJ; jj++) {
        const int j = jj * 32 + c;
        if (j >= a.r) continue;
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++) {
          const int q = q0 + sub * 32 + 8 * r4 + 4 * h;
          const float f[4] = {acc[sub][jj][4 * r4], acc[sub][jj][4 * r4 + 1], acc[sub][jj][4 * r4 + 2], acc[sub][jj][4 * r4 + 3]};
          if (!whole) {
            store4(part + (long)j * a.KQ + q, f, a.KQ - q);
          } else if (a.o_q == 1) {
            store4(out + (long)j * a.o_j + q, f, a.KQ - q);
          } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (q + i < a.KQ) out[(long)j * a.o_j + (long)(q + i) * a.o_q] = (T)f[i];
          }
        }
      }
    pos = end;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void outer_join_kernel(OuterArgs a, RowGroups g) {
  const int e = blockIdx.y;
  const int begin = g.offsets[e], end = g.offsets[e + 1];
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long total = (long)a.r * a.KQ;
  if (i >= total) return;
  const int first = begin / a.chunk, last = (end - 1) / a.chunk;
  if (begin < end && first == last) return;
  const int j = (int)(i / a.KQ), q = (int)(i - (long)j * a.KQ);
  float s = 0.f;
  if (begin < end)
    for (int k = first; k <= last; k++) s += a.part[((long)k * 2 + (begin < k * a.chunk ? 0 : 1)) * total + i];
  ((T*)a.out)[(long)e * total + (long)j * a.o_j + (long)q * a.o_q] = (T)s;
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

// Up to this many rows the projection's weight is streamed past all rows at once (base_rows_kernel).
#define BASE_ROWS_MAX 64

struct BaseSlices { int slices, kslice; };
static BaseSlices base_slices(int n, int K, int N) {
  BaseSlices b;
  if (n <= BASE_ROWS_MAX) b.slices = k_slices((N + 15) / 16, 768, K, 512, 32, &b.kslice);
  else b.slices = k_slices((long)((n + 127) / 128) * ((N + 127) / 128), 512, K, 512, 16, &b.kslice);
  return b;
}
static BaseSlices shrink_slices(int n, int K, int E) {
  BaseSlices b;
  b.slices = k_slices(row_tiles_cap(n, E), 512, K, 256, 32, &b.kslice);
  return b;
}

template <typename T, bool V_STRIDED>
static int launch_shrink(const ShrinkArgs& a, const RowGroups& g, int slices, hipStream_t st) {
  const dim3 grid(g.cap, slices);
  if (a.n <= 16) {
    if (a.rp <= 16) hipLaunchKernelGGL((shrink_kernel<T, 1, 1, V_STRIDED>), grid, dim3(256), 0, st, a, g);
    else if (a.rp <= 32) hipLaunchKernelGGL((shrink_kernel<T, 1, 2, V_STRIDED>), grid, dim3(256), 0, st, a, g);
    else if (a.rp <= 64) hipLaunchKernelGGL((shrink_kernel<T, 1, 4, V_STRIDED>), grid, dim3(256), 0, st, a, g);
    else hipLaunchKernelGGL((shrink_kernel<T, 1, 8, V_STRIDED>), grid, dim3(256), 0, st, a, g);
  } else {
    if (a.rp <= 16) hipLaunchKernelGGL((shrink_kernel<T, 2, 1, V_STRIDED>), grid, dim3(256), 0, st, a, g);
    else if (a.rp <= 32) hipLaunchKernelGGL((shrink_kernel<T, 2, 2, V_STRIDED>), grid, dim3(256), 0, st, a, g);
    else if (a.rp <= 64) hipLaunchKernelGGL((shrink_kernel<T, 2, 4, V_STRIDED>), grid, dim3(256), 0, st, a, g);
    else hipLaunchKernelGGL((shrink_kernel<T, 2, 8, V_STRIDED>), grid, dim3(256), 0, st, a, g);
  }
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}

// part = X * W^T (W [N,K]), any type
template <typename T>
static int launch_base(const BaseArgs& a, int slices, hipStream_t st) {
  if (a.n <= BASE_ROWS_MAX) {
    const dim3 grid((a.N + 15) / 16, slices);
    if (a.n <= 16) hipLaunchKernelGGL((base_rows_kernel<T, 1>), grid, dim3(256), 0, st, a);
    else if (a.n <= 32) hipLaunchKernelGGL((base_rows_kernel<T, 2>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((base_rows_kernel<T, 4>), grid, dim3(256), 0, st, a);
  } else if constexpr (sizeof(T) == 4) {
    return gemm_x3_slices((const float*)a.x, a.ldx, (const float*)a.w, a.ldw, true, a.part, a.n, a.N, a.K, slices, a.kslice, st);
  } else {
    hipLaunchKernelGGL(base_tile_kernel<T>, dim3((a.N + 127) / 128, (a.n + 127) / 128, slices), dim3(256), 0, st, a);
  }
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}

template <typename T, bool V_STRIDED>
static int launch_finish(const FinishArgs& a, const RowGroups& g, hipStream_t st) {
  hipLaunchKernelGGL((finish_kernel<T, V_STRIDED>), dim3((a.N + 127) / 128, (a.n + 31) / 32), dim3(256), 0, st, a, g);
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}

template <typename T>
static int launch_outer(const OuterArgs& a, const RowGroups& g, hipStream_t st) {
  const dim3 grid((a.KQ + 255) / 256, (a.n + a.chunk - 1) / a.chunk);
  if (a.r <= 32) hipLaunchKernelGGL((outer_kernel<T, 1>), grid, dim3(256), 0, st, a, g);
  else if (a.r <= 64) hipLaunchKernelGGL((outer_kernel<T, 2>), grid, dim3(256), 0, st, a, g);
  else hipLaunchKernelGGL((outer_kernel<T, 4>), grid, dim3(256), 0, st, a, g);
  FLM_CHECK_LAUNCH();
  hipLaunchKernelGGL(outer_join_kernel<T>, dim3((unsigned)(((long)a.r * a.KQ + 255) / 256), a.E), dim3(256), 0, st, a, g);
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}

static long round16(long bytes) { return (bytes + 255) & ~255L; }

// rows of sorted positions a workgroup of outer_kernel takes
static int outer_chunk(int n, int KQ) {
  const long cols = (KQ + 255) / 256;
  long chunks = (768 + cols - 1) / cols;
  long c = ((n + chunks - 1) / chunks + 15) & ~15L;
  if (c < 64) c = 64;
  return (int)c;
}

template <typename T>
static int forward(const void* x, long ldx, const void* w, long ldw, const void* bias, const void* a, const void* b,
                   const RowGroups& g, const float* scale, float scale_all, int n, int K, int N, int r, int E, char* ws, void* y,
                   long ldy, float* low, hipStream_t st) {
  const int rp = ranks_padded(r);
  const BaseSlices ss = shrink_slices(n, K, E), bs = base_slices(n, K, N);
  float* low_part = (float*)ws;
  float* part = (float*)(ws + round16(4L * ss.slices * n * rp));
  int rc = launch_shrink<T, false>(ShrinkArgs{x, a, ldx, (long)r * K, K, 1, K, r, rp, n, ss.kslice, low_part}, g, ss.slices, st);
  if (rc) return rc;
  if ((rc = launch_base<T>(BaseArgs{x, w, ldx, ldw, n, K, N, bs.kslice, part}, bs.slices, st))) return rc;
  if ((rc = launch_finish<T, false>(FinishArgs{part, bs.slices, bias, low_part, ss.slices, r, rp, b, (long)N * r, r, 1, scale,
                                               scale_all, n, N, E, y, ldy},
                                    g, st)))
    return rc;
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
  const BaseSlices ss = shrink_slices(n, N, E);
  float* u = (float*)ws;                                             // s_e is applied where u is used
  ws += round16(4L * ss.slices * n * rp);
  int rc = launch_shrink<T, true>(ShrinkArgs{dy, b, lddy, (long)N * r, 1, r, N, r, rp, n, ss.kslice, u}, g, ss.slices, st);
  if (rc) return rc;
  const int ca = outer_chunk(n, K), cb = outer_chunk(n, N);
  float* part = (float*)ws;                                          // both gradients in turn
  if ((rc = launch_outer<T>(OuterArgs{u, ss.slices, rp, 0, (long)n * rp, x, ldx, K, r, E, n, ca, scale, scale_all, part, da, K, 1},
                            g, st)))
    return rc;
  if ((rc = launch_outer<T>(OuterArgs{low, 1, r, 1, 0, dy, lddy, N, r, E, n, cb, scale, scale_all, part, db, 1, r}, g, st)))
    return rc;
  if (!dx) return FLM_OK;
  const BaseSlices bs = base_slices(n, N, K);
  float* dx_part = (float*)ws;
  if constexpr (sizeof(T) == 4) {
    if (n > BASE_ROWS_MAX) {
      rc = gemm_x3_slices((const float*)dy, lddy, (const float*)w, ldw, false, dx_part, n, K, N, bs.slices, bs.kslice, st);
      if (rc) return rc;
    }
  }
  if (sizeof(T) != 4 || n <= BASE_ROWS_MAX) {
    T* wt = (T*)(ws + round16(4L * bs.slices * n * K));
    hipLaunchKernelGGL(transpose_kernel<T>, dim3((K + 63) / 64, (N + 63) / 64), dim3(256), 0, st, (const T*)w, ldw, N, K, wt);
    FLM_CHECK_LAUNCH();
    if ((rc = launch_base<T>(BaseArgs{dy, wt, lddy, N, n, N, K, bs.kslice, dx_part}, bs.slices, st))) return rc;
  }
  return launch_finish<T, true>(FinishArgs{dx_part, bs.slices, nullptr, u, ss.slices, r, rp, a, (long)r * K, 1, K, scale, scale_all,
                                           n, K, E, dx, lddx},
                                g, st);
}

}  // namespace flm

using namespace flm;

static bool adapter_sizes(int n, int K, int N, int r, int E, int dtype) {
  return n > 0 && n <= (1 << 20) && K > 0 && N > 0 && K <= (1 << 20) && N <= (1 << 20) && r > 0 && r <= FLM_ADAPTER_MAX_RANK && E > 0 &&
         E <= FLM_GROUPS_MAX && dtype >= FLM_F32 && dtype <= FLM_F16;
}

extern "C" long flm_adapter_workspace(int n, int K, int N, int r, int E) {
  if (!adapter_sizes(n, K, N, r, E, FLM_F32)) return 0;
  return round16(4L * shrink_slices(n, K, E).slices * n * ranks_padded(r)) + round16(4L * base_slices(n, K, N).slices * n * N);
}

extern "C" long flm_adapter_backward_workspace(int n, int K, int N, int r, int E, int dtype, int need_dx) {
  if (!adapter_sizes(n, K, N, r, E, dtype)) return 0;
  const int ca = outer_chunk(n, K), cb = outer_chunk(n, N);
  const long pa = 8L * ((n + ca - 1) / ca) * r * K, pb = 8L * ((n + cb - 1) / cb) * r * N;
  long rest = pa > pb ? pa : pb;
  if (need_dx) {
    const long base = round16(4L * base_slices(n, N, K).slices * n * K) +
                      (dtype == FLM_F32 && n > BASE_ROWS_MAX ? 0 : (dtype == FLM_F32 ? 4L : 2L) * K * N);
    if (base > rest) rest = base;
  }
  return round16(4L * shrink_slices(n, N, E).slices * n * ranks_padded(r)) + rest;
}

extern "C" int flm_adapter_linear(const void* x, long ldx, const void* w, long ldw, const void* bias, const void* a, const void* b,
                                  const int32_t* groups, const float* scale, float scale_all, int n, int K, int N, int r, int E,
                                  int dtype, void* workspace, void* y, long ldy, float* low, void* stream) {
  if (!x || !w || !a || !b || !groups || !workspace || !y || !adapter_sizes(n, K, N, r, E, dtype) || ldx < 0 || ldw < 0 || ldy < N ||
      ((uintptr_t)workspace & 15))
    return FLM_E_ARG;
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
  const RowGroups g = row_groups(groups, n, E);
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  if (dtype == FLM_F32) return backward<float>(dy, lddy, x, ldx, w, ldw, a, b, g, scale, scale_all, low, n, K, N, r, E, ws, dx, lddx, da, db, st);
  if (dtype == FLM_BF16) return backward<__bf16>(dy, lddy, x, ldx, w, ldw, a, b, g, scale, scale_all, low, n, K, N, r, E, ws, dx, lddx, da, db, st);
  return backward<_Float16>(dy, lddy, x, ldx, w, ldw, a, b, g, scale, scale_all, low, n, K, N, r, E, ws, dx, lddx, da, db, st);
}
