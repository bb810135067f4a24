// Global gradient norm over many tensors, and clipping, on gfx950.
//
//   norm = sqrt(sum over every element of every tensor of g^2)   (or max |g|)
//   g   *= min(1, max_norm / (norm + 1e-6))
//
// Two launches: every workgroup sums (or maximises) its share of the tensors into one partial result; then every
// workgroup folds all partial results itself, in the same order, and scales its share.  Sums are kept in 64 bits: the
// square of an fp32 number then neither overflows nor vanishes (1e-30 and 1e30 are ordinary gradients to this kernel),
// and 64-bit multiply-adds run at a rate that a stream of memory does not notice.  Nothing depends on the order in which
// workgroups finish.  55 MB of fp32: 12 us for the norm (4.6 TB/s) and 21 for the scaling (5.2); 512 MB of bf16 in 291 tensors:
// 345 us, 1.6 GB at 4.6 TB/s with what the cache behind the L2s keeps of the first pass.
// The tensors' addresses travel in the launch's arguments, FLM_GRAD_LIST tensors a launch: no table in device memory has to be
// kept or refreshed by the caller.
#include <algorithm>
#include <new>
#include <vector>

#include "flm_common.h"

namespace flm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

#define FLM_GRAD_LIST 112                // tensors per launch: 32 bytes each of the 4 KiB a launch's arguments may take
#define GRAD_STEPS 12                    // a place in the list is found by halves where there are more tensors than this
#define GRAD_PARTS FLM_GRAD_WORKSPACE    // partial results at most

struct GradItem {
  const void* src;
  void* dst;                             // nullptr: the tensor only counts in the norm
  long numel;
  int first;                             // number of chunks of the list before this tensor
  int dtype;
};
struct GradList {
  GradItem item[FLM_GRAD_LIST];
  int count, chunks;
  int chunk;                             // elements a workgroup takes at a time, a multiple of 2048
};
// What the gradient holds beside the listed tensors: `times` copies of the outer products g_i (x) r, r [64], over the
// 512 + 512 values of two vectors (the first dense layer's gradient under empty rows, formed by the optimizer pass).
struct GradOuter {
  const float *r, *g0, *g1;              // r == nullptr: nothing
  double times;                          // at least one
};

template <typename T> struct Pack8;
template <> struct Pack8<float> { struct V { float v[8]; }; struct __attribute__((packed, aligned(4))) W { unsigned w[8]; }; };
template <> struct Pack8<__bf16> { struct V { __bf16 v[8]; }; struct __attribute__((packed, aligned(2))) W { unsigned w[4]; }; };
template <> struct Pack8<_Float16> { struct V { _Float16 v[8]; }; struct __attribute__((packed, aligned(2))) W { unsigned w[4]; }; };
// (memory is accessed as words at the element's alignment: the first elements of a tensor up to a 16-byte boundary are
// taken apart, but source and destination need not be aligned alike)
template <typename T> __device__ __forceinline__ typename Pack8<T>::V get8(const T* p, int i) {
  return __builtin_bit_cast(typename Pack8<T>::V, reinterpret_cast<const typename Pack8<T>::W*>(p)[i]);
}
template <typename T> __device__ __forceinline__ void put8(T* p, int i, const typename Pack8<T>::V& v) {
  reinterpret_cast<typename Pack8<T>::W*>(p)[i] = __builtin_bit_cast(typename Pack8<T>::W, v);
}
typedef unsigned u32x4 __attribute__((ext_vector_type(4), aligned(2)));
// the same past the caches
template <typename T> __device__ __forceinline__ void put8_past(T* p, int i, const typename Pack8<T>::V& v) {
  struct Q { u32x4 q[sizeof(T) / 2]; };
  const Q q = __builtin_bit_cast(Q, v);
#pragma unroll
  for (int k = 0; k < (int)sizeof(T) / 2; k++) __builtin_nontemporal_store(q.q[k], reinterpret_cast<u32x4*>(p + 8 * i) + k);
}

__device__ __forceinline__ double larger(double m, double v) { return (m == m && !(v <= m)) ? v : m; }   // NaN stays

// f(value array, count) over one chunk of a tensor, eight elements a thread and step
template <typename T>
__device__ __forceinline__ void grad_norm_chunk(const T* p, int n, int lead, int tid, int threads, bool inf_norm, double (&acc)[4]) {
  typedef typename Pack8<T>::V V;
  const int whole = n >> 3;
  auto take = [&](const V& v) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double g = (double)(float)v.v[j];
      if (inf_norm) acc[j & 3] = larger(acc[j & 3], __builtin_fabs(g));
      else acc[j & 3] = __builtin_fma(g, g, acc[j & 3]);
    }
  };
  int i = tid;
  for (; i + 3 * threads < whole; i += 4 * threads) {
    V v[4];
#pragma unroll
    for (int u = 0; u < 4; u++) v[u] = get8(p, i + u * threads);
#pragma unroll
    for (int u = 0; u < 4; u++) take(v[u]);
  }
  for (; i < whole; i += threads) take(get8(p, i));
  if (tid < (n & 7) + lead) {
    const double g = (double)(float)p[tid < lead ? tid - lead : (whole << 3) + tid - lead];
    acc[0] = inf_norm ? larger(acc[0], __builtin_fabs(g)) : __builtin_fma(g, g, acc[0]);
  }
}

// g * coef, rounded to fp32 and from there to the type.  (The fp32 value is pinned: the compiler otherwise takes some of the
// conversions from 64 to 16 bits in one step, in software, and the same element may come out differently in another kernel.)
template <typename T>
__device__ __forceinline__ T grad_scaled(T g, double coef) {
  float f = (float)((double)(float)g * coef);
  asm("" : "+v"(f));
  return (T)f;
}

template <typename T, bool PAST>
__device__ __forceinline__ void grad_scale_chunk(const T* p, T* q, int n, int lead, int tid, int threads, double coef) {
  typedef typename Pack8<T>::V V;
  const int whole = n >> 3;
  auto scaled = [&](const V& v) {
    V o;
#pragma unroll
    for (int j = 0; j < 8; j++) o.v[j] = grad_scaled(v.v[j], coef);
    return o;
  };
  int i = tid;
  for (; i + 3 * threads < whole; i += 4 * threads) {
    V v[4];
#pragma unroll
    for (int u = 0; u < 4; u++) v[u] = get8(p, i + u * threads);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      if (PAST) put8_past(q, i + u * threads, scaled(v[u]));
      else put8(q, i + u * threads, scaled(v[u]));
    }
  }
  for (; i < whole; i += threads) put8(q, i, scaled(get8(p, i)));
  if (tid < (n & 7) + lead) {
    const int j = tid < lead ? tid - lead : (whole << 3) + tid - lead;
    q[j] = grad_scaled(p[j], coef);
  }
}

// the workgroup's total of one value per thread, in a fixed order; every thread gets it.  red: 16 doubles of LDS
__device__ __forceinline__ double grad_fold(double v, bool inf_norm, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double w = __shfl_xor(v, o);
    v = inf_norm ? larger(larger(0.0, v), w) : v + w;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 6); i++) t = inf_norm ? larger(t, red[i]) : t + red[i];
  return t;
}

// Walks the chunks first, first + stride, ... of the list, or (BACK) the same chunks from the other end: the scaling pass
// starts with what the norm pass has read last.  A tensor's first chunk also holds the elements in front of its first
// 16-byte boundary; f(item, offset, count, leading) gets them as `leading` (0..7) elements before `offset`.
template <bool BACK, typename F>
__device__ __forceinline__ void grad_chunks(const GradList& list, int first, int stride, F&& f) {
  // the tensor of the first chunk: by halves down to a few, from there a step at a time (100 tensors of 1000 elements, replayed:
  // 18 -> 8.1 us; lists of ten are better off with steps alone)
  int lo = 0, hi = list.count - 1;
  const int start = BACK ? list.chunks - 1 - first : first;
  while (hi - lo > GRAD_STEPS) {
    const int mid = (lo + hi + 1) >> 1;
    if (list.item[mid].first <= start) lo = mid;
    else hi = mid - 1;
  }
  int t = BACK ? hi : lo;
  for (int i = first; i < list.chunks; i += stride) {
    const int c = BACK ? list.chunks - 1 - i : i;
    if (BACK) {
      while (list.item[t].first > c) t--;
    } else {
      while (t + 1 < list.count && list.item[t + 1].first <= c) t++;
    }
    const GradItem& it = list.item[t];
    const int size = it.dtype == FLM_F32 ? 4 : 2;
    const long odd = min(it.numel, (long)((-(uintptr_t)it.src & 15) / size));
    const long off = odd + (long)(c - it.first) * list.chunk;
    const long left = max(it.numel - off, 0L);               // (0: the leading elements made one chunk fewer)
    f(it, off, (int)(left < list.chunk ? left : list.chunk), c == it.first ? (int)odd : 0);
  }
}

// tid, threads: who walks a chunk together, the workgroup or a wave; the result is the workgroup's
__device__ __forceinline__ double grad_norm_share(const GradList& list, int first, int stride, int tid, int threads, bool inf_norm,
                                                  double* red) {
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  grad_chunks<false>(list, first, stride, [&](const GradItem& it, long off, int n, int lead) {
    if (it.dtype == FLM_F32) grad_norm_chunk((const float*)it.src + off, n, lead, tid, threads, inf_norm, acc);
    else if (it.dtype == FLM_BF16) grad_norm_chunk((const __bf16*)it.src + off, n, lead, tid, threads, inf_norm, acc);
    else grad_norm_chunk((const _Float16*)it.src + off, n, lead, tid, threads, inf_norm, acc);
  });
  const double v = inf_norm ? larger(larger(acc[0], acc[1]), larger(acc[2], acc[3])) : (acc[0] + acc[1]) + (acc[2] + acc[3]);
  return grad_fold(v, inf_norm, red);
}

template <bool PAST>
__device__ __forceinline__ void grad_scale_share(const GradList& list, int first, int stride, int tid, int threads, double coef) {
  grad_chunks<true>(list, first, stride, [&](const GradItem& it, long off, int n, int lead) {
    if (!it.dst || (it.dst == it.src && coef == 1.0)) return;
    if (it.dtype == FLM_F32) grad_scale_chunk<float, PAST>((const float*)it.src + off, (float*)it.dst + off, n, lead, tid, threads, coef);
    else if (it.dtype == FLM_BF16) grad_scale_chunk<__bf16, PAST>((const __bf16*)it.src + off, (__bf16*)it.dst + off, n, lead, tid, threads, coef);
    else grad_scale_chunk<_Float16, PAST>((const _Float16*)it.src + off, (_Float16*)it.dst + off, n, lead, tid, threads, coef);
  });
}

// a NaN norm gives a NaN factor (NaN gradients), an infinite one the factor 0, as the formula does
__device__ __forceinline__ double grad_factor(double norm, double max_norm) {
  const double c = max_norm / (norm + 1e-6);
  return c >= 1.0 ? 1.0 : c;
}

__global__ __launch_bounds__(256) void grad_norm_kernel(GradList list, GradOuter outer, int inf_norm, double* __restrict__ part) {
  __shared__ double red[16];
  const bool inf = inf_norm != 0;
  double v = grad_norm_share(list, blockIdx.x, gridDim.x, threadIdx.x, 256, inf, red);
  if (outer.r && blockIdx.x == gridDim.x - 1) {          // the implicit part: a product of two short sums
    double sr = 0.0, sg = 0.0;
    auto add = [&](double s, double g) { return inf ? larger(s, __builtin_fabs(g)) : __builtin_fma(g, g, s); };
    for (int i = threadIdx.x; i < 512; i += 256) { sg = add(sg, outer.g0[i]); sg = add(sg, outer.g1[i]); }
    if (threadIdx.x < 64) sr = add(sr, outer.r[threadIdx.x]);
    sr = grad_fold(sr, inf, red);
    sg = grad_fold(sg, inf, red);
    v = inf ? larger(v, sr * sg) : v + outer.times * sr * sg;
  }
  if (threadIdx.x == 0) part[blockIdx.x] = v;
}

// PAST: the results are written past the caches
template <bool PAST>
__global__ __launch_bounds__(256) void grad_clip_kernel(GradList list, int inf_norm, const double* __restrict__ part, int n_part,
                                                        double max_norm, float* __restrict__ norm_out) {
  __shared__ double red[16];
  const bool inf = inf_norm != 0;
  double v = 0.0;
  for (int i = threadIdx.x; i < n_part; i += 256) v = inf ? larger(v, part[i]) : v + part[i];
  v = grad_fold(v, inf, red);
  const double norm = inf ? v : __builtin_sqrt(v);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  if (list.chunks) grad_scale_share<PAST>(list, blockIdx.x, gridDim.x, threadIdx.x, 256, grad_factor(norm, max_norm));
}

// Short lists: one workgroup sums, then scales what it has just read; its waves take the chunks in turn, each with its own
// loads under way.
__global__ __launch_bounds__(1024) void grad_clip_small_kernel(GradList list, int inf_norm, double max_norm,
                                                               float* __restrict__ norm_out) {
  __shared__ double red[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const double v = grad_norm_share(list, w, 16, lane, 64, inf_norm != 0, red);
  const double norm = inf_norm ? v : __builtin_sqrt(v);
  if (threadIdx.x == 0) *norm_out = (float)norm;
  grad_scale_share<false>(list, w, 16, lane, 64, grad_factor(norm, max_norm));
}

// tensors [lo, lo + count) of the caller's arrays as one launch's list
static bool grad_list(GradList& list, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype,
                      int lo, int count, int chunk) {
  long chunks = 0;
  list.count = 0;
  list.chunk = chunk;
  for (int i = lo; i < lo + count; i++) {
    if (numel[i] < 0 || (numel[i] > 0 && !src[i]) || dtype[i] < FLM_F32 || dtype[i] > FLM_F16) return false;
    if (numel[i] == 0) continue;
    const uintptr_t between = dtype[i] == FLM_F32 ? 3 : 1;
    if (((uintptr_t)src[i] | (uintptr_t)(dst ? dst[i] : nullptr)) & between) return false;
    GradItem& it = list.item[list.count++];
    it.src = src[i];
    it.dst = dst ? dst[i] : nullptr;
    it.numel = numel[i];
    it.dtype = dtype[i];
    it.first = (int)chunks;
    chunks += (numel[i] + chunk - 1) / chunk;
    if (chunks >= (1L << 30)) return false;
  }
  list.chunks = (int)chunks;
  return true;
}

// Whether a place would be written twice, written as one tensor's and read as another's, or clipped as two tensors' (into
// places elsewhere): spans in the order of their addresses, each against the ends of those before it.  Tensors that only count
// in the norm may overlap each other.
static int grad_overlap(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int count) {
  enum { COUNTED, CLIPPED, WRITTEN };
  struct Span {
    uintptr_t begin, end;
    int kind;
    bool operator<(const Span& o) const { return begin < o.begin; }
  };
  try {
    std::vector<Span> span;
    span.reserve(2 * (size_t)count);
    for (int i = 0; i < count; i++) {
      if (numel[i] == 0) continue;
      const uintptr_t bytes = (uintptr_t)numel[i] * (dtype[i] == FLM_F32 ? 4 : 2), s = (uintptr_t)src[i], d = (uintptr_t)dst[i];
      span.push_back({s, s + bytes, !d ? COUNTED : (d == s ? WRITTEN : CLIPPED)});
      if (d && d != s) span.push_back({d, d + bytes, WRITTEN});
    }
    if (!std::is_sorted(span.begin(), span.end())) std::sort(span.begin(), span.end());
    uintptr_t end[3] = {0, 0, 0};
    for (const Span& s : span) {
      if (s.begin < end[WRITTEN] || (s.kind != COUNTED && s.begin < end[CLIPPED]) || (s.kind == WRITTEN && s.begin < end[COUNTED]))
        return FLM_E_OVERLAP;
      end[s.kind] = std::max(end[s.kind], s.end);
    }
  } catch (const std::bad_alloc&) {
    return FLM_E_CAPACITY;
  }
  return FLM_OK;
}

// A list that one workgroup handles alone: up to this many chunks of 2048 elements, one a wave.  (Replayed from a graph, one
// launch / two: 64 elements 3.9 / 5.1 us, 10 tensors of 100 6.7 / 7.1, one of 8192 5.3 / 6.1, 10 of 2048 8.4 / 7.0, 10 of 6000
// 17 / 7.3; called, the second launch costs 3 us of the host's time more.)
#define GRAD_SMALL 16

static int grad_clip_run(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int count,
                         const GradOuter& outer, double max_norm, int inf_norm, double* workspace, float* norm_out,
                         hipStream_t stream) {
  GradList list;
  long total = 0;
  for (int lo = 0; lo < count; lo += FLM_GRAD_LIST) {       // every tensor is checked before anything is launched
    if (!grad_list(list, src, dst, numel, dtype, lo, count - lo < FLM_GRAD_LIST ? count - lo : FLM_GRAD_LIST, 8192)) return FLM_E_ARG;
    for (int i = 0; i < list.count; i++) total += list.item[i].numel;
  }
  if (dst) {
    const int rc = grad_overlap(src, dst, numel, dtype, count);
    if (rc) return rc;
  }
  if (count <= FLM_GRAD_LIST && total <= 2048L * GRAD_SMALL && !outer.r &&
      grad_list(list, src, dst, numel, dtype, 0, count, 2048) && list.chunks <= GRAD_SMALL) {
    hipLaunchKernelGGL(grad_clip_small_kernel, dim3(1), dim3(1024), 0, stream, list, inf_norm, max_norm, norm_out);
    FLM_CHECK_LAUNCH();
    return FLM_OK;
  }
  // chunks: short enough to occupy the card, long enough that a workgroup's four 16-byte loads per thread are many
  long chunk = (total / 2048 + 2047) / 2048 * 2048;
  chunk = chunk < 2048 ? 2048 : (chunk > 32768 ? 32768 : chunk);
  // partial results are dealt to the launches in proportion to their chunks, at least one each
  const int launches = (count + FLM_GRAD_LIST - 1) / FLM_GRAD_LIST;
  const long all_chunks = total / chunk + count;
  const int parts_max = GRAD_PARTS - launches;             // (at most 586 launches)
  int n_part = 0;
  for (int lo = 0; lo < count; lo += FLM_GRAD_LIST) {
    grad_list(list, src, dst, numel, dtype, lo, count - lo < FLM_GRAD_LIST ? count - lo : FLM_GRAD_LIST, (int)chunk);
    long blocks = all_chunks <= parts_max ? list.chunks : (long)((double)list.chunks / all_chunks * parts_max);
    if (blocks < 1) blocks = 1;
    GradOuter o = outer;
    if (lo != 0) o.r = nullptr;
    hipLaunchKernelGGL(grad_norm_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, list, o, inf_norm, workspace + n_part);
    FLM_CHECK_LAUNCH();
    n_part += (int)blocks;
  }
  // Results that go elsewhere than to their gradients' places, and are more than the 256 MB cache behind the L2s could keep
  // beside the gradients, are written past it: what the norm pass has read is still there (512 MB of bf16: 386 -> 356 us; 55
  // MB of fp32 stay in the cache either way, 33.5 us, past it 35).
  const bool past = dst && dst[0] != src[0] && total >= (64L << 20);
  for (int i = launches - 1; i >= 0; i--) {
    const int lo = i * FLM_GRAD_LIST;
    grad_list(list, src, dst, numel, dtype, lo, count - lo < FLM_GRAD_LIST ? count - lo : FLM_GRAD_LIST, (int)chunk);
    if (!dst) list.chunks = 0;                              // the norm alone
    const int blocks = list.chunks < 1 ? 1 : (list.chunks < 2048 ? list.chunks : 2048);
    float* const norm = i == launches - 1 ? norm_out : (float*)nullptr;
    if (past) hipLaunchKernelGGL(grad_clip_kernel<true>, dim3(blocks), dim3(256), 0, stream, list, inf_norm, workspace, n_part, max_norm, norm);
    else hipLaunchKernelGGL(grad_clip_kernel<false>, dim3(blocks), dim3(256), 0, stream, list, inf_norm, workspace, n_part, max_norm, norm);
    FLM_CHECK_LAUNCH();
    if (!dst) break;
  }
  return FLM_OK;
}

}  // namespace flm

extern "C" int flm_grad_clip(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int count,
                             double max_norm, int inf_norm, double* workspace, float* norm_out, void* stream) {
  if (!src || !numel || !dtype || count <= 0 || count > FLM_GRAD_MAX_TENSORS || !workspace || !norm_out ||
      !(max_norm >= 0.0) || ((uintptr_t)workspace & 7) || ((uintptr_t)norm_out & 3))
    return FLM_E_ARG;
  return flm::grad_clip_run(src, dst, numel, dtype, count, flm::GradOuter{}, max_norm, inf_norm, workspace, norm_out,
                            (hipStream_t)stream);
}

extern "C" int flm_dqn_grad_clip(float* grads, int Rp, int T1, int NA, int rails4, int packed, const float* rcb,
                                 double max_norm, int inf_norm, double* workspace, float* norm_out, void* stream) {
  if (!grads || Rp <= 0 || T1 <= 0 || rails4 < 0 || rails4 > Rp || (rails4 > 0 && !rcb) || (packed && rails4 <= 0) ||
      !workspace || !norm_out || !(max_norm >= 0.0) || (((uintptr_t)grads | (uintptr_t)rcb | (uintptr_t)norm_out) & 3) ||
      ((uintptr_t)workspace & 7))
    return FLM_E_ARG;
  const long n = flm_dqn_param_count(3 * Rp, T1, NA);
  if (n <= 0) return FLM_E_ARG;
  const long a1_w = 64L * T1 + 64, block = 512L * 64 * 3 * Rp, v1_w = a1_w + block + 512;
  if (!packed) {
    // the used rails lie scattered among rows that were left unwritten: only whole gradients or packed ones are taken
    if (rails4 > 0) return FLM_E_ARG;
    const void* src[1] = {grads};
    void* dst[1] = {grads};
    const int64_t numel[1] = {n};
    const int32_t dtype[1] = {FLM_F32};
    return flm::grad_clip_run(src, dst, numel, dtype, 1, flm::GradOuter{}, max_norm, inf_norm, workspace, norm_out,
                              (hipStream_t)stream);
  }
  const long used = 512L * 64 * 3 * rails4;
  float* piece[3] = {grads, grads + a1_w + block, grads + v1_w + block};
  const int64_t numel[3] = {a1_w + used, 512 + used, n - (v1_w + block)};
  const void* src[3] = {piece[0], piece[1], piece[2]};
  void* dst[3] = {piece[0], piece[1], piece[2]};
  const int32_t dtype[3] = {FLM_F32, FLM_F32, FLM_F32};
  flm::GradOuter outer{};
  if (rails4 < Rp) outer = {rcb, grads + a1_w + block, grads + v1_w + block, 3.0 * (Rp - rails4)};     // (else: no empty rows)
  return flm::grad_clip_run(src, dst, numel, dtype, 3, outer, max_norm, inf_norm, workspace, norm_out, (hipStream_t)stream);
}
