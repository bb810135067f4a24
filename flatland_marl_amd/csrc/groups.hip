// Rows sorted by the group (here: the low-rank adapter) each of them uses: a stable counting sort on the device, and the
// table of row tiles the adapter kernels run over.  Ids outside 0..E-1 mean "no group" and sort behind all others.
//
// A wave owns a run of consecutive rows.  It counts them per group, the counts are turned into first positions (groups
// slowest, runs within a group in row order), and the wave then walks its rows again, 64 at a time: a lane's place is the
// group's next position plus the number of lower lanes with the same group, which log2(E) ballots give.  Nothing depends
// on the order in which waves run.
// Up to GROUP_SMALL rows one workgroup does all of it in LDS (317 rows, 20 groups: 4.7 us, the latency of a launch and of two
// loads); beyond that the three steps are three launches (262144 rows, 1024 groups: 3 + 6 + 14 us; the last one's scan of the
// groups by every workgroup and its two scattered stores a row).
#include "flm_adapters.h"

namespace flm {

#define GROUP_SMALL 8192
#define GROUP_RUN 512                    // rows of a wave (at least) in the large form
#define GROUP_KEYS 8                     // rows a lane holds at a time: their ids are fetched together
#define GROUP_RUNS_MAX 4096
#define GROUP_WAVES 4                    // runs of a workgroup when rows are placed

// lanes of the wave that hold the same key (all 64 lanes take part; bits: bits of a key)
__device__ __forceinline__ unsigned long long same_key(int key, int bits) {
  unsigned long long m = ~0ull;
  for (int b = 0; b < bits; b++) {
    const bool one = (key >> b) & 1;
    const unsigned long long v = __ballot(one);
    m &= one ? v : ~v;
  }
  return m;
}

// exclusive prefix over the workgroup of one int per thread; total to all.  scratch: 17 ints
__device__ __forceinline__ int block_scan(int v, int* scratch, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(inc, o);
    if (lane >= o) inc += t;
  }
  __syncthreads();
  if (lane == 63) scratch[w] = inc;
  __syncthreads();
  int base = 0, tot = 0;
  for (int i = 0; i < nw; i++) {
    const int c = scratch[i];
    if (i < w) base += c;
    tot += c;
  }
  *total = tot;
  return base + inc - v;
}

// The keys of rows lo + 64*u + lane (E for rows from hi on), lo < hi.  All ids are on their way before the first is looked at.
__device__ __forceinline__ void load_keys(const void* ids, int ids64, long lo, long hi, int E, int (&key)[GROUP_KEYS]) {
  const int lane = threadIdx.x & 63;
  if (ids64) {
    int64_t v[GROUP_KEYS];
#pragma unroll
    for (int u = 0; u < GROUP_KEYS; u++) v[u] = reinterpret_cast<const int64_t*>(ids)[min(lo + 64 * u + lane, hi - 1)];
#pragma unroll
    for (int u = 0; u < GROUP_KEYS; u++) key[u] = lo + 64 * u + lane < hi && v[u] >= 0 && v[u] < E ? (int)v[u] : E;
  } else {
    int v[GROUP_KEYS];
#pragma unroll
    for (int u = 0; u < GROUP_KEYS; u++) v[u] = reinterpret_cast<const int32_t*>(ids)[min(lo + 64 * u + lane, hi - 1)];
#pragma unroll
    for (int u = 0; u < GROUP_KEYS; u++) key[u] = lo + 64 * u + lane < hi && (unsigned)v[u] < (unsigned)E ? v[u] : E;
  }
}

// f(i, src[i]) for i = first, first + stride, .. < n, eight loads in flight
template <typename F>
__device__ __forceinline__ void each_of(const int* src, int n, int first, int stride, F&& f) {
  for (int i0 = first; i0 < n; i0 += 8 * stride) {
    int v[8];
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = src[min(i0 + u * stride, n - 1)];
#pragma unroll
    for (int u = 0; u < 8; u++)
      if (i0 + u * stride < n) f(i0 + u * stride, v[u]);
  }
}

__device__ __forceinline__ void count_keys(const int (&key)[GROUP_KEYS], long lo, long hi, int* cnt) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < GROUP_KEYS; u++)
    if (lo + 64 * u + lane < hi) atomicAdd(&cnt[key[u]], 1);
}

// places the rows of these keys; next [E+1]: the wave's next position per group
__device__ __forceinline__ void place_keys(const int (&key)[GROUP_KEYS], long lo, long hi, int bits, int* next, int* order,
                                           int* keys) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < GROUP_KEYS; u++) {
    if (lo + 64 * u >= hi) break;
    const long i = lo + 64 * u + lane;
    const bool in = i < hi;
    const unsigned long long same = same_key(key[u], bits) & __ballot(in);
    const int rank = __popcll(same & lanemask_lt());
    int pos = 0;
    if (in) pos = next[key[u]] + rank;
    // (all lanes have read before one lane a group writes, and that write is there before the next 64 rows read)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) next[key[u]] = pos + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in) {
      order[pos] = (int)i;
      keys[pos] = key[u];
    }
  }
}

// Writes tiles [first, cap) in steps of stride.  off [E+1] and tstart [E+1] (number of tiles before a group) in LDS.
__device__ __forceinline__ void write_tiles(const int* off, const int* tstart, int E, int cap, int first, int stride, int2* tiles) {
  for (int t = first; t < cap; t += stride) {
    int2 out = make_int2(0, 0);
    if (t < tstart[E]) {
      int lo = 0, hi = E - 1;                    // the last group whose first tile is at or before t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tstart[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      const int pos = off[lo] + (t - tstart[lo]) * FLM_ROW_TILE;
      out = make_int2(pos, lo | (min(FLM_ROW_TILE, off[lo + 1] - pos) << 16));
    }
    tiles[t] = out;
  }
}

// off [E+1] (counts in, first positions out; off[E] = rows with a group), tstart [E+1] out.  All threads; E + 1 <= 2048.
__device__ __forceinline__ void scan_groups(int* off, int* tstart, int E, int* scratch) {
  const int per = (E + 1 + blockDim.x - 1) / blockDim.x;          // consecutive groups per thread
  const int g0 = threadIdx.x * per;
  int rows = 0, tl = 0;
  for (int j = 0; j < per; j++)
    if (g0 + j < E) {
      rows += off[g0 + j];
      tl += (off[g0 + j] + FLM_ROW_TILE - 1) / FLM_ROW_TILE;
    }
  int total_rows, total_tiles;
  int r = block_scan(rows, scratch, &total_rows);
  int t = block_scan(tl, scratch, &total_tiles);
  __syncthreads();
  for (int j = 0; j < per; j++)
    if (g0 + j < E) {
      const int c = off[g0 + j];
      off[g0 + j] = r;
      tstart[g0 + j] = t;
      r += c;
      t += (c + FLM_ROW_TILE - 1) / FLM_ROW_TILE;
    }
  if (threadIdx.x == 0) {
    off[E] = total_rows;
    tstart[E] = total_tiles;
  }
  __syncthreads();
}

// LDS: cnt [waves][E+1], off [E+1], tstart [E+1], scratch [17]
__global__ __launch_bounds__(1024) void group_small_kernel(const void* ids, int ids64, int n, int E, int bits, int* order, int* keys,
                                                           int* offsets, int* first_tile, int2* tiles, int cap) {
  extern __shared__ int lds[];
  const int nw = blockDim.x >> 6, w = threadIdx.x >> 6, E1 = E + 1;
  int* cnt = lds;
  int* off = cnt + nw * E1;
  int* tstart = off + E1;
  int* scratch = tstart + E1;
  // (a wave's run is at most 64 * GROUP_KEYS rows: GROUP_SMALL rows over 16 waves)
  const int run = ((n + nw - 1) / nw + 63) & ~63;
  const int lo = min(n, w * run), hi = min(n, lo + run);
  int key[GROUP_KEYS];
  if (lo < hi) load_keys(ids, ids64, lo, hi, E, key);
  for (int i = threadIdx.x; i < nw * E1; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  count_keys(key, lo, hi, cnt + w * E1);
  __syncthreads();
  // per group: counts of the waves -> rows before each wave; the group's total to off
  for (int g = threadIdx.x; g < E1; g += blockDim.x) {
    int s = 0;
    for (int k = 0; k < nw; k++) {
      const int c = cnt[k * E1 + g];
      cnt[k * E1 + g] = s;
      s += c;
    }
    off[g] = s;
  }
  __syncthreads();
  scan_groups(off, tstart, E, scratch);
  for (int g = threadIdx.x; g < E1; g += blockDim.x) {
    const int o = off[g];
    for (int k = 0; k < nw; k++) cnt[k * E1 + g] += o;
    offsets[g] = o;
    first_tile[g] = tstart[g];
  }
  __syncthreads();
  place_keys(key, lo, hi, bits, cnt + w * E1, order, keys);
  write_tiles(off, tstart, E, cap, threadIdx.x, blockDim.x, tiles);
}

// counts[run][E+1]; one wave per run
__global__ __launch_bounds__(64) void group_count_kernel(const void* ids, int ids64, int n, int run, int E, int* counts) {
  extern __shared__ int lds[];
  const int E1 = E + 1;
  for (int i = threadIdx.x; i < E1; i += 64) lds[i] = 0;
  __syncthreads();
  const long lo = (long)blockIdx.x * run, hi = min((long)n, lo + run);
  for (long at = lo; at < hi; at += 64 * GROUP_KEYS) {
    int key[GROUP_KEYS];
    load_keys(ids, ids64, at, hi, E, key);
    count_keys(key, at, hi, lds);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < E1; i += 64) counts[(long)blockIdx.x * E1 + i] = lds[i];
}

// Per group the rows before each run, in place, and the group's total.  64 groups a workgroup, one per lane; the 16 waves
// take a sixteenth of the runs each.
__global__ __launch_bounds__(1024) void group_scan_kernel(int* counts, int runs, int E, int* totals) {
  __shared__ int part[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, E1 = E + 1, g = blockIdx.x * 64 + lane;
  const int per = (runs + 15) / 16, lo = min(runs, w * per), hi = min(runs, lo + per);
  const int gg = min(g, E1 - 1);
  // up to 32 runs a thread stay in registers between the two passes (512 runs: 262144 rows); longer shares are read twice
  constexpr int KEEP = 32;
  int c[KEEP];
  int s = 0;
  for (int k0 = lo; k0 < hi; k0 += KEEP) {
#pragma unroll
    for (int u = 0; u < KEEP; u++) c[u] = counts[(long)min(k0 + u, hi - 1) * E1 + gg];
#pragma unroll
    for (int u = 0; u < KEEP; u++) s += k0 + u < hi ? c[u] : 0;
  }
  part[w][lane] = s;
  __syncthreads();
  int base = 0, total = 0;
#pragma unroll
  for (int k = 0; k < 16; k++) {
    if (k < w) base += part[k][lane];
    total += part[k][lane];
  }
  if (g >= E1) return;
  for (int k0 = lo; k0 < hi; k0 += KEEP) {
    if (per > KEEP) {
#pragma unroll
      for (int u = 0; u < KEEP; u++) c[u] = counts[(long)min(k0 + u, hi - 1) * E1 + g];
    }
#pragma unroll
    for (int u = 0; u < KEEP; u++)
      if (k0 + u < hi) {
        counts[(long)(k0 + u) * E1 + g] = base;
        base += c[u];
      }
  }
  if (w == 0) totals[g] = total;
}

// GROUP_WAVES runs a workgroup.  LDS: next [GROUP_WAVES][E+1], off [E+1], tstart [E+1], scratch [17]
__global__ __launch_bounds__(64 * GROUP_WAVES) void group_place_kernel(const void* ids, int ids64, int n, int run, int runs, int E, int bits,
                                                          const int* counts, const int* totals, int* order, int* keys,
                                                          int* offsets, int* first_tile, int2* tiles, int cap) {
  extern __shared__ int lds[];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, E1 = E + 1;
  int* next = lds;
  int* off = next + GROUP_WAVES * E1;
  int* tstart = off + E1;
  int* scratch = tstart + E1;
  const int r = blockIdx.x * GROUP_WAVES + w;
  int key[GROUP_KEYS];                     // (fetched ahead of the scan)
  if (r < runs) load_keys(ids, ids64, (long)r * run, min((long)n, (long)(r + 1) * run), E, key);
  constexpr int NT = 64 * GROUP_WAVES;
  each_of(totals, E1, threadIdx.x, NT, [&](int g, int v) { off[g] = v; });
  if (r < runs) each_of(counts + (long)r * E1, E1, lane, 64, [&](int g, int v) { next[w * E1 + g] = v; });
  __syncthreads();
  scan_groups(off, tstart, E, scratch);
  if (r < runs)
    for (int g = lane; g < E1; g += 64) next[w * E1 + g] += off[g];
  if (blockIdx.x == 0)
    for (int g = threadIdx.x; g < E1; g += NT) {
      offsets[g] = off[g];
      first_tile[g] = tstart[g];
    }
  __syncthreads();
  if (r < runs) {
    const long lo = (long)r * run, hi = min((long)n, lo + run);
    for (long at = lo; at < hi; at += 64 * GROUP_KEYS) {
      if (at > lo) load_keys(ids, ids64, at, hi, E, key);
      place_keys(key, at, hi, bits, next + w * E1, order, keys);
    }
  }
  write_tiles(off, tstart, E, cap, blockIdx.x * NT + threadIdx.x, gridDim.x * NT, tiles);
}

}  // namespace flm

using namespace flm;

static int group_run_rows(int n) {
  long run = GROUP_RUN;
  while ((n + run - 1) / run > GROUP_RUNS_MAX) run *= 2;
  return (int)run;
}

extern "C" long flm_group_rows_ints(int n, int n_groups) {
  return n > 0 && n_groups > 0 ? row_groups_ints(n, n_groups) : 0;
}

extern "C" long flm_group_rows_workspace(int n, int n_groups) {
  if (n <= GROUP_SMALL || n_groups <= 0) return 0;
  const int run = group_run_rows(n);
  return ((long)(n + run - 1) / run + 1) * (n_groups + 1);
}

extern "C" int flm_group_rows(const void* ids, int ids64, int n, int n_groups, int32_t* groups, int32_t* workspace, void* stream) {
  if (!ids || !groups || n <= 0 || n > (1 << 30) || n_groups <= 0 || n_groups > FLM_GROUPS_MAX) return FLM_E_ARG;
  if (((uintptr_t)groups & 15) || ((uintptr_t)ids & (ids64 ? 7 : 3)) || ((uintptr_t)workspace & 3)) return FLM_E_ARG;
  const int E = n_groups, E1 = E + 1;
  const RowGroups g = row_groups(groups, n, E);
  int* order = const_cast<int*>(g.order);
  int* keys = const_cast<int*>(g.key);
  int* offsets = const_cast<int*>(g.offsets);
  int* first_tile = const_cast<int*>(g.first_tile);
  int2* tiles = const_cast<int2*>(g.tiles);
  int bits = 0;
  while ((1 << bits) <= E) bits++;
  hipStream_t st = (hipStream_t)stream;
  if (n <= GROUP_SMALL) {
    int waves = (n + 63) / 64;
    waves = waves < 4 ? 4 : (waves > 16 ? 16 : waves);
    const size_t lds = sizeof(int) * ((size_t)(waves + 2) * E1 + 17);
    if (lds > 64 * 1024) FLM_RAISE_LDS_ONCE(group_small_kernel);
    hipLaunchKernelGGL(group_small_kernel, dim3(1), dim3(64 * waves), lds, st, ids, ids64, n, E, bits, order, keys, offsets,
                       first_tile, tiles, g.cap);
    FLM_CHECK_LAUNCH();
    return FLM_OK;
  }
  if (!workspace) return FLM_E_ARG;
  const int run = group_run_rows(n), runs = (n + run - 1) / run;
  int* totals = workspace + (long)runs * E1;
  hipLaunchKernelGGL(group_count_kernel, dim3(runs), dim3(64), sizeof(int) * E1, st, ids, ids64, n, run, E, workspace);
  FLM_CHECK_LAUNCH();
  hipLaunchKernelGGL(group_scan_kernel, dim3((E1 + 63) / 64), dim3(1024), 0, st, workspace, runs, E, totals);
  FLM_CHECK_LAUNCH();
  const size_t lds = sizeof(int) * ((size_t)(GROUP_WAVES + 2) * E1 + 17);
  if (lds > 64 * 1024) FLM_RAISE_LDS_ONCE(group_place_kernel);
  hipLaunchKernelGGL(group_place_kernel, dim3((runs + GROUP_WAVES - 1) / GROUP_WAVES), dim3(64 * GROUP_WAVES), lds, st, ids, ids64, n,
                     run, runs, E, bits, workspace, totals, order, keys, offsets, first_tile, tiles, g.cap);
  FLM_CHECK_LAUNCH();
  return FLM_OK;
}
