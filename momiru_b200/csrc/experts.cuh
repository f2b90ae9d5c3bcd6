// experts.cuh -- tokens sorted by expert and back.
//
// An assignment i = t * top_k + j sends token t to expert ids[t, j]; one whose
// id is outside [0, experts) is dropped. Expert e's segment of the sorted rows
// starts at offsets[e], a multiple of row_align, and holds its counts[e]
// assignments in increasing i, so the order (and every later sum) is fixed.
//   slots[i]   the assignment's row, or -1
//   sources[r] the row's assignment, or -1 for a row that holds no token
//
// The sort is a stable counting sort: every CTA takes a run of tokens, learns
// how many assignments of each expert come before its run and in all, ranks
// its own, and copies its rows where they go, a token's row read once for its
// top_k destinations. Up to ES_DIRECT assignments each CTA counts the ids
// itself (one launch); above, a first kernel leaves one histogram per CTA.
//
// Bound: memory, the rows in and out.
#pragma once
#include <cstring>

#include "linear_epi.cuh"
#include "ptx.cuh"

namespace mmr {

constexpr int ES_THREADS = 256;
constexpr int ES_WARPS = ES_THREADS / 32;
constexpr int ES_MAX_EXPERTS = 1024;
constexpr int ES_DIRECT = 4096;

// Loads and stores of V elements (VB bytes): the widest vector that the row
// pitches, the base addresses and the row length all allow.
template <int VB>
struct VecOf;
template <>
struct VecOf<16> { using type = uint4; };
template <>
struct VecOf<8> { using type = uint2; };
template <>
struct VecOf<4> { using type = unsigned int; };
template <>
struct VecOf<2> { using type = unsigned short; };

struct RowMat {
  void* p = nullptr;
  long long ld = 0;  // bytes from row to row
};

struct DispatchParams {
  const int* ids = nullptr;
  long long ids_t = 0, ids_j = 0;
  int tokens = 0, top_k = 0, experts = 0, align = 1;
  long long rows = 0;
  int run = 0;  // tokens of one CTA
  int *slots = nullptr, *sources = nullptr, *offsets = nullptr, *counts = nullptr;
  int* hist = nullptr;  // [CTAs][experts], or null: count directly
  RowMat x, out;
  int row_vecs = 0;  // vectors of a row
};

__device__ __forceinline__ int es_id(const DispatchParams& p, int i) {
  const int t = i / p.top_k, j = i - t * p.top_k;
  const int id = p.ids[t * p.ids_t + j * p.ids_j];
  return id >= 0 && id < p.experts ? id : -1;
}

// First token of CTA b's run.
__device__ __forceinline__ int run_start(const DispatchParams& p, long long b) {
  return static_cast<int>(min(b * p.run, static_cast<long long>(p.tokens)));
}

// One histogram of expert ids per CTA's run.
static __global__ void __launch_bounds__(ES_THREADS) mmr_expert_hist_kernel(const DispatchParams p) {
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e < p.experts; e += ES_THREADS) hist[e] = 0;
  griddep_wait();
  griddep_release();
  __syncthreads();
  const int i0 = run_start(p, blockIdx.x) * p.top_k, i1 = run_start(p, blockIdx.x + 1ll) * p.top_k;
  for (int i = i0 + static_cast<int>(threadIdx.x); i < i1; i += ES_THREADS) {
    const int id = es_id(p, i);
    if (id >= 0) atomicAdd(&hist[id], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += ES_THREADS)
    p.hist[static_cast<long long>(blockIdx.x) * p.experts + e] = hist[e];
}

// Shared memory: total[E], before[E] (then the run's next row per expert),
// start[E + 1], and per-warp counts [ES_WARPS][E].
constexpr int dispatch_smem_bytes(int experts) { return 4 * (3 * experts + 1 + ES_WARPS * experts); }

template <int VB>
__global__ void __launch_bounds__(ES_THREADS) mmr_dispatch_kernel(const DispatchParams p) {
  using Vec = typename VecOf<VB>::type;
  extern __shared__ int sh[];
  const int E = p.experts;
  int* total = sh;
  int* before = total + E;
  int* start = before + E;
  int* wcount = start + E + 1;
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  for (int e = tid; e < 2 * E; e += ES_THREADS) sh[e] = 0;
  for (int e = tid; e < ES_WARPS * E; e += ES_THREADS) wcount[e] = 0;
  griddep_wait();
  griddep_release();
  __syncthreads();
  const int n = p.tokens * p.top_k;
  const int t0 = run_start(p, blockIdx.x), t1 = run_start(p, blockIdx.x + 1ll);
  const int i0 = t0 * p.top_k, i1 = t1 * p.top_k;
  if (p.hist) {
    // columns of the histograms, the CTAs' rows dealt to `groups` of threads
    const int groups = max(1, ES_THREADS / E);
    for (int idx = tid; idx < E * groups; idx += ES_THREADS) {
      const int e = idx % E, g = idx / E, nb = static_cast<int>(gridDim.x);
      const int b0 = static_cast<int>(static_cast<long long>(nb) * g / groups);
      const int b1 = static_cast<int>(static_cast<long long>(nb) * (g + 1) / groups);
      int all = 0, pre = 0;
#pragma unroll 8
      for (int b = b0; b < b1; ++b) {
        const int c = __ldcg(p.hist + static_cast<long long>(b) * E + e);
        all += c;
        pre += b < static_cast<int>(blockIdx.x) ? c : 0;
      }
      atomicAdd(&total[e], all);
      atomicAdd(&before[e], pre);
    }
  } else {
    for (int i = tid; i < n; i += ES_THREADS) {
      const int id = es_id(p, i);
      if (id < 0) continue;
      atomicAdd(&total[id], 1);
      if (i < i0) atomicAdd(&before[id], 1);
    }
  }
  // the run's own assignments, by warp: warp w takes a contiguous part
  const int per = (i1 - i0 + ES_WARPS - 1) / ES_WARPS;
  const int w0 = min(i0 + warp * per, i1), w1 = min(w0 + per, i1);
  for (int i = w0 + lane; i < w1; i += 32) {
    const int id = es_id(p, i);
    if (id >= 0) atomicAdd(&wcount[warp * E + id], 1);
  }
  __syncthreads();
  if (warp == 0) {
    int base = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      const int c = e < E ? total[e] : 0;
      const int padded = (c + p.align - 1) / p.align * p.align;
      int incl = padded;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      if (e < E) start[e] = base + incl - padded;
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) start[E] = base;
  }
  __syncthreads();
  // each warp's first row per expert
  for (int e = tid; e < E; e += ES_THREADS) {
    int at = start[e] + before[e];
#pragma unroll
    for (int w = 0; w < ES_WARPS; ++w) {
      const int c = wcount[w * E + e];
      wcount[w * E + e] = at;
      at += c;
    }
  }
  if (blockIdx.x == 0) {
    for (int e = tid; e < E; e += ES_THREADS) {
      p.offsets[e] = start[e];
      p.counts[e] = total[e];
    }
    if (tid == 0) p.offsets[E] = start[E];
  }
  __syncthreads();
  // stable ranks, 32 assignments at a time in order
  for (int ib = w0; ib < w1; ib += 32) {
    const int i = ib + lane;
    const int id = i < w1 ? es_id(p, i) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int slot = -1;
    if (id >= 0) slot = wcount[warp * E + id] + rank;
    __syncwarp();
    if (id >= 0 && rank == 0) wcount[warp * E + id] += __popc(same);
    __syncwarp();
    if (i < w1) {
      p.slots[i] = slot;
      if (slot >= 0) p.sources[slot] = i;
    }
  }
  __syncthreads();  // the run's slots (written above by this CTA) are read back below

  // Rows that hold no token, every warp-count-th row a warp's, so that the long
  // run of them after the last segment is spread over all warps; 32 at a time,
  // finding a row's segment by bisection.
  const long long warps = static_cast<long long>(gridDim.x) * ES_WARPS;
  Vec zero;
  memset(&zero, 0, sizeof zero);
  for (long long rb = static_cast<long long>(blockIdx.x) * ES_WARPS + warp; rb < p.rows; rb += 32 * warps) {
    const long long r = rb + lane * warps;
    bool none = false;
    if (r < p.rows) {
      int lo = 0, hi = E;  // the last segment that starts at or before r
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= r) lo = mid;
        else hi = mid - 1;
      }
      none = lo == E || r - start[lo] >= total[lo];
      if (none) p.sources[r] = -1;
    }
    for (unsigned left = __ballot_sync(0xffffffffu, none); left; left &= left - 1) {
      Vec* dst = reinterpret_cast<Vec*>(static_cast<char*>(p.out.p) + (rb + (__ffs(left) - 1) * warps) * p.out.ld);
      for (int c = lane; c < p.row_vecs; c += 32) dst[c] = zero;
    }
  }
  // The rows of this run's tokens, in pieces of 32 vectors: four pieces' loads in
  // flight in a warp where there are enough of them.
  const int pieces = (p.row_vecs + 31) / 32;
  const bool many = (t1 - t0) * pieces >= 4 * ES_WARPS;
  const int group = many ? 4 : 1, groups = (pieces + group - 1) / group;
  for (int u = warp; u < (t1 - t0) * groups; u += ES_WARPS) {
    const int t = t0 + u / groups, c = (u % groups) * group * 32 + lane;
    const Vec* src = reinterpret_cast<const Vec*>(static_cast<const char*>(p.x.p) + t * p.x.ld);
    Vec v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < group && c + 32 * q < p.row_vecs) v[q] = __ldcg(src + c + 32 * q);
    for (int j0 = 0; j0 < p.top_k; j0 += 4) {
      int slot[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) slot[j] = j0 + j < p.top_k ? p.slots[t * p.top_k + j0 + j] : -1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (slot[j] < 0) continue;
        Vec* dst = reinterpret_cast<Vec*>(static_cast<char*>(p.out.p) + slot[j] * p.out.ld);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q < group && c + 32 * q < p.row_vecs) dst[c + 32 * q] = v[q];
      }
    }
  }
}

// -------------------------------------------------------------- combine --
struct CombineParams {
  const int* slots = nullptr;
  int tokens = 0, top_k = 0;
  int n_rows = 0;  // a slot outside [0, n_rows) counts as dropped
  const float* weights = nullptr;  // null: all one
  long long w_t = 0, w_j = 0;
  RowMat rows, residual, out;  // residual.p may be null
  int row_vecs = 0;
};

template <typename T, int VB>
__device__ __forceinline__ void vec_to_f32(const typename VecOf<VB>::type& w, float (&v)[VB / sizeof(T)]) {
  T t[VB / sizeof(T)];
  memcpy(t, &w, VB);
#pragma unroll
  for (int i = 0; i < int(VB / sizeof(T)); ++i) v[i] = to_f32<T>(t[i]);
}
template <typename T, int VB>
__device__ __forceinline__ typename VecOf<VB>::type vec_from_f32(const float (&v)[VB / sizeof(T)]) {
  T t[VB / sizeof(T)];
#pragma unroll
  for (int i = 0; i < int(VB / sizeof(T)); ++i) t[i] = from_f32<T>(v[i]);
  typename VecOf<VB>::type w;
  memcpy(&w, t, VB);
  return w;
}

// out[t] = sum_j weights[t, j] rows[slots[t, j]] (+ residual[t]): f32 sums in
// increasing j, one rounding. A thread takes one vector of a token's row, so a
// warp reads 512 contiguous bytes of every row it adds; the reads of kChoices
// choices are in flight together.
template <typename T, int VB, int kChoices>
__global__ void __launch_bounds__(128) mmr_combine_kernel(const CombineParams p) {
  using Vec = typename VecOf<VB>::type;
  constexpr int V = VB / sizeof(T);
  griddep_wait();
  griddep_release();
  const int lane = static_cast<int>(threadIdx.x) & 31;
  const int pieces = (p.row_vecs + 127) / 128;
  const long long units = static_cast<long long>(p.tokens) * pieces;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int t = static_cast<int>(u / pieces), c = static_cast<int>(u % pieces) * 128 + static_cast<int>(threadIdx.x);
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    // a lane per choice reads its slot and weight; the rows' addresses then
    // depend on nothing else
    for (int jb = 0; jb < p.top_k; jb += 32) {
      const int many = min(p.top_k - jb, 32);
      int my_slot = -1;
      float my_scale = 1.0f;
      if (lane < many) {
        my_slot = p.slots[static_cast<long long>(t) * p.top_k + jb + lane];
        if (my_slot >= p.n_rows) my_slot = -1;
        if (p.weights && my_slot >= 0) my_scale = *(p.weights + t * p.w_t + (jb + lane) * p.w_j);
      }
      for (int j0 = 0; j0 < many; j0 += kChoices) {
        Vec w[kChoices];
        float scale[kChoices];
        int slot[kChoices];
#pragma unroll
        for (int q = 0; q < kChoices; ++q) {
          slot[q] = __shfl_sync(0xffffffffu, my_slot, (j0 + q) & 31);
          scale[q] = __shfl_sync(0xffffffffu, my_scale, (j0 + q) & 31);
          if (j0 + q >= many || c >= p.row_vecs) slot[q] = -1;
          if (slot[q] >= 0)
            w[q] = __ldcg(reinterpret_cast<const Vec*>(static_cast<const char*>(p.rows.p) + slot[q] * p.rows.ld) + c);
        }
#pragma unroll
        for (int q = 0; q < kChoices; ++q) {
          if (slot[q] < 0) continue;
          float v[V];
          vec_to_f32<T, VB>(w[q], v);
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = fmaf(scale[q], v[i], acc[i]);
        }
      }
    }
    if (c >= p.row_vecs) continue;
    if (p.residual.p) {
      float v[V];
      vec_to_f32<T, VB>(reinterpret_cast<const Vec*>(static_cast<const char*>(p.residual.p) + t * p.residual.ld)[c], v);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += v[i];
    }
    reinterpret_cast<Vec*>(static_cast<char*>(p.out.p) + t * p.out.ld)[c] = vec_from_f32<T, VB>(acc);
  }
}

// --------------------------------------------------------- combine grad --
struct CombineGradParams {
  const int *slots = nullptr, *sources = nullptr;
  int tokens = 0, top_k = 0;
  long long n_rows = 0;
  const float* weights = nullptr;
  long long w_t = 0, w_j = 0;
  RowMat d_out, rows, d_rows;  // d_rows.p may be null
  float* d_weights = nullptr;  // may be null
  long long dw_t = 0, dw_j = 0;
  int row_vecs = 0;
  int zero_blocks = 0;  // trailing blocks that zero the rows without a token
};

// d_rows[slot] = w d_out[t] and d_w = <d_out[t], rows[slot]> in one pass, four
// choices at a time. W warps take a token: one where the tokens alone fill the
// GPU (no block-wide joins), else the block's eight. The dot products are
// joined in a fixed order.
template <typename T, int VB, int W>
__global__ void __launch_bounds__(256) mmr_combine_grad_kernel(const CombineGradParams p) {
  using Vec = typename VecOf<VB>::type;
  constexpr int V = VB / sizeof(T);
  constexpr int U = VB == 16 ? 1 : 2;  // vectors of a row that a thread has in flight
  __shared__ float part[8][4];
  griddep_wait();
  griddep_release();
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int token_blocks = (p.tokens * W + 7) / 8;
  if (static_cast<int>(blockIdx.x) >= token_blocks) {
    Vec zero;
    memset(&zero, 0, sizeof zero);
    // rows strided over the warps: those without a token come in runs
    const long long warps = p.zero_blocks * 8ll;
    for (long long rb = (static_cast<int>(blockIdx.x) - token_blocks) * 8 + warp; rb < p.n_rows; rb += 32 * warps) {
      const bool none = rb + lane * warps < p.n_rows && p.sources[rb + lane * warps] < 0;
      for (unsigned left = __ballot_sync(0xffffffffu, none); left; left &= left - 1) {
        Vec* dst = reinterpret_cast<Vec*>(static_cast<char*>(p.d_rows.p) + (rb + (__ffs(left) - 1) * warps) * p.d_rows.ld);
        for (int c = lane; c < p.row_vecs; c += 32) dst[c] = zero;
      }
    }
    return;
  }
  const int t = W == 8 ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x) * 8 + warp;
  const int me = W == 8 ? tid : lane;
  if (t >= p.tokens) return;  // whole warps, and only where warps are on their own
  const Vec* d_out = reinterpret_cast<const Vec*>(static_cast<const char*>(p.d_out.p) + t * p.d_out.ld);
  for (int j0 = 0; j0 < p.top_k; j0 += 4) {
    int slot[4];
    float scale[4], dot[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      slot[q] = j0 + q < p.top_k ? p.slots[static_cast<long long>(t) * p.top_k + j0 + q] : -1;
      if (slot[q] >= p.n_rows) slot[q] = -1;
      scale[q] = slot[q] >= 0 ? (p.weights ? p.weights[t * p.w_t + (j0 + q) * p.w_j] : 1.0f) : 0.0f;
      dot[q] = 0.0f;
    }
    for (int c0 = me; c0 < p.row_vecs; c0 += 32 * W * U) {
      Vec dv[U], w[U][4];
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int c = c0 + x * 32 * W;
        if (c >= p.row_vecs) continue;
        dv[x] = __ldcg(d_out + c);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (slot[q] >= 0 && p.d_weights)
            w[x][q] = __ldcg(reinterpret_cast<const Vec*>(static_cast<const char*>(p.rows.p) + slot[q] * p.rows.ld) + c);
      }
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int c = c0 + x * 32 * W;
        if (c >= p.row_vecs) continue;
        float d[V];
        vec_to_f32<T, VB>(dv[x], d);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (slot[q] < 0) continue;
          float v[V];
          if (p.d_weights) {
            vec_to_f32<T, VB>(w[x][q], v);
#pragma unroll
            for (int i = 0; i < V; ++i) dot[q] = fmaf(d[i], v[i], dot[q]);
          }
          if (p.d_rows.p) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = scale[q] * d[i];
            reinterpret_cast<Vec*>(static_cast<char*>(p.d_rows.p) + slot[q] * p.d_rows.ld)[c] = vec_from_f32<T, VB>(v);
          }
        }
      }
    }
    if (!p.d_weights) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
      for (int d = 16; d; d >>= 1) dot[q] += __shfl_xor_sync(0xffffffffu, dot[q], d);
    }
    if (W == 1) {
      float s = dot[0];
#pragma unroll
      for (int q = 1; q < 4; ++q) s = lane == q ? dot[q] : s;
      if (lane < 4 && j0 + lane < p.top_k) p.d_weights[t * p.dw_t + (j0 + lane) * p.dw_j] = s;
    } else {
      if (lane == 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) part[warp][q] = dot[q];
      }
      __syncthreads();
      if (tid < 4 && j0 + tid < p.top_k) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += part[w][tid];
        p.d_weights[t * p.dw_t + (j0 + tid) * p.dw_j] = s;
      }
      __syncthreads();
    }
  }
}

}  // namespace mmr
