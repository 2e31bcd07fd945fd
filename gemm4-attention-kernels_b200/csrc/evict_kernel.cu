// Eviction: of every sequence keep the slots that have received the most attention weight, and copy their keys and
// values, in order, to new pages.
//
// Selection. A sequence of n slots keeps m = min(n, keep): its first keep_first and last keep_recent slots, and of the
// others the m - (those) with the largest weight; of equal weights the lower slot stays. Weights are mapped to 32-bit
// keys whose order as whole numbers is the order of the weights (-0 = +0, NaN above everything), and the smallest kept
// key is found digit by digit from the top (8 bits a pass): a histogram of the digit among the keys that agree with the
// digits found so far, and a scan from its upper end. No sums of weights are formed, so the result is exact.
//
// One cluster of eight CTAs per sequence, each with an eighth of its slots; histograms and counts meet through
// distributed shared memory. A last pass over the slots gives every kept one its place by a running count.
//
// Copy. One warp per kept slot and tensor, 16 bytes per lane, four head rows in flight; nothing is read or written
// that does not move. It is bound by HBM: 2 * heads_kv KB read and written per slot.
#include <cooperative_groups.h>

#include <cstring>

#include "launch.cuh"
#include "paged.cuh"
#include "warp_mma.cuh"

namespace sd {

namespace ev {
constexpr int kCluster = 8;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kCopyWarps = 8;
constexpr int kCopyUnroll = 4;
}  // namespace ev

struct EvictParams {
  const uint16_t *k_src, *v_src;
  uint16_t *k_dst, *v_dst;
  int64_t k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;
  int heads_kv, batch;
  PageMap from, to;
  const int* seqlens;
  const float* weights;
  int64_t weights_stride;
  int weights_len;
  int keep, keep_first, keep_recent;
  int* new_seqlens;   // (batch)
  int* kept;          // (batch, keep), -1 behind the last one
  float* new_weights; // (batch, keep), 0 behind the last one
  int* status;
};

namespace ev {

__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 + 0 = +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int cache_len(const EvictParams& p, int b) {
  return min(min(max(__ldg(p.seqlens + b), 0), page_capacity(p.from)), p.weights_len);
}

__device__ __forceinline__ int block_sum(int v, int* scratch, int warp, int lane) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) s += scratch[i];
  return s;
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) splitd_evict_select_kernel(const __grid_constant__ EvictParams p) {
  namespace cg = cooperative_groups;
  __shared__ unsigned hist[256];
  __shared__ unsigned total[256];
  __shared__ int scratch[kWarps];
  __shared__ int counts[2];  // kept for certain, equal to the threshold: of this CTA's slots
  __shared__ unsigned found[2];
  cg::cluster_group cluster = cg::this_cluster();
  pdl_launch_dependents();
  const int b = blockIdx.x / kCluster, rank = cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = cache_len(p, b);
  if (rank == 0 && tid == 0 && p.status && __ldg(p.seqlens + b) > n) atomicCAS(p.status, 0, ST_BAD_CACHE_LEN);
  const int m = min(n, p.keep);
  const float* w = p.weights + b * p.weights_stride;
  // slots in [lo, hi) compete for the places that the first and the recent ones leave
  const int lo = min(p.keep_first, n), hi = max(lo, n - p.keep_recent);
  const int per = ((hi - lo) + kCluster - 1) / kCluster;
  const int c0 = min(lo + rank * per, hi), c1 = min(c0 + per, hi);
  int want = m - (n - (hi - lo));  // of [lo, hi)
  uint32_t threshold = 0;
  if (n <= p.keep) {
    want = hi - lo;  // everything stays (threshold 0: no key is below it)
  } else {
    uint32_t mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
      __syncthreads();
      for (int i0 = c0; i0 < c1; i0 += kThreads) {
        const int i = i0 + tid;
        const uint32_t key = i < c1 ? order_key(__ldg(w + i)) : 0u;
        const bool in = i < c1 && (key & mask) == threshold;
        const unsigned active = __ballot_sync(0xffffffffu, in);
        if (in) {
          const uint32_t digit = (key >> shift) & 255u;
          const unsigned same = __match_any_sync(active, digit);
          if (lane == __ffs(same) - 1) atomicAdd(hist + digit, __popc(same));
        }
      }
      cluster.sync();
      if (tid < 256) {
        unsigned s = 0;
#pragma unroll
        for (int r = 0; r < kCluster; ++r) s += cluster.map_shared_rank(hist, r)[tid];
        total[tid] = s;
      }
      cluster.sync();  // every CTA has read the histograms
      // from the top: the digit in which the running count reaches `want`
      if (warp == 0) {
        unsigned mine[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += mine[e] = total[255 - (lane * 8 + e)];
        unsigned incl = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const unsigned o = __shfl_up_sync(0xffffffffu, incl, d);
          if (lane >= d) incl += o;
        }
        unsigned above = incl - sum;
        if (above < static_cast<unsigned>(want) && incl >= static_cast<unsigned>(want)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (above < static_cast<unsigned>(want) && above + mine[e] >= static_cast<unsigned>(want))
              found[0] = 255 - (lane * 8 + e), found[1] = above;
            above += mine[e];
          }
        }
        if (want == 0 && lane == 0) found[0] = 255, found[1] = 0;
      }
      __syncthreads();
      threshold |= found[0] << shift;
      mask |= 255u << shift;
      want -= static_cast<int>(found[1]);
      __syncthreads();
    }
  }
  // `want` slots of weight `threshold` stay, and every slot above it
  const bool all = n <= p.keep;
  int above = 0, equal = 0;
  for (int i = c0 + tid; i < c1; i += kThreads) {
    const uint32_t key = order_key(__ldg(w + i));
    above += all || key > threshold, equal += !all && key == threshold;
  }
  above = block_sum(above, scratch, warp, lane);
  equal = block_sum(equal, scratch, warp, lane);
  if (tid == 0) counts[0] = above, counts[1] = equal;
  cluster.sync();
  int place = lo, eq = 0;  // place of this CTA's first kept slot; slots equal to the threshold before this CTA's
  for (int r = 0; r < rank; ++r) {
    const int* c = cluster.map_shared_rank(counts, r);
    place += c[0] + min(max(want - eq, 0), c[1]), eq += c[1];
  }
  cluster.sync();  // nobody reads the counts of a CTA that has ended
  int* kept = p.kept + static_cast<int64_t>(b) * p.keep;
  float* nw = p.new_weights + static_cast<int64_t>(b) * p.keep;
  for (int i0 = c0; i0 < c1; i0 += kThreads) {
    const int i = i0 + tid;
    const float v = i < c1 ? __ldg(w + i) : 0.f;
    const uint32_t key = order_key(v);
    const bool is_above = i < c1 && (all || key > threshold), is_equal = i < c1 && !all && key == threshold;
    const unsigned em = __ballot_sync(0xffffffffu, is_equal), below = (1u << lane) - 1;
    // counts of the warps before this one: equal ones first, since they decide which of them stay
    __syncthreads();
    if (lane == 0) scratch[warp] = __popc(em);
    __syncthreads();
    int eq_before = eq, eq_all = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      if (k < warp) eq_before += scratch[k];
      eq_all += scratch[k];
    }
    const bool stays = is_above || (is_equal && eq_before + __popc(em & below) < want);
    const unsigned sm = __ballot_sync(0xffffffffu, stays);
    __syncthreads();
    if (lane == 0) scratch[warp] = __popc(sm);
    __syncthreads();
    int at = place, st_all = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      if (k < warp) at += scratch[k];
      st_all += scratch[k];
    }
    if (stays) {
      at += __popc(sm & below);
      kept[at] = i, nw[at] = v;
    }
    place += st_all, eq += eq_all;
  }
  // the first and the recent ones, and the empty places behind them
  const int gtid = rank * kThreads + tid, step = kCluster * kThreads;
  for (int i = gtid; i < lo; i += step) kept[i] = i, nw[i] = __ldg(w + i);
  for (int i = hi + gtid; i < n; i += step) kept[m - (n - i)] = i, nw[m - (n - i)] = __ldg(w + i);
  for (int i = m + gtid; i < p.keep; i += step) kept[i] = -1, nw[i] = 0.f;
  if (gtid == 0) p.new_seqlens[b] = m;
}

__global__ void __launch_bounds__(kCopyWarps * 32) splitd_evict_copy_kernel(const __grid_constant__ EvictParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  const int place = blockIdx.x * (kCopyWarps / 2) + (warp >> 1);
  pdl_wait();
  if (place >= p.keep) return;
  const int slot = p.kept[static_cast<int64_t>(b) * p.keep + place];
  if (slot < 0) return;
  int entry, row_from, row_to;
  split_slot(p.from, slot, entry, row_from);
  const int page_from = page_of(p.from, b, entry);
  split_slot(p.to, place, entry, row_to);
  const int page_to = page_of(p.to, b, entry);
  if (!page_ok(p.from, page_from) || !page_ok(p.to, page_to)) {
    if (lane == 0 && p.status) atomicCAS(p.status, 0, ST_BAD_PAGE);
    return;
  }
  const bool is_v = warp & 1;
  const int64_t sp = is_v ? p.v_sp : p.k_sp, ss = is_v ? p.v_ss : p.k_ss, sh = is_v ? p.v_sh : p.k_sh;
  const uint16_t* src = (is_v ? p.v_src : p.k_src) + page_from * sp + row_from * ss;
  uint16_t* dst = (is_v ? p.v_dst : p.k_dst) + page_to * sp + row_to * ss;
  for (int h = 0; h < p.heads_kv; h += kCopyUnroll) {
    uint4 x[kCopyUnroll][2];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (h + u < p.heads_kv) {
        const uint4* s = reinterpret_cast<const uint4*>(src + (h + u) * sh);
        x[u][0] = __ldcs(s + lane), x[u][1] = __ldcs(s + lane + 32);
      }
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (h + u < p.heads_kv) {
        uint4* d = reinterpret_cast<uint4*>(dst + (h + u) * sh);
        __stcs(d + lane, x[u][0]);
        __stcs(d + lane + 32, x[u][1]);
      }
  }
}

}  // namespace ev

int launch_evict(const splitd_evict_params* a, cudaStream_t stream) {
  EvictParams p;
  memset(&p, 0, sizeof(p));
  p.k_src = static_cast<const uint16_t*>(a->k_pages), p.v_src = static_cast<const uint16_t*>(a->v_pages);
  p.k_dst = static_cast<uint16_t*>(a->k_pages), p.v_dst = static_cast<uint16_t*>(a->v_pages);
  p.k_sp = a->k_strides[0], p.k_ss = a->k_strides[1], p.k_sh = a->k_strides[2];
  p.v_sp = a->v_strides[0], p.v_ss = a->v_strides[1], p.v_sh = a->v_strides[2];
  p.heads_kv = a->heads_kv, p.batch = a->batch;
  const int shift = page_shift(a->page_size);
  p.from = {a->page_table, a->page_table_stride, a->max_pages, a->page_size, a->num_pages, shift};
  p.to = {a->new_page_table, a->new_page_table_stride, a->new_max_pages, a->page_size, a->num_pages, shift};
  p.seqlens = a->seqlens_k;
  p.weights = a->key_weights, p.weights_stride = a->key_weights_stride, p.weights_len = a->key_weights_len;
  p.keep = a->keep, p.keep_first = a->keep_first, p.keep_recent = a->keep_recent;
  p.new_seqlens = a->new_seqlens, p.kept = a->kept, p.new_weights = a->new_weights;
  p.status = a->status_flag;
  ev::splitd_evict_select_kernel<<<dim3(a->batch * ev::kCluster), ev::kThreads, 0, stream>>>(p);
  cudaError_t ce = cudaGetLastError();
  if (ce == cudaSuccess)
    ce = launch_dependent(ev::splitd_evict_copy_kernel,
                          dim3((a->keep + ev::kCopyWarps / 2 - 1) / (ev::kCopyWarps / 2), a->batch),
                          dim3(ev::kCopyWarps * 32), 0, stream, p);
  if (ce != cudaSuccess) {
    cudaGetLastError();
    return fail(SPLITD_ERR_CUDA, "eviction: launch failed: %s", cudaGetErrorString(ce));
  }
  return 0;
}

}  // namespace sd
