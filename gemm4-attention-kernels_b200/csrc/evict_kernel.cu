// Eviction: of every sequence keep the slots that have received the most attention weight, and copy their keys and
// values, in order, to new pages.
//
// Selection. A sequence of n slots keeps m = min(n, keep): its first keep_first and last keep_recent slots, and of the
// others the m - (those) with the largest weight; of equal weights the lower slot stays. Weights are mapped to 32-bit
// keys whose order as whole numbers is the order of the weights (-0 = +0, NaN above everything), and the smallest kept
// key, the threshold, is found digit by digit from the top (11, 11 and 10 bits): a histogram of the digit among the keys
// that agree with the digits found so far, and a scan from its upper end. No sums of weights are formed, so the result
// is exact. A slot's place is then the number of slots above the threshold before it, plus the number of equal ones
// before it as far as those stay: counts per warp, one scan over warps and CTAs, and a last pass.
//
// A cluster of eight CTAs per sequence, each with its share of the slots; histograms and counts meet through distributed
// shared memory. Up to kOneCta slots a single CTA is faster than the cluster's barriers. The weights are read once and
// their keys kept in shared memory (a sequence of more than eight times kCacheMost slots is read from L2 again). What
// bounds it is the chain of passes and barriers (131072 slots: 18 us; the copy of 20000 of them, 4 heads: 50 us), not
// bytes.
//
// Copy. The kept slots' head rows are laid end to end; a warp takes four of them of one tensor, whose places four of its
// lanes look up side by side, and has all four in flight, 16 bytes per lane. Nothing is read or written that does not
// move. It is bound by HBM: 2 * heads_kv KB read and written per slot (8 sequences of up to 16384 slots cut to 4096: 99 us
// in all, of which the copy's bytes take 82).
#include <cooperative_groups.h>

#include <cstring>

#include "launch.cuh"
#include "paged.cuh"
#include "warp_mma.cuh"

namespace sd {

namespace ev {
constexpr int kCluster = 8;  // sixteen: the same time for one sequence of 131072 slots, 14 % more for 8 of 16384
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kOneCta = 16384;  // 8000 slots: 12 us, 14 us with the cluster; 16000: 17 us both ways; 32000: 27, 23
constexpr int kCacheMost = 49152;  // keys that a CTA keeps in shared memory (192 KB)
constexpr int kCopyWarps = 8;
constexpr int kCopyRows = 4;  // head rows of a warp
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
  float* new_weights; // (batch, new_weights_len), 0 behind the last one
  int new_weights_len;  // >= keep
  int* status;
  int cached;  // keys a CTA has room for in shared memory
};

namespace ev {

__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 + 0 = +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int cache_len(const EvictParams& p, int len) {
  return min(min(max(len, 0), page_capacity(p.from)), p.weights_len);
}

template <int kCtas>
__global__ void __launch_bounds__(kThreads, 1) splitd_evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t cache[];  // keys of this CTA's slots
  namespace cg = cooperative_groups;
  __shared__ unsigned hist[kBins];   // of this CTA
  __shared__ unsigned total[kBins];  // of the cluster
  __shared__ unsigned warp_total[kWarps];
  __shared__ unsigned found[2];
  __shared__ int counts[2];  // this CTA's slots above the threshold and equal to it
  __shared__ int2 warp_counts[kWarps];
  cg::cluster_group cluster = cg::this_cluster();
  pdl_launch_dependents();
  const int b = blockIdx.x / kCtas, rank = kCtas > 1 ? static_cast<int>(cluster.block_rank()) : 0;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gtid = rank * kThreads + tid, step = kCtas * kThreads;
  // One thread of the cluster reads the length: threads that saw different ones would wait for each other for good.
  __shared__ int length[2];
  if (gtid == 0) length[0] = __ldg(p.seqlens + b), length[1] = cache_len(p, length[0]);
  int n = 0, stated = 0;
  if constexpr (kCtas > 1) {
    cluster.sync();
    const int* first = cluster.map_shared_rank(length, 0);
    stated = first[0], n = first[1];
  } else {
    __syncthreads();
    stated = length[0], n = length[1];
  }
  const int m = min(n, p.keep);
  if (gtid == 0 && p.status && stated > n) atomicCAS(p.status, 0, ST_BAD_CACHE_LEN);
  int* kept = p.kept + static_cast<int64_t>(b) * p.keep;
  // the copy writes the first `keep` of them
  for (int i = p.keep + gtid; i < p.new_weights_len; i += step) p.new_weights[static_cast<int64_t>(b) * p.new_weights_len + i] = 0.f;
  if (n <= p.keep) {  // the whole cluster: everything stays
    for (int i = gtid; i < p.keep; i += step) kept[i] = i < n ? i : -1;
    if (gtid == 0) p.new_seqlens[b] = m;
    if constexpr (kCtas > 1) cluster.sync();  // no CTA ends while another may read its memory
    return;
  }
  // slots in [lo, hi) compete for the places that the first and the recent ones leave
  const int lo = p.keep_first, hi = n - p.keep_recent;
  const float* w = p.weights + b * p.weights_stride;
  const int per = ((hi - lo) + kCtas - 1) / kCtas;
  const int c0 = min(lo + rank * per, hi), c1 = min(c0 + per, hi);
  const bool cached = c1 - c0 <= p.cached;
  int want = m - (n - (hi - lo));  // of [lo, hi); at the end: of those equal to the threshold
  uint32_t threshold = 0, mask = 0;
  int above = 0;  // of this CTA, spread over its threads
  constexpr int kShift[3] = {21, 10, 0};
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = kShift[pass];
    const uint32_t digit_mask = pass < 2 ? 2047u : 1023u;
    hist[tid] = 0, hist[tid + kThreads] = 0;
    __syncthreads();
    auto count = [&](uint32_t key) {
      if ((key & mask) == threshold) atomicAdd(hist + ((key >> shift) & digit_mask), 1u);
    };
    if (pass > 0 && cached) {
#pragma unroll 4
      for (int i = tid; i < c1 - c0; i += kThreads) count(cache[i]);
    } else {
#pragma unroll 8
      for (int i = tid; i < c1 - c0; i += kThreads) {
        const uint32_t key = order_key(__ldg(w + c0 + i));
        if (cached) cache[i] = key;
        count(key);
      }
    }
    if constexpr (kCtas > 1) {
      cluster.sync();
      if (tid < kBins / kCtas) {
        const int bin = rank * (kBins / kCtas) + tid;
        unsigned s = 0;
#pragma unroll
        for (int r = 0; r < kCtas; ++r) s += cluster.map_shared_rank(hist, r)[bin];
#pragma unroll
        for (int r = 0; r < kCtas; ++r) cluster.map_shared_rank(total, r)[bin] = s;
      }
      cluster.sync();
    } else {
      __syncthreads();
    }
    // from the top: the digit in which the running count reaches `want`; thread t has the t-th pair of bins from there
    const unsigned* sum = kCtas > 1 ? total : hist;
    const int top = kBins - 1 - 2 * tid;
    const unsigned n0 = sum[top], n1 = sum[top - 1];
    unsigned incl = n0 + n1;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    if (lane == 31) warp_total[warp] = incl;
    if (tid == 0) found[0] = digit_mask, found[1] = 0;  // want == 0: above every key
    __syncthreads();
    unsigned before = lane < warp ? warp_total[lane] : 0u;
    before = __reduce_add_sync(0xffffffffu, before) + incl - (n0 + n1);
    const unsigned goal = static_cast<unsigned>(want);
    if (before < goal && before + n0 >= goal)
      found[0] = top, found[1] = before;
    else if (before + n0 < goal && before + n0 + n1 >= goal)
      found[0] = top - 1, found[1] = before + n0;
    __syncthreads();
    const unsigned digit = found[0];
    want -= static_cast<int>(found[1]);
    threshold |= digit << shift;
    mask |= digit_mask << shift;
    above += (top > static_cast<int>(digit) ? hist[top] : 0u) + (top - 1 > static_cast<int>(digit) ? hist[top - 1] : 0u);
    if (pass == 2 && tid == 0) counts[1] = static_cast<int>(hist[digit]);
    __syncthreads();
  }
  // counts of this CTA, of the CTAs before it, and of the warps before this one; a warp has a run of neighbouring slots
  above = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0) warp_total[warp] = above;
  const int run = ((c1 - c0 + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int w0 = min(warp * run, c1 - c0), w1 = min(w0 + run, c1 - c0);
  int2 mine = make_int2(0, 0);
  auto tally = [&](uint32_t key) { mine.x += key > threshold, mine.y += key == threshold; };
  if (cached) {
#pragma unroll 4
    for (int i = w0 + lane; i < w1; i += 32) tally(cache[i]);
  } else {
#pragma unroll 4
    for (int i = w0 + lane; i < w1; i += 32) tally(order_key(__ldg(w + c0 + i)));
  }
  mine.x = __reduce_add_sync(0xffffffffu, mine.x), mine.y = __reduce_add_sync(0xffffffffu, mine.y);
  if (lane == 0) warp_counts[warp] = mine;
  __syncthreads();
  int2 c = lane < warp ? warp_counts[lane] : make_int2(0, 0);
  if constexpr (kCtas > 1) {
    if (warp == 0) {
      const int s = __reduce_add_sync(0xffffffffu, static_cast<int>(warp_total[lane]));
      if (lane == 0) counts[0] = s;
    }
    cluster.sync();
    if (lane < rank) {
      const int* other = cluster.map_shared_rank(counts, lane);
      c.x += other[0], c.y += other[1];
    }
  }
  int a = __reduce_add_sync(0xffffffffu, c.x), e = __reduce_add_sync(0xffffffffu, c.y);
  if constexpr (kCtas > 1) cluster.barrier_arrive();  // done with the others' memory
  const unsigned below = (1u << lane) - 1;
  auto place = [&](int i, uint32_t key) {
    const bool is_above = i < w1 && key > threshold, is_equal = i < w1 && key == threshold;
    const unsigned am = __ballot_sync(0xffffffffu, is_above), em = __ballot_sync(0xffffffffu, is_equal);
    const int my_e = e + __popc(em & below);
    const int at = lo + a + __popc(am & below) + min(my_e, want);
    if ((is_above || (is_equal && my_e < want)) && at < m) kept[at] = c0 + i;  // `at` is, unless the weights change
    a += __popc(am), e += __popc(em);
  };
  if (cached) {
#pragma unroll 4
    for (int i0 = w0; i0 < w1; i0 += 32) place(i0 + lane, i0 + lane < w1 ? cache[i0 + lane] : 0u);
  } else {
#pragma unroll 4
    for (int i0 = w0; i0 < w1; i0 += 32) place(i0 + lane, i0 + lane < w1 ? order_key(__ldg(w + c0 + i0 + lane)) : 0u);
  }
  // the first and the recent ones; not before the barriers, which would wait for the stores
  for (int i = gtid; i < lo; i += step) kept[i] = i;
  for (int i = hi + gtid; i < n; i += step) kept[m - (n - i)] = i;
  if (gtid == 0) p.new_seqlens[b] = m;
  if constexpr (kCtas > 1) cluster.barrier_wait();  // no CTA ends while another may read its memory
}

__global__ void __launch_bounds__(kCopyWarps * 32) splitd_evict_copy_kernel(const __grid_constant__ EvictParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  const bool is_v = warp & 1;
  const int64_t sp = is_v ? p.v_sp : p.k_sp, ss = is_v ? p.v_ss : p.k_ss, sh = is_v ? p.v_sh : p.k_sh;
  // lanes 0 .. 3: one head row each
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * (kCopyWarps / 2) + (warp >> 1)) * kCopyRows + lane;
  const int place = static_cast<int>(min(row / p.heads_kv, static_cast<int64_t>(p.keep)));
  const int h = static_cast<int>(row % p.heads_kv);
  int64_t from = 0, to = 0;
  bool moves = false;
  pdl_wait();
  if (lane < kCopyRows && place < p.keep) {
    const int64_t at = static_cast<int64_t>(b) * p.keep + place;
    // `kept` has a hole (what its memory held before) if somebody changed the weights during the selection of a sequence
    // whose keys do not fit in shared memory; what is no slot of this cache is not followed.
    int slot = p.kept[at];
    if (slot >= min(page_capacity(p.from), p.weights_len)) slot = -1;
    if (h == 0 && !is_v)
      p.new_weights[static_cast<int64_t>(b) * p.new_weights_len + place] = slot < 0 ? 0.f : __ldg(p.weights + b * p.weights_stride + slot);
    if (slot >= 0) {
      int entry, in_page;
      split_slot(p.from, slot, entry, in_page);
      const int page_from = page_of(p.from, b, entry);
      from = page_from * sp + in_page * ss + h * sh;
      split_slot(p.to, place, entry, in_page);
      const int page_to = page_of(p.to, b, entry);
      to = page_to * sp + in_page * ss + h * sh;
      moves = page_ok(p.from, page_from) && page_ok(p.to, page_to);
      if (!moves && p.status) atomicCAS(p.status, 0, ST_BAD_PAGE);
    }
  }
  const unsigned rows = __ballot_sync(0xffffffffu, moves);
  uint4 x[kCopyRows][2];
#pragma unroll
  for (int u = 0; u < kCopyRows; ++u) {
    const int64_t at = __shfl_sync(0xffffffffu, from, u);
    if (rows >> u & 1) {
      const uint4* s = reinterpret_cast<const uint4*>((is_v ? p.v_src : p.k_src) + at);
      x[u][0] = __ldcs(s + lane), x[u][1] = __ldcs(s + lane + 32);
    }
  }
#pragma unroll
  for (int u = 0; u < kCopyRows; ++u) {
    const int64_t at = __shfl_sync(0xffffffffu, to, u);
    if (rows >> u & 1) {
      uint4* d = reinterpret_cast<uint4*>((is_v ? p.v_dst : p.k_dst) + at);
      __stcs(d + lane, x[u][0]);
      __stcs(d + lane + 32, x[u][1]);
    }
  }
}

}  // namespace ev

namespace {

// once per device and kernel
int allow_cache(void (*kern)(EvictParams), bool one) {
  static std::atomic<int> done[2][64];
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64;
  if (known && done[one][dev].load(std::memory_order_acquire)) return 0;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ev::kCacheMost * 4) != cudaSuccess) {
    cudaGetLastError();
    return fail(SPLITD_ERR_CUDA, "eviction: the kernel's shared memory cannot be set");
  }
  if (known) done[one][dev].store(1, std::memory_order_release);
  return 0;
}

}  // namespace

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
  p.new_weights_len = a->new_weights_len > 0 ? a->new_weights_len : a->keep;
  p.status = a->status_flag;
  int64_t slots = static_cast<int64_t>(a->max_pages) * a->page_size;
  if (a->key_weights_len < slots) slots = a->key_weights_len;
  const bool one = slots <= ev::kOneCta;
  const int64_t share = one ? slots : (slots + ev::kCluster - 1) / ev::kCluster;
  p.cached = static_cast<int>(share < ev::kCacheMost ? share : ev::kCacheMost);
  if (int e = allow_cache(one ? ev::splitd_evict_select_kernel<1> : ev::splitd_evict_select_kernel<ev::kCluster>, one)) return e;
  constexpr int kBlockRows = ev::kCopyRows * ev::kCopyWarps / 2;
  const int64_t copy_blocks = (static_cast<int64_t>(a->keep) * a->heads_kv + kBlockRows - 1) / kBlockRows;
  if (copy_blocks > 0x7fffffff) return fail(SPLITD_ERR_INVALID_ARGUMENT, "eviction: keep * heads_kv is too large");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(one ? a->batch : a->batch * ev::kCluster);
  cfg.blockDim = dim3(ev::kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.cached) * 4;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ev::kCluster, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = one ? 0 : 1;
  cudaError_t ce = one ? cudaLaunchKernelEx(&cfg, ev::splitd_evict_select_kernel<1>, p)
                       : cudaLaunchKernelEx(&cfg, ev::splitd_evict_select_kernel<ev::kCluster>, p);
  if (ce == cudaSuccess)
    ce = launch_dependent(ev::splitd_evict_copy_kernel,
                          dim3(static_cast<unsigned>(copy_blocks), a->batch),
                          dim3(ev::kCopyWarps * 32), 0, stream, p);
  if (ce != cudaSuccess) {
    cudaGetLastError();
    return fail(SPLITD_ERR_CUDA, "eviction: launch failed: %s", cudaGetErrorString(ce));
  }
  return 0;
}

}  // namespace sd
