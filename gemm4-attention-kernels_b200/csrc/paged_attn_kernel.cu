// Attention of a few query tokens per sequence over a paged cache (head_dim 512): o = softmax(q K^T scale) V, lse, and
// optionally the attention weight that every cached key received.
//
// Mathematics. For one KV head, R = seqlen_q * (heads_q / heads_kv) query rows share its keys. With x = q.k scale
// log2(e) (after the soft cap and the mask) a row keeps m = max x, l = sum 2^(x - m), O = sum 2^(x - m) v over the keys
// seen so far; two such triples of disjoint key sets join to one by scaling both to the larger m. o = O / l and
// lse = (m + log2 l) ln 2; a row that sees no key has l = 0: o = 0, lse = -inf.
//
// What bounds it. Every visible key costs 2 KB of cache and 4 * 512 * R flops: at R = 8, 8 flops a byte, far left of the
// ridge. So the kernel is built around the stream of cache rows: one CTA per SM, four producer warps that keep two rings
// of 32-row stages (keys, values) full with one 1 KB bulk copy per row (a page of any size and a row of any page are then
// the same thing: no tile has to match a page). One producer warp alone can issue such a copy every 74 cycles, 59 % of
// the bandwidth. Measured (replays of a graph): 1 x 131072 keys, 4 KV heads, 8 rows each: 158 us, 6.8 TB/s; 32 sequences of
// up to 8192: 209 us, 6.7 TB/s (a plain copy moves 6.6). With 32 rows (4 tokens) a tile's instructions cost as much as its
// bytes: 107 us where the stream alone takes 94 and the bytes 81.
//
// Split. The (sequence, KV head, row block) units are laid end to end, in tiles of 32 keys, and every CTA takes an
// equal share of the whole line, whatever the lengths are; the lengths never leave the device. A unit that lies inside
// one CTA is finished there. Each CTA has at most two unfinished ones (its first and its last), whose (m, l, O) go to
// the workspace in fp32, and a second kernel adds them up in CTA order: no atomics, the same bits every time.
//
// Products. keys x rows on the warp matrix instruction (16 keys x 8 rows x 16): the cache row is the A operand, so a
// group of 8 query heads fills the 8 columns exactly. S^T = K Q^T is split over four quarters of the head dimension; the
// partial sums meet in shared memory, where score warp w then owns the softmax of every fourth (eighth) row, one key per
// lane. O^T = V^T P^T is split over the head dimension, 64 columns per value warp, accumulators in registers. Score and
// value warps only meet through two buffers of P, so that products and softmax of neighbouring tiles overlap (one set of
// eight warps for both, with one barrier a tile: 119 us with 32 rows, 103 us this way; up to 24 rows the same).
//
// Roundings. The matrix instruction multiplies V, which is exact, by P in V's 16-bit type. P is kept as the sum of TWO such
// numbers (two products): a single one would put an error of the size of the output's own rounding on top of it. Two
// leave a weight off by 2^-16 of itself in bf16 and by 2^-22 in fp16, a 256th and a 2048th of the output's rounding; three
// would cost a third product for an error that the scores' own sums in 32 bits have as well. The weights are at most 1, and
// fp16 ends at 2^-24, so there P is 2^16 times the weight, taken out again where l divides: what a weight loses is then at
// most 2^-41 of the row's largest one (without the factor, 131071 keys at 2^-26 of one whose value is 0 came out as 0).
#include <cstring>

#include "launch.cuh"
#include "paged.cuh"
#include "warp_mma.cuh"

namespace sd {

namespace pa {
constexpr int kTile = 32;                      // keys per tile = rows per ring stage
constexpr int kPitch = kRowBytes + 16;         // ldmatrix reads 8 rows at once: 16 bytes of padding spread them over the banks
constexpr int kStageBytes = kTile * kPitch;
constexpr int kProducers = 4;                  // producer warps: each asks for a quarter of a tile's rows
constexpr int kRowsPerProducer = kTile / kProducers;
constexpr int kValueWarps = 8;                 // 64 columns of the head dimension each
// Score warps have a quarter of the head dimension each; from 25 rows on half of the rows, too (32 rows: 103 us, 115 us
// with four score warps; they read the keys from shared memory twice then, which 24 rows would not repay).
template <int kNB>
constexpr int kRowGroups = kNB == 4 ? 2 : 1;
template <int kNB>
constexpr int kScoreWarps = 4 * kRowGroups<kNB>;
template <int kNB>
constexpr int kThreads = 32 * (kValueWarps + kScoreWarps<kNB> + kProducers);
constexpr int kPartPitch = 36;                 // floats per row of the partial scores (32 keys + padding)
constexpr int kPPitch = 20;                    // 32-bit words per row of P (32 keys x 2 bytes + padding)
constexpr int kMaxRows = 32;                   // rows of a row block

// From 17 rows on some warps need more registers than a block's threads can have each (512: 128, 640: 96), and the others
// give up some of theirs. The launch checks that the block comes with at least as many as the shares together. With 32 rows
// the compiler still keeps 96 bytes of a thread in local memory (200 bytes loaded): it allots 96 registers to all roles.
// Splits of 40 / 112 / 104 and 48 / 112 / 104 were no faster.
template <int kNB>
constexpr bool kSplitRegs = kNB >= 3;
template <int kNB>
constexpr int kProducerRegs = kNB == 4 ? 40 : 48;
template <int kNB>
constexpr int kScoreRegs = kNB == 4 ? 104 : 168;
template <int kNB>
constexpr int kValueRegs = kNB == 4 ? 112 : 120;
template <int kNB>
constexpr int kSplitTotal =
    32 * (kProducers * kProducerRegs<kNB> + kScoreWarps<kNB> * kScoreRegs<kNB> + kValueWarps * kValueRegs<kNB>);
static_assert(kSplitTotal<3> <= 65536 / kThreads<3> / 8 * 8 * kThreads<3> && kSplitTotal<4> <= 65536 / kThreads<4> / 8 * 8 * kThreads<4>,
              "registers of a block");

struct Desc {  // what the producer tells the others about a stretch of tiles
  int b, head, row0, n_tiles;  // n_tiles == 0: no more work
  int len, first_key;          // keys [first_key, len), tile by tile
  int slot;                    // -1: the whole unit is here; 0 / 1: partial result of this CTA to keep
  int pad;
};

template <int kNB>
struct Layout {
  static constexpr int kRows = 8 * kNB;
  // two of each of these: one tile's are read while the next one's are written
  static constexpr int kPartFloats = 4 * kRows * kPartPitch;
  static constexpr int kPWords = kRows * kPPitch;  // of each half of P
  // Of keys (and query rows), and of values: enough to cover the latency of HBM, and no more, since a deeper queue of
  // requests costs HBM efficiency (1 x 131072 keys: 172 us with six stages in all, 168 with five, 159 with four, 160 with
  // three; 32 sequences up to 8192: 222, 215, 208, 210).
  static constexpr int kKStages = 2, kVStages = 2;
  static constexpr int kStages = kKStages + kVStages;
  static constexpr int kOffPart = kStages * kStageBytes;
  static constexpr int kOffP = kOffPart + 2 * kPartFloats * 4;
  static constexpr int kOffCorr = kOffP + 2 * 2 * kPWords * 4;
  static constexpr int kCorr = kRows + 4;  // factors of the rows, then whether some rows do not see some of the tile's keys
  static constexpr int kOffStat = kOffCorr + 2 * kCorr * 4;
  static constexpr int kOffBounds = kOffStat + kRows * 8;
  static constexpr int kOffDesc = kOffBounds + kRows * 8;
  static constexpr int kOffBar = kOffDesc + kStages * static_cast<int>(sizeof(Desc));
  static constexpr int kBars = 2 * kStages + 6;
  static constexpr int kOffAbort = kOffBar + kBars * 8;
  static constexpr int kBytes = kOffAbort + 16;
  static_assert(kOffDesc % 16 == 0 && kOffBar % 8 == 0 && kOffPart % 16 == 0, "alignment");
  static_assert(kBytes <= 232448, "shared memory of an SM");
};
}  // namespace pa

struct PagedAttnParams {
  const uint16_t *q, *k, *v;
  uint16_t* o;
  float* lse;
  PageMap map;
  const int* seqlens;
  int64_t q_sb, q_ss, q_sh, o_sb, o_ss, o_sh;  // elements
  int64_t k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;  // page, row of the page, head
  int batch, sq, heads_q, heads_kv, group;
  int rows;        // sq * group: query rows of a KV head
  int row_blocks, rows_per_block;
  int win_left, win_right;  // -1: unbounded
  float scale, softcap;
  int max_ctas;
  // workspace
  float* part_o;   // [CTA][2][rows_per_block][512], kPScale times O
  float2* part_ml; // [CTA][2][rows_per_block]
  float* lse2;     // [batch][heads_kv * rows] in log2 units, of the rows that one CTA finished; only with key_weights
  float* scores;   // [batch][heads_kv * rows][weights_len], only with key_weights
  float* weights;
  int64_t weights_stride;
  int weights_len;
  int* status;
};

// First visible key of a sequence (over all its rows) and its length; tiles start at the first visible key.
__device__ __forceinline__ int seq_len(const PagedAttnParams& p, int b) {
  return min(max(__ldg(p.seqlens + b), 0), page_capacity(p.map));
}
__device__ __forceinline__ int first_key(const PagedAttnParams& p, int len) {
  if (p.win_left < 0) return 0;
  const long long lo = static_cast<long long>(len) - p.sq - p.win_left;
  return lo > 0 ? static_cast<int>(lo) : 0;
}
__device__ __forceinline__ int seq_tiles(const PagedAttnParams& p, int len) {
  return (len - first_key(p, len) + pa::kTile - 1) / pa::kTile;
}

// The line of tiles: `total` over all sequences, cut into `ctas` shares; share c is [c total / ctas, (c+1) total / ctas).
// A 64-bit division costs hundreds of cycles; most sizes fit 32 bits.
__device__ __forceinline__ long long divide(long long a, long long b) {  // a >= 0, b > 0
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}
struct Line {
  long long total;
  int ctas;
  __device__ __forceinline__ long long begin(int c) const { return total * c / ctas; }
  __device__ __forceinline__ int owner(long long t) const {  // largest c with begin(c) <= t
    return static_cast<int>(divide((t + 1) * ctas - 1, total));
  }
};
__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}
// One warp: tiles of the sequences below `end` (all of a sequence's units).
__device__ __forceinline__ long long tiles_before(const PagedAttnParams& p, int end, int lane) {
  long long s = 0;
  for (int b = lane; b < end; b += 32) s += seq_tiles(p, seq_len(p, b));
  return warp_sum(s) * (p.heads_kv * p.row_blocks);
}
__device__ __forceinline__ Line make_line(const PagedAttnParams& p, long long total) {
  Line ln;
  ln.total = total;
  ln.ctas = total < p.max_ctas ? static_cast<int>(total) : p.max_ctas;  // no more than tiles
  return ln;
}

namespace pa {

// What P is multiplied by, a power of two: 2^16 is the largest whose product with a weight of 1 two fp16 numbers hold
// (65504 + 32).
template <bool kFp16>
constexpr float kPScale = kFp16 ? 65536.f : 1.f;
template <bool kFp16>
constexpr float kPUnscale = 1.f / kPScale<kFp16>;

// p >= 0 as a sum of two 16-bit numbers. The upper one is the largest that is LESS than p, so that both are positive
// where p is: a visible infinity of V times p stays an infinity (inf * 0 and inf - inf would be NaN). In fp16 that ends
// at p = 2^-24, a weight of 2^-40 of the largest.
template <bool kFp16>
__device__ __forceinline__ void split16(float p, uint16_t& hi, uint16_t& lo) {
  const float below = p > 0.f ? __uint_as_float(__float_as_uint(p) - 1) : p;
  if constexpr (kFp16) {
    const __half h = __float2half_rz(below);
    hi = __half_as_ushort(h), lo = __half_as_ushort(__float2half_rn(p - __half2float(h)));
  } else {
    const __nv_bfloat16 h = __float2bfloat16_rz(below);
    hi = __bfloat16_as_ushort(h), lo = __bfloat16_as_ushort(__float2bfloat16_rn(p - __bfloat162float(h)));
  }
}

// Which keys the rows of a stretch of tiles see.
struct Seen {
  long long lo, hi;      // query token i: keys [i + lo, i + hi) of the sequence's [0, len)
  int free_lo, free_hi;  // all rows of the block: keys [free_lo, free_hi)
  int n_rows;
  __device__ __forceinline__ Seen(const PagedAttnParams& p, const Desc& d) {
    lo = p.win_left < 0 ? -(1ll << 40) : static_cast<long long>(d.len) - p.sq - p.win_left;
    hi = p.win_right < 0 ? 1ll << 40 : static_cast<long long>(d.len) - p.sq + p.win_right + 1;
    n_rows = min(p.rows_per_block, p.rows - d.row0);
    free_lo = first((d.row0 + n_rows - 1) / p.group);
    free_hi = end(d.row0 / p.group, d.len);
  }
  __device__ __forceinline__ int first(int i) const { return static_cast<int>(max(0ll, i + lo)); }
  __device__ __forceinline__ int end(int i, int len) const {
    return static_cast<int>(max(0ll, min(static_cast<long long>(len), i + hi)));
  }
  // whether every row of the block sees every key of the tile
  __device__ __forceinline__ bool all_of(int key0) const { return key0 >= free_lo && key0 + kTile <= free_hi; }
};

// whether one of two 16-bit numbers is an infinity or NaN
template <bool kFp16>
__device__ __forceinline__ bool not_finite2(uint32_t x) {
  constexpr uint32_t kExp = kFp16 ? 0x7c00u : 0x7f80u;
  return (x & kExp) == kExp || (x >> 16 & kExp) == kExp;
}

// largest value of the warp in all lanes; NaN are passed over
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// A ring of kStages slots: 32-row stages (of keys or of values), buffers of P, or the one place for a unit's (m, l).
template <int kStages>
struct Ring {
  uint32_t full, empty;  // barrier arrays
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ Ring(uint32_t bars) : full(bars), empty(bars + 8 * kStages) {}
  __device__ __forceinline__ void next() {
    if (++stage == kStages) stage = 0, phase ^= 1;
  }
  __device__ __forceinline__ bool wait_full(volatile int* abort_flag, int* status, int code) const {
    return mbar_wait(full + 8 * stage, phase, abort_flag, status, code);
  }
  __device__ __forceinline__ bool wait_empty(volatile int* abort_flag, int* status, int code) const {
    return mbar_wait(empty + 8 * stage, phase ^ 1, abort_flag, status, code);
  }
  // one arrival per warp
  __device__ __forceinline__ void arrive_full(int lane) const {
    __syncwarp();
    if (lane == 0) mbar_arrive(full + 8 * stage);
  }
  __device__ __forceinline__ void arrive_empty(int lane) const {
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + 8 * stage);
  }
};
template <int kNB>
struct Rings {
  using L = Layout<kNB>;
  Ring<L::kKStages> k;
  Ring<L::kVStages> v;
  Ring<2> p;
  Ring<1> stat;
  __device__ __forceinline__ explicit Rings(uint32_t bars)
      : k(bars), v(bars + 16 * L::kKStages), p(bars + 16 * L::kStages), stat(bars + 16 * L::kStages + 32) {}
  __device__ __forceinline__ void init() const {
    auto one = [](const auto& r, int n, int full, int empty) {
      for (int i = 0; i < n; ++i) mbar_init(r.full + 8 * i, full), mbar_init(r.empty + 8 * i, empty);
    };
    one(k, L::kKStages, kProducers, kScoreWarps<kNB>);
    one(v, L::kVStages, kProducers, kValueWarps);
    one(p, 2, kScoreWarps<kNB>, kValueWarps);
    one(stat, 1, kScoreWarps<kNB>, kValueWarps);
  }
};

template <int kNB>
__device__ __forceinline__ void producer(const PagedAttnParams& p, uint8_t* smem, Rings<kNB> rings, volatile int* abort_flag, int pw,
                                         int lane) {
  using L = Layout<kNB>;
  const int my_row = pw * kRowsPerProducer + lane % kRowsPerProducer;  // row of a tile; lanes beyond kRowsPerProducer are idle
  const bool active = lane < kRowsPerProducer;
  Desc* descs = reinterpret_cast<Desc*>(smem + L::kOffDesc);
  auto& kr = rings.k;
  auto& vr = rings.v;
  const uint32_t k_ring = smem_u32(smem), v_ring = k_ring + L::kKStages * kStageBytes;
  Desc* const v_descs = descs + L::kKStages;
  int k_used = 0, v_used = 0;  // stages handed out
  bool ok = true;
  auto acquire = [&](const auto& r) {
    if (ok) ok = r.wait_empty(abort_flag, p.status, ST_TIMEOUT_LOAD);
    ok = __all_sync(0xffffffffu, ok);
    return ok;
  };
  // up to 32 sequences: their lengths are read once
  const int len0 = lane < p.batch ? seq_len(p, lane) : 0;
  const Line line = make_line(p, p.batch <= 32 ? warp_sum(seq_tiles(p, len0)) * (p.heads_kv * p.row_blocks) : tiles_before(p, p.batch, lane));
  const int cta = blockIdx.x;
  if (cta < line.ctas) {
    long long t = line.begin(cta);
    const long long t_end = line.begin(cta + 1);
    const int units = p.heads_kv * p.row_blocks;
    // the sequence that holds tile t: whole warps of sequences at a time, then inside one
    long long base = 0;
    int b = 0, len = 0, n_tiles = 0;
    for (int b0 = 0;; b0 += 32) {
      const int my_len = b0 == 0 ? len0 : b0 + lane < p.batch ? seq_len(p, b0 + lane) : 0;
      const int mine = seq_tiles(p, my_len);
      long long incl = static_cast<long long>(mine) * units;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, incl, m);
        if (lane >= m) incl += o;
      }
      const unsigned past = __ballot_sync(0xffffffffu, base + incl > t);
      if (past) {
        const int w = __ffs(past) - 1;
        b = b0 + w;
        len = __shfl_sync(0xffffffffu, my_len, w);
        n_tiles = __shfl_sync(0xffffffffu, mine, w);
        const long long before = __shfl_sync(0xffffffffu, incl, w) - static_cast<long long>(n_tiles) * units;
        base += before;
        break;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
      if (b0 + 32 >= p.batch) {  // the lengths changed under the kernel: nothing to do
        t = t_end;
        break;
      }
    }
    while (t < t_end && ok) {
      const long long off = t - base;
      const int unit = static_cast<int>(off / n_tiles);
      const int tile0 = static_cast<int>(off - static_cast<long long>(unit) * n_tiles);
      const int n = static_cast<int>(min(static_cast<long long>(n_tiles - tile0), t_end - t));
      const int head = unit / p.row_blocks;
      const int row0 = (unit - head * p.row_blocks) * p.rows_per_block;
      const int n_rows = min(p.rows_per_block, p.rows - row0);
      const int lo = first_key(p, len);
      // query rows: one ring stage, with the description of the work in front of it
      if (!acquire(kr)) break;
      Desc d;
      d.b = b, d.head = head, d.row0 = row0, d.n_tiles = n;
      d.len = len, d.first_key = lo + tile0 * kTile;
      d.slot = n == n_tiles ? -1 : (tile0 > 0 ? 0 : 1);
      d.pad = 0;
      {
        const uint32_t bar = kr.full + 8 * kr.stage;
        const uint32_t dst = k_ring + kr.stage * kStageBytes + my_row * kPitch;
        const uint32_t rows = __popc(__ballot_sync(0xffffffffu, active && my_row < n_rows));
        if (lane == 0 && pw == 0) descs[kr.stage] = d;
        if (active && my_row >= n_rows && my_row < L::kRows) {  // rows that pad the block: scores of 0, and no NaN
          for (int c = 0; c < kRowBytes; c += 16) st_shared_v4(dst + c, 0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(bar, rows * kRowBytes);
        __syncwarp();
        if (active && my_row < n_rows) {
          const int i = (row0 + my_row) / p.group, g = (row0 + my_row) - i * p.group;
          bulk_load(dst, p.q + b * p.q_sb + i * p.q_ss + (head * p.group + g) * p.q_sh, kRowBytes, bar);
        }
        kr.next(), ++k_used;
      }
      // keys and values: lane = row of the tile; the page of the next tile is looked up one tile ahead
      auto lookup = [&](int slot, int& page, int& row) {
        page = -1, row = 0;
        if (slot < len) {
          int entry;
          split_slot(p.map, slot, entry, row);
          page = page_of(p.map, b, entry);
        }
      };
      int slot = lo + tile0 * kTile + my_row, page, row;
      lookup(slot, page, row);
      const uint16_t* v_src = nullptr;
      bool v_have = false;
      auto ask = [&](auto& r, uint32_t ring, int& used, const uint16_t* src, bool have) {
        const uint32_t bar = r.full + 8 * r.stage;
        const uint32_t dst = ring + r.stage * kStageBytes + my_row * kPitch;
        if (active && !have) {  // a row that is not there counts as zeros: 0 * (what lay there) could be NaN
          for (int c = 0; c < kRowBytes; c += 16) st_shared_v4(dst + c, 0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, have)) * kRowBytes;
        __syncwarp();  // all lanes' zeros before the arrival that hands the stage over (a ballot orders no memory)
        if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
        __syncwarp();
        if (have) bulk_load(dst, src, kRowBytes, bar);
        r.next(), ++used;
      };
      // K(0), K(1), V(0), K(2), V(1), ..., K(n - 1), V(n - 2), V(n - 1)
      for (int i = 0; i <= n && ok; ++i) {
        int next_page = -1, next_row = 0;
        if (i + 1 < n) lookup(slot + kTile, next_page, next_row);
        const bool inside = active && i < n && slot < len;
        const bool have = inside && page_ok(p.map, page);
        if (inside && !have && p.status) atomicCAS(p.status, 0, ST_BAD_PAGE);
        if (i < n && acquire(kr)) ask(kr, k_ring, k_used, p.k + page * p.k_sp + row * p.k_ss + head * p.k_sh, have);
        if (i > 0 && acquire(vr)) {
          if (i == 1 && lane == 0 && pw == 0) v_descs[vr.stage] = d;
          ask(vr, v_ring, v_used, v_src, v_have);
        }
        v_src = p.v + page * p.v_sp + row * p.v_ss + head * p.v_sh, v_have = have;
        slot += kTile, page = next_page, row = next_row;
      }
      t += n;
      if (t < t_end && t == base + static_cast<long long>(n_tiles) * units) {  // on to the next sequence that has keys
        base = t;
        do {
          ++b;
          len = b < p.batch ? seq_len(p, b) : 0;
          n_tiles = seq_tiles(p, len);
        } while (b < p.batch && n_tiles == 0);
        if (b >= p.batch) break;
      }
    }
  }
  // no more work, on both rings
  auto finish = [&](auto& r, Desc* at) {
    if (lane == 0) {
      if (pw == 0) at[r.stage].n_tiles = 0;
      mbar_arrive(r.full + 8 * r.stage);
    }
  };
  if (acquire(kr)) finish(kr, descs);
  if (acquire(vr)) finish(vr, v_descs);
  if (!ok) {  // a wait was given up: let the copies in flight land before the block ends
    auto drain = [&](auto& r, int stages, int used) {
      for (int i = 0; i < stages && i < used; ++i) {
        r.phase ^= r.stage == 0;
        r.stage = r.stage == 0 ? stages - 1 : r.stage - 1;
        volatile int never = 0;
        mbar_wait_limit(r.full + 8 * r.stage, r.phase, &never, nullptr, 0, 1000ull * 1000ull * 1000ull);
      }
    };
    drain(kr, L::kKStages, k_used);
    drain(vr, L::kVStages, v_used);
  }
}

// Four or eight warps: S^T = K Q^T, a quarter of the head dimension (and half of the rows) each, and the softmax of every
// fourth or eighth row.
template <bool kFp16, int kNB>
__device__ __forceinline__ void score_warp(const PagedAttnParams& p, uint8_t* smem, Rings<kNB> rings, volatile int* abort_flag,
                                           int warp, int lane) {
  using L = Layout<kNB>;
  constexpr int kRows = L::kRows;
  constexpr int kW = kScoreWarps<kNB>;
  constexpr int kNBS = kNB / kRowGroups<kNB>;  // n tiles of a warp
  constexpr int kR = kRows / kW;               // softmax: rows of a warp
  const int quarter = warp & 3, nb0 = (warp >> 2) * kNBS;
  const Desc* descs = reinterpret_cast<const Desc*>(smem + L::kOffDesc);
  float* part0 = reinterpret_cast<float*>(smem + L::kOffPart);
  uint16_t* p0 = reinterpret_cast<uint16_t*>(smem + L::kOffP);
  float* corr0 = reinterpret_cast<float*>(smem + L::kOffCorr);
  float2* stat = reinterpret_cast<float2*>(smem + L::kOffStat);
  int2* bounds = reinterpret_cast<int2*>(smem + L::kOffBounds);
  auto& r = rings.k;
  const uint32_t ring0 = smem_u32(smem);
  const int frag_row = lane >> 2, frag_col = (lane & 3) * 2;
  const float scale_log2 = p.scale * kLog2e;
  const float cap_in = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
  const float cap_out = p.softcap * kLog2e;
  auto wait = [&](const auto& ring) { return ring.wait_full(abort_flag, p.status, ST_TIMEOUT_SOFTMAX); };

  while (true) {
    const int mine = wait(r) && !*abort_flag;
    // These warps meet at a barrier below: they have to agree on whether to go on.
    int go;
    asm volatile(
        "{\n\t.reg .pred P, Q;\n\tsetp.ne.s32 P, %1, 0;\n\tbarrier.cta.red.and.pred Q, 1, %2, P;\n\tselp.s32 %0, 1, 0, Q;\n\t}"
        : "=r"(go)
        : "r"(mine), "n"(32 * kW)
        : "memory");
    if (!go) return;
    const Desc d = descs[r.stage];
    if (d.n_tiles == 0) return;
    // query rows as B operand: [k step][n tile][2]
    uint32_t qf[8][kNBS][2];
    {
      const uint32_t base = ring0 + r.stage * kStageBytes + (lane & 7) * kPitch + quarter * 256 + (lane >> 3) * 16;
#pragma unroll
      for (int nb = 0; nb < kNBS; ++nb)
#pragma unroll
        for (int ks = 0; ks < 8; ks += 2) {
          uint32_t x[4];
          ldmatrix_x4(base + (nb0 + nb) * 8 * kPitch + ks * 32, x);
          qf[ks][nb][0] = x[0], qf[ks][nb][1] = x[1], qf[ks + 1][nb][0] = x[2], qf[ks + 1][nb][1] = x[3];
        }
    }
    r.arrive_empty(lane);
    r.next();
    const Seen seen(p, d);
    float m_row[kR], l_row[kR];
#pragma unroll
    for (int k = 0; k < kR; ++k) {
      m_row[k] = -INFINITY, l_row[k] = 0.f;
      const int row = warp + kW * k, i = (d.row0 + row) / p.group;
      if (lane == 0)  // only this warp reads its rows' bounds; rows that pad the block see nothing
        bounds[row] = row < seen.n_rows ? make_int2(seen.first(i), seen.end(i, d.len)) : make_int2(0, 0);
    }
    __syncwarp();
    // with key_weights: where the scores of this warp's rows go, and how many of their keys are counted
    const int counted = p.scores ? min(d.len, p.weights_len) : 0;
    const int64_t score_pitch = static_cast<int64_t>(kW) * p.weights_len;
    float* const score_row =
        p.scores + (static_cast<int64_t>(d.b) * p.heads_kv * p.rows + d.head * p.rows + d.row0 + warp) * p.weights_len;

    for (int tile = 0; tile < d.n_tiles; ++tile) {
      // ---- partial scores: 2 x 16 keys x rows
      float s[2][kNBS][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nb = 0; nb < kNBS; ++nb) s[h][nb][0] = s[h][nb][1] = s[h][nb][2] = s[h][nb][3] = 0.f;
      wait(r);
      const uint32_t base = ring0 + r.stage * kStageBytes + (lane & 15) * kPitch + quarter * 256 + (lane >> 4) * 16;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a[4];
          ldmatrix_x4(base + h * 16 * kPitch + ks * 32, a);
#pragma unroll
          for (int nb = 0; nb < kNBS; ++nb) mma_16816<kFp16>(s[h][nb], a, qf[ks][nb][0], qf[ks][nb][1]);
        }
      r.arrive_empty(lane);
      r.next();
      float* const part = part0 + (tile & 1) * L::kPartFloats;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nb = 0; nb < kNBS; ++nb) {
          float* dst = part + (quarter * kRows + (nb0 + nb) * 8 + frag_col) * kPartPitch + h * 16 + frag_row;
          dst[0] = s[h][nb][0], dst[kPartPitch] = s[h][nb][1], dst[8] = s[h][nb][2], dst[kPartPitch + 8] = s[h][nb][3];
        }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kW) : "memory");
      // ---- softmax: a row at a time, one key per lane; step by step over all rows, so that their latencies overlap
      const int key0 = d.first_key + tile * kTile, key = key0 + lane;
      float x[kR], top[kR];
#pragma unroll
      for (int k = 0; k < kR; ++k) {
        const float* src = part + (warp + kW * k) * kPartPitch + lane;
        x[k] = (src[0] + src[kRows * kPartPitch]) + (src[2 * kRows * kPartPitch] + src[3 * kRows * kPartPitch]);
      }
      if (p.softcap > 0.f) {
#pragma unroll
        for (int k = 0; k < kR; ++k) x[k] = cap_out * tanhf(x[k] * cap_in);
      } else {
#pragma unroll
        for (int k = 0; k < kR; ++k) x[k] *= scale_log2;
      }
      if (!seen.all_of(key0)) {
#pragma unroll
        for (int k = 0; k < kR; ++k) {
          const int2 vis = bounds[warp + kW * k];
          if (key < vis.x || key >= vis.y) x[k] = -INFINITY;
        }
      }
      if (key < counted) {
        float* to = score_row + key;
#pragma unroll
        for (int k = 0; k < kR; ++k)
          if (warp + kW * k < seen.n_rows) to[k * score_pitch] = x[k];
      }
#pragma unroll
      for (int k = 0; k < kR; ++k) top[k] = warp_max(x[k]);
      rings.p.wait_empty(abort_flag, p.status, ST_TIMEOUT_SOFTMAX);
      uint16_t* const p_hi = p0 + rings.p.stage * 4 * L::kPWords;
      uint16_t* const p_lo = p_hi + 2 * L::kPWords;
      float* const corr = corr0 + rings.p.stage * L::kCorr;
#pragma unroll
      for (int k = 0; k < kR; ++k) {
        const int row = warp + kW * k;
        const float m_new = fmaxf(m_row[k], top[k]);
        // a row that has seen no key yet: any finite reference gives p = 0 (and NaN for scores that are NaN)
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float c = ex2(m_row[k] - ref), e = ex2(x[k] - ref);
        m_row[k] = m_new;
        l_row[k] = l_row[k] * c + e;
        uint16_t hi, lo;
        split16<kFp16>(e * kPScale<kFp16>, hi, lo);
        p_hi[row * kPPitch * 2 + lane] = hi, p_lo[row * kPPitch * 2 + lane] = lo;
        if (lane == 0) corr[row] = c;
      }
      if (warp == 0 && lane == 0) corr[kRows] = key0 < seen.free_lo || min(key0 + kTile, d.len) > seen.free_hi ? 1.f : 0.f;
      rings.p.arrive_full(lane);
      rings.p.next();
    }
    // ---- the stretch is done
    rings.stat.wait_empty(abort_flag, p.status, ST_TIMEOUT_SOFTMAX);
#pragma unroll
    for (int k = 0; k < kR; ++k) {
      float l = l_row[k];
#pragma unroll
      for (int w = 16; w; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
      const int row = warp + kW * k;
      if (lane == 0) {
        stat[row] = make_float2(m_row[k], l);
        if (row < seen.n_rows) {
          const int unit_row = d.row0 + row;
          if (d.slot < 0) {
            const int i = unit_row / p.group, g = unit_row - i * p.group;
            const float l2 = l == 0.f ? -INFINITY : m_row[k] + log2f(l);
            if (p.lse) p.lse[(static_cast<int64_t>(d.b) * p.heads_q + d.head * p.group + g) * p.sq + i] = l2 * kLn2;
            if (p.lse2) p.lse2[(static_cast<int64_t>(d.b) * p.heads_kv + d.head) * p.rows + unit_row] = l2;
          } else {
            p.part_ml[(blockIdx.x * 2 + d.slot) * p.rows_per_block + row] = make_float2(m_row[k], l);
          }
        }
      }
    }
    rings.stat.arrive_full(lane);
    rings.stat.next();
  }
}

// Eight warps: O^T += V^T P^T, 64 columns of the head dimension each, behind the score warps. They do not wait for one
// another, so one that gives up a wait just ends.
template <bool kFp16, int kNB>
__device__ __forceinline__ void value_warp(const PagedAttnParams& p, uint8_t* smem, Rings<kNB> rings, volatile int* abort_flag,
                                           int warp, int lane) {
  using L = Layout<kNB>;
  constexpr int kRows = L::kRows;
  constexpr int kMT = kHeadDim / kValueWarps / 16;  // 16-column tiles
  const Desc* descs = reinterpret_cast<const Desc*>(smem + L::kOffDesc) + L::kKStages;
  const uint32_t* p0 = reinterpret_cast<const uint32_t*>(smem + L::kOffP);
  const float* corr0 = reinterpret_cast<const float*>(smem + L::kOffCorr);
  const float2* stat = reinterpret_cast<const float2*>(smem + L::kOffStat);
  auto& r = rings.v;
  const uint32_t ring0 = smem_u32(smem) + L::kKStages * kStageBytes;
  const int frag_row = lane >> 2, frag_col = (lane & 3) * 2;
  auto wait = [&](const auto& ring) {
    return __all_sync(0xffffffffu, ring.wait_full(abort_flag, p.status, ST_TIMEOUT_SOFTMAX));
  };

  while (true) {
    if (!wait(r)) return;
    const Desc d = descs[r.stage];
    if (d.n_tiles == 0) return;
    float o[kMT][kNB][4];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][nb][e] = 0.f;
    for (int tile = 0; tile < d.n_tiles; ++tile) {
      if (!wait(rings.p)) return;
      const float* const corr = corr0 + rings.p.stage * L::kCorr;
      float2 cf[kNB];
      bool any = false;
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb) {
        cf[nb] = *reinterpret_cast<const float2*>(corr + nb * 8 + frag_col);
        any |= cf[nb].x != 1.f || cf[nb].y != 1.f;
      }
      if (__any_sync(0xffffffffu, any)) {
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
          for (int nb = 0; nb < kNB; ++nb) {
            o[mt][nb][0] *= cf[nb].x, o[mt][nb][1] *= cf[nb].y;
            o[mt][nb][2] *= cf[nb].x, o[mt][nb][3] *= cf[nb].y;
          }
      }
      if (tile > 0 && !wait(r)) return;
      const uint32_t base =
          ring0 + r.stage * kStageBytes + ((lane & 7) + (lane >> 4) * 8) * kPitch + warp * (kMT * 32) + ((lane >> 3) & 1) * 16;
      // P as B operand, one load per k step and n tile: its upper numbers' two registers, then its lower ones'
      const uint32_t p_base =
          smem_u32(p0 + (rings.p.stage * 2 + (lane >> 4)) * L::kPWords) + (lane & 7) * (kPPitch * 4) + ((lane >> 3) & 1) * 16;
      // Where some rows do not see some keys, an infinity or NaN among those keys' values must not reach them through a
      // weight of 0 (0 * inf). Such tiles are few, and such values next to none.
      bool products = true;
      if (corr[kRows] != 0.f) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 2 * kMT; ++i) {
          uint32_t a[4];
          ldmatrix_x4_trans(base + (i & 1) * 16 * kPitch + (i >> 1) * 32, a);
          bad |= not_finite2<kFp16>(a[0]) || not_finite2<kFp16>(a[1]) || not_finite2<kFp16>(a[2]) || not_finite2<kFp16>(a[3]);
        }
        products = !__any_sync(0xffffffffu, bad);
      }
      if (products) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t pf[kNB][4];
#pragma unroll
          for (int nb = 0; nb < kNB; ++nb) ldmatrix_x4(p_base + nb * 8 * kPPitch * 4 + ks * 32, pf[nb]);
#pragma unroll
          for (int mt = 0; mt < kMT; ++mt) {
            uint32_t a[4];
            ldmatrix_x4_trans(base + ks * 16 * kPitch + mt * 32, a);
#pragma unroll
            for (int nb = 0; nb < kNB; ++nb) mma_16816<kFp16>(o[mt][nb], a, pf[nb][0], pf[nb][1]);
#pragma unroll
            for (int nb = 0; nb < kNB; ++nb) mma_16816<kFp16>(o[mt][nb], a, pf[nb][2], pf[nb][3]);
          }
        }
      } else {
        const uint8_t* v_at = smem + L::kKStages * kStageBytes + r.stage * kStageBytes + (warp * (kMT * 16) + frag_row) * 2;
        const uint16_t* p_at = reinterpret_cast<const uint16_t*>(p0 + rings.p.stage * 2 * L::kPWords) + frag_col * kPPitch * 2;
#pragma unroll 1
        for (int key = 0; key < kTile; ++key) {
          float unused;
#pragma unroll
          for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const volatile uint16_t* at = p_at + (nb * 8 + e) * kPPitch * 2 + key;
              float hi, lo;
              unpack2<kFp16>(at[0], hi, unused);
              unpack2<kFp16>(at[2 * L::kPWords], lo, unused);
              const float w = hi + lo;
              if (w != 0.f) {
#pragma unroll
                for (int i = 0; i < 2 * kMT; ++i) {
                  float v;
                  unpack2<kFp16>(*reinterpret_cast<const volatile uint16_t*>(v_at + key * kPitch + i * 16), v, unused);
                  o[i >> 1][nb][e + 2 * (i & 1)] += w * v;
                }
              }
            }
        }
      }
      r.arrive_empty(lane);
      r.next();
      rings.p.arrive_empty(lane);
      rings.p.next();
    }
    // ---- the stretch is done
    if (!wait(rings.stat)) return;
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = nb * 8 + frag_col + e;
        const int unit_row = d.row0 + row;
        if (row >= p.rows_per_block || unit_row >= p.rows) continue;
        const int col = warp * (kMT * 16) + frag_row;
        if (d.slot < 0) {
          const int i = unit_row / p.group, g = unit_row - i * p.group;
          const float l = stat[row].y;
          const float inv = l == 0.f ? 0.f : kPUnscale<kFp16> / l;
          uint16_t* dst = p.o + d.b * p.o_sb + i * p.o_ss + (d.head * p.group + g) * p.o_sh + col;
#pragma unroll
          for (int mt = 0; mt < kMT; ++mt) {
            dst[mt * 16] = static_cast<uint16_t>(pack2<kFp16>(o[mt][nb][e] * inv, 0.f) & 0xffffu);
            dst[mt * 16 + 8] = static_cast<uint16_t>(pack2<kFp16>(o[mt][nb][e + 2] * inv, 0.f) & 0xffffu);
          }
        } else {
          float* dst = p.part_o + (static_cast<int64_t>(blockIdx.x * 2 + d.slot) * p.rows_per_block + row) * kHeadDim + col;
#pragma unroll
          for (int mt = 0; mt < kMT; ++mt) dst[mt * 16] = o[mt][nb][e], dst[mt * 16 + 8] = o[mt][nb][e + 2];
        }
      }
    rings.stat.arrive_empty(lane);
    rings.stat.next();
  }
}

template <bool kFp16, int kNB>
__global__ void __launch_bounds__(kThreads<kNB>, 1) splitd_paged_attn_kernel(const __grid_constant__ PagedAttnParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using L = Layout<kNB>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffAbort);
  const Rings<kNB> rings(smem_u32(smem + L::kOffBar));
  if (threadIdx.x == 0) {
    rings.init();
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (warp >= kValueWarps + kScoreWarps<kNB>) {
    if constexpr (kSplitRegs<kNB>) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs<kNB>));
    producer<kNB>(p, smem, rings, abort_flag, warp - kValueWarps - kScoreWarps<kNB>, lane);
  } else if (warp >= kValueWarps) {
    if constexpr (kSplitRegs<kNB>) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kScoreRegs<kNB>));
    score_warp<kFp16, kNB>(p, smem, rings, abort_flag, warp - kValueWarps, lane);
  } else {
    if constexpr (kNB == 3) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kValueRegs<kNB>));
    if constexpr (kNB == 4) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kValueRegs<kNB>));
    value_warp<kFp16, kNB>(p, smem, rings, abort_flag, warp, lane);
  }
}

// How the line of tiles falls on one sequence, from the lengths alone. One warp.
struct Span {
  long long total, first;  // tiles of all sequences, and before this one
  int n_tiles, len;        // tiles of a unit of this sequence
};
__device__ __forceinline__ Span span_of(const PagedAttnParams& p, int b, int lane) {
  long long before = 0, after = 0;
#pragma unroll 4
  for (int b0 = 0; b0 < p.batch; b0 += 32) {  // the tiles of 32 sequences fit 32 bits
    const int i = b0 + lane;
    const unsigned t = i < p.batch ? seq_tiles(p, seq_len(p, i)) : 0u;
    before += __reduce_add_sync(0xffffffffu, i < b ? t : 0u), after += __reduce_add_sync(0xffffffffu, i >= b ? t : 0u);
  }
  const int units = p.heads_kv * p.row_blocks;
  Span s;
  s.len = seq_len(p, b), s.n_tiles = seq_tiles(p, s.len);
  s.first = before * units, s.total = (before + after) * units;
  return s;
}
// The CTAs [first, last] whose shares hold parts of a unit.
__device__ __forceinline__ int2 owners(const PagedAttnParams& p, const Span& s, int unit) {
  const Line line = make_line(p, s.total);
  const long long t0 = s.first + static_cast<long long>(unit) * s.n_tiles;
  return make_int2(line.owner(t0), line.owner(t0 + s.n_tiles - 1));
}
// Partial result of CTA c: the first owner's share ends inside the unit (its second one); the others begin inside it.
__device__ __forceinline__ int slot_of(int c, int first) { return c == first ? 2 * c + 1 : 2 * c; }

// One block per output row: adds up the partial results of the CTAs that share the row's unit, or writes the row of a
// sequence without keys. Rows whose unit lay inside one CTA are finished already. kGroups groups of kCols / 4 threads, 4
// columns each; group g takes every kGroups-th partial result; `slice` counts the kCols columns of this block.
template <bool kFp16, int kGroups, int kCols>
__device__ __forceinline__ void join_row(const PagedAttnParams& p, const Span& span, int b, int hr, int slice) {
  constexpr int kPer = kCols / 4;  // threads of a group
  __shared__ float4 acc[kGroups][kGroups > 1 ? kPer : 1];
  const int tid = threadIdx.x, lane = tid & 31, col0 = slice * kCols;
  const int head = hr / p.rows, unit_row = hr - head * p.rows;
  const int rb = unit_row / p.rows_per_block, row = unit_row - rb * p.rows_per_block;
  const int i = unit_row / p.group, g = unit_row - i * p.group;
  const int hq = head * p.group + g;
  uint16_t* out = p.o + b * p.o_sb + i * p.o_ss + hq * p.o_sh;
  const int64_t lse_at = (static_cast<int64_t>(b) * p.heads_q + hq) * p.sq + i;
  const int2 own = span.n_tiles > 0 ? owners(p, span, head * p.row_blocks + rb) : make_int2(0, -1);
  pdl_wait();
  if (span.n_tiles == 0) {
    if (tid < kCols / 8) *reinterpret_cast<uint4*>(out + col0 + tid * 8) = make_uint4(0, 0, 0, 0);
    if (tid == 0 && col0 == 0 && p.lse) p.lse[lse_at] = -INFINITY;
    return;
  }
  if (own.x == own.y) return;
  auto ml_of = [&](int c) { return p.part_ml[slot_of(c, own.x) * p.rows_per_block + row]; };
  const float2 none = make_float2(-INFINITY, 0.f);
  float2 ml = own.x + lane <= own.y ? ml_of(own.x + lane) : none;
  float m = ml.x;
  for (int c = own.x + 32 + lane; c <= own.y; c += 32) m = fmaxf(m, ml_of(c).x);
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  const int grp = tid / kPer, col = col0 + tid % kPer * 4;
  const float* base = p.part_o + static_cast<int64_t>(row) * kHeadDim + col;
  const int64_t pitch = static_cast<int64_t>(p.rows_per_block) * kHeadDim;
  float l = 0.f;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int cc = own.x; cc <= own.y; cc += 32) {  // lane: weight of partial result cc + lane
    if (cc > own.x) ml = cc + lane <= own.y ? ml_of(cc + lane) : none;
    const float w = ex2(ml.x - ref);
    l += w * ml.y;
    const int n = min(32, own.y - cc + 1);
#pragma unroll 4
    for (int k = grp; k < n; k += kGroups) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(base + slot_of(cc + k, own.x) * pitch));
      const float wk = __shfl_sync(0xffffffffu, w, k);
      s.x += wk * v.x, s.y += wk * v.y, s.z += wk * v.z, s.w += wk * v.w;
    }
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
  if constexpr (kGroups > 1) {
    acc[grp][tid % kPer] = s;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) {
      const float4 v = acc[k][tid];
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  const float inv = l == 0.f ? 0.f : kPUnscale<kFp16> / l;
  uint2 w;
  w.x = pack2<kFp16>(s.x * inv, s.y * inv), w.y = pack2<kFp16>(s.z * inv, s.w * inv);
  *reinterpret_cast<uint2*>(out + col) = w;
  if (tid == 0 && col0 == 0 && p.lse) p.lse[lse_at] = (l == 0.f ? -INFINITY : m + log2f(l)) * kLn2;
}

// key_weights[b][key] += sum over the query rows of 2^(x - lse2), in row order; one key per thread. The lse of a row is
// formed here once more from the partial (m, l), so that this does not have to wait for the join: by one thread per row,
// or by one warp where many CTAs share a unit (kWide).
template <int kThreads, bool kWide>
__device__ __forceinline__ void add_weights(const PagedAttnParams& p, const Span& span, int b, int block) {
  constexpr int kRows = kWide ? 64 : kThreads;  // rows at a time
  constexpr int kUnits = 64;
  __shared__ float lse2[kRows];
  __shared__ int2 unit_owners[kWide ? kUnits : 1];  // of the sequence's first units
  const int tid = threadIdx.x, lane = tid & 31;
  const int n = min(span.len, p.weights_len);
  const int key0 = first_key(p, span.len) + block * kThreads;
  const int rows = p.heads_kv * p.rows;
  if (block == 0 && tid == 0 && span.len > p.weights_len && p.status) atomicCAS(p.status, 0, ST_BAD_CACHE_LEN);
  if (key0 >= n) {
    pdl_wait();
    return;
  }
  const int key = key0 + tid;
  const float* x = p.scores + static_cast<int64_t>(b) * rows * p.weights_len + key;
  const int units = p.heads_kv * p.row_blocks;
  if constexpr (kWide) {
    for (int u = tid; u < min(units, kUnits); u += kThreads) unit_owners[u] = owners(p, span, u);
    __syncthreads();
    pdl_wait();
  }
  float sum = 0.f;
  for (int r0 = 0; r0 < rows; r0 += kRows) {
    const int nr = min(kRows, rows - r0);
    if (r0 > 0) __syncthreads();
    for (int r = kWide ? tid >> 5 : tid; r < nr; r += kWide ? kThreads / 32 : kThreads) {
      const int hr = r0 + r;
      const int head = hr / p.rows, unit_row = hr - head * p.rows;
      const int rb = unit_row / p.rows_per_block, row = unit_row - rb * p.rows_per_block;
      const int u = head * p.row_blocks + rb;
      const int2 own = kWide && u < kUnits ? unit_owners[u] : owners(p, span, u);
      if (!kWide) pdl_wait();
      float m = -INFINITY, l = 0.f;
      if (own.x == own.y) {
        m = p.lse2[static_cast<int64_t>(b) * rows + hr], l = 1.f;
      } else {
#pragma unroll 4
        for (int c = kWide ? own.x + lane : own.x; c <= own.y; c += kWide ? 32 : 1) {
          const float2 ml = p.part_ml[slot_of(c, own.x) * p.rows_per_block + row];
          const float top = fmaxf(m, ml.x), ref = top == -INFINITY ? 0.f : top;
          l = l * ex2(m - ref) + ml.y * ex2(ml.x - ref);
          m = top;
        }
        if constexpr (kWide) {
          const float top = warp_max(m), ref = top == -INFINITY ? 0.f : top;
          l *= ex2(m - ref);
#pragma unroll
          for (int w = 16; w; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
          m = top;
        }
      }
      if (!kWide || lane == 0) lse2[r] = l == 0.f ? -INFINITY : m + log2f(l);
    }
    if (!kWide) pdl_wait();  // threads without a row
    __syncthreads();
    if (key < n) {
#pragma unroll 16
      for (int r = 0; r < nr; ++r) {
        const float l2 = lse2[r], v = __ldcs(x + static_cast<int64_t>(r0 + r) * p.weights_len);
        sum += l2 == -INFINITY ? 0.f : ex2(v - l2);
      }
    }
  }
  if (key < n) p.weights[b * p.weights_stride + key] += sum;
}

// What is left when all shares are done: blockIdx.y is the sequence; the first heads_kv * rows * (512 / kCols) blocks join
// a row (or a slice of it) each, the others (with key_weights) add up the weights of kGroups * kCols / 4 keys each.
template <bool kFp16, int kGroups, int kCols>
__global__ void __launch_bounds__(kGroups * kCols / 4) splitd_paged_finish_kernel(const __grid_constant__ PagedAttnParams p) {
  constexpr int kSlices = kHeadDim / kCols;
  __shared__ Span shared_span;
  const int b = blockIdx.y, n_join = p.heads_kv * p.rows * kSlices;
  if (threadIdx.x < 32) {
    const Span s = span_of(p, b, threadIdx.x);
    if (threadIdx.x == 0) shared_span = s;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0 && __ldg(p.seqlens + b) > page_capacity(p.map) && p.status)
    atomicCAS(p.status, 0, ST_BAD_CACHE_LEN);
  __syncthreads();
  const Span span = shared_span;
  const int block = blockIdx.x;
  if (block < n_join)
    join_row<kFp16, kGroups, kCols>(p, span, b, block / kSlices, block % kSlices);
  else
    add_weights<kGroups * kCols / 4, (kGroups > 1)>(p, span, b, block - n_join);
}

}  // namespace pa

namespace {

int row_blocks_of(int rows) { return (rows + pa::kMaxRows - 1) / pa::kMaxRows; }
int rows_per_block_of(int rows) { return (rows + row_blocks_of(rows) - 1) / row_blocks_of(rows); }

int64_t max_keys(const splitd_paged_params* p) { return static_cast<int64_t>(p->max_pages) * p->page_size; }

constexpr int kMaxCtas = 256;  // sizes the workspace without asking a device

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

size_t paged_workspace_bytes(const splitd_paged_params* p) {
  if (p->batch <= 0 || p->seqlen_q <= 0 || p->heads_q <= 0 || p->heads_kv <= 0) return 0;
  const int64_t rows = static_cast<int64_t>(p->seqlen_q) * (p->heads_q / p->heads_kv);
  const size_t rpb = rows < pa::kMaxRows ? rows : pa::kMaxRows;
  size_t n = align256(static_cast<size_t>(kMaxCtas) * 2 * rpb * kHeadDim * 4) + align256(static_cast<size_t>(kMaxCtas) * 2 * rpb * 8);
  if (p->key_weights) {
    const size_t all = static_cast<size_t>(p->batch) * rows * p->heads_kv;
    n += align256(all * 4) + align256(all * p->key_weights_len * 4);
  }
  return n;
}

namespace {

template <typename Kernel>
int raise_smem(Kernel kern, int bytes, int threads, int split_total, std::atomic<int> (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && done[dev].load(std::memory_order_acquire)) return 0;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return fail(SPLITD_ERR_CUDA, "paged attention: the kernel's shared memory cannot be set");
  }
  if (split_total > 0) {
    cudaFuncAttributes at;
    if (cudaFuncGetAttributes(&at, kern) != cudaSuccess ||
        at.numRegs * threads < split_total) {
      cudaGetLastError();
      return fail(SPLITD_ERR_CUDA, "paged attention: built with too few registers for its split");
    }
  }
  if (dev >= 0 && dev < 64) done[dev].store(1, std::memory_order_release);
  return 0;
}

template <bool kFp16, int kNB>
int launch_main(const PagedAttnParams& p, int grid, cudaStream_t stream) {
  static std::atomic<int> done[64];
  auto kern = pa::splitd_paged_attn_kernel<kFp16, kNB>;
  if (int e = raise_smem(kern, pa::Layout<kNB>::kBytes, pa::kThreads<kNB>, pa::kSplitRegs<kNB> ? pa::kSplitTotal<kNB> : 0, done)) return e;
  kern<<<grid, pa::kThreads<kNB>, pa::Layout<kNB>::kBytes, stream>>>(p);
  return 0;
}

}  // namespace

int launch_paged_attn(const splitd_paged_params* a, cudaStream_t stream) {
  PagedAttnParams p;
  memset(&p, 0, sizeof(p));
  p.q = static_cast<const uint16_t*>(a->q), p.k = static_cast<const uint16_t*>(a->k_pages), p.v = static_cast<const uint16_t*>(a->v_pages);
  p.o = static_cast<uint16_t*>(a->o), p.lse = a->lse;
  p.map = {a->page_table, a->page_table_stride, a->max_pages, a->page_size, a->num_pages, page_shift(a->page_size)};
  p.seqlens = a->seqlens_k;
  p.q_sb = a->q_strides[0], p.q_ss = a->q_strides[1], p.q_sh = a->q_strides[2];
  p.o_sb = a->o_strides[0], p.o_ss = a->o_strides[1], p.o_sh = a->o_strides[2];
  p.k_sp = a->k_strides[0], p.k_ss = a->k_strides[1], p.k_sh = a->k_strides[2];
  p.v_sp = a->v_strides[0], p.v_ss = a->v_strides[1], p.v_sh = a->v_strides[2];
  p.batch = a->batch, p.sq = a->seqlen_q, p.heads_q = a->heads_q, p.heads_kv = a->heads_kv;
  p.group = a->heads_q / a->heads_kv;
  p.rows = p.sq * p.group;
  p.row_blocks = row_blocks_of(p.rows), p.rows_per_block = rows_per_block_of(p.rows);
  p.win_left = a->local ? a->window_left : -1;
  p.win_right = a->causal ? 0 : a->local ? a->window_right : -1;
  p.scale = a->softmax_scale, p.softcap = a->softcap;
  p.status = a->status_flag;
  // no more CTAs than tiles there can be
  const int64_t most = static_cast<int64_t>(p.batch) * p.heads_kv * p.row_blocks * ((max_keys(a) + pa::kTile - 1) / pa::kTile);
  int grid = sm_count() < kMaxCtas ? sm_count() : kMaxCtas;
  if (most < grid) grid = most > 0 ? static_cast<int>(most) : 1;
  p.max_ctas = grid;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.part_o = reinterpret_cast<float*>(ws);
  ws += align256(static_cast<size_t>(kMaxCtas) * 2 * p.rows_per_block * kHeadDim * 4);
  p.part_ml = reinterpret_cast<float2*>(ws);
  ws += align256(static_cast<size_t>(kMaxCtas) * 2 * p.rows_per_block * 8);
  if (a->key_weights) {
    const size_t all = static_cast<size_t>(p.batch) * p.rows * p.heads_kv;
    p.lse2 = reinterpret_cast<float*>(ws);
    ws += align256(all * 4);
    p.scores = reinterpret_cast<float*>(ws);
    p.weights = a->key_weights, p.weights_stride = a->key_weights_stride, p.weights_len = a->key_weights_len;
  }
  const bool fp16 = a->dtype == SPLITD_DTYPE_FP16;
  const int nb = (p.rows_per_block + 7) / 8;
  int e;
  if (nb == 1)
    e = fp16 ? launch_main<true, 1>(p, grid, stream) : launch_main<false, 1>(p, grid, stream);
  else if (nb == 2)
    e = fp16 ? launch_main<true, 2>(p, grid, stream) : launch_main<false, 2>(p, grid, stream);
  else if (nb == 3)
    e = fp16 ? launch_main<true, 3>(p, grid, stream) : launch_main<false, 3>(p, grid, stream);
  else
    e = fp16 ? launch_main<true, 4>(p, grid, stream) : launch_main<false, 4>(p, grid, stream);
  if (e) return e;
  cudaError_t ce = cudaGetLastError();
  // Few rows (so few units, each shared by many CTAs): four blocks a row, in which sixteen groups of threads read partial
  // results side by side (1 x 131072 keys, 32 rows, 37 results each: 4 us, 7 us with one block of four groups a row). Eight
  // results a row or more and up to two rows per SM: one block of four groups each (3 x 5452 keys, 192 rows: 27 us in all,
  // 29 with small blocks; 8 x 230 keys, 512 rows: 16, 13). Otherwise one small block each. The choice, which decides the
  // order of the sums, does not look at the width of the page table.
  const int64_t units = static_cast<int64_t>(p.batch) * p.heads_kv * p.row_blocks;
  const int64_t all_rows = static_cast<int64_t>(p.batch) * p.heads_kv * p.rows;
  const bool few = all_rows <= sm_count();
  const bool shared = units * 8 <= sm_count() && all_rows <= 2 * sm_count();
  const int64_t longest = !p.weights ? 0 : max_keys(a) < p.weights_len ? max_keys(a) : p.weights_len;
  const unsigned rows = p.heads_kv * p.rows;
  if (ce != cudaSuccess) {
  } else if (few) {
    const dim3 blocks(rows * 4 + static_cast<unsigned>((longest + 511) / 512), p.batch);
    ce = launch_dependent(fp16 ? pa::splitd_paged_finish_kernel<true, 16, 128> : pa::splitd_paged_finish_kernel<false, 16, 128>, blocks,
                          dim3(512), 0, stream, p);
  } else if (shared) {
    const dim3 blocks(rows + static_cast<unsigned>((longest + 511) / 512), p.batch);
    ce = launch_dependent(fp16 ? pa::splitd_paged_finish_kernel<true, 4, 512> : pa::splitd_paged_finish_kernel<false, 4, 512>, blocks,
                          dim3(512), 0, stream, p);
  } else {
    const dim3 blocks(rows + static_cast<unsigned>((longest + 127) / 128), p.batch);
    ce = launch_dependent(fp16 ? pa::splitd_paged_finish_kernel<true, 1, 512> : pa::splitd_paged_finish_kernel<false, 1, 512>, blocks,
                          dim3(128), 0, stream, p);
  }
  if (ce != cudaSuccess) {
    cudaGetLastError();
    return fail(SPLITD_ERR_CUDA, "paged attention: launch failed: %s", cudaGetErrorString(ce));
  }
  return 0;
}

}  // namespace sd
