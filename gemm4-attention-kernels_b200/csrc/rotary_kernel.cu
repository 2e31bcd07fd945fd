// Rotary positions on query and key heads of 512, and the append of new tokens to a paged cache (the same rotation on
// the way into the cache, and the values beside it).
//
// Mathematics. The first R dimensions of a head (R even, R <= 512) are R / 2 pairs; pair i of a token at position t is
// turned by the angle a = t * inv_freq[i]: y1 = f (x1 cos a - x2 sin a), y2 = f (x1 sin a + x2 cos a). A pair is
// (i, i + R / 2) or, interleaved, (2 i, 2 i + 1). The other dimensions pass through bit for bit. The gradient is the
// same map with -a.
//
// Angles. t * inv_freq loses its fraction in 32 bits at long contexts (t = 10^6: 0.06 rad), so turns = t * inv_freq /
// (2 pi) is formed in 64 bits, its whole part is dropped there, and only the rest goes to the 32-bit sincospi: three
// 64-bit operations and one sincospi per (token, pair, warp), shared by the heads the warp goes through.
//
// What bounds it. 2 bytes in and 2 out per element, a handful of operations: HBM. One warp takes a token and a run of
// its heads; a lane holds the two 16-byte pieces of a head row that belong together, so that both halves of a pair are
// in its registers, and asks for four head rows before it uses the first. Measured: 2 x 8192 tokens, 36 heads: 194 us a
// direction, 6.2 TB/s, 95 % of a plain copy's rate (212 us where the halves start at no 16-byte boundary and rows go
// through shared memory); 24576 tokens into a cache, 40 heads: 230 us, 6.3 TB/s.
#include <cstring>

#include "launch.cuh"
#include "paged.cuh"

namespace sd {

namespace rot {
constexpr int kWarps = 8;
constexpr int kUnroll = 4;

enum Layout { kHalf = 0, kInterleaved = 1, kHalfOdd = 2 };  // kHalfOdd: R / 2 is no multiple of 8
}  // namespace rot

struct RotaryParams {
  const uint16_t *q, *k, *v;  // v only when appending
  uint16_t *q_out, *k_out, *v_out;
  int64_t q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
  int64_t qo_sb, qo_ss, qo_sh;
  int64_t ko_sb, ko_ss, ko_sh, vo_sb, vo_ss, vo_sh;  // appending: page, row of the page, head
  int heads_q, heads_k, heads_v;
  int batch, seqlen;  // batched: tokens = batch * seqlen; packed: batch sequences in `tokens` rows of stride *_ss
  int64_t tokens;
  const void* positions;  // nullptr: the slot (appending only)
  int64_t pos_sb, pos_ss;
  int pos64;
  const double* inv_freq;
  int pairs;       // R / 2
  float factor, sign;
  int heads_per_warp, groups;  // a token's heads are split over `groups` warps
  // appending
  int append;
  PageMap map;
  const int* seqlens;
  const int* cu;  // packed tokens: first token of each sequence, batch + 1 entries
  int* status;
};

namespace rot {

// lane's share of one head row: two 16-byte pieces
struct Pieces {
  uint4 a, b;
};

template <bool kFp16>
__device__ __forceinline__ void turn_words(uint32_t& x1, uint32_t& x2, const float2* cs) {
  float a0, a1, b0, b1;
  unpack2<kFp16>(x1, a0, a1);
  unpack2<kFp16>(x2, b0, b1);
  x1 = pack2<kFp16>(a0 * cs[0].x - b0 * cs[0].y, a1 * cs[1].x - b1 * cs[1].y);
  x2 = pack2<kFp16>(a0 * cs[0].y + b0 * cs[0].x, a1 * cs[1].y + b1 * cs[1].x);
}

// first token of sequence b is cu[b]; the sequence that holds token t (the last one that begins at or before it and
// is not empty). One warp: 32 entries at a time.
__device__ __forceinline__ int sequence_of(const int* cu, int batch, int t, int lane) {
  for (int b0 = 0; b0 < batch; b0 += 32) {
    const bool past = b0 + lane < batch && __ldg(cu + b0 + lane + 1) > t;
    const unsigned m = __ballot_sync(0xffffffffu, past);
    if (m) return b0 + __ffs(m) - 1;
  }
  return -1;
}

template <bool kFp16, int kLayout, int kBlocksPerSm>
__global__ void __launch_bounds__(kWarps * 32, kBlocksPerSm) splitd_rotary_kernel(const __grid_constant__ RotaryParams p) {
  __shared__ __align__(16) uint16_t stage[kLayout == kHalfOdd ? kWarps : 1][kLayout == kHalfOdd ? kHeadDim : 8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t work = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  const int64_t token = work / p.groups;
  if (token >= p.tokens) return;
  const int h0 = static_cast<int>(work - token * p.groups) * p.heads_per_warp;
  const int heads = p.heads_q + p.heads_k + p.heads_v;
  const int h1 = min(h0 + p.heads_per_warp, heads);

  int b = 0;
  int64_t s = token;
  if (p.cu == nullptr) {
    b = static_cast<int>(token / p.seqlen);
    s = token - static_cast<int64_t>(b) * p.seqlen;
  }
  // where the token goes in the cache
  int64_t slot = 0;
  bool stored = true;
  int page = 0, row = 0;
  if (p.append) {
    int seq = b;
    if (p.cu) {
      seq = sequence_of(p.cu, p.batch, static_cast<int>(token), lane);
      slot = seq < 0 ? -1 : static_cast<int64_t>(__ldg(p.seqlens + seq)) - __ldg(p.cu + seq + 1) + token;
    } else {
      slot = static_cast<int64_t>(__ldg(p.seqlens + b)) - p.seqlen + s;
    }
    stored = slot >= 0;
    if (stored) {
      int code = 0;
      if (slot >= page_capacity(p.map)) {
        code = ST_BAD_CACHE_LEN;
      } else {
        int entry;
        split_slot(p.map, static_cast<int>(slot), entry, row);
        page = page_of(p.map, seq, entry);
        if (!page_ok(p.map, page)) code = ST_BAD_PAGE;
      }
      if (code) {
        stored = false;
        if (lane == 0 && p.status) atomicCAS(p.status, 0, code);
      }
    }
  }
  // cos and sin of the lane's pairs
  float2 cs[8];
  {
    double t = 0.0;
    if (p.positions) {
      const int64_t at = b * p.pos_sb + s * p.pos_ss;
      t = p.pos64 ? static_cast<double>(__ldg(static_cast<const long long*>(p.positions) + at))
                  : static_cast<double>(__ldg(static_cast<const int*>(p.positions) + at));
    } else {
      t = static_cast<double>(slot < 0 ? 0 : slot);  // a token that is not stored: as at position 0
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int pair;
      if constexpr (kLayout == kHalf) pair = lane * 8 + e;
      if constexpr (kLayout == kInterleaved) pair = (lane + (e >> 2) * 32) * 4 + (e & 3);
      if constexpr (kLayout == kHalfOdd) pair = lane + 32 * e;
      cs[e] = make_float2(1.f, 0.f);
      if (pair < p.pairs && h0 < p.heads_q + p.heads_k) {
        const double turns = t * (__ldg(p.inv_freq + pair) * 0.15915494309189533577);
        const float part = static_cast<float>(turns - rint(turns));
        float sn, cn;
        sincospif(2.f * part, &sn, &cn);
        cs[e] = make_float2(cn * p.factor, sn * p.factor * p.sign);
      }
    }
  }
  // pieces of a head row that this lane holds (16-byte units of it)
  int piece_a = lane, piece_b = lane + 32;
  if constexpr (kLayout == kHalf) {
    const int np = p.pairs >> 3;  // pieces of each rotated half
    piece_a = lane < np ? lane : 2 * np + 2 * (lane - np);
    piece_b = lane < np ? np + lane : piece_a + 1;
  }
  auto src_of = [&](int h) -> const uint4* {
    const uint16_t* x;
    if (h < p.heads_q)
      x = p.q + b * p.q_sb + s * p.q_ss + h * p.q_sh;
    else if (h < p.heads_q + p.heads_k)
      x = p.k + b * p.k_sb + s * p.k_ss + (h - p.heads_q) * p.k_sh;
    else
      x = p.v + b * p.v_sb + s * p.v_ss + (h - p.heads_q - p.heads_k) * p.v_sh;
    return reinterpret_cast<const uint4*>(x);
  };
  auto dst_of = [&](int h) -> uint4* {
    uint16_t* y;
    if (h < p.heads_q)
      y = p.q_out + b * p.qo_sb + s * p.qo_ss + h * p.qo_sh;
    else if (h < p.heads_q + p.heads_k)
      y = p.append ? p.k_out + page * p.ko_sb + row * p.ko_ss + (h - p.heads_q) * p.ko_sh
                   : p.k_out + b * p.ko_sb + s * p.ko_ss + (h - p.heads_q) * p.ko_sh;
    else
      y = p.v_out + page * p.vo_sb + row * p.vo_ss + (h - p.heads_q - p.heads_k) * p.vo_sh;
    return reinterpret_cast<uint4*>(y);
  };
  for (int h = h0; h < h1; h += kUnroll) {
    Pieces x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (h + u < h1) {
        const uint4* src = src_of(h + u);
        x[u].a = __ldcs(src + piece_a), x[u].b = __ldcs(src + piece_b);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (h + u >= h1) break;
      const bool is_q = h + u < p.heads_q;
      if (h + u < p.heads_q + p.heads_k && p.pairs > 0) {
        uint32_t* wa = reinterpret_cast<uint32_t*>(&x[u].a);
        uint32_t* wb = reinterpret_cast<uint32_t*>(&x[u].b);
        if constexpr (kLayout == kHalf) {
          if (lane < (p.pairs >> 3)) {
#pragma unroll
            for (int w = 0; w < 4; ++w) turn_words<kFp16>(wa[w], wb[w], cs + 2 * w);
          }
        }
        if constexpr (kLayout == kInterleaved) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            uint32_t& w = e < 4 ? wa[e] : wb[e - 4];
            float x1, x2;
            unpack2<kFp16>(w, x1, x2);
            const uint32_t y = pack2<kFp16>(x1 * cs[e].x - x2 * cs[e].y, x1 * cs[e].y + x2 * cs[e].x);
            if ((lane + (e >> 2) * 32) * 4 + (e & 3) < p.pairs) w = y;
          }
        }
        if constexpr (kLayout == kHalfOdd) {
          // the second half starts at no 16-byte boundary: the row goes through shared memory element by element
          uint16_t* st = stage[warp];
          uint4* st4 = reinterpret_cast<uint4*>(st);
          __syncwarp();
          st4[lane] = x[u].a, st4[lane + 32] = x[u].b;
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int pair = lane + 32 * e;
            if (pair < p.pairs) {
              float x1, x2, unused;
              unpack2<kFp16>(st[pair], x1, unused);
              unpack2<kFp16>(st[pair + p.pairs], x2, unused);
              st[pair] = static_cast<uint16_t>(pack2<kFp16>(x1 * cs[e].x - x2 * cs[e].y, 0.f) & 0xffffu);
              st[pair + p.pairs] = static_cast<uint16_t>(pack2<kFp16>(x1 * cs[e].y + x2 * cs[e].x, 0.f) & 0xffffu);
            }
          }
          __syncwarp();
          x[u].a = st4[lane], x[u].b = st4[lane + 32];
        }
      }
      if (is_q || stored) {
        uint4* dst = dst_of(h + u);
        __stcs(dst + piece_a, x[u].a);
        __stcs(dst + piece_b, x[u].b);
      }
    }
  }
}

}  // namespace rot

namespace {

template <bool kFp16, int kLayout>
void launch_layout(const RotaryParams& p, unsigned blocks, cudaStream_t stream) {
  if (blocks <= 2u * sm_count())
    rot::splitd_rotary_kernel<kFp16, kLayout, 2><<<blocks, rot::kWarps * 32, 0, stream>>>(p);
  else
    rot::splitd_rotary_kernel<kFp16, kLayout, 3><<<blocks, rot::kWarps * 32, 0, stream>>>(p);
}
template <int kLayout>
void launch_type(const RotaryParams& p, bool fp16, unsigned blocks, cudaStream_t stream) {
  if (fp16)
    launch_layout<true, kLayout>(p, blocks, stream);
  else
    launch_layout<false, kLayout>(p, blocks, stream);
}

int launch_rotary_kernel(RotaryParams& p, bool fp16, bool interleaved, cudaStream_t stream) {
  const int heads = p.heads_q + p.heads_k + p.heads_v;
  // Up to 20 heads per warp, in rounds of four and equal runs where the number of heads allows it: a warp's angles cost as
  // much as five of its heads, and much longer runs leave a tail (37 x 46 tokens, 40 heads: 25 us with two runs, 33 us with
  // three of 14, 34 us with ten of 4; 2 x 8192 tokens, 36 heads: 194 us with three runs, 201 us with two of 18). Shorter
  // runs when there would not be half as many warps as the GPU holds (6 x 103 tokens, 36 heads: 11 us with three runs, 13
  // us with two), but four heads, one round of loads, at least. Calls of up to one wave of blocks get the registers of two
  // blocks per SM (64 tokens: 5.7 us, 6.5 us with three), longer ones three blocks (2 x 8192 tokens: 194 us, 201 us with
  // two), whose 80 registers a thread leave 32 to 36 bytes of it in local memory (102 to 114 registers, and none there, with
  // two).
  const int64_t half_full = sm_count() * (3 * rot::kWarps) / 2;
  int64_t groups = (heads + 19) / 20;
  for (int64_t g = groups; g <= 2 * groups; ++g)
    if (heads % (4 * g) == 0) {
      groups = g;
      break;
    }
  const int64_t fill = (half_full + p.tokens - 1) / p.tokens, most = (heads + rot::kUnroll - 1) / rot::kUnroll;
  if (groups < fill) groups = fill < most ? fill : most;
  p.heads_per_warp = static_cast<int>((heads + groups - 1) / groups);
  p.groups = (heads + p.heads_per_warp - 1) / p.heads_per_warp;
  const int64_t blocks = (p.tokens * p.groups + rot::kWarps - 1) / rot::kWarps;
  if (blocks > 0x7fffffff) return fail(SPLITD_ERR_INVALID_ARGUMENT, "too many tokens for one call");
  const unsigned n = static_cast<unsigned>(blocks);
  if (interleaved)
    launch_type<rot::kInterleaved>(p, fp16, n, stream);
  else if (p.pairs % 8 == 0)
    launch_type<rot::kHalf>(p, fp16, n, stream);
  else
    launch_type<rot::kHalfOdd>(p, fp16, n, stream);
  const cudaError_t ce = cudaGetLastError();
  if (ce != cudaSuccess) return fail(SPLITD_ERR_CUDA, "rotary: launch failed: %s", cudaGetErrorString(ce));
  return 0;
}

void set3(int64_t& a, int64_t& b, int64_t& c, const int64_t* s) { a = s[0], b = s[1], c = s[2]; }

}  // namespace

int launch_rotary(const splitd_rotary_params* a, cudaStream_t stream) {
  RotaryParams p;
  memset(&p, 0, sizeof(p));
  p.q = static_cast<const uint16_t*>(a->q), p.k = static_cast<const uint16_t*>(a->k);
  p.q_out = static_cast<uint16_t*>(a->q_out), p.k_out = static_cast<uint16_t*>(a->k_out);
  set3(p.q_sb, p.q_ss, p.q_sh, a->q_strides);
  set3(p.k_sb, p.k_ss, p.k_sh, a->k_strides);
  set3(p.qo_sb, p.qo_ss, p.qo_sh, a->q_out_strides);
  set3(p.ko_sb, p.ko_ss, p.ko_sh, a->k_out_strides);
  p.heads_q = a->q ? a->heads_q : 0, p.heads_k = a->k ? a->heads_kv : 0;
  p.batch = a->batch, p.seqlen = a->seqlen;
  p.tokens = static_cast<int64_t>(a->batch) * a->seqlen;
  p.positions = a->positions, p.pos_sb = a->position_strides[0], p.pos_ss = a->position_strides[1], p.pos64 = a->positions_64bit;
  p.inv_freq = a->inv_freq, p.pairs = a->rotary_dim / 2;
  p.factor = a->factor, p.sign = a->backward ? -1.f : 1.f;
  return launch_rotary_kernel(p, a->dtype == SPLITD_DTYPE_FP16, a->interleaved != 0, stream);
}

int launch_paged_append(const splitd_append_params* a, cudaStream_t stream) {
  RotaryParams p;
  memset(&p, 0, sizeof(p));
  p.append = 1;
  p.q = static_cast<const uint16_t*>(a->q), p.k = static_cast<const uint16_t*>(a->k), p.v = static_cast<const uint16_t*>(a->v);
  p.q_out = static_cast<uint16_t*>(a->q_out);
  p.k_out = static_cast<uint16_t*>(a->k_pages), p.v_out = static_cast<uint16_t*>(a->v_pages);
  set3(p.q_sb, p.q_ss, p.q_sh, a->q_strides);
  set3(p.k_sb, p.k_ss, p.k_sh, a->k_strides);
  set3(p.v_sb, p.v_ss, p.v_sh, a->v_strides);
  set3(p.qo_sb, p.qo_ss, p.qo_sh, a->q_out_strides);
  set3(p.ko_sb, p.ko_ss, p.ko_sh, a->k_page_strides);
  set3(p.vo_sb, p.vo_ss, p.vo_sh, a->v_page_strides);
  p.heads_q = a->q ? a->heads_q : 0, p.heads_k = p.heads_v = a->heads_kv;
  p.batch = a->batch, p.seqlen = a->seqlen;
  p.cu = a->cu_seqlens;
  p.tokens = a->cu_seqlens ? a->total_tokens : static_cast<int64_t>(a->batch) * a->seqlen;
  p.positions = a->positions, p.pos_sb = a->position_strides[0], p.pos_ss = a->position_strides[1], p.pos64 = a->positions_64bit;
  p.inv_freq = a->inv_freq, p.pairs = a->inv_freq ? a->rotary_dim / 2 : 0;
  p.factor = a->factor, p.sign = 1.f;
  p.map = {a->page_table, a->page_table_stride, a->max_pages, a->page_size, a->num_pages, page_shift(a->page_size)};
  p.seqlens = a->seqlens_k;
  p.status = a->status_flag;
  return launch_rotary_kernel(p, a->dtype == SPLITD_DTYPE_FP16, a->interleaved != 0, stream);
}

}  // namespace sd
