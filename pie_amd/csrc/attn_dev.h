// Device code of paged attention that the kernels in attn.hip and attn_shared.hip share: the cache and
// its page table, a wave's online softmax, the decode unit (one split of a request for one kv head), the
// prefill item (128 query rows over a kv range) and the sum of partial results.
#pragma once

#include "common.h"

namespace pie {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4_t mfma_16x16x32(const u32x4_t& a, const u32x4_t& b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// ds_read_b64_tr_b16: within each 16-lane group, output lane r element j is element r%4 of
// the 8 bytes addressed by lane 4j + r/4 (measured on gfx950).
__device__ __forceinline__ uint2 lds_read_tr16(const uint16_t* p) {
  typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;
  const i16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p));
  return __builtin_bit_cast(uint2, v);
}

__device__ __forceinline__ float lane_read(float v, int src_lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(src_lane << 2, __builtin_bit_cast(int, v)));
}

__device__ __forceinline__ u32x4_t ld16v(const uint16_t* p) {
  return *reinterpret_cast<const u32x4_t*>(p);
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// Attention sinks (gpt_oss.py:693-697): a per-head logit in the units of the scaled scores that
// joins each row's softmax denominator and no value: the row's mass gains exp2(sink log2(e) - m)
// relative to the row's running maximum m (0 when the row saw nothing).
__device__ __forceinline__ float sink_mass(const float* sinks, int head, float m) {
  return sinks ? fast_exp2(sinks[head] * 1.4426950408889634f - (m == -INFINITY ? 0.f : m)) : 0.f;
}

// The base-2 log-sum-exp of a row of softmax mass L relative to 2^M: -inf for a row that saw nothing.
__device__ __forceinline__ float row_lse(float L, float M) { return L == 0.f ? -INFINITY : M + log2f(L); }

// Online softmax with a lazy maximum: a row's reference maximum (and with it the rescale of its
// output accumulators and sum) moves only when a tile's scores exceed it by more than kLazyMax
// (log2 units), so every exponent stays <= 2^kLazyMax. Numerator and denominator share the
// reference, so the softmax is the same; the rescale runs a few times per row, not per tile.
constexpr float kLazyMax = 8.f;

// Kernel argument: the paged KV cache and its page table.
struct PagedKV {
  const uint16_t* k;       // k of page 0, slot 0, head 0
  const uint16_t* v;       // v of page 0, slot 0, head 0
  int64_t page_stride, slot_stride, head_stride;  // elements
  const int32_t* indptr;   // [B+1] pages per request
  const int32_t* indices;  // [sum pages] physical page ids
  const int32_t* last_len; // [B]
  int32_t num_pages;       // pages in the pool (ids outside [0, num_pages) are masked out)
  int32_t page_size;
  FastDiv pdiv;
};

// Host: fills *kv after checking the cache and page table arguments of the entry point `what`.
int paged_kv_desc(PagedKV* kv, const uint16_t* k_cache, const uint16_t* v_cache, int64_t page_stride,
                  int64_t slot_stride, int64_t head_stride, int64_t num_pages, const int32_t* kv_indptr,
                  const int32_t* kv_indices, const int32_t* kv_last_page_len, int64_t page_size, int64_t D,
                  const char* what);

__device__ __forceinline__ int kv_length(const PagedKV& kv, int b) {
  const int np = kv.indptr[b + 1] - kv.indptr[b];
  return np > 0 ? (np - 1) * kv.page_size + kv.last_len[b] : 0;
}

// Element offset of (token t of the request whose pages start at indices[page0], kv head h);
// -1 if its page id is out of range.
__device__ __forceinline__ int64_t kv_offset(const PagedKV& kv, int page0, int t, int h) {
  const uint32_t lp = kv.pdiv.div((uint32_t)t);
  const int slot = t - (int)lp * kv.page_size;
  const int page = kv.indices[page0 + (int)lp];
  if ((unsigned)page >= (unsigned)kv.num_pages) return -1;
  return (int64_t)page * kv.page_stride + (int64_t)slot * kv.slot_stride + (int64_t)h * kv.head_stride;
}

constexpr int kTileTokens = 32;  // kv tokens per wave iteration (two 16-token MFMA subtiles)

// XOR swizzle of the 16-byte chunks of LDS row r (rows of D bf16, no padding): the 16 rows one
// transpose read touches land on distinct chunks, so its 64 lanes hit every bank at most twice.
template <int D>
__device__ __forceinline__ int chunk_swizzle(int r) {
  return D == 64 ? (r >> 1) & 7 : r & 15;
}

// Swizzle of V rows, read by ds_read_b64_tr_b16: a transpose read takes two 16-byte chunks
// (one pair) from each of 16 rows, and every 8 consecutive rows must hit different 32-byte bank
// groups, so the pair index is XORed with r mod 8 (D = 64 keeps the row-pair scheme above).
template <int D>
__device__ __forceinline__ int v_swizzle(int r) {
  return D == 64 ? chunk_swizzle<64>(r) : (r & 7) << 1;
}

// Wait until this wave's LDS reads have returned (a transpose read must finish before a load
// into the same LDS tile is issued).
__device__ __forceinline__ void wait_lgkmcnt0() {
  __builtin_amdgcn_s_waitcnt((63 << 14) | (0 << 8) | (7 << 4) | 15);
}

// Wait until at most n vector-memory operations of this wave are outstanding (loads into LDS
// included); exp and lgkm counters are not waited on.
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt(((N >> 4) << 14) | (15 << 8) | (7 << 4) | (N & 15));
}

// One wave's running state for 16 query rows over a stream of 32-token kv tiles.
template <int D>
struct WaveAttn {
  static constexpr int NS = D / 32;  // MFMA k-steps over the head dim
  static constexpr int NB = D / 16;  // 16-dim output blocks
  u32x4_t qb[NS];     // B operand: query row n, dims 8(4s+g)..+8
  f32x4_t o[NB];      // C layout: rows 4g+i, dim 16nb+n
  float m;            // running max (exp2 domain) of row n, same in all four lane groups
  float l;            // this lane's partial sum of row n's probabilities

  __device__ __forceinline__ void init() {
    #pragma unroll
    for (int nb = 0; nb < NB; ++nb) o[nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }

  // The PV B-operands of a 32-token tile from the wave's LDS tile vt ([32][D], chunk-swizzled):
  // for each 16-dim block, lane 16g + 4j + q of two transpose reads addresses row (16h + 4g + j),
  // dims 16nb + 4q..+3, which sit in logical chunk 2nb + q/2 of that row.
  __device__ __forceinline__ void read_v(const uint16_t* vt, int lane, u32x4_t (&vb)[NB]) const {
    const int g = lane >> 4, j = (lane >> 2) & 3, q = lane & 3;
    const int r0 = 4 * g + j, r1 = r0 + 16;
    const uint16_t* b0 = vt + r0 * D + 4 * (q & 1);
    const uint16_t* b1 = vt + r1 * D + 4 * (q & 1);
    const int z0 = v_swizzle<D>(r0), z1 = v_swizzle<D>(r1);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int lc = 2 * nb + (q >> 1);
      const uint2 lo = lds_read_tr16(b0 + 8 * (lc ^ z0));
      const uint2 hi = lds_read_tr16(b1 + 8 * (lc ^ z1));
      vb[nb] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
    }
  }

  // Scores of a 32-token tile in the exp2 domain: s[u][i] = row n . token 16u+4g+i, -inf where
  // bit 4u+i of vmask is clear.
  __device__ __forceinline__ void scores(const u32x4_t (&ka)[2][NS], uint32_t vmask, float scale_log2,
                                         float (&s)[2][4]) const {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < NS; ++st) acc = mfma_16x16x32(ka[u][st], qb[st], acc);
      if (vmask == 0xFFu) {  // wave-uniform fast path for fully visible tiles
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] = acc[i] * scale_log2;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] = ((vmask >> (4 * u + i)) & 1u) ? acc[i] * scale_log2 : -INFINITY;
      }
    }
  }

  // Online-softmax step: updates m and l, returns the tile's probabilities as the PV A-operand
  // (bf16) and in a[i] the factor by which O row 4g+i must be rescaled; rescale = false (a
  // unset) when no row of the wave changed its maximum, so O needs no rescaling (wave-uniform).
  __device__ __forceinline__ u32x4_t softmax(const float (&s)[2][4], int lane, float (&a)[4],
                                             bool& rescale) {
    const int g = lane >> 4;
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = fmaxf(mx, lane_read(mx, lane ^ 16));
    mx = fmaxf(mx, lane_read(mx, lane ^ 32));
    const bool grow = mx > m + kLazyMax;  // lazy maximum
    const float m_new = grow ? mx : m;
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = grow ? fast_exp2(m - mx) : 1.f;
    float p[2][4], psum = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) { p[u][i] = fast_exp2(s[u][i] - m_use); psum += p[u][i]; }
    l = l * alpha + psum;
    m = m_new;
    rescale = __builtin_amdgcn_ballot_w64(alpha != 1.f) != 0;
    if (rescale) {
      // O rows 4g+i take the factor of row 4g+i (held by lane 4g+i of every group)
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = lane_read(alpha, 4 * g + i);
    }
    return u32x4_t{pack_bf2(p[0][0], p[0][1]), pack_bf2(p[0][2], p[0][3]),
                   pack_bf2(p[1][0], p[1][1]), pack_bf2(p[1][2], p[1][3])};
  }

  // O block nb = O block nb * a + P V_nb (no rescaling when softmax() reported none).
  __device__ __forceinline__ void pv(const u32x4_t& pa, const u32x4_t& vb, const float (&a)[4], bool rescale,
                                     int nb) {
    f32x4_t c = o[nb];
    if (rescale) {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] *= a[i];
    }
    o[nb] = mfma_16x16x32(pa, vb, c);
  }

  // One 32-token tile: ka = K A-operands of the two subtiles, vb = the V B-operands (read_v),
  // bit 4u+i of vmask says whether this lane's row n sees token 16u+4g+i.
  __device__ __forceinline__ void tile(const u32x4_t (&ka)[2][NS], uint32_t vmask,
                                       const u32x4_t (&vb)[NB], float scale_log2, int lane) {
    float s[2][4], a[4];
    bool rescale;
    scores(ka, vmask, scale_log2, s);
    const u32x4_t pa = softmax(s, lane, a, rescale);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) pv(pa, vb[nb], a, rescale, nb);
  }

  // Row n's total probability mass (sum of the four lane groups' partials).
  __device__ __forceinline__ float row_sum(int lane) const {
    float t = l + lane_read(l, lane ^ 16);
    return t + lane_read(t, lane ^ 32);
  }
};

// Page ids of a window of logical pages, staged in LDS once per work group.
constexpr int kPageWin = 512;

// Element offset of token t (its logical page lp = t / P lies in the staged window starting at
// lp0) for kv head h, branch-free; ok = false (and page 0 addressed) if the page id is out of
// range.
__device__ __forceinline__ uint64_t kv_offset_lds(const PagedKV& kv, const int32_t* ptab, int lp0,
                                                  int t, int h, bool& ok) {
  const int lp = (int)kv.pdiv.div((uint32_t)t);
  const int slot = t - lp * kv.page_size;
  const int page = ptab[lp - lp0];
  ok = (unsigned)page < (unsigned)kv.num_pages;
  const uint32_t pg = ok ? (uint32_t)page : 0u;
  return (uint64_t)pg * (uint32_t)kv.page_stride + (uint64_t)(uint32_t)slot * (uint32_t)kv.slot_stride +
         (uint64_t)(uint32_t)h * (uint32_t)kv.head_stride;
}

// One wave's loads for a 32-token tile: the K MFMA operands of both subtiles with their
// visibility ballots (registers), and the V rows, which go from HBM straight into the wave's
// LDS tile ([32][D], chunk-swizzled) without passing through registers. Tokens at or past `end`
// and tokens on out-of-range pages are invisible; their loads are clamped to valid addresses
// (an invisible row gets probability 0).
//
// Where first tokens stay visible beside a window (KEPT), the tiles walk the visible positions without
// the hidden ones between: visible position i is token i below `kept`, token i + skip from there on, and
// the staged page table holds the pages of the kept tokens, then those of the window, whose logical page
// lp is entry lp - lp0 before the hidden pages and lp - lp0 - gap after them.
// Bound: HBM. 256 streams of 128-20000 tokens, 2048 + 5 visible, 8 kv heads of 128: 2.1 GB in 372 us,
// 5.6 TB/s (their whole contexts hold about five times the bytes). One row of 1024 + 4 tokens: 8.3 us,
// and 4 for its splits' merge.
struct KeptMap {
  int kept = 0x7fffffff, skip = 0, gap = 0;
};
template <int D, bool KEPT = false>
struct KVTile {
  static constexpr int NS = D / 32, CH = D / 8, RPI = 64 / CH, NVL = kTileTokens / RPI;
  u32x4_t ka[2][NS];
  uint64_t vis[2];

  // Element offset of visible position i.
  static __device__ __forceinline__ uint64_t offset(const PagedKV& kv, const int32_t* ptab, int lp0, const KeptMap& km,
                                                    int i, int h, bool& ok) {
    if constexpr (KEPT) {
      const bool past = i >= km.kept;
      return kv_offset_lds(kv, ptab, past ? lp0 + km.gap : lp0, past ? i + km.skip : i, h, ok);
    } else {
      return kv_offset_lds(kv, ptab, lp0, i, h, ok);
    }
  }

  // Row-independent visibility in tile()'s vmask form: bit 4u+i = token 16u+4g+i.
  __device__ __forceinline__ uint32_t vmask(int lane) const {
    const int g = lane >> 4;
    return (uint32_t)((vis[0] >> (4 * g)) & 15u) | ((uint32_t)((vis[1] >> (4 * g)) & 15u) << 4);
  }

  __device__ __forceinline__ void load(const PagedKV& kv, const int32_t* ptab, int lp0, const KeptMap& km, int t0,
                                       int end, int kvh, int lane, uint16_t* vt) {
    const int n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < NVL; ++i) {
      const int r = RPI * i + lane / CH;
      bool ok;
      const uint64_t off = offset(kv, ptab, lp0, km, min(t0 + r, end - 1), kvh, ok);
      const int lc = (lane % CH) ^ v_swizzle<D>(r);
      __builtin_amdgcn_global_load_lds(kv.v + off + 8 * lc,
                                       (__attribute__((address_space(3))) void*)(vt + RPI * i * D),
                                       16, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int tok = t0 + 16 * u + n;
      bool ok;
      const uint16_t* kp = kv.k + offset(kv, ptab, lp0, km, min(tok, end - 1), kvh, ok);
#pragma unroll
      for (int s = 0; s < NS; ++s) ka[u][s] = ld16v(kp + 8 * (4 * s + g));
      vis[u] = __builtin_amdgcn_ballot_w64(tok < end && ok);
    }
  }
};

// ------------------------------------------------------------------------------ decode
// Grid (batch * splits * kv heads), one dimension: work group x takes the request of rank
// x / (splits * kv heads), split (x / kv heads) % splits, kv head x % kv heads. For batches of
// at most kRankMax requests the rank orders requests by attended length, longest first (ties
// by request index), so the longest requests' work groups are dispatched first and the short
// ones fill the tail; larger batches keep request order (rank = request). The split is derived
// on the device from the request's current kv length (chunks of ceil(kv_len / splits) rounded
// up to whole 32-token tiles, at least kMinChunk), and so is the rank, so a launch depends only
// on (batch, splits) and a captured graph replays correctly for any lengths.
// With one split the work group writes the output; otherwise it writes an fp32 partial output
// and its log2-sum-exp to slot x, and attn_merge_kernel combines the splits.
constexpr int kMinChunk = 128;
constexpr int kRankMax = 256;  // one request per thread of the work group

// The first position a window shows, the first tokens kept visible before it (positions [0, kept), none
// of them in the window) and the number of visible positions, for the query at position kv_len - 1.
__device__ __forceinline__ int window_start(int kv_len, int window_left) {
  return window_left >= 0 ? max(0, kv_len - 1 - window_left) : 0;
}
__device__ __forceinline__ int visible_len(int kv_len, int window_left, int first) {
  const int ws = window_start(kv_len, window_left);
  return kv_len - ws + min(first, ws);
}

// The request of rank r (B <= kRankMax), with its kv length and first page-table entry. Every
// work group of the launch ranks the same lengths the same way, so together they cover each
// (request, split, kv head) once. lens: kRankMax ints of LDS.
__device__ __forceinline__ int request_of_rank(const PagedKV& kv, int B, int window_left, int first, int r,
                                               int32_t* lens, int32_t* pick, int& kv_len, int& page0) {
  const int i = threadIdx.x;
  int kl = 0, li = -1, p0 = 0;  // padding: below every length
  if (i < B) {
    p0 = kv.indptr[i];
    kl = kv_length(kv, i);
    li = visible_len(kl, window_left, first);
  }
  lens[i] = li;
  __syncthreads();
  if (i < B) {
    int before = 0;  // requests ordered before i
    for (int k = 0; k < B; k += 4) {
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(lens + k);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int le = (int)v[e];
        before += le > li || (le == li && k + e < i);
      }
    }
    if (before == r) { pick[0] = i; pick[1] = kl; pick[2] = p0; }
  }
  __syncthreads();
  const int b = uniform(pick[0]);
  kv_len = uniform(pick[1]);
  page0 = uniform(pick[2]);  // (not loaded again: a round trip before the page table's)
  return b;
}

__device__ __forceinline__ int split_chunk(int kv_len, int splits) {
  const int chunk = (kv_len + splits - 1) / splits;
  return max(kMinChunk, (chunk + kTileTokens - 1) / kTileTokens * kTileTokens);
}
// The splits of a request that hold at least one token: 0 .. split_count - 1.
__device__ __forceinline__ int split_count(int kv_len, int splits) {
  const int chunk = split_chunk(kv_len, splits);
  return (kv_len + chunk - 1) / chunk;
}
__device__ __forceinline__ void split_range(int kv_len, int splits, int j, int& kv0, int& kv1) {
  const int chunk = split_chunk(kv_len, splits);
  kv0 = min(kv_len, j * chunk);
  kv1 = min(kv_len, kv0 + chunk);
}
// LDS of a decode unit: the four waves' V tiles, then the merge of their results.
template <int D>
constexpr int decode_smem() {
  return 4 * kTileTokens * D * 2 > 4 * 16 * (D + 2) * 4 ? 4 * kTileTokens * D * 2 : 4 * 16 * (D + 2) * 4;
}

// One decode unit: split j of request b for kv head kvh, as above, for the launch's unit `unit`.
// With one split it writes the output; otherwise an fp32 partial output and its
// log2-sum-exp to rows (b * splits + j) * Hq + head of part_o / part_lse.
template <int D, bool FIRST>
__device__ __forceinline__ void decode_unit(
    char* smem, int32_t* ptab, int unit, const uint16_t* __restrict__ q, int64_t q_ts, int64_t q_hs, const PagedKV& kv,
    int B, int G, int Hq, float scale_log2, int splits, int window_left, int first,
    uint16_t* __restrict__ out, int64_t o_ts, int64_t o_hs, float* __restrict__ part_o, float* __restrict__ part_lse,
    const float* __restrict__ sinks, float* __restrict__ lse) {
  using W = WaveAttn<D>;
  constexpr int kVtile = kTileTokens * D;  // elements of one wave's V tile
  static_assert(decode_smem<D>() >= kRankMax * 4, "the ranked lengths fit in the V tiles' LDS");
  __shared__ int32_t rank_pick[3];

  const int Hkv = Hq / G;
  const int per = splits * Hkv;
  const int r = unit / per, rem = unit - r * per;
  const int j = rem / Hkv, kvh = rem - j * Hkv;
  int b = r, kv_len, page0;
  if (B <= kRankMax) {
    // the LDS holds the lengths until the first page window's barrier
    b = request_of_rank(kv, B, window_left, first, r, reinterpret_cast<int32_t*>(smem), rank_pick, kv_len, page0);
  } else {
    kv_len = kv_length(kv, b);
    page0 = kv.indptr[b];
  }
  const int slot = b * splits + j;
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  // sliding window: the query (position kv_len - 1) sees positions >= kv_len - 1 - window_left
  const int ws = window_start(kv_len, window_left);
  KeptMap km;
  int kv0, kv1;
  if constexpr (FIRST) {  // kv0..kv1 count visible positions
    km.kept = min(first, ws);
    km.skip = ws - km.kept;
    split_range(kv_len - km.skip, splits, j, kv0, kv1);
  } else {
    split_range(kv_len - ws, splits, j, kv0, kv1);
  }
  const bool whole = splits == 1;
  if (!whole && kv0 >= kv1) return;  // an empty split: the merge does not read it
  if constexpr (!FIRST) {
    kv0 += ws;
    kv1 += ws;
  }

  W st;
  st.init();
  // query rows of this kv head: heads kvh*G + n (rows n >= G are zero)
  {
    const bool valid = n < G;
    const uint16_t* qp = q + (int64_t)b * q_ts + (int64_t)(kvh * G + (valid ? n : 0)) * q_hs;
    #pragma unroll
    for (int s = 0; s < W::NS; ++s) {
      const u32x4_t z = {0u, 0u, 0u, 0u};
      st.qb[s] = valid ? ld16v(qp + 8 * (4 * s + g)) : z;
    }
  }
  uint16_t* vt = reinterpret_cast<uint16_t*>(smem) + w * kVtile;
  // kv tokens per page window: the pages any such run spans fit in kPageWin (two runs' where FIRST)
  const int win = max(kTileTokens, (kPageWin - (FIRST ? 4 : 2)) * kv.page_size / kTileTokens * kTileTokens);
  for (int wt0 = kv0; wt0 < kv1; wt0 += win) {
    const int wt1 = min(kv1, wt0 + win);
    int lp0;
    if constexpr (FIRST) {
      const int a1 = min(wt1, km.kept), b0 = max(wt0, km.kept) + km.skip, b1 = wt1 + km.skip;
      const int lpb = (int)kv.pdiv.div((uint32_t)b0);
      const int nb = b0 < b1 ? (int)kv.pdiv.div((uint32_t)(b1 - 1)) - lpb + 1 : 0;
      lp0 = wt0 < a1 ? (int)kv.pdiv.div((uint32_t)wt0) : lpb;
      const int na = wt0 < a1 ? (int)kv.pdiv.div((uint32_t)(a1 - 1)) - lp0 + 1 : 0;
      km.gap = lpb - na - lp0;
      __syncthreads();  // the previous window's lookups are done
      for (int i = threadIdx.x; i < na + nb; i += 256) ptab[i] = kv.indices[page0 + lp0 + i + (i < na ? 0 : km.gap)];
    } else {
      lp0 = (int)kv.pdiv.div((uint32_t)wt0);
      const int npg = (int)kv.pdiv.div((uint32_t)(wt1 - 1)) - lp0 + 1;
      __syncthreads();  // the previous window's lookups are done
      for (int i = threadIdx.x; i < npg; i += 256) ptab[i] = kv.indices[page0 + lp0 + i];
    }
    __syncthreads();
    // Each wave takes every fourth tile. Two tile slots alternate (no register copies, which
    // would force a wait on the in-flight loads): the next tile's loads are issued before the
    // current tile's MFMA/softmax work, so HBM latency overlaps compute.
    int t0 = wt0 + kTileTokens * w;
    if (t0 < wt1) {
      // Two K register slots alternate (no copies, which would force waits on loads in
      // flight); V has one LDS tile. Each step: wait for the current tile's loads, move its V
      // from LDS into registers, issue the next tile's loads (V into the now free LDS tile),
      // then run the current tile's MFMA/softmax work while they stream in.
      KVTile<D, FIRST> ta, tb;
      u32x4_t vb[W::NB];
      ta.load(kv, ptab, lp0, km, t0, wt1, kvh, lane, vt);
      for (;;) {
        wait_vmcnt<0>();
        st.read_v(vt, lane, vb);
        wait_lgkmcnt0();
        const bool more_b = t0 + 4 * kTileTokens < wt1;
        if (more_b) tb.load(kv, ptab, lp0, km, t0 + 4 * kTileTokens, wt1, kvh, lane, vt);
        st.tile(ta.ka, ta.vmask(lane), vb, scale_log2, lane);
        if (!more_b) break;
        t0 += 4 * kTileTokens;
        wait_vmcnt<0>();
        st.read_v(vt, lane, vb);
        wait_lgkmcnt0();
        const bool more_a = t0 + 4 * kTileTokens < wt1;
        if (more_a) ta.load(kv, ptab, lp0, km, t0 + 4 * kTileTokens, wt1, kvh, lane, vt);
        st.tile(tb.ka, tb.vmask(lane), vb, scale_log2, lane);
        if (!more_a) break;
        t0 += 4 * kTileTokens;
      }
    }
  }
  const float lsum = st.row_sum(lane);

  // merge the four waves through LDS: m[4][16], l[4][16], o[4][16][D] (fp32)
  __syncthreads();
  float* ms = reinterpret_cast<float*>(smem);
  float* ls = ms + 4 * 16;
  float* os = ls + 4 * 16;
  if (g == 0) { ms[w * 16 + n] = st.m; ls[w * 16 + n] = lsum; }
  #pragma unroll
  for (int nb = 0; nb < W::NB; ++nb)
    #pragma unroll
    for (int i = 0; i < 4; ++i) os[(w * 16 + 4 * g + i) * D + 16 * nb + n] = st.o[nb][i];
  __syncthreads();
  constexpr int CH = D / 8;
  for (int u = threadIdx.x; u < G * CH; u += 256) {
    const int row = u / CH, c = u % CH;
    float M = -INFINITY;
    #pragma unroll
    for (int ww = 0; ww < 4; ++ww) M = fmaxf(M, ms[ww * 16 + row]);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
    if (M != -INFINITY) {
      #pragma unroll
      for (int ww = 0; ww < 4; ++ww) {
        const float f = fast_exp2(ms[ww * 16 + row] - M);
        L += ls[ww * 16 + row] * f;
        const float* src = os + (ww * 16 + row) * D + 8 * c;
        #pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += src[e] * f;
      }
    }
    const int hq = kvh * G + row;
    // the sink joins the denominator once, after the splits are merged
    if (whole && M != -INFINITY) L += sink_mass(sinks, hq, M);
    const float inv = L > 0.f ? 1.f / L : 0.f;
    #pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= inv;
    if (whole) {
      if (lse && c == 0) lse[(int64_t)b * Hq + hq] = row_lse(L, M);
      st16(out + (int64_t)b * o_ts + (int64_t)hq * o_hs + 8 * c, pack8(acc));
    } else {
      float* dst = part_o + ((int64_t)slot * Hq + hq) * D + 8 * c;
      #pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = acc[e];
      if (c == 0) part_lse[(int64_t)slot * Hq + hq] = L > 0.f ? M + log2f(L) : -INFINITY;
    }
  }
}

// Sums partial results of 64 / (D/8) output rows, one row per group of D/8 lanes, each lane 8 dims;
// the four waves of the work group take every fourth partial, KB of them loaded at once before the
// first is used, and meet in LDS. Partial s of the lane's row is row r = row(s) of the results: its 8 dims
// po[r * D .. +8) (fp32, normalised) and log2-sum-exp pl[r]. Every thread of the
// work group calls it; wave 0 gets the row's weighted sum (acc, NaN if a partial is), weight sum (L)
// and maximum (M, -inf if no partial saw anything) of partials [0, ns); there is memory for room >= max(ns, 1).
// Bound: load latency. The partials are read in ns / 32 rounds of independent loads, and only the
// splits that hold tokens: 3.0 us for one request of 1,000 tokens planned at 64 splits (32 heads,
// 8 splits hold tokens) and 5.3 us for three of 16-32k tokens at 43; one wave reading every split
// in turn took 27.9 us at either.
template <int D, int KB, typename Row>
__device__ __forceinline__ void merge_partials(const float* __restrict__ po, const float* __restrict__ pl, Row row,
                                               int ns, int room, float (&acc)[8], float& L, float& M) {
  constexpr int CH = D / 8;
  __shared__ float sm[4][64][10];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  M = -INFINITY;
  L = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  // The first round's loads do not wait for ns (which may itself be in flight): partials [ns, room)
  // are memory, but hold nothing, and count as zero.
  for (int s0 = w; s0 == w || s0 < ns; s0 += 4 * KB) {
    const int top = (s0 == w ? room : ns) - 1;
    float4 a[KB], b[KB];
    float ls[KB];
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const int64_t r = row(min(s0 + 4 * k, top));
      ls[k] = pl[r];
      a[k] = *reinterpret_cast<const float4*>(po + r * D);
      b[k] = *reinterpret_cast<const float4*>(po + r * D + 4);
    }
    float mx = M;
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      if (s0 + 4 * k >= ns) {
        ls[k] = -INFINITY;
        a[k] = b[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      mx = fmaxf(mx, ls[k]);
    }
    // with nothing seen yet every weight is 0; a NaN among the partials still has to reach the sum
    const float ref = mx == -INFINITY ? 0.f : mx;
    const float f0 = fast_exp2(M - ref);
    L *= f0;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= f0;
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const float f = fast_exp2(ls[k] - ref);
      L += f;
      const float v[8] = {a[k].x, a[k].y, a[k].z, a[k].w, b[k].x, b[k].y, b[k].z, b[k].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(v[e], f, acc[e]);
    }
    M = mx;
  }
  static_assert(64 % CH == 0, "whole rows per wave");
  if (w > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sm[w][lane][e] = acc[e];
    sm[w][lane][8] = L;
    sm[w][lane][9] = M;
  }
  __syncthreads();
  if (w == 0) {
    float mx = M;
#pragma unroll
    for (int ww = 1; ww < 4; ++ww) mx = fmaxf(mx, sm[ww][lane][9]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    const float f0 = fast_exp2(M - ref);
    L *= f0;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= f0;
#pragma unroll
    for (int ww = 1; ww < 4; ++ww) {
      const float f = fast_exp2(sm[ww][lane][9] - ref);
      L = fmaf(sm[ww][lane][8], f, L);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(sm[ww][lane][e], f, acc[e]);
    }
    M = mx;
  }
}

// ------------------------------------------------------------------------------ prefill
// Work item: request b, first packed query row row0 (row R = query token R / G, head R % G of
// the kv head's group). A work group of four waves owns kPrefillRows = 128 rows, 32 per wave, and
// streams the request's kv tokens in tiles of prefill_tile<D> tokens; the four waves load each K
// and V tile cooperatively into registers (two tiles ahead) and then into LDS (chunk-swizzled,
// double-buffered).
// Visibility: mode 0 every cached position, 1 causal (t <= kv_len - qo_len + i), 2 the custom
// mask, bit-packed by attn_mask_kernel: query token i of request b reads 32-bit word
// w (kv positions 32w..32w+31) at packed + word_off[b] + i * ceil(kv_len / 32) + w.
//
// The products run on v_mfma_f32_32x32x16_bf16, the output transposed:
//   S^T = K Q^T    A = 32 kv tokens x 16 dims (lane (t, kg): token t's dims 8(2s+kg)..+8 at
//                  step s, from LDS), B = 32 query rows (lane (r, kg): row r, the same dims)
//   O^T = V^T P^T  A = 32 dims x 16 tokens (two transpose reads of 4 V rows each),
//                  B = P^T: lane (r, kg) holds row r's probabilities of tokens
//                  16j + 8(e/4) + 4kg + e%4, exactly 8 consecutive registers of S^T's C layout
// so every lane owns one query row r = lane % 32 in both products: its running max, sum and
// rescale factor are its own (one exchange with lane ^ 32 for the max), and no factor has to be
// broadcast to other lanes.
//
// What bounds it (rocprofv3 counters, 4 x 4000 causal tokens, shares of a SIMD's cycles). Head dim 64:
// VALU 66%, MFMA 32%, LDS 12%; waves wait 26% of their time: a tile's softmax costs twice its MFMAs,
// and the two hardly overlap. Head dim 256: MFMA 22%, VALU 30%, LDS 8%: one wave fits a SIMD and nothing
// runs under its softmax and waits. No bank conflicts at either. Work groups of four 32-row waves in
// 64-token tiles, each MFMA's V operands read a step ahead, against the four 2 x 16-row waves on
// 16x16x32 MFMAs in 32-token tiles before (4 x 4000 causal tokens, 8 kv heads): head dim 64, 64 heads
// 1,331 -> 690 us (760 TFLOP/s); head dim 256, 16 heads (one 16-row tile per wave before) 1,852 -> 934
// us (562 TFLOP/s).
constexpr int kPrefillRows = 128;
// kv tokens per tile: 64, or 32 at head dim 256, whose accumulators fill the registers
template <int D>
constexpr int prefill_tile() { return D == 256 ? 32 : 64; }
// work groups per CU the registers are budgeted for (at head dim 64 three fit: 164 registers, 34 KiB)
template <int D>
constexpr int prefill_groups() { return D == 256 ? 1 : 2; }
constexpr int kPlanHeader = 16;  // plan words before the items: [0] items, [1] batch, [2] rows per item
// Plan word 2: rows per item; head dim 256 sets another value, so that its plans and those of
// the other head dims do not drive each other's kernels.
constexpr int plan_rows_word(int64_t D) { return D == 256 ? kPrefillRows | (1 << 16) : kPrefillRows; }
constexpr int kPlanChunkWord = 5;  // kv tokens per piece of a split item
// Plan words the head-dim-128 kernel uses as counters: the next unit of each XCD's queue, and
// the work groups that have finished (the last one sets all nine back to zero).
constexpr int kPlanQueueWord = 8, kPlanDoneWord = 7;
// words per work item: request b, first packed row, the request's q0 (first query token),
// qo_len, kv_len and first page-table slot, so the kernels' prologue reads one 32-byte item
// instead of chasing b through qo_indptr / kv_indptr / kv_last_page_len; then, for an item split
// over its kv range, the piece's index and 1 + its partial-result slot (0: not split)
constexpr int kPlanItemWords = 8;
// words per merge entry of a split plan: first packed row, q0, qo_len, first slot, pieces, and
// kMergeTag + the plan's rows word
constexpr int kPlanMergeWords = 8;
constexpr int kMergeTag = 0x4d520000;

// XCD-aware order of the prefill grid: work groups are dispatched round-robin over the 8 XCDs
// (id mod 8), each with its own L2, so XCD x takes the contiguous run [x * per, (x + 1) * per) of
// the (kv head, item) units. The plan lists each request's items together, so the work groups an
// XCD runs at one time mostly read the same request's K/V prefix through one L2. Returns the
// unit's number, or -1 for the padding work groups past the last unit.
__device__ __forceinline__ int prefill_unit(int units) {
  const int per = (units + 7) / 8;
  const int u = (int)(blockIdx.x & 7u) * per + (int)(blockIdx.x >> 3);
  return u < units ? u : -1;
}

// attn_mask_kernel marks a query token whose mask row is exactly causal (positions
// 0..kv_len - qo_len + i, nothing else) with this bit of its extent.
constexpr int kExtentCausal = 1 << 30;

// Custom-mask prologue: the furthest position any of the work group's nrows rows (from row0) can
// see, and whether every one of those rows' masks is exactly causal (then the causal path serves
// them without reading mask words). Every thread of the work group calls it.
__device__ __forceinline__ void mask_rows_extent(const int32_t* __restrict__ extent, int q0, int row0, int rows,
                                                 int G, int nrows, int& ext, bool& causal) {
  __shared__ int s_ext, s_mixed;
  const int zero = opaque_v(0);  // a constant pair would be kept in registers over the caller's loop
  if (threadIdx.x == 0) { s_ext = zero; s_mixed = zero; }
  __syncthreads();
  const int r = row0 + (int)threadIdx.x;
  if ((int)threadIdx.x < nrows && r < rows) {
    const int e = extent[q0 + r / G];
    atomicMax(&s_ext, e & ~kExtentCausal);
    if (!(e & kExtentCausal)) atomicOr(&s_mixed, 1);
  }
  __syncthreads();
  ext = s_ext;
  causal = s_mixed == 0;
}
typedef float f32x16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16_t mfma_32x32x16(const u32x4_t& a, const u32x4_t& b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Scheduling group: the next `n` instructions of class `mask` (0x8 MFMA, 0x100 LDS read).
#define sched_group(mask, n) __builtin_amdgcn_sched_group_barrier((mask), (n), 0)

// V-row swizzle for this kernel's transpose reads: one read takes 4 consecutive rows x 4 chunks
// (64 bytes) per half-wave, and the 4 rows must fall on different 64-byte bank groups: rows of
// 256 bytes or more XOR chunk bits 2-3 with r mod 4, rows of 128 bytes chunk bit 2 with bit 1 of r.
template <int D>
__device__ __forceinline__ int v32_swizzle(int r) { return D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2; }

// The n lowest bits set (n <= 0: none, n >= 64: all).
__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// v of lane ^ 32
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

// Partial results of a split item (piece slot s, kv head h): 128 rows of D fp32 outputs
// (normalised) at part_o + (s * n_kv_heads + h) * 128 * D and their log2-sum-exps at
// part_lse + (s * n_kv_heads + h) * 128; attn_prefill_merge_kernel combines an item's pieces.
// part_row: the row of part_o / part_lse that the item's first query row's partial result goes to; < 0:
// the item is whole and writes the output. off, chunk: the item's kv range is [off, off + chunk) of the
// positions its rows can see (whole items: 0 and any chunk >= their number). With FIRST those are the
// kept first tokens, padded to whole tiles, followed by the window's. (18082 tokens in windows of 1024 + 4, 32
// heads of 128: 353-376 us, 695-740 TFLOP/s over the visible pairs, as the causal prefill of long requests; both
// ranges' tiles in one loop, with a choice of range per tile, take as long.)
// JOINT: pre_len tokens of another run of pages (pre_indices from pre_page0 on), which all rows see, come before
// the item's own kv range.
struct PrefillItem {
  int b, row0, q0, qo_len, kv_len, page0, off, chunk;
  int64_t part_row;
  const int32_t* pre_indices = nullptr;
  int pre_page0 = 0, pre_len = 0;
};
template <int D>
constexpr int prefill_smem() { return 2 * 2 * prefill_tile<D>() * D * 2; }

template <int D, bool FIRST, bool JOINT = false>
__device__ __forceinline__ void prefill_item(
    char* smem, int32_t* ptab, const PrefillItem& it, const uint16_t* __restrict__ q, int64_t q_ts, int64_t q_hs,
    const PagedKV& kv, int G, int n_kv_heads, int kvh, float scale_log2, int mode_in, int window_left, int first_in,
    const uint32_t* __restrict__ packed, const int64_t* __restrict__ word_off, const int32_t* __restrict__ extent,
    uint16_t* __restrict__ out, int64_t o_ts, int64_t o_hs, const float* __restrict__ sinks,
    float* __restrict__ part_o, float* __restrict__ part_lse, float* __restrict__ lse) {
  constexpr int TT = prefill_tile<D>(), H2 = TT / 32;  // tile tokens, 32-token halves
  constexpr int NS = D / 16;  // QK k-steps
  constexpr int NB = D / 32;  // 32-dim output blocks
  constexpr int CH = D / 8, RPI = 64 / CH;  // 16-byte chunks per row, rows per load instruction
  constexpr int NT = 256;
  constexpr int TILE = TT * D;
  constexpr int WR = TT / 4;    // rows of each K / V tile one wave loads
  constexpr int NL = WR / RPI;  // load instructions for them
  static_assert(NL >= 1 && WR % RPI == 0, "tile rows per wave");
  __shared__ int window_bad;

  const int b = it.b, row0 = it.row0, q0 = it.q0, qo_len = it.qo_len, kv_len = it.kv_len, page0 = it.page0;
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  const int r32 = lane & 31, kg = lane >> 5;
  const int rows = qo_len * G;
  int mode = mode_in, mext = 0;  // a custom mask that is causal for all the rows: the causal path
  if (mode_in == 2) {
    bool causal;
    mask_rows_extent(extent, q0, row0, rows, G, kPrefillRows, mext, causal);
    mode = uniform(causal ? 1 : 2);  // wave-uniform (a scalar register), like the argument
    mext = uniform(mext);
  }

  // this lane's query row
  const int R = row0 + 32 * w + r32;
  const bool valid = R < rows;
  const int row_tok = valid ? R / G : -1;
  // the positions a row (its query token; -1: no row) sees: lo..lim (and the mask)
  const auto row_lim = [&](int t) { return t < 0 ? -1 : mode == 1 ? kv_len - qo_len + t : kv_len - 1; };
  const auto row_lo = [&](int t) { return window_left >= 0 ? kv_len - qo_len + t - window_left : 0; };
  u32x4_t qb[NS];
  {
    const int tok = max(row_tok, 0), hg = valid ? R - tok * G : 0;
    const uint16_t* qp = q + (int64_t)(q0 + tok) * q_ts + (int64_t)(kvh * G + hg) * q_hs;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const u32x4_t z = {0u, 0u, 0u, 0u};
      qb[s] = valid ? ld16v(qp + 8 * (2 * s + kg)) : z;
    }
  }
  f32x16_t o[NB];
#pragma unroll
  for (int bb = 0; bb < NB; ++bb)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[bb][i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  // kv positions any row of this work group can see (mode 2: the furthest set mask bit of its
  // rows' query tokens, from attn_mask_kernel); a sliding window hides positions before
  // its first row's window (tiles start 32-aligned so mask words line up)
  const int last_row = min(rows, row0 + kPrefillRows) - 1;
  int kv_end = mode == 1 ? min(kv_len, kv_len - qo_len + last_row / G + 1) : kv_len;
  if (mode == 2) kv_end = min(kv_len, mext);
  int kv_begin = window_left >= 0 ? max(0, kv_len - qo_len + row0 / G - window_left) & ~31 : 0;
  // FIRST: kept first tokens that lie before every row's window are a range of their own, [a0, a1); where
  // they reach it the walk starts at 0, and rows see t < first beside their window
  int a0 = 0, a1 = 0, first = 0, lo_all = 0;
  if constexpr (FIRST) {
    lo_all = window_left >= 0 ? kv_len - qo_len + row0 / G - window_left : 0;  // no row sees [first_in, lo_all)
    if (kv_begin > 0 && first_in < kv_begin) {
      a1 = min(first_in, kv_end);
    } else {
      kv_begin = 0;
      first = first_in;
    }
    // (a1 is padded to whole tiles in the count of positions, so that the window's pieces start tile-aligned)
    const int64_t pad = (a1 + 63) & ~63, end = (int64_t)it.off + it.chunk;
    a0 = min(it.off, a1);
    a1 = (int)min(end, (int64_t)a1);
    kv_end = (int)min((int64_t)kv_end, kv_begin + max(end, pad) - pad);
    kv_begin += (int)(max((int64_t)it.off, pad) - pad);
  } else {
    kv_begin += it.off;
    kv_end = (int)min((int64_t)kv_end, (int64_t)kv_begin + it.chunk);
    if constexpr (JOINT) a1 = it.pre_len;
  }
  const int nw = (kv_len + 31) / 32;
  const uint32_t* mword = mode == 2 ? packed + word_off[b] + (int64_t)max(row_tok, 0) * nw : nullptr;
  // uniform bounds of the wave's rows: tiles inside [wave_lo, wave_lim] need no per-element test,
  // tiles past wave_hi are seen by none of them
  // (a row's limits grow with its token, so the wave's first and last rows give them)
  const int wr0 = row0 + 32 * w, wr1 = min(wr0 + 31, rows - 1);
  const bool wave_rows = wr0 < rows;
  const int wtok0 = wave_rows ? wr0 / G : -1, wtok1 = wave_rows ? wr1 / G : -1;
  const int wave_lim = wave_rows ? row_lim(wtok0) : 0x7fffffff, wave_hi = row_lim(wtok1);
  const int wave_lo = wave_rows ? row_lo(wtok1) : 0;

  uint16_t* kt = reinterpret_cast<uint16_t*>(smem);  // [2 buffers][K, V][TT][D]
  // A tile in flight in registers: this wave's rows WR*w.. of K and V (chunk-swizzled as they will
  // sit in LDS), and the mask words of this lane's row.
  struct Slot { u32x4_t k[NL], v[NL]; uint32_t mw[H2]; };
  // Pages of at least WR tokens (a multiple of it) hold the wave's rows of a tile together: one
  // uniform page lookup and a scalar base address per tile. Load i's rows are RPI*i further on, a
  // scalar too, and its lanes' chunks differ from load 0's by XORs of constants, with cache rows
  // that are whole multiples of D elements apart.
  const bool one_page = kv.page_size % WR == 0 && kv.slot_stride % D == 0 && kv.slot_stride < (1 << 26);
  const auto k_xor = [](int i) { return (uint32_t)(D == 256 ? 32 * i : 64 * i); };  // bytes
  const auto v_xor = [](int i) { return (uint32_t)(D == 256 ? 128 * (i & 1) : 0); };
  uint32_t koff, voff;
  {
    const int rl = lane / CH, r = WR * w + rl;
    koff = 2u * ((uint32_t)rl * (uint32_t)kv.slot_stride + 8u * ((lane % CH) ^ chunk_swizzle<D>(r)));
    voff = 2u * ((uint32_t)rl * (uint32_t)kv.slot_stride + 8u * ((lane % CH) ^ v32_swizzle<D>(r)));
  }
  const uint32_t step = 2u * RPI * (uint32_t)kv.slot_stride;
  // LDS byte offsets of this lane's operands in a tile: k step 0 of half 0 (step s: ^ 32s), and V
  // block 0 of the first transpose read (block bb: ^ 64bb). Transpose-read source lanes: group
  // G16 = lane / 16 reads rows 16j + 8h + 4kg + (lane%16)/4 (h: first or second 4 tokens), dims
  // 32bb + 16(G16%2) + 4(lane%4)
  uint32_t kl0, vl0;
  {
    kl0 = 2u * r32 * D + 16u * (kg ^ chunk_swizzle<D>(r32));
    const int r = 4 * kg + ((lane >> 2) & 3), dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    vl0 = 2u * (TILE + r * D + 8 * ((dim >> 3) ^ v32_swizzle<D>(r)) + (dim & 7));
  }
  const int win = max(TT, (kPageWin - 2) * kv.page_size / TT * TT);
  // the range of the kept first tokens (FIRST), then the window's
  bool kept = (FIRST || JOINT) && a0 < a1;
  int seg_end = kept ? a1 : kv_end;
  for (int wt0 = kept ? a0 : kv_begin; wt0 < seg_end;) {
    const int wt1 = min(seg_end, wt0 + win);
    const int lp0 = (int)kv.pdiv.div((uint32_t)wt0);
    const int npg = (int)kv.pdiv.div((uint32_t)(wt1 - 1)) - lp0 + 1;
    const int ntiles = (wt1 - wt0 + TT - 1) / TT;
    if (threadIdx.x == 0) window_bad = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < npg; i += NT) {
      const int pg = JOINT && kept ? it.pre_indices[it.pre_page0 + lp0 + i] : kv.indices[page0 + lp0 + i];
      ptab[i] = pg;
      if ((unsigned)pg >= (unsigned)kv.num_pages) window_bad = 1;
    }
    __syncthreads();
    const bool all_pages_ok = uniform(window_bad) == 0;
    // the wave's first token of a tile (in the last tile at most the last whole group of WR rows)
    const auto wave_tok = [&](int tile) { return min(wt0 + tile * TT + WR * w, (wt1 - 1) & ~(WR - 1)); };
    int next_page = one_page ? ptab[(int)kv.pdiv.div((uint32_t)wave_tok(0)) - lp0] : 0;
    // Tiles are loaded in order, 0, 1, ...; the next tile's page id is read from LDS one tile ahead.
    auto gload = [&](Slot& sl, int tile) {
      const int t0 = wt0 + tile * TT;
      if (one_page) {
        const int tb = wave_tok(tile);
        const int slot0 = tb - (int)kv.pdiv.div((uint32_t)tb) * kv.page_size;
        const int page = uniform(next_page);
        next_page = ptab[(int)kv.pdiv.div((uint32_t)wave_tok(tile + 1)) - lp0];
        const uint32_t pg = (unsigned)page < (unsigned)kv.num_pages ? (uint32_t)page : 0u;
        const int64_t base = (int64_t)pg * kv.page_stride + (int64_t)slot0 * kv.slot_stride + (int64_t)kvh * kv.head_stride;
        // rows past the end lie behind the buffers' and read as zero (their probability is 0)
        const int bytes = 2 * ((min(WR, wt1 - tb) - 1) * (int)kv.slot_stride + D);
        const auto kb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(kv.k + base), 0, bytes, 0x00020000);
        const auto vb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(kv.v + base), 0, bytes, 0x00020000);
        const uint32_t ko = (uint32_t)opaque_v((int)koff);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          sl.k[i] = __builtin_amdgcn_raw_buffer_load_b128(kb, (int)((ko ^ k_xor(i)) + i * step), 0, 0);
          sl.v[i] = __builtin_amdgcn_raw_buffer_load_b128(vb, (int)((voff ^ v_xor(i)) + i * step), 0, 0);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int r = WR * w + RPI * i + lane / CH;
          bool ok;
          const uint64_t off = kv_offset_lds(kv, ptab, lp0, min(t0 + r, wt1 - 1), kvh, ok);
          sl.k[i] = ld16v(kv.k + off + 8 * ((lane % CH) ^ chunk_swizzle<D>(r)));
          sl.v[i] = ld16v(kv.v + off + 8 * ((lane % CH) ^ v32_swizzle<D>(r)));
        }
      }
      if (mode == 2) {
#pragma unroll
        for (int h = 0; h < H2; ++h) sl.mw[h] = mword[min((t0 >> 5) + h, nw - 1)];
      }
    };
    uint32_t mcur[H2];  // the mask words of the tile being computed
#pragma unroll
    for (int h = 0; h < H2; ++h) mcur[h] = 0;
    auto lwrite = [&](Slot& sl, int tile) {
      uint16_t* kd = kt + (tile & 1) * 2 * TILE;
      if constexpr (FIRST) {  // rows between the kept range and every window: a NaN there is nobody's
        const int t0 = wt0 + tile * TT;
        if (!kept && t0 < lo_all) {
#pragma unroll
          for (int i = 0; i < NL; ++i) {
            const int t = t0 + WR * w + RPI * i + lane / CH;
            if (t < lo_all && t >= first) sl.v[i] = u32x4_t{0u, 0u, 0u, 0u};
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        *reinterpret_cast<u32x4_t*>(kd + (WR * w + RPI * i) * D + 8 * lane) = sl.k[i];
        *reinterpret_cast<u32x4_t*>(kd + TILE + (WR * w + RPI * i) * D + 8 * lane) = sl.v[i];
      }
      if (mode == 2) {
#pragma unroll
        for (int h = 0; h < H2; ++h) mcur[h] = sl.mw[h];
      }
    };
    auto compute = [&](int tile) {
      const int t0 = wt0 + tile * TT;
      if (JOINT && kept ? !wave_rows : t0 > wave_hi) return;  // no row of the wave sees the tile
      const uint32_t buf = (tile & 1) * 4 * TILE;  // bytes
      const uint32_t kl = (uint32_t)opaque_v((int)(buf + kl0));
      // S^T: token 32h + r32 of the tile against this lane group's 32 rows
      f32x16_t sacc[H2];
#pragma unroll
      for (int h = 0; h < H2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) sacc[h][i] = 0.f;
      {
        // K operands read four ahead of the MFMAs. The schedule is pinned: left to itself the
        // compiler reads two ahead and exposes the LDS latency several times per tile.
        u32x4_t kr[NS][H2];
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int h = 0; h < H2; ++h)
            kr[s][h] = *reinterpret_cast<const u32x4_t*>(smem + ((kl ^ (32 * s)) + 64 * h * D));
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int h = 0; h < H2; ++h) sacc[h] = mfma_32x32x16(kr[s][h], qb[s], sacc[h]);
        sched_group(0x100, 4);
#pragma unroll
        for (int s = 0; s < NS * H2 - 4; ++s) { sched_group(0x008, 1); sched_group(0x100, 1); }
        sched_group(0x008, 4);
      }
      // V operands, read 16 tokens ahead of their MFMAs (the first ones here, over the softmax)
      const uint32_t vl = (uint32_t)opaque_v((int)(buf + vl0));
      u32x4_t va[2][NB];
      const auto read_v = [&](int j) {
#pragma unroll
        for (int bb = 0; bb < NB; ++bb) {
          uint2 hv[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            hv[h] = lds_read_tr16(reinterpret_cast<const uint16_t*>(smem + ((vl ^ (64 * bb)) + (32 * j + 16 * h) * D)));
          va[j & 1][bb] = u32x4_t{hv[0].x, hv[0].y, hv[1].x, hv[1].y};
        }
      };
      read_v(0);
      // visibility of token tt(i) = 32h + 8(i/4) + 4kg + i%4 for this lane's row: mask bits by
      // shifts, then the per-element bounds only in tiles that cross a row's limit or window start
      uint32_t vis[H2];
#pragma unroll
      for (int h = 0; h < H2; ++h) vis[h] = 0xffffu;
      if (mode == 2) {
#pragma unroll
        for (int h = 0; h < H2; ++h) {
          vis[h] = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) vis[h] |= ((mcur[h] >> (8 * c + 4 * kg)) & 15u) << (4 * c);
        }
      }
      if (!all_pages_ok || (JOINT && kept ? t0 + TT > wt1 : t0 + TT - 1 > wave_lim || t0 < wave_lo)) {
        uint64_t tv = ~0ull;
        if (!all_pages_ok) {
          bool pok = false;
          if (lane < TT && t0 + lane < wt1) kv_offset_lds(kv, ptab, lp0, t0 + lane, kvh, pok);
          tv = __builtin_amdgcn_ballot_w64(pok);
        }
        const int hi = (JOINT && kept ? wt1 - 1 : row_lim(row_tok)) - t0 - 4 * kg;
        tv >>= 4 * kg;
        if constexpr (FIRST || JOINT) {  // as token bits: [lo, hi] of the window, and the kept ones
          if constexpr (FIRST) {
            const int lo = (kept ? 0x7fffffff : row_lo(row_tok)) - t0 - 4 * kg;
            tv &= (low_bits(hi + 1) & ~low_bits(lo)) | low_bits(min(hi + 1, (kept ? wt1 : first) - t0 - 4 * kg));
          } else {
            tv &= low_bits(hi + 1);
          }
#pragma unroll
          for (int h = 0; h < H2; ++h) {
            uint32_t seen = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) seen |= (uint32_t)((tv >> (32 * h + 8 * c)) & 15u) << (4 * c);
            vis[h] &= seen;
          }
        } else {
          // compared against the constants 32h + 8(i/4) + i%4, so that nothing per element stays live
          const int lo = row_lo(row_tok) - t0 - 4 * kg;
#pragma unroll
          for (int h = 0; h < H2; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int c = 32 * h + 8 * (i >> 2) + (i & 3);
              if (!(c <= hi && c >= lo && ((tv >> c) & 1ull))) vis[h] &= ~(1u << i);
            }
        }
      }
      // Scores stay raw (q.k) until the exponent, where one fma applies the scale: the row maximum
      // is taken over raw scores, negated when the scale is negative (a uniform branch), with
      // hidden entries set to the raw value that scales to -inf (the scale is never 0 here).
      const bool neg = scale_log2 < 0.f;
      bool seen_all = true;
#pragma unroll
      for (int h = 0; h < H2; ++h) seen_all = seen_all && vis[h] == 0xffffu;
      if (__builtin_amdgcn_ballot_w64(!seen_all) != 0) {
        const float hidden = neg ? INFINITY : -INFINITY;
#pragma unroll
        for (int h = 0; h < H2; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) sacc[h][i] = ((vis[h] >> i) & 1u) ? sacc[h][i] : hidden;
      }
      float mx = -INFINITY;
      if (!neg) {
        // (three-operand maxima in two chains; a tree of two-operand ones takes twice the instructions, since the
        // products' results are quieted first)
        float mh[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 16 * H2; i += 4)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            mh[c] = fmaxf(fmaxf(mh[c], sacc[i >> 4][(i & 15) + 2 * c]), sacc[i >> 4][(i & 15) + 2 * c + 1]);
        mx = fmaxf(mh[0], mh[1]);
      } else {
#pragma unroll
        for (int h = 0; h < H2; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, -sacc[h][i]);
      }
      mx *= fabsf(scale_log2);
      // lazy maximum (kLazyMax); the row's other half of the tokens is looked at only where one half exceeds it
      if (__builtin_amdgcn_ballot_w64(mx > m_run + kLazyMax) != 0) {
        mx = fmaxf(mx, other_half(mx));
        const bool grow = mx > m_run + kLazyMax;
        const float alpha = grow ? fast_exp2(m_run - mx) : 1.f;
        if (grow) m_run = mx;
        l_run *= alpha;
#pragma unroll
        for (int bb = 0; bb < NB; ++bb)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[bb][i] *= alpha;
      }
      const float m_use = m_run == -INFINITY ? 0.f : m_run;
      // O^T += V^T P^T, 16 tokens at a time. Step j's MFMAs, the next step's V reads and its
      // exponentials are independent and stay together, the reads pinned before the MFMAs: left to
      // itself the compiler reads each V operand right before its MFMA and waits for it there. (The
      // exponentials are the compiler's to place: each pinned behind an MFMA is 2-4% slower.)
      float ps[2 * H2];
      u32x4_t pb[2];
      const auto probs = [&](int j) {
        float sc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[i] = fast_exp2(fmaf(sacc[j >> 1][8 * (j & 1) + i], scale_log2, -m_use));
        // the row's partial sum as a tree (a chain of dependent adds sat on the critical path)
        ps[j] = ((sc[0] + sc[1]) + (sc[2] + sc[3])) + ((sc[4] + sc[5]) + (sc[6] + sc[7]));
        pb[j & 1] = u32x4_t{pack_bf2(sc[0], sc[1]), pack_bf2(sc[2], sc[3]), pack_bf2(sc[4], sc[5]), pack_bf2(sc[6], sc[7])};
      };
      probs(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 2 * H2; ++j) {
        const bool more = j + 1 < 2 * H2;
        if (more) { read_v(j + 1); probs(j + 1); }
#pragma unroll
        for (int bb = 0; bb < NB; ++bb) o[bb] = mfma_32x32x16(va[j & 1][bb], pb[j & 1], o[bb]);
        if (more) sched_group(0x100, 2 * NB);
#pragma unroll
        for (int bb = 0; bb < NB; ++bb) sched_group(0x008, 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (H2 == 2) l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
      else l_run += ps[0] + ps[1];
    };
    Slot sl;
    gload(sl, 0);
    lwrite(sl, 0);
    if (ntiles > 1) gload(sl, 1);
    __syncthreads();
    for (int k = 0;;) {
      compute(k);
      if (k + 1 < ntiles) {
        lwrite(sl, k + 1);
        if (k + 2 < ntiles) gload(sl, k + 2);
      }
      __syncthreads();
      if (++k >= ntiles) break;
    }
    wt0 += win;
    if ((FIRST || JOINT) && kept && wt0 >= seg_end) {
      kept = false;
      wt0 = kv_begin;
      seg_end = kv_end;
    }
  }
  // normalise and write: o[bb][i] is dim 32bb + 8(i/4) + 4kg + i%4 of row R; lanes r and r^32
  // together cover 8 consecutive dims
  float L = l_run + other_half(l_run);
  // the row again, so that nothing of it is kept over the loop
  const int le = opaque_v((int)(threadIdx.x & 63)), re = 32 * w + (le & 31), Re = row0 + re, ge = le >> 5;
  if (it.part_row >= 0) {
    if (Re < rows) {
      const float inv = L > 0.f ? 1.f / L : 0.f;
      const int64_t pr = it.part_row + re;
      float* op = part_o + pr * D;
#pragma unroll
      for (int bb = 0; bb < NB; ++bb)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<float4*>(op + 32 * bb + 8 * c + 4 * ge) =
              make_float4(o[bb][4 * c] * inv, o[bb][4 * c + 1] * inv, o[bb][4 * c + 2] * inv, o[bb][4 * c + 3] * inv);
      if (ge == 0) part_lse[pr] = L > 0.f ? m_run + log2f(L) : -INFINITY;
    }
  } else if (Re < rows) {
    const int tok = Re / G, hg = Re - tok * G;
    L += sink_mass(sinks, kvh * G + hg, m_run);
    if (lse && ge == 0) lse[(int64_t)(q0 + tok) * (G * n_kv_heads) + kvh * G + hg] = row_lse(L, m_run);
    const float inv = L > 0.f ? 1.f / L : 0.f;
    uint16_t* op = out + (int64_t)(q0 + tok) * o_ts + (int64_t)(kvh * G + hg) * o_hs;
#pragma unroll
    for (int bb = 0; bb < NB; ++bb)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint2 v = {pack_bf2(o[bb][4 * c] * inv, o[bb][4 * c + 1] * inv),
                         pack_bf2(o[bb][4 * c + 2] * inv, o[bb][4 * c + 3] * inv)};
        *reinterpret_cast<uint2*>(op + 32 * bb + 8 * c + 4 * ge) = v;
      }
  }
}

}  // namespace pie
