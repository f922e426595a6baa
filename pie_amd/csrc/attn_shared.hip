// Attention of a batch whose requests share long prefixes. Requests come in groups; group g's prefix is
// cached once, and every query token of the group sees all of it, then its own request's tokens (the
// suffix) up to itself:
//   out = sum_t p_t v_t over prefix and suffix,  p = softmax(q . k_t * sm_scale).
// The softmax over both is the join of the softmaxes over the parts: with each part's normalised output
// o_i and base-2 log-sum-exp l_i, M = max l_i: out = sum 2^(l_i - M) o_i / sum 2^(l_i - M).
//
// MI355X mapping. A prefix read once per request costs its bytes n times over; read for the group it is
// a matrix product of all the group's query rows (tokens x the kv head's query heads) with the prefix,
// cut into items of 128 rows over a piece of the prefix (prefill_item), which MFMA bounds at many rows
// and HBM at few. The suffixes are private: a decode step's, and prefixes that at most 16 rows share, are
// streamed by stream units (below), bound by HBM; runs of several query tokens per request are causal
// prefill items, which walk a short prefix themselves. All run in one launch, the prefill items' work groups first: they use the matrix cores
// while the others use the memory. Every other part leaves an fp32 partial result, joined by a second launch
// (attn_shared_merge_kernel).
//
// Measured (32 query and 8 kv heads of 128): 256 requests of 128-1000 tokens behind 16000, 628 MB and 69
// GFLOP, 138-140 us (4.5 TB/s and 500 TFLOP/s at once; the bytes alone take 128 us at a large copy's rate)
// and the join 7; 37 requests behind 9 prompts of 300-3500, 104 MB, 24.5 us and 5; 163 query tokens of 23
// requests behind two prompts of 3000-3500, 29 us and 5.4 (MFMA busy 21% of the cycles, waits 42% of the
// waves' time: items of 11 tiles, one round of the device).
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "attn_dev.h"

namespace pie {

// The plan on the device: kItemWords each for the prefill items of prefixes and (several query tokens
// per request) of suffixes, then for the stream items of prefixes; then kTokenWords per query token; then,
// in a decode step, the requests, longest suffix first.
// Item: first row, first query token, query tokens, kv length, first page-table slot, start and length of
// the piece, first partial row of kv head 0 (kv head h: + h * rows of the run; -1: the item walks its
// group's prefix and then its suffix and writes the output), first page-table slot and length of that prefix.
// Query token: {first partial row, rows of the run, the token's first row in the run, pieces} of its
// prefix, and of its suffix. Row r of piece s for kv head h is first + (s * kv heads + h) * rows + r. In a
// decode step a run of G rows is the request's own and -pieces of them are planned (the device counts
// those that hold tokens). -1 prefix pieces: nothing to join, an item wrote the output.
constexpr int kItemWords = 10, kTokenWords = 8;

struct SharedArgs {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  PagedKV kv;                     // the suffixes' pages
  const int32_t* prefix_indices;  // the prefixes' page ids
  const int32_t* plan;
  const int32_t* order;           // decode: the requests in the order they are worked on
  int G, Hq, Hkv, prefix_items, suffix_items, stream_items, B, splits, heads;
  float scale_log2;
  float *part_o, *part_lse;
  int64_t suffix_row;  // decode: first partial row of the suffixes
  uint16_t* out;
  int64_t o_ts, o_hs;
  float* lse;
};

// A stream unit: at most 16 query rows (row n: query token q0 + n / G, head n % G of the kv head's group)
// over positions [kv0, kv1) of a run of pages, for one or two (`heads`) adjacent kv heads. The four waves
// are shared out among the heads; a head's waves take its tiles in turn and meet in LDS. With two heads the
// page table and the set-up are paid once for both and the waves read the heads' rows of a token side by
// side (four heads gain nothing more). A wave loads its next tile as soon as it has the current one's V in
// registers and its scores. HBM bounds it.
struct StreamRun {
  int q0, rows, kv0, kv1, page0, kvh0;
  const int32_t* indices;
  int64_t part_row;  // of kv head 0, row 0; head h: + h * rows
};
template <int D>
__device__ __forceinline__ void stream_unit(char* smem, int32_t* ptab, const StreamRun& run, const uint16_t* __restrict__ q,
                                            int64_t q_ts, int64_t q_hs, const PagedKV& kv, int G, int heads,
                                            float scale_log2, float* __restrict__ part_o, float* __restrict__ part_lse) {
  using W = WaveAttn<D>;
  constexpr int kVtile = kTileTokens * D;  // elements of one V tile
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int share = 4 / heads, phase = w / heads, kvh = run.kvh0 + w % heads;  // waves of a head, this one's place
  W st;
  st.init();
  {
    const bool valid = n < run.rows;
    const int tok = valid ? n / G : 0, hg = valid ? n - tok * G : 0;
    const uint16_t* qp = q + (int64_t)(run.q0 + tok) * q_ts + (int64_t)(kvh * G + hg) * q_hs;
#pragma unroll
    for (int s = 0; s < W::NS; ++s) {
      const u32x4_t z = {0u, 0u, 0u, 0u};
      st.qb[s] = valid ? ld16v(qp + 8 * (4 * s + g)) : z;
    }
  }
  uint16_t* vt = reinterpret_cast<uint16_t*>(smem) + w * kVtile;
  const int step = share * kTileTokens;
  const int win = max(kTileTokens, (kPageWin - 2) * kv.page_size / kTileTokens * kTileTokens);
  for (int wt0 = run.kv0; wt0 < run.kv1; wt0 += win) {
    const int wt1 = min(run.kv1, wt0 + win);
    const int lp0 = (int)kv.pdiv.div((uint32_t)wt0);
    const int npg = (int)kv.pdiv.div((uint32_t)(wt1 - 1)) - lp0 + 1;
    __syncthreads();  // the previous window's lookups are done
    for (int i = threadIdx.x; i < npg; i += 256) ptab[i] = run.indices[run.page0 + lp0 + i];
    __syncthreads();
    KVTile<D> t;
    int t0 = wt0 + kTileTokens * phase;
    if (t0 < wt1) t.load(kv, ptab, lp0, KeptMap{}, t0, wt1, kvh, lane, vt);
    for (; t0 < wt1; t0 += step) {
      u32x4_t vb[W::NB];
      float s[2][4], a[4];
      bool rescale;
      wait_vmcnt<0>();
      st.read_v(vt, lane, vb);
      st.scores(t.ka, t.vmask(lane), scale_log2, s);
      wait_lgkmcnt0();
      __builtin_amdgcn_sched_barrier(0);  // (loads moved up would need registers of their own)
      if (t0 + step < wt1) t.load(kv, ptab, lp0, KeptMap{}, t0 + step, wt1, kvh, lane, vt);
      __builtin_amdgcn_sched_barrier(0);
      const u32x4_t pa = st.softmax(s, lane, a, rescale);
#pragma unroll
      for (int nb = 0; nb < W::NB; ++nb) st.pv(pa, vb[nb], a, rescale, nb);
    }
  }
  // the waves' results through LDS: m[4][16], l[4][16], o[4][16][D] (fp32); wave p * heads + h is part p of
  // head h
  const float lsum = st.row_sum(lane);
  __syncthreads();
  float* ms = reinterpret_cast<float*>(smem);
  float* ls = ms + 4 * 16;
  float* os = ls + 4 * 16;
  if (g == 0) { ms[w * 16 + n] = st.m; ls[w * 16 + n] = lsum; }
#pragma unroll
  for (int nb = 0; nb < W::NB; ++nb)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * g + i < run.rows) os[(w * 16 + 4 * g + i) * D + 16 * nb + n] = st.o[nb][i];
  __syncthreads();
  constexpr int CH = D / 8;
  for (int u = threadIdx.x; u < heads * run.rows * CH; u += 256) {
    const int hr = u / CH, c = u % CH, h = hr / run.rows, row = hr - h * run.rows;
    float M = -INFINITY;
    for (int p = 0; p < share; ++p) M = fmaxf(M, ms[(p * heads + h) * 16 + row]);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
    const float ref = M == -INFINITY ? 0.f : M;
    for (int p = 0; p < share; ++p) {
      const int x = (p * heads + h) * 16 + row;
      const float f = fast_exp2(ms[x] - ref);
      L = fmaf(ls[x], f, L);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(os[x * D + 8 * c + e], f, acc[e]);
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const int64_t r = run.part_row + (int64_t)(run.kvh0 + h) * run.rows + row;
    float4* dst = reinterpret_cast<float4*>(part_o + r * D + 8 * c);
    dst[0] = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    dst[1] = make_float4(acc[4] * inv, acc[5] * inv, acc[6] * inv, acc[7] * inv);
    if (c == 0) part_lse[r] = L > 0.f ? M + log2f(L) : -INFINITY;
  }
}

// Work groups of a list of prefill items: one per (item, kv head), padded to the XCDs.
__host__ __device__ __forceinline__ int shared_blocks(int items, int Hkv) { return (items * Hkv + 7) / 8 * 8; }

// STREAM: stream units (a decode step, or prefixes of few rows). RAGGED: several query tokens per request; items may
// walk a prefix and a suffix.
template <int D, bool STREAM, bool RAGGED>
__global__ __launch_bounds__(256, prefill_groups<D>()) void attn_shared_kernel(SharedArgs a) {
  constexpr int kUnit = STREAM ? decode_smem<D>() : 0, kItem = prefill_smem<D>();
  constexpr int kSmem = kItem > kUnit ? kItem : kUnit;
  __shared__ __attribute__((aligned(16))) char smem[kSmem];
  __shared__ int32_t ptab[kPageWin];
  // Prefill items of one kind in prefill_unit's order: each XCD takes a run of them, those of one piece together.
  const int prefix_blocks = shared_blocks(a.prefix_items, a.Hkv), item_blocks = prefix_blocks + shared_blocks(a.suffix_items, a.Hkv);
  if (STREAM && (int)blockIdx.x >= item_blocks) {
    const int heads = a.heads, blocks = a.Hkv / heads;
    const int u = (int)blockIdx.x - item_blocks, hb = u % blocks, v = u / blocks;
    StreamRun run;
    run.kvh0 = hb * heads;
    if (v < a.stream_items) {
      const int32_t* w = a.plan + kItemWords * (a.prefix_items + a.suffix_items + v);
      run.q0 = uniform(w[1]);
      run.rows = uniform(w[2]) * a.G;
      run.page0 = uniform(w[4]);
      run.kv0 = uniform(w[5]);
      run.kv1 = min(uniform(w[3]), run.kv0 + uniform(w[6]));
      run.part_row = uniform(w[7]);
      run.indices = a.prefix_indices;
    } else {
      const int r = (v - a.stream_items) / a.splits, j = v - a.stream_items - r * a.splits;
      const int b = uniform(a.order[r]);
      split_range(kv_length(a.kv, b), a.splits, j, run.kv0, run.kv1);
      if (run.kv0 >= run.kv1) return;  // an empty split: the merge does not read it
      run.q0 = b;
      run.rows = a.G;
      run.page0 = a.kv.indptr[b];
      run.part_row = a.suffix_row + (int64_t)(b * a.splits + j) * a.Hq;
      run.indices = a.kv.indices;
    }
    stream_unit<D>(smem, ptab, run, a.q, a.q_ts, a.q_hs, a.kv, a.G, heads, a.scale_log2, a.part_o, a.part_lse);
    return;
  }
  const bool suffix = (int)blockIdx.x >= prefix_blocks;
  const int n = suffix ? a.suffix_items : a.prefix_items, x = (int)blockIdx.x - (suffix ? prefix_blocks : 0);
  const int per = (n * a.Hkv + 7) / 8, u = (x & 7) * per + (x >> 3);
  if (u >= n * a.Hkv) return;  // padding work group
  const int kvh = u / n;
  const int32_t* w = a.plan + kItemWords * ((suffix ? a.prefix_items : 0) + u - kvh * n);
  PrefillItem it;
  it.b = 0;
  it.row0 = uniform(w[0]);
  it.q0 = uniform(w[1]);
  it.qo_len = uniform(w[2]);
  it.kv_len = uniform(w[3]);
  it.page0 = uniform(w[4]);
  it.off = uniform(w[5]);
  it.chunk = uniform(w[6]);
  const int part_row = uniform(w[7]);
  it.part_row = part_row < 0 ? -1 : (int64_t)part_row + (int64_t)kvh * (it.qo_len * a.G);
  it.pre_indices = a.prefix_indices;
  it.pre_page0 = uniform(w[8]);
  it.pre_len = uniform(w[9]);
  PagedKV kv = a.kv;
  if (!suffix) kv.indices = a.prefix_indices;
  prefill_item<D, false, RAGGED>(smem, ptab, it, a.q, a.q_ts, a.q_hs, kv, a.G, a.Hkv, kvh, a.scale_log2, suffix ? 1 : 0,
                                  -1, 0, nullptr, nullptr, nullptr, a.out, a.o_ts, a.o_hs, nullptr, a.part_o, a.part_lse,
                                  a.lse);
}

// Joins the parts of each (query token, head), D / 8 lanes to a head. WIDE (more than kNarrowParts parts): a work
// group for 512 / D heads of a token, its waves sharing the parts out. Else each wave takes 512 / D heads of its
// own and loads all their parts at once: a quarter of the waves, and no meeting in LDS (256 tokens of 32 heads
// and 5 parts: 11.5 us with the waves sharing, 7.0 with a wave each). HBM and load latency bound it.
constexpr int kNarrowParts = 8;
template <int D, bool WIDE>
__global__ __launch_bounds__(256) void attn_shared_merge_kernel(SharedArgs a, int64_t units, const int32_t* __restrict__ tokens) {
  constexpr int CH = D / 8, HEADS = 64 / CH;
  const int lane = threadIdx.x & 63, per = (a.Hq + HEADS - 1) / HEADS;
  const int64_t u = WIDE ? blockIdx.x : 4 * (int64_t)blockIdx.x + uniform(threadIdx.x >> 6);
  if (u >= units) return;
  const int t = (int)(u / per);
  const int hq = (int)(u - (int64_t)t * per) * HEADS + lane / CH, c = lane % CH;
  const int hl = min(hq, a.Hq - 1);  // lanes past the last head read its partials and write nothing
  const int kvh = hl / a.G, hg = hl - kvh * a.G;
  const int32_t* w = tokens + kTokenWords * (int64_t)t;
  const int np = w[3], planned = w[7];
  if (np < 0) return;  // (of the whole token: every thread of its waves)
  const int room = np + abs(planned);
  const int64_t p0 = (int64_t)w[0] + (int64_t)kvh * w[1] + w[2] + hg, s0 = (int64_t)w[4] + (int64_t)kvh * w[5] + w[6] + hg;
  const int64_t p_step = (int64_t)w[1] * a.Hkv, s_step = (int64_t)w[5] * a.Hkv;
  const auto row = [&](int s) { return s < np ? p0 + s * p_step : s0 + (s - np) * s_step; };
  const int n = planned < 0 ? np + split_count(kv_length(a.kv, t), -planned) : room;
  float acc[8], L = 0.f, M = -INFINITY;
  if constexpr (WIDE) {
    merge_partials<D, 8>(a.part_o + 8 * c, a.part_lse, row, n, room, acc, L, M);
    if (threadIdx.x >= 64) return;
  } else {
    float l[kNarrowParts];
    float4 v[kNarrowParts][2];
#pragma unroll
    for (int s = 0; s < kNarrowParts; ++s) {
      l[s] = -INFINITY;
      if (s < n) {
        const int64_t r = row(s);
        const float4* p = reinterpret_cast<const float4*>(a.part_o + r * D + 8 * c);
        l[s] = a.part_lse[r];
        v[s][0] = p[0];
        v[s][1] = p[1];
      }
    }
#pragma unroll
    for (int s = 0; s < kNarrowParts; ++s) M = fmaxf(M, l[s]);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll
    for (int s = 0; s < kNarrowParts; ++s)
      if (s < n) {
        const float f = fast_exp2(l[s] - ref);
        L += f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(f, (&v[s][e >> 2].x)[e & 3], acc[e]);
      }
  }
  if (hq >= a.Hq) return;
  if (a.lse && c == 0) a.lse[(int64_t)t * a.Hq + hq] = row_lse(L, M);
  const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= inv;
  st16(a.out + (int64_t)t * a.o_ts + (int64_t)hq * a.o_hs + 8 * c, pack8(acc));
}

template <int D>
static void launch_shared(hipStream_t st, const SharedArgs& a, int T, int max_parts, const int32_t* tokens) {
  const int items = shared_blocks(a.prefix_items, a.Hkv) + shared_blocks(a.suffix_items, a.Hkv);
  const int streams = (a.stream_items + a.B * a.splits) * (a.Hkv / a.heads);
  if (items + streams)
    hipLaunchKernelGGL((!streams ? attn_shared_kernel<D, false, true> : a.splits ? attn_shared_kernel<D, true, false>
                                                                            : attn_shared_kernel<D, true, true>),
                       dim3(items + streams), dim3(256), 0, st, a);
  const int64_t units = (int64_t)T * ((a.Hq + 512 / D - 1) / (512 / D));
  if (max_parts > kNarrowParts)
    hipLaunchKernelGGL((attn_shared_merge_kernel<D, true>), dim3((unsigned)units), dim3(256), 0, st, a, units, tokens);
  else if (max_parts)
    hipLaunchKernelGGL((attn_shared_merge_kernel<D, false>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, a, units,
                       tokens);
}

}  // namespace pie

using namespace pie;

// info[]: what a run needs of its plan, and what it checks against its own arguments.
enum {
  kInfoWords, kInfoScratch, kInfoPrefixItems, kInfoSuffixItems, kInfoStreamItems, kInfoTokensWord, kInfoSplits,
  kInfoSuffixRow, kInfoMaxParts, kInfoTokens, kInfoBatch, kInfoHq, kInfoHkv, kInfoDim, kInfoPage, kInfoRows,
  kInfoHeads
};

// The shortest pieces, in kv tokens, of a prefill item and of a stream unit: below them a work group is mostly
// set-up (22 requests of at most 96 tokens behind 742: 18 us, 20 with prefill items of 512; four behind 600:
// 12.9 us, 14.2 with stream units of 256).
constexpr int64_t kMinPrefill = 256, kMinStream = 128;
// The longest prefix that an item of several query tokens per request walks itself, before its suffix, where no
// suffix of the group is cut: the prefix is walked once per request instead of once per 128 rows of the group,
// but no partial results are written and joined (213 requests of up to 19 tokens behind 143: 59 us against 81;
// 230 behind up to 366: 55 against 66; 112 behind up to 859: 57 against 38). Head dim 256 walks a tile more
// slowly (165 requests of up to 22 tokens behind 185: 96 us against 87; 234 behind 72: 214 against 234). Beside
// groups that need the join all the same, only prefixes of one piece (14 requests of 2 kv heads behind up to
// 604: 23 us with all up to 512, 17.7 with those up to 256).
static int64_t joint_prefix(int64_t D, bool no_join) { return D == 256 ? 128 : no_join ? 512 : kMinPrefill; }
// Query rows of a kv head that a stream unit holds.
constexpr int64_t kStreamRows = 16;

static int shared_plan(const int32_t* group_indptr, int64_t groups, const int32_t* prefix_indptr,
                       const int32_t* prefix_last, const int32_t* qo_indptr, const int32_t* kv_indptr,
                       const int32_t* kv_last, int64_t batch, int64_t P, int64_t Hq, int64_t Hkv, int64_t D,
                       int64_t num_cus, int64_t scratch_max, int32_t* plan, int64_t capacity, int64_t* info) {
  const char* what = "attention_shared_plan";
  PIE_REQUIRE(group_indptr && prefix_indptr && prefix_last && kv_indptr && kv_last && info, "%s: null argument", what);
  PIE_REQUIRE(groups >= 0 && groups <= (1 << 24) && batch >= 0 && batch <= (1 << 24) && P > 0 && P <= 65536,
              "%s: bad groups %lld / batch %lld / page_size %lld", what, (long long)groups, (long long)batch, (long long)P);
  PIE_REQUIRE(Hkv > 0 && Hkv <= 65535 && Hq > 0 && Hq % Hkv == 0 && Hq <= 65535 && (qo_indptr || Hq / Hkv <= kStreamRows),
              "%s: need num_qo_heads = G * num_kv_heads (got %lld / %lld), G <= 16 for one query token per request", what,
              (long long)Hq, (long long)Hkv);
  PIE_REQUIRE(D == 64 || D == 128 || D == 256, "%s: head_dim %lld not in {64, 128, 256}", what, (long long)D);
  PIE_REQUIRE(group_indptr[0] == 0 && group_indptr[groups] == batch, "%s: group_indptr must run from 0 to the batch size %lld",
              what, (long long)batch);
  const int64_t G = Hq / Hkv;
  const int64_t cus = num_cus > 0 ? num_cus : 256;
  const int64_t slots = (D == 256 ? prefill_groups<256>() : prefill_groups<128>()) * cus;
  // a run of cached tokens: its length, or -1 for a bad table
  const auto length = [&](const int32_t* indptr, const int32_t* last, int64_t i) -> int64_t {
    const int64_t np = (int64_t)indptr[i + 1] - indptr[i];
    if (np < 0 || indptr[i] < 0) return -1;
    if (np == 0) return 0;
    if (last[i] < 0 || last[i] > P) return -1;
    const int64_t n = (np - 1) * P + last[i];
    return n < 0x7ffff000ll ? n : -1;  // (a tile past the end still has an int position)
  };
  const auto first_token = [&](int64_t b) -> int64_t { return qo_indptr ? qo_indptr[b] : b; };
  PIE_REQUIRE(first_token(0) == 0, "%s: qo_indptr must start at 0", what);
  // A run of cached tokens and the query tokens that read it. tiles: its prefill items per piece, 0: streamed.
  struct Run { int64_t len, q0, tokens, page0, tiles; };
  std::vector<Run> prefix((size_t)groups), suffix((size_t)batch);
  const auto tiles = [&](int64_t tokens) { return (tokens * G + kPrefillRows - 1) / kPrefillRows; };
  int64_t total = 0, longest = 0, longest_suffix = 0;  // total: kv tokens that work groups walk, over all kv heads
  for (int64_t b = 0; b < batch; ++b) {
    const int64_t n = length(kv_indptr, kv_last, b), qo = first_token(b + 1) - first_token(b);
    PIE_REQUIRE(n >= 0 && qo >= 0 && qo * G < 0x7fffff00ll, "%s: bad table at request %lld", what, (long long)b);
    suffix[(size_t)b] = Run{n, first_token(b), qo, kv_indptr[b], qo_indptr ? tiles(qo) : 0};
    total += n * (qo_indptr ? tiles(qo) : 1) * Hkv;
    longest_suffix = std::max(longest_suffix, n);
  }
  for (int64_t g = 0; g < groups; ++g) {
    const int64_t n = length(prefix_indptr, prefix_last, g);
    PIE_REQUIRE(n >= 0 && group_indptr[g + 1] >= group_indptr[g] && group_indptr[g + 1] <= batch,
                "%s: bad table at group %lld", what, (long long)g);
    const int64_t q0 = first_token(group_indptr[g]), tokens = first_token(group_indptr[g + 1]) - q0;
    PIE_REQUIRE(tokens * G < 0x7fffff00ll, "%s: group %lld has too many query tokens", what, (long long)g);
    prefix[(size_t)g] = Run{n, q0, tokens, prefix_indptr[g], tokens * G <= kStreamRows ? 0 : tiles(tokens)};
    total += n * tiles(tokens) * Hkv;
    if (tokens) longest = std::max(longest, n);
  }
  const int64_t T = first_token(batch);
  PIE_REQUIRE(T < (1 << 27) && T * Hq < 0x7fffff00ll, "%s: too many query tokens", what);
  // Pieces of equal length near a work group's share of the launch, which for a prefill item is of one kv
  // head's tokens, for a stream unit of `heads` heads'.
  int64_t share = total / slots, heads = 1;
  const auto target = [&](const Run& r) {
    return r.tiles ? std::max(kMinPrefill, share) : std::max(kMinStream, share / heads);
  };
  const auto piece_len = [&](const Run& r) {
    const int64_t n = std::max<int64_t>(1, (r.len + target(r) - 1) / target(r));
    return std::max<int64_t>(64, ((r.len + n - 1) / n + 63) / 64 * 64);  // whole tiles
  };
  const auto pieces = [&](const Run& r) { return r.tokens ? (r.len + piece_len(r) - 1) / piece_len(r) : 0; };
  std::vector<char> joint((size_t)groups);  // groups whose items walk prefix and suffix
  int64_t rows, prefix_rows, items, suffix_items, stream_items, splits, max_parts, streams;
  const auto lay_out = [&] {
    rows = items = suffix_items = stream_items = splits = max_parts = 0;
    for (bool no_join : {true, false}) {
      bool all = true;
      for (int64_t g = 0; g < groups; ++g) {
        bool one = qo_indptr && prefix[(size_t)g].len <= joint_prefix(D, no_join);
        for (int64_t b = group_indptr[g]; one && b < group_indptr[g + 1]; ++b) one = pieces(suffix[(size_t)b]) <= 1;
        joint[(size_t)g] = one;
        all = all && (one || prefix[(size_t)g].tokens == 0);
      }
      if (all) break;
    }
    for (int64_t g = 0; g < groups; ++g) {
      const Run& r = prefix[(size_t)g];
      if (joint[(size_t)g]) continue;
      rows += pieces(r) * r.tokens * Hq;
      if (r.tiles) items += pieces(r) * r.tiles;
      else stream_items += pieces(r);
      max_parts = std::max(max_parts, pieces(r));
    }
    prefix_rows = rows;
    if (qo_indptr) {
      int64_t most = 0;
      for (int64_t g = 0; g < groups; ++g)
        for (int64_t b = group_indptr[g]; b < group_indptr[g + 1]; ++b) {
          const Run& r = suffix[(size_t)b];
          const int64_t n = std::max<int64_t>(1, pieces(r));
          suffix_items += n * r.tiles;
          if (joint[(size_t)g]) continue;
          rows += n * r.tokens * Hq;
          most = std::max(most, n);
        }
      max_parts += most;
    } else {
      // A decode step's suffixes grow under one plan: as many splits as 512 tokens more ask for, as long as
      // the launch holds them all at once (242 requests of at most 26 tokens, 2 kv heads: 14.8 us with one
      // split, 15.9 with five, four of them empty).
      const auto of = [&](int64_t len) { return pieces(Run{len, 0, 1, 0, 0}); };
      const int64_t room = slots / std::max<int64_t>(1, batch * (Hkv / heads));
      splits = std::min<int64_t>(64, std::max({(int64_t)1, of(longest_suffix), std::min(of(longest_suffix + 512), room)}));
      rows += batch * splits * Hq;
      max_parts += splits;
    }
    streams = (stream_items + batch * splits) * (Hkv / heads);
  };
  lay_out();
  // More stream units than the launch holds at once: two kv heads to each (256 requests behind 16000 tokens,
  // 8 kv heads: 155 us against 167; 4 behind 600, which leave CUs idle: 14.5 us against 12.9).
  if (Hkv % 2 == 0 && streams > slots) {
    heads = 2;
    lay_out();
  }
  // More prefill items than CUs: twice as long ones. Two at once on a CU share its matrix cores and end no
  // sooner than one of both, with twice the partial results (23 requests of up to 13 tokens behind 3000-3500: 33 us
  // against 40; fewer items, 61 requests of 16 heads behind 5000, are the worse for it: 45 us against 37).
  if ((items + suffix_items) * Hkv > cus) {
    share *= 2;
    lay_out();
  }
  // Longer pieces where the scratch or the partial rows' count does not allow these.
  while (rows >= 0x7fffff00ll || rows * (D + 1) * 4 > scratch_max || (items + suffix_items) * Hkv + streams >= 0x7fffff00ll) {
    PIE_REQUIRE(share < std::max(longest, longest_suffix + 512) * heads,
                "%s: the partial results need %lld bytes of workspace, have %lld", what, (long long)(rows * (D + 1) * 4),
                (long long)scratch_max);
    share = std::max(share, kMinStream) * 2;
    lay_out();
  }
  const int64_t tokens_word = kItemWords * (items + suffix_items + stream_items);
  const int64_t words = tokens_word + kTokenWords * T + (qo_indptr ? 0 : batch);
  info[kInfoWords] = words;
  info[kInfoScratch] = rows * (D + 1) * 4;
  info[kInfoPrefixItems] = items;
  info[kInfoSuffixItems] = suffix_items;
  info[kInfoStreamItems] = stream_items;
  info[kInfoTokensWord] = tokens_word;
  info[kInfoSplits] = splits;
  info[kInfoMaxParts] = max_parts;
  info[kInfoTokens] = T;
  info[kInfoBatch] = batch;
  info[kInfoHq] = Hq;
  info[kInfoHkv] = Hkv;
  info[kInfoDim] = D;
  info[kInfoPage] = P;
  info[kInfoSuffixRow] = prefix_rows;
  info[kInfoRows] = rows;
  info[kInfoHeads] = heads;
  if (!plan) return PIE_HIP_OK;
  PIE_REQUIRE(capacity >= words, "%s: needs %lld words, capacity %lld", what, (long long)words, (long long)capacity);
  int32_t *it = plan, *stream = plan + kItemWords * (items + suffix_items), *tok = plan + tokens_word;
  int64_t row = 0;
  // the items of a run in order of pieces, and the part of its query tokens' words; pre: the prefix that a joint
  // item walks before it
  const auto put = [&](const Run& r, int64_t n, int at, const Run* pre) {
    const int64_t chunk = piece_len(r), run_rows = r.tokens * G;
    int32_t*& to = r.tiles ? it : stream;
    for (int64_t s = 0; s < n; ++s)
      for (int64_t r0 = 0; r0 < run_rows; r0 += kPrefillRows) {  // (a streamed run has rows of one tile at most)
        const int32_t w[kItemWords] = {(int32_t)r0, (int32_t)r.q0, (int32_t)r.tokens, (int32_t)r.len, (int32_t)r.page0,
                                       (int32_t)(s * chunk), (int32_t)chunk,
                                       pre ? -1 : (int32_t)(row + s * Hkv * run_rows + r0),
                                       pre ? (int32_t)pre->page0 : 0, pre ? (int32_t)pre->len : 0};
        memcpy(to, w, sizeof(w));
        to += kItemWords;
      }
    for (int64_t i = 0; i < r.tokens; ++i) {
      const int32_t w[4] = {(int32_t)row, (int32_t)run_rows, (int32_t)(i * G), (int32_t)(pre ? 0 : n)};
      memcpy(tok + kTokenWords * (r.q0 + i) + at, w, sizeof(w));
    }
    if (!pre) row += n * run_rows * Hkv;
  };
  for (int64_t g = 0; g < groups; ++g) {
    const Run& r = prefix[(size_t)g];
    if (!joint[(size_t)g]) {
      put(r, pieces(r), 0, nullptr);
      continue;
    }
    const int32_t w[4] = {0, 0, 0, -1};
    for (int64_t i = 0; i < r.tokens; ++i) memcpy(tok + kTokenWords * (r.q0 + i), w, sizeof(w));
  }
  if (qo_indptr) {
    for (int64_t g = 0; g < groups; ++g)
      for (int64_t b = group_indptr[g]; b < group_indptr[g + 1]; ++b) {
        const Run& r = suffix[(size_t)b];
        put(r, std::max<int64_t>(1, pieces(r)), 4, joint[(size_t)g] ? &prefix[(size_t)g] : nullptr);
      }
  } else {
    for (int64_t b = 0; b < batch; ++b) {
      const int32_t w[4] = {(int32_t)(row + b * splits * Hq), (int32_t)G, 0, (int32_t)-splits};
      memcpy(tok + kTokenWords * b + 4, w, sizeof(w));
    }
  }
  if (!qo_indptr) {  // the longest suffixes first, so that the short ones fill the launch's tail
    int32_t* order = tok + kTokenWords * T;
    for (int64_t b = 0; b < batch; ++b) order[b] = (int32_t)b;
    std::stable_sort(order, order + batch, [&](int32_t x, int32_t y) { return suffix[(size_t)x].len > suffix[(size_t)y].len; });
  }
  return PIE_HIP_OK;
}

extern "C" int pie_hip_attention_shared_plan(const int32_t* group_indptr, int64_t groups, const int32_t* prefix_indptr,
                                             const int32_t* prefix_last_page_len, const int32_t* qo_indptr,
                                             const int32_t* kv_indptr, const int32_t* kv_last_page_len, int64_t batch,
                                             int64_t page_size, int64_t num_qo_heads, int64_t num_kv_heads,
                                             int64_t head_dim, int64_t num_cus, int64_t scratch_bytes, int32_t* plan,
                                             int64_t plan_capacity, int64_t* info) {
  try {
    return shared_plan(group_indptr, groups, prefix_indptr, prefix_last_page_len, qo_indptr, kv_indptr, kv_last_page_len,
                       batch, page_size, num_qo_heads, num_kv_heads, head_dim, num_cus, scratch_bytes, plan,
                       plan_capacity, info);
  } catch (const std::bad_alloc&) {
    return set_error(PIE_HIP_EINVAL, "attention_shared_plan: out of host memory");
  }
}

extern "C" int pie_hip_attention_shared(
    const pie_bf16* q, int64_t q_tok_stride, int64_t q_head_stride, const pie_bf16* k_cache, const pie_bf16* v_cache,
    int64_t page_stride, int64_t slot_stride, int64_t head_stride, int64_t num_pages, const int32_t* prefix_indices,
    const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* kv_last_page_len, int64_t num_tokens,
    int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim, int64_t page_size, float sm_scale, const int32_t* plan,
    const int64_t* info, void* scratch, int64_t scratch_bytes, pie_bf16* out, int64_t o_tok_stride,
    int64_t o_head_stride, float* lse, void* stream) {
  const char* what = "attention_shared";
  SharedArgs a{};
  const int rc = paged_kv_desc(&a.kv, k_cache, v_cache, page_stride, slot_stride, head_stride, num_pages, kv_indptr,
                               kv_indices, kv_last_page_len, page_size, head_dim, what);
  if (rc) return rc;
  PIE_REQUIRE(info && (prefix_indices || info[kInfoPrefixItems] + info[kInfoSuffixItems] + info[kInfoStreamItems] == 0), "%s: null argument", what);
  PIE_REQUIRE(info[kInfoTokens] == num_tokens && info[kInfoHq] == num_qo_heads && info[kInfoHkv] == num_kv_heads &&
                  info[kInfoDim] == head_dim && info[kInfoPage] == page_size,
              "%s: the plan is for %lld tokens, %lld/%lld heads of %lld, pages of %lld", what, (long long)info[kInfoTokens],
              (long long)info[kInfoHq], (long long)info[kInfoHkv], (long long)info[kInfoDim], (long long)info[kInfoPage]);
  if (num_tokens == 0) return PIE_HIP_OK;
  PIE_REQUIRE(q && out && plan, "%s: null q, out or plan", what);
  PIE_REQUIRE(aligned16(q) && aligned16(out) && q_tok_stride % 8 == 0 && q_head_stride % 8 == 0 && o_tok_stride % 8 == 0 &&
                  o_head_stride % 8 == 0,
              "%s: q/out pointers and strides must be 16-byte aligned", what);
  PIE_REQUIRE(info[kInfoScratch] == 0 || (scratch && aligned16(scratch) && scratch_bytes >= info[kInfoScratch]),
              "%s: needs %lld bytes of 16-byte-aligned scratch, got %lld", what, (long long)info[kInfoScratch],
              (long long)scratch_bytes);
  // a run hands its partial results from its first launch to its second
  InflightClaim claim;
  if (info[kInfoScratch]) {
    const InflightClaim::State got = claim.take(scratch, stream);
    if (got == InflightClaim::kBusy || got == InflightClaim::kShared) return inflight_busy(what);
  }
  a.q = q;
  a.q_ts = q_tok_stride;
  a.q_hs = q_head_stride;
  a.prefix_indices = prefix_indices;
  a.plan = plan;
  a.G = (int)(num_qo_heads / num_kv_heads);
  a.Hq = (int)num_qo_heads;
  a.Hkv = (int)num_kv_heads;
  a.prefix_items = (int)info[kInfoPrefixItems];
  a.suffix_items = (int)info[kInfoSuffixItems];
  a.stream_items = (int)info[kInfoStreamItems];
  a.B = (int)info[kInfoBatch];
  a.splits = (int)info[kInfoSplits];
  a.heads = (int)info[kInfoHeads];
  // (prefill_item scales raw scores inside the exponent, where a zero scale would turn -inf into NaN)
  a.scale_log2 = sm_scale == 0.f ? 1e-30f : sm_scale * 1.4426950408889634f;
  a.part_o = static_cast<float*>(scratch);
  a.part_lse = a.part_o + info[kInfoRows] * head_dim;
  a.suffix_row = info[kInfoSuffixRow];
  a.out = out;
  a.o_ts = o_tok_stride;
  a.o_hs = o_head_stride;
  a.lse = lse;
  const int32_t* tokens = plan + info[kInfoTokensWord];
  a.order = tokens + kTokenWords * num_tokens;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int T = (int)num_tokens, parts = (int)info[kInfoMaxParts];
  switch (head_dim) {
    case 64: launch_shared<64>(st, a, T, parts, tokens); break;
    case 128: launch_shared<128>(st, a, T, parts, tokens); break;
    default: launch_shared<256>(st, a, T, parts, tokens); break;
  }
  return check_launch(what);
}
