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
// and HBM at few. The suffixes are private: a decode step's are streamed by decode units (decode_unit),
// bound by HBM, runs of several query tokens per request are causal prefill items. Both kinds run in one
// launch, the prefix's work groups first: they use the matrix cores while the suffixes' use the memory.
// Every part leaves an fp32 partial result, joined by a second launch (attn_shared_merge_kernel).
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "attn_dev.h"

namespace pie {

// The plan on the device: prefix items and (several query tokens per request) suffix items of
// kItemWords each, then kTokenWords per query token.
// Item: first row, first query token, query tokens, kv length, first page-table slot, start and length of
// the piece, first partial row of kv head 0 (kv head h: + h * rows of the run).
// Query token: {first partial row, rows of the run, the token's first row in the run, pieces} of its
// prefix, and of its suffix. Row r of piece s for kv head h is first + (s * kv heads + h) * rows + r. In a
// decode step a run of G rows is the request's own and -pieces of them are planned (the device counts
// those that hold tokens).
constexpr int kItemWords = 8, kTokenWords = 8;

struct SharedArgs {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  PagedKV kv;                     // the suffixes' pages
  const int32_t* prefix_indices;  // the prefixes' page ids
  const int32_t* plan;
  int G, Hq, Hkv, prefix_items, suffix_items, B, splits;
  float scale_log2;
  float *part_o, *part_lse;
  int64_t suffix_row;  // decode: first partial row of the suffixes
};

// Work groups of a list of items: one per (item, kv head), padded to the XCDs.
__host__ __device__ __forceinline__ int shared_blocks(int items, int Hkv) { return (items * Hkv + 7) / 8 * 8; }

// The kernel's arguments, loaded where they are used: one branch's need not stay in scalar registers
// over the other's (the decode units' spilled 36 of them at head dim 64).
__device__ __forceinline__ SharedArgs branch_args(const SharedArgs& a) {
#ifdef PIE_HOST_EMULATION
  return a;
#else
  typedef const __attribute__((address_space(4))) uint32_t* words_t;
  words_t p = (words_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  union { uint32_t w[sizeof(SharedArgs) / 4]; SharedArgs a; } u;
#pragma unroll
  for (unsigned i = 0; i < sizeof(SharedArgs) / 4; ++i) u.w[i] = p[i];
  return u.a;
#endif
}

// RAGGED: several query tokens per request.
template <int D, bool RAGGED>
__global__ __launch_bounds__(256, prefill_groups<D>()) void attn_shared_kernel(SharedArgs a) {
  constexpr int kSmem = prefill_smem<D>() > decode_smem<D>() ? prefill_smem<D>() : decode_smem<D>();
  __shared__ __attribute__((aligned(16))) char smem[kSmem];
  __shared__ int32_t ptab[kPageWin];
  // Items of one kind in prefill_unit's order: each XCD takes a run of them, those of one piece together.
  const int prefix_blocks = shared_blocks(a.prefix_items, a.Hkv);
  const bool suffix = (int)blockIdx.x >= prefix_blocks;
  if (!RAGGED && suffix) {
    const SharedArgs d = branch_args(a);
    decode_unit<D, false>(smem, ptab, (int)blockIdx.x - prefix_blocks, d.q, d.q_ts, d.q_hs, d.kv, d.B, d.G, d.Hq,
                          d.scale_log2, d.splits, -1, 0, true, nullptr, 0, 0, d.part_o + d.suffix_row * D,
                          d.part_lse + d.suffix_row, nullptr, nullptr);
    return;
  }
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
  it.part_row = (int64_t)uniform(w[7]) + (int64_t)kvh * (it.qo_len * a.G);
  PagedKV kv = a.kv;
  if (!suffix) kv.indices = a.prefix_indices;
  prefill_item<D, false>(smem, ptab, it, a.q, a.q_ts, a.q_hs, kv, a.G, a.Hkv, kvh, a.scale_log2, suffix ? 1 : 0, -1, 0,
                         nullptr, nullptr, nullptr, nullptr, 0, 0, nullptr, a.part_o, a.part_lse, nullptr);
}

// Joins the parts of each (query token, head): one work group per token and 512 / D heads.
template <int D, int KB>
__global__ __launch_bounds__(256) void attn_shared_merge_kernel(SharedArgs a, const int32_t* __restrict__ tokens,
                                                                uint16_t* __restrict__ out, int64_t o_ts, int64_t o_hs,
                                                                float* __restrict__ lse) {
  constexpr int CH = D / 8;
  const int t = blockIdx.x, lane = threadIdx.x & 63;
  const int hq = blockIdx.y * (64 / CH) + lane / CH, c = lane % CH;
  const int hl = min(hq, a.Hq - 1);  // lanes past the last head read its partials and write nothing
  const int kvh = hl / a.G, hg = hl - kvh * a.G;
  const int32_t* w = tokens + kTokenWords * (int64_t)t;
  const int np = w[3], planned = w[7];
  const int room = np + abs(planned);
  const int64_t p0 = (int64_t)w[0] + (int64_t)kvh * w[1] + w[2] + hg, s0 = (int64_t)w[4] + (int64_t)kvh * w[5] + w[6] + hg;
  const int64_t p_step = (int64_t)w[1] * a.Hkv, s_step = (int64_t)w[5] * a.Hkv;
  const int n = planned < 0 ? np + split_count(kv_length(a.kv, t), -planned) : room;
  float acc[8], L, M;
  merge_partials<D, KB>(a.part_o + 8 * c, a.part_lse,
                        [&](int s) { return s < np ? p0 + s * p_step : s0 + (s - np) * s_step; }, n, room, acc, L, M);
  if (threadIdx.x >= 64 || hq >= a.Hq) return;
  if (lse && c == 0) lse[(int64_t)t * a.Hq + hq] = row_lse(L, M);
  const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= inv;
  st16(out + (int64_t)t * o_ts + (int64_t)hq * o_hs + 8 * c, pack8(acc));
}

template <int D>
static void launch_shared(hipStream_t st, const SharedArgs& a, int T, int max_parts, const int32_t* tokens,
                          uint16_t* out, int64_t o_ts, int64_t o_hs, float* lse) {
  const int prefix = shared_blocks(a.prefix_items, a.Hkv);
  if (a.splits)
    hipLaunchKernelGGL((attn_shared_kernel<D, false>), dim3(prefix + a.B * a.splits * a.Hkv), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attn_shared_kernel<D, true>), dim3(prefix + shared_blocks(a.suffix_items, a.Hkv)), dim3(256), 0,
                       st, a);
  hipLaunchKernelGGL((max_parts <= 4 ? attn_shared_merge_kernel<D, 1> : attn_shared_merge_kernel<D, 8>),
                     dim3(T, (a.Hq + 512 / D - 1) / (512 / D)), dim3(256), 0, st, a, tokens, out, o_ts, o_hs, lse);
}

}  // namespace pie

using namespace pie;

// info[]: what a run needs of its plan, and what it checks against its own arguments.
enum {
  kInfoWords, kInfoScratch, kInfoPrefixItems, kInfoSuffixItems, kInfoTokensWord, kInfoSplits, kInfoSuffixRow,
  kInfoMaxParts, kInfoTokens, kInfoBatch, kInfoHq, kInfoHkv, kInfoDim, kInfoPage, kInfoPrefixSlots, kInfoRows
};

// The shortest piece of a prefix or suffix: below it a work group is mostly set-up.
constexpr int64_t kSharedMinChunk = 256;

static int shared_plan(const int32_t* group_indptr, int64_t groups, const int32_t* prefix_indptr,
                       const int32_t* prefix_last, const int32_t* qo_indptr, const int32_t* kv_indptr,
                       const int32_t* kv_last, int64_t batch, int64_t P, int64_t Hq, int64_t Hkv, int64_t D,
                       int64_t num_cus, int64_t scratch_max, int32_t* plan, int64_t capacity, int64_t* info) {
  const char* what = "attention_shared_plan";
  PIE_REQUIRE(group_indptr && prefix_indptr && prefix_last && kv_indptr && kv_last && info, "%s: null argument", what);
  PIE_REQUIRE(groups >= 0 && groups <= (1 << 24) && batch >= 0 && batch <= (1 << 24) && P > 0 && P <= 65536,
              "%s: bad groups %lld / batch %lld / page_size %lld", what, (long long)groups, (long long)batch, (long long)P);
  PIE_REQUIRE(Hkv > 0 && Hkv <= 65535 && Hq > 0 && Hq % Hkv == 0 && Hq <= 65535 && (qo_indptr || Hq / Hkv <= 16),
              "%s: need num_qo_heads = G * num_kv_heads (got %lld / %lld), G <= 16 for one query token per request", what,
              (long long)Hq, (long long)Hkv);
  PIE_REQUIRE(D == 64 || D == 128 || D == 256, "%s: head_dim %lld not in {64, 128, 256}", what, (long long)D);
  PIE_REQUIRE(group_indptr[0] == 0 && group_indptr[groups] == batch, "%s: group_indptr must run from 0 to the batch size %lld",
              what, (long long)batch);
  const int64_t G = Hq / Hkv, slots = (D == 256 ? prefill_groups<256>() : prefill_groups<128>()) * (num_cus > 0 ? num_cus : 256);
  // a run of cached tokens: its length, or -1 for a bad table
  const auto length = [&](const int32_t* indptr, const int32_t* last, int64_t i) -> int64_t {
    const int64_t np = (int64_t)indptr[i + 1] - indptr[i];
    if (np < 0 || indptr[i] < 0) return -1;
    if (np == 0) return 0;
    if (last[i] < 0 || last[i] > P) return -1;
    const int64_t n = (np - 1) * P + last[i];
    return n < 0x7fffff00ll ? n : -1;
  };
  const auto first_token = [&](int64_t b) -> int64_t { return qo_indptr ? qo_indptr[b] : b; };
  PIE_REQUIRE(first_token(0) == 0, "%s: qo_indptr must start at 0", what);
  struct Run { int64_t len, q0, tokens, page0; };
  std::vector<Run> prefix((size_t)groups), suffix((size_t)batch);
  int64_t total = 0, longest = 0, longest_suffix = 0;  // kv tokens that work groups walk, over all kv heads
  for (int64_t b = 0; b < batch; ++b) {
    const int64_t n = length(kv_indptr, kv_last, b), qo = first_token(b + 1) - first_token(b);
    PIE_REQUIRE(n >= 0 && qo >= 0 && qo * G < 0x7fffff00ll, "%s: bad table at request %lld", what, (long long)b);
    suffix[(size_t)b] = Run{n, first_token(b), qo, kv_indptr[b]};
    total += n * (qo_indptr ? (qo * G + kPrefillRows - 1) / kPrefillRows : 1) * Hkv;
    longest_suffix = std::max(longest_suffix, n);
  }
  for (int64_t g = 0; g < groups; ++g) {
    const int64_t n = length(prefix_indptr, prefix_last, g);
    PIE_REQUIRE(n >= 0 && group_indptr[g + 1] >= group_indptr[g] && group_indptr[g + 1] <= batch,
                "%s: bad table at group %lld", what, (long long)g);
    const int64_t q0 = first_token(group_indptr[g]), tokens = first_token(group_indptr[g + 1]) - q0;
    PIE_REQUIRE(tokens * G < 0x7fffff00ll, "%s: group %lld has too many query tokens", what, (long long)g);
    prefix[(size_t)g] = Run{n, q0, tokens, prefix_indptr[g]};
    total += n * ((tokens * G + kPrefillRows - 1) / kPrefillRows) * Hkv;
    if (tokens) longest = std::max(longest, n);
  }
  const int64_t T = first_token(batch);
  PIE_REQUIRE(T < (1 << 27) && T * Hq < 0x7fffff00ll, "%s: too many query tokens", what);
  // Pieces of equal length near every work group's share of the launch; longer ones where the scratch or
  // the partial rows' count does not allow it.
  int64_t target = std::max(kSharedMinChunk, (total + slots - 1) / slots);
  const auto piece_len = [&](int64_t len) {
    const int64_t n = std::max<int64_t>(1, (len + target - 1) / target);
    return std::max<int64_t>(64, ((len + n - 1) / n + 63) / 64 * 64);  // whole tiles
  };
  const auto pieces = [&](int64_t len) { return (len + piece_len(len) - 1) / piece_len(len); };
  int64_t rows = 0, items = 0, suffix_items = 0, splits = 0, max_parts = 0;
  for (;; target *= 2) {
    rows = items = suffix_items = max_parts = 0;
    for (const Run& r : prefix) {
      rows += pieces(r.len) * r.tokens * Hq;
      items += pieces(r.len) * ((r.tokens * G + kPrefillRows - 1) / kPrefillRows);
      if (r.tokens) max_parts = std::max(max_parts, pieces(r.len));
    }
    const int64_t prefix_rows = rows;
    if (qo_indptr) {
      int64_t most = 0;
      for (const Run& r : suffix) {
        const int64_t n = std::max<int64_t>(1, pieces(r.len));
        rows += n * r.tokens * Hq;
        suffix_items += n * ((r.tokens * G + kPrefillRows - 1) / kPrefillRows);
        most = std::max(most, n);
      }
      max_parts += most;
    } else {
      // (a decode step's suffixes grow under one plan: room for 512 tokens more)
      splits = std::min<int64_t>(64, pieces(longest_suffix + 512));
      rows += batch * splits * Hq;
      max_parts += splits;
    }
    const bool fits = rows < 0x7fffff00ll && rows * (D + 1) * 4 <= scratch_max && (items + suffix_items) * Hkv < 0x7fffff00ll &&
                      batch * splits * Hkv + (items + suffix_items) * Hkv < 0x7fffff00ll;
    info[kInfoSuffixRow] = prefix_rows;
    if (fits) break;
    PIE_REQUIRE(target < std::max(longest, longest_suffix + 512),
                "%s: the partial results need %lld bytes of workspace, have %lld", what, (long long)(rows * (D + 1) * 4),
                (long long)scratch_max);
  }
  const int64_t tokens_word = kItemWords * (items + suffix_items), words = tokens_word + kTokenWords * T;
  info[kInfoWords] = words;
  info[kInfoScratch] = rows * (D + 1) * 4;
  info[kInfoPrefixItems] = items;
  info[kInfoSuffixItems] = suffix_items;
  info[kInfoTokensWord] = tokens_word;
  info[kInfoSplits] = splits;
  info[kInfoMaxParts] = max_parts;
  info[kInfoTokens] = T;
  info[kInfoBatch] = batch;
  info[kInfoHq] = Hq;
  info[kInfoHkv] = Hkv;
  info[kInfoDim] = D;
  info[kInfoPage] = P;
  info[kInfoPrefixSlots] = groups ? prefix_indptr[groups] : 0;
  info[kInfoRows] = rows;
  if (!plan) return PIE_HIP_OK;
  PIE_REQUIRE(capacity >= words, "%s: needs %lld words, capacity %lld", what, (long long)words, (long long)capacity);
  int32_t *it = plan, *tok = plan + tokens_word;
  int64_t row = 0;
  // the items of a run in order of pieces, and the part of its query tokens' words
  const auto put = [&](const Run& r, int64_t n, int at) {
    const int64_t chunk = piece_len(r.len), run_rows = r.tokens * G;
    for (int64_t s = 0; s < n; ++s)
      for (int64_t r0 = 0; r0 < run_rows; r0 += kPrefillRows) {
        const int32_t w[kItemWords] = {(int32_t)r0, (int32_t)r.q0, (int32_t)r.tokens, (int32_t)r.len, (int32_t)r.page0,
                                       (int32_t)(s * chunk), (int32_t)chunk, (int32_t)(row + s * Hkv * run_rows + r0)};
        memcpy(it, w, sizeof(w));
        it += kItemWords;
      }
    for (int64_t i = 0; i < r.tokens; ++i) {
      const int32_t w[4] = {(int32_t)row, (int32_t)run_rows, (int32_t)(i * G), (int32_t)n};
      memcpy(tok + kTokenWords * (r.q0 + i) + at, w, sizeof(w));
    }
    row += n * run_rows * Hkv;
  };
  for (const Run& r : prefix) put(r, pieces(r.len), 0);
  for (int64_t b = 0; b < batch; ++b) {
    if (qo_indptr) {
      put(suffix[(size_t)b], std::max<int64_t>(1, pieces(suffix[(size_t)b].len)), 4);
    } else {
      const int32_t w[4] = {(int32_t)(row + b * splits * Hq), (int32_t)G, 0, (int32_t)-splits};
      memcpy(tok + kTokenWords * b + 4, w, sizeof(w));
    }
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
  PIE_REQUIRE(info && (prefix_indices || info[kInfoPrefixItems] == 0), "%s: null argument", what);
  PIE_REQUIRE(info[kInfoTokens] == num_tokens && info[kInfoHq] == num_qo_heads && info[kInfoHkv] == num_kv_heads &&
                  info[kInfoDim] == head_dim && info[kInfoPage] == page_size,
              "%s: the plan is for %lld tokens, %lld/%lld heads of %lld, pages of %lld", what, (long long)info[kInfoTokens],
              (long long)info[kInfoHq], (long long)info[kInfoHkv], (long long)info[kInfoDim], (long long)info[kInfoPage]);
  if (num_tokens == 0) return PIE_HIP_OK;
  PIE_REQUIRE(q && out && plan, "%s: null q, out or plan", what);
  PIE_REQUIRE(aligned16(q) && aligned16(out) && q_tok_stride % 8 == 0 && q_head_stride % 8 == 0 && o_tok_stride % 8 == 0 &&
                  o_head_stride % 8 == 0,
              "%s: q/out pointers and strides must be 16-byte aligned", what);
  PIE_REQUIRE(scratch && aligned16(scratch) && scratch_bytes >= info[kInfoScratch],
              "%s: needs %lld bytes of 16-byte-aligned scratch, got %lld", what, (long long)info[kInfoScratch],
              (long long)scratch_bytes);
  // a run hands its partial results from its first launch to its second
  InflightClaim claim;
  const InflightClaim::State got = claim.take(scratch, stream);
  if (got == InflightClaim::kBusy || got == InflightClaim::kShared) return inflight_busy(what);
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
  a.B = (int)info[kInfoBatch];
  a.splits = (int)info[kInfoSplits];
  // (prefill_item scales raw scores inside the exponent, where a zero scale would turn -inf into NaN)
  a.scale_log2 = sm_scale == 0.f ? 1e-30f : sm_scale * 1.4426950408889634f;
  a.part_o = static_cast<float*>(scratch);
  a.part_lse = a.part_o + info[kInfoRows] * head_dim;
  a.suffix_row = info[kInfoSuffixRow];
  const int32_t* tokens = plan + info[kInfoTokensWord];
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int T = (int)num_tokens, parts = (int)info[kInfoMaxParts];
  switch (head_dim) {
    case 64: launch_shared<64>(st, a, T, parts, tokens, out, o_tok_stride, o_head_stride, lse); break;
    case 128: launch_shared<128>(st, a, T, parts, tokens, out, o_tok_stride, o_head_stride, lse); break;
    default: launch_shared<256>(st, a, T, parts, tokens, out, o_tok_stride, o_head_stride, lse); break;
  }
  return check_launch(what);
}
