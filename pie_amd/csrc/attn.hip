// Paged attention over the KV cache the append kernels write: flashinfer's
// BatchDecodeWithPagedKVCacheWrapper.run and BatchPrefillWithPagedKVCacheWrapper.run as Pie
// calls them (pie/src/pie_worker/model/llama3.py:293-313, :689, :765-790; semantics restated in
// pie/src/flashinfer_metal/ops.py:163-282 and kernels/metal_attention_simdgroup_opt.metal).
//
// For request b with kv_len = (npages-1)*P + last_len[b] cached tokens and qo_len query tokens,
// query token i attends kv positions t <= kv_len - qo_len + i (or where the custom mask is set),
// head h reads kv head h / (Hq/Hkv), scores are q.k * sm_scale, output is softmax(scores) @ v.
//
// MI355X mapping. Decode runs the matrix products on MFMA v_mfma_f32_16x16x32_bf16 (prefill, below,
// on v_mfma_f32_32x32x16_bf16 with the output transposed):
//   S^T = K Q^T   A = 16 kv tokens x 32 head dims (straight from HBM into registers: lane
//                 (n, g) holds token n's dims 8(4s+g)..+8 at step s, one 64-byte run per token
//                 per step), B = 16 query rows (the same dims permutation), C = S^T tile with
//                 lane (n, g) holding tokens 4g..4g+3 of query row n;
//   O  = P V      A = the probabilities in exactly that C layout read as 8 tokens per lane
//                 (two 16-token subtiles: tokens 4g+i and 16+4g+i), B = V staged row-major in
//                 LDS and read with ds_read_b64_tr_b16, whose 16-lane transpose turns 4 rows x
//                 4 dims into the 8-tokens-of-one-dim operand the MFMA wants.
// The query rows of one MFMA tile are (token, head) pairs of one kv-head group (GQA packing),
// so a decode step with 4 heads per kv head shares every K/V byte between its 4 heads.
// Softmax is online in the exp2 domain (scores pre-multiplied by sm_scale*log2 e); P is
// rounded to bf16 for the second product as flashinfer does; everything else is fp32.
#include <math.h>

#include <string.h>

#include <algorithm>
#include <mutex>
#include <vector>

#include "attn_dev.h"

namespace pie {

template <int D, bool FIRST>
__global__ __launch_bounds__(256) void attn_decode_kernel(
    const uint16_t* __restrict__ q, int64_t q_ts, int64_t q_hs, PagedKV kv, int B, int G, int Hq,
    float scale_log2, int splits, int window_left, int first, uint16_t* __restrict__ out, int64_t o_ts,
    int64_t o_hs, float* __restrict__ part_o, float* __restrict__ part_lse,
    const float* __restrict__ sinks, float* __restrict__ lse) {
  __shared__ __attribute__((aligned(16))) char smem[decode_smem<D>()];
  __shared__ int32_t ptab[kPageWin];
  decode_unit<D, FIRST>(smem, ptab, blockIdx.x, q, q_ts, q_hs, kv, B, G, Hq, scale_log2, splits, window_left, first,
                        out, o_ts, o_hs, part_o, part_lse, sinks, lse);
}

// Combines the partial results of each (request, head): one work group per request and 512 / D
// heads. Splits past the end of the request's kv range wrote nothing and are not read. KB: plans of at
// most four splits need one load per wave; with eight (seven of them repeats of it) a decode layer of 45
// requests at 3 splits took 69.1 us, 68.0 with one.
template <int D, int KB>
__global__ __launch_bounds__(256) void attn_merge_kernel(PagedKV kv, int window_left, int first, int Hq, int splits,
                                                         const float* __restrict__ part_o,
                                                         const float* __restrict__ part_lse,
                                                         uint16_t* __restrict__ out, int64_t o_ts,
                                                         int64_t o_hs, const float* __restrict__ sinks,
                                                         float* __restrict__ lse) {
  constexpr int CH = D / 8;
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  const int hq = blockIdx.y * (64 / CH) + lane / CH, c = lane % CH;
  const int hl = min(hq, Hq - 1);  // lanes past the last head read its partials and write nothing
  const int kv_len = kv_length(kv, b);
  const int ns = split_count(visible_len(kv_len, window_left, first), splits);
  const int64_t row = (int64_t)b * splits * Hq + hl;
  float acc[8], L, M;
  merge_partials<D, KB>(part_o + 8 * c, part_lse, [&](int s) { return row + (int64_t)s * Hq; }, ns, splits, acc, L, M);
  if (threadIdx.x >= 64 || hq >= Hq) return;
  if (M != -INFINITY) L += sink_mass(sinks, hq, M);
  if (lse && c == 0) lse[(int64_t)b * Hq + hq] = row_lse(L, M);
  const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= inv;
  st16(out + (int64_t)b * o_ts + (int64_t)hq * o_hs + 8 * c, pack8(acc));
}

// A plan made for another head_dim cannot drive this kernel: every work group fills the whole
// output (the plan's tokens, all q heads) with NaN instead, so the mistake shows in the result
// rather than leaving the output unwritten.
template <int D>
__device__ void prefill_plan_mismatch(const int32_t* __restrict__ plan, const int32_t* __restrict__ qo_indptr,
                                      int Hq, uint16_t* __restrict__ out, int64_t o_ts, int64_t o_hs,
                                      float* __restrict__ lse) {
  const int t0 = qo_indptr[0], T = qo_indptr[plan[1]] - t0;
  constexpr int CH = D / 8;  // 16-byte chunks per head row
  const int64_t n = (int64_t)T * Hq * CH;
  const uint4 nan4 = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / (Hq * CH);
    const int h = (int)(i / CH % Hq), c = (int)(i % CH);
    *reinterpret_cast<uint4*>(out + (t0 + t) * o_ts + (int64_t)h * o_hs + 8 * c) = nan4;
    if (lse && c == 0) lse[(t0 + t) * Hq + h] = __builtin_nanf("");
  }
}

// Partial results of a split item (piece slot s, kv head h): 128 rows of D fp32 outputs
// (normalised) at part_o + (s * n_kv_heads + h) * 128 * D and their log2-sum-exps at
// part_lse + (s * n_kv_heads + h) * 128; attn_prefill_merge_kernel combines an item's pieces.
template <int D, bool FIRST>
__global__ __launch_bounds__(256, prefill_groups<D>()) void attn_prefill_kernel(
    const uint16_t* __restrict__ q, int64_t q_ts, int64_t q_hs, PagedKV kv,
    const int32_t* __restrict__ qo_indptr, int G, float scale_log2, const int32_t* __restrict__ plan,
    int items_word, int n_items, int n_kv_heads,
    int mode_in, int window_left, int first, const uint32_t* __restrict__ packed,
    const int64_t* __restrict__ word_off, const int32_t* __restrict__ extent,
    uint16_t* __restrict__ out, int64_t o_ts, int64_t o_hs, const float* __restrict__ sinks,
    float* __restrict__ part_o, float* __restrict__ part_lse, float* __restrict__ lse) {
  __shared__ __attribute__((aligned(16))) char smem[prefill_smem<D>()];
  __shared__ int32_t ptab[kPageWin];
  if (plan[2] != plan_rows_word(D)) {
    prefill_plan_mismatch<D>(plan, qo_indptr, G * n_kv_heads, out, o_ts, o_hs, lse);
    return;
  }
  const int u = prefill_unit(n_items * n_kv_heads);
  if (u < 0) return;  // padding work group
  const int kvh = u / n_items;
  const int32_t* item = plan + items_word + kPlanItemWords * (u - kvh * n_items);
  const int slot = uniform(item[7]) - 1;
  const int chunk = slot >= 0 ? uniform(plan[kPlanChunkWord]) : 0x7fffffff;
  const PrefillItem it = {uniform(item[0]), uniform(item[1]), uniform(item[2]), uniform(item[3]), uniform(item[4]),
                          uniform(item[5]), slot >= 0 ? uniform(item[6]) * chunk : 0, chunk,
                          slot >= 0 ? ((int64_t)slot * n_kv_heads + kvh) * kPrefillRows : -1};
  prefill_item<D, FIRST>(smem, ptab, it, q, q_ts, q_hs, kv, G, n_kv_heads, kvh, scale_log2, mode_in, window_left, first,
                         packed, word_off, extent, out, o_ts, o_hs, sinks, part_o, part_lse, lse);
}

// Head dim 128 with more units than the chip runs at once: the same products and work items in
// 32-token tiles with two tiles in flight in registers, on persistent work groups.
// Long prompts run alike on either kernel (8 x 8192 tokens: 4.76 ms here, 4.68 in
// attn_prefill_kernel); short ones, where a tile's overhang past the causal limit counts, are
// faster here (64 x U[1, 2048]: 963 against 980 us; 128 x 512: 623 against 659 us).
template <int D>
__global__ __launch_bounds__(256, 2) void attn_prefill32_kernel(
    const uint16_t* __restrict__ q, int64_t q_ts, int64_t q_hs, PagedKV kv,
    const int32_t* __restrict__ qo_indptr, int G, float scale_log2, const int32_t* __restrict__ plan,
    int n_items, int n_kv_heads,
    int mode_in, int window_left, const uint32_t* __restrict__ packed,
    const int64_t* __restrict__ word_off, const int32_t* __restrict__ extent,
    uint16_t* __restrict__ out, int64_t o_ts, int64_t o_hs, const float* __restrict__ sinks,
    float* __restrict__ lse) {
  static_assert(D == 128, "32x32 prefill is built for head_dim 128");
  constexpr int NS = D / 16;  // QK k-steps
  constexpr int NB = D / 32;  // 32-dim output blocks
  constexpr int CH = D / 8, RPI = 64 / CH;
  constexpr int kRows = 128, NT = 256;
  constexpr int TILE = kTileTokens * D;
  __shared__ __attribute__((aligned(16))) char smem[2 * 2 * TILE * 2];
  __shared__ int32_t ptab[kPageWin];
  __shared__ int window_bad;
  __shared__ uint32_t mwt[2][NT];

  // Persistent: each work group takes (kv head, item) units from its XCD's queue until every
  // queue is empty. XCD x's queue is the contiguous run [x * per, (x + 1) * per) of the units, in
  // plan order (each request's items together), so the work groups of one XCD share the K/V
  // prefix they read through its L2; a work group whose queue is empty takes from the others.
  if (plan[2] != plan_rows_word(D)) {
    prefill_plan_mismatch<D>(plan, qo_indptr, G * n_kv_heads, out, o_ts, o_hs, lse);
    return;
  }
  int32_t* counters = const_cast<int32_t*>(plan);
  __shared__ int s_unit;
  const int units = n_items * n_kv_heads, per = (units + 7) / 8;
  const int xcd = (int)(__builtin_amdgcn_s_getreg((20) | (0 << 6) | ((4 - 1) << 11)) & 7);  // HW_REG_XCC_ID
  int queue = 0;
  for (;;) {
  __syncthreads();  // the previous unit's LDS use (and s_unit) is done
  if (threadIdx.x == 0) {
    int u = -1;
    for (; queue < 8 && u < 0; ) {
      const int x = (xcd + queue) & 7;
      const int n = min(per, units - x * per);
      const int i = atomicAdd(&counters[kPlanQueueWord + x], 1);
      if (i < n) u = x * per + i; else ++queue;
    }
    s_unit = u;
  }
  __syncthreads();
  const int u = s_unit;
  if (u < 0) break;
  const int kvh = u / n_items;
  const int32_t* item = plan + kPlanHeader + kPlanItemWords * (u - kvh * n_items);
  const int b = item[0], row0 = item[1], q0 = item[2], qo_len = item[3], kv_len = item[4];
  const int page0 = item[5];
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  const int r32 = lane & 31, kg = lane >> 5;
  const int rows = qo_len * G;
  int mode = mode_in, mext = 0;  // a custom mask that is causal for all the rows: the causal path
  if (mode_in == 2) {
    bool causal;
    mask_rows_extent(extent, q0, row0, rows, G, kRows, mext, causal);
    mode = uniform(causal ? 1 : 2);  // wave-uniform (a scalar register), like the argument
  }

  // this lane's query row
  const int R = row0 + 32 * w + r32;
  const bool valid = R < rows;
  const int tok = valid ? R / G : 0, hg = valid ? R - tok * G : 0;
  const int lim = !valid ? -1 : mode == 1 ? min(kv_len - qo_len + tok, kv_len - 1) : kv_len - 1;
  const int lo = window_left >= 0 ? kv_len - qo_len + tok - window_left : 0;
  u32x4_t qb[NS];
  {
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

  const int last_row = min(rows, row0 + kRows) - 1;
  int kv_end = mode == 1 ? min(kv_len, kv_len - qo_len + last_row / G + 1) : kv_len;
  if (mode == 2) kv_end = min(kv_len, mext);
  const int kv_begin = window_left >= 0 ? max(0, kv_len - qo_len + row0 / G - window_left) & ~31 : 0;
  const int nw = (kv_len + 31) / 32;
  const uint32_t* mword = mode == 2 ? packed + word_off[b] + (int64_t)tok * nw : nullptr;
  // uniform bounds of the wave's rows: tiles inside [wave_lo, wave_lim] need no per-element test
  int wave_lim = valid ? lim : 0x7fffffff, wave_lo = valid ? lo : 0;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    wave_lim = min(wave_lim, __builtin_amdgcn_ds_bpermute((lane ^ off) << 2, wave_lim));
    wave_lo = max(wave_lo, __builtin_amdgcn_ds_bpermute((lane ^ off) << 2, wave_lo));
  }
  wave_lim = uniform(wave_lim);
  wave_lo = uniform(wave_lo);

  uint16_t* kt = reinterpret_cast<uint16_t*>(smem);  // [2 buffers][K, V][32][D]
  constexpr int WR = kTileTokens / 4;  // rows of each K / V tile one wave loads
  constexpr int NL = WR / RPI;
  struct Slot { u32x4_t k[NL], v[NL]; uint32_t mw; };
  const int win = max(kTileTokens, (kPageWin - 2) * kv.page_size / kTileTokens * kTileTokens);
  for (int wt0 = kv_begin; wt0 < kv_end; wt0 += win) {
    const int wt1 = min(kv_end, wt0 + win);
    const int lp0 = (int)kv.pdiv.div((uint32_t)wt0);
    const int npg = (int)kv.pdiv.div((uint32_t)(wt1 - 1)) - lp0 + 1;
    const int ntiles = (wt1 - wt0 + kTileTokens - 1) / kTileTokens;
    if (threadIdx.x == 0) window_bad = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < npg; i += NT) {
      const int pg = kv.indices[page0 + lp0 + i];
      ptab[i] = pg;
      if ((unsigned)pg >= (unsigned)kv.num_pages) window_bad = 1;
    }
    __syncthreads();
    const bool all_pages_ok = window_bad == 0;
    auto gload = [&](Slot& sl, int tile) {
      const int t0 = wt0 + tile * kTileTokens;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int r = WR * w + RPI * i + lane / CH;
        bool ok;
        const uint64_t off = kv_offset_lds(kv, ptab, lp0, min(t0 + r, wt1 - 1), kvh, ok);
        sl.k[i] = ld16v(kv.k + off + 8 * ((lane % CH) ^ chunk_swizzle<D>(r)));
        sl.v[i] = ld16v(kv.v + off + 8 * ((lane % CH) ^ v32_swizzle<D>(r)));
      }
      if (mode == 2) sl.mw = mword[t0 >> 5];
    };
    auto lwrite = [&](const Slot& sl, int tile) {
      uint16_t* kd = kt + (tile & 1) * 2 * TILE;
      if (mode == 2) mwt[tile & 1][threadIdx.x] = sl.mw;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        *reinterpret_cast<u32x4_t*>(kd + (WR * w + RPI * i) * D + 8 * lane) = sl.k[i];
        *reinterpret_cast<u32x4_t*>(kd + TILE + (WR * w + RPI * i) * D + 8 * lane) = sl.v[i];
      }
    };
    auto compute = [&](int tile) {
      const int t0 = wt0 + tile * kTileTokens;
      const uint16_t* kd = kt + (tile & 1) * 2 * TILE;
      // S^T: token r32 of the tile against this lane group's 32 rows
      f32x16_t sacc;
#pragma unroll
      for (int i = 0; i < 16; ++i) sacc[i] = 0.f;
      {
        const int z = chunk_swizzle<D>(r32);
        // K operands read four k-steps ahead of the MFMA chain. The schedule is pinned: left to
        // itself the compiler reads two ahead and exposes the LDS latency four times per tile.
        u32x4_t kr[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) kr[s] = *reinterpret_cast<const u32x4_t*>(kd + r32 * D + 8 * ((2 * s + kg) ^ z));
#pragma unroll
        for (int s = 0; s < NS; ++s) sacc = mfma_32x32x16(kr[s], qb[s], sacc);
        sched_group(0x100, 4);
#pragma unroll
        for (int s = 0; s < NS - 4; ++s) { sched_group(0x008, 1); sched_group(0x100, 1); }
        sched_group(0x008, 4);
      }
      // visibility of token tt(i) = 8(i/4) + 4kg + i%4 for this lane's row: mask bits by shifts,
      // then the per-element bounds only in tiles that cross a row's limit or window start
      uint32_t vis = 0xffffu;
      if (mode == 2) {
        const uint32_t mw = mwt[tile & 1][threadIdx.x];
        vis = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) vis |= ((mw >> (8 * c + 4 * kg)) & 15u) << (4 * c);
      }
      if (!all_pages_ok || t0 + kTileTokens - 1 > wave_lim || t0 < wave_lo) {
        uint64_t tv = 0xffffffffull;
        if (!all_pages_ok) {
          bool pok = false;
          if (lane < kTileTokens && t0 + lane < wt1) kv_offset_lds(kv, ptab, lp0, t0 + lane, kvh, pok);
          tv = __builtin_amdgcn_ballot_w64(pok);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int tt = 8 * (i >> 2) + 4 * kg + (i & 3), t = t0 + tt;
          if (!(t <= lim && t >= lo && ((tv >> tt) & 1ull))) vis &= ~(1u << i);
        }
      }
      // Scores stay raw (q.k) until the exponent, where one fma applies the scale: the row maximum
      // is taken over raw scores, negated when the scale is negative (a uniform branch), with
      // hidden entries set to the raw value that scales to -inf (the scale is never 0 here).
      const bool neg = scale_log2 < 0.f;
      const bool masked = __builtin_amdgcn_ballot_w64(vis != 0xffffu) != 0;
      if (masked) {
        const float hidden = neg ? INFINITY : -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) sacc[i] = ((vis >> i) & 1u) ? sacc[i] : hidden;
      }
      float mx = -INFINITY;
      if (!neg) {
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sacc[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, -sacc[i]);
      }
      mx = fmaxf(mx, lane_read(mx, lane ^ 32)) * fabsf(scale_log2);
      // lazy maximum (kLazyMax)
      if (__builtin_amdgcn_ballot_w64(mx > m_run + kLazyMax) != 0) {
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
      float sc[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = fast_exp2(fmaf(sacc[i], scale_log2, -m_use));
      // the row's partial sum as a tree (a chain of 16 dependent adds sat on the critical path)
      float ps[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ps[i] = (sc[4 * i] + sc[4 * i + 1]) + (sc[4 * i + 2] + sc[4 * i + 3]);
      l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
      u32x4_t pb[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        pb[j] = u32x4_t{pack_bf2(sc[8 * j], sc[8 * j + 1]), pack_bf2(sc[8 * j + 2], sc[8 * j + 3]),
                        pack_bf2(sc[8 * j + 4], sc[8 * j + 5]), pack_bf2(sc[8 * j + 6], sc[8 * j + 7])};
      // O^T += V^T P^T. Transpose-read source lanes: group G16 = lane / 16 reads rows
      // 16j + 8h + 4kg + (lane%16)/4 (h: first or second 4 tokens), dims 32bb + 16(G16%2) + 4(lane%4)
      const int g16 = lane >> 4, jj = (lane >> 2) & 3, qq = lane & 3;
      const uint16_t* vbase = kd + TILE;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int bb = 0; bb < NB; ++bb) {
          uint2 hv[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = 16 * j + 8 * h + 4 * kg + jj;
            const int dim = 32 * bb + 16 * (g16 & 1) + 4 * qq;
            const int c = (dim >> 3) ^ v32_swizzle<D>(r);
            hv[h] = lds_read_tr16(vbase + r * D + 8 * c + (dim & 7));
          }
          const u32x4_t va = {hv[0].x, hv[0].y, hv[1].x, hv[1].y};
          o[bb] = mfma_32x32x16(va, pb[j], o[bb]);
        }
    };
    Slot sa, sb;
    gload(sa, 0);
    if (ntiles > 1) gload(sb, 1);
    lwrite(sa, 0);
    if (ntiles > 2) gload(sa, 2);
    __syncthreads();
    for (int k = 0;;) {
      compute(k);
      if (k + 1 < ntiles) {
        lwrite(sb, k + 1);
        if (k + 3 < ntiles) gload(sb, k + 3);
      }
      __syncthreads();
      if (++k >= ntiles) break;
      compute(k);
      if (k + 1 < ntiles) {
        lwrite(sa, k + 1);
        if (k + 3 < ntiles) gload(sa, k + 3);
      }
      __syncthreads();
      if (++k >= ntiles) break;
    }
  }
  // normalise and write: o[bb][i] is dim 32bb + 8(i/4) + 4kg + i%4 of row R; lanes r and r^32
  // together cover 8 consecutive dims
  float L = l_run + lane_read(l_run, lane ^ 32);
  if (valid) L += sink_mass(sinks, kvh * G + hg, m_run);
  if (lse && valid && kg == 0) lse[(int64_t)(q0 + tok) * (G * n_kv_heads) + kvh * G + hg] = row_lse(L, m_run);
  const float inv = L > 0.f ? 1.f / L : 0.f;
  if (valid) {
    uint16_t* op = out + (int64_t)(q0 + tok) * o_ts + (int64_t)(kvh * G + hg) * o_hs;
#pragma unroll
    for (int bb = 0; bb < NB; ++bb)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint2 v = {pack_bf2(o[bb][4 * c] * inv, o[bb][4 * c + 1] * inv),
                         pack_bf2(o[bb][4 * c + 2] * inv, o[bb][4 * c + 3] * inv)};
        *reinterpret_cast<uint2*>(op + 32 * bb + 8 * c + 4 * kg) = v;
      }
  }
  }
  // the last work group out resets the counters for the next launch with this plan; the fence
  // orders this group's queue atomics before its done count
  __threadfence();
  if (threadIdx.x == 0 && atomicAdd(&counters[kPlanDoneWord], 1) == (int)gridDim.x - 1) {
    for (int x = 0; x < 8; ++x) atomicExch(&counters[kPlanQueueWord + x], 0);
    atomicExch(&counters[kPlanDoneWord], 0);
  }
}

// Combines the pieces of split items: work group x takes (merge entry, kv head) x and 512 / D of
// its 128 rows. (A plan that attn_prefill_kernel could not use has no pieces: its NaN stays.)
template <int D>
__global__ __launch_bounds__(256) void attn_prefill_merge_kernel(
    const int32_t* __restrict__ plan, int merges_word, int n_kv_heads, int G, const float* __restrict__ part_o,
    const float* __restrict__ part_lse, uint16_t* __restrict__ out, int64_t o_ts, int64_t o_hs,
    const float* __restrict__ sinks, float* __restrict__ lse) {
  constexpr int CH = D / 8;
  const int e = blockIdx.x / n_kv_heads, kvh = blockIdx.x - e * n_kv_heads;
  const int32_t* m = plan + merges_word + kPlanMergeWords * e;
  const int row0 = m[0], q0 = m[1], rows = m[2] * G, slot = m[3], pieces = m[4];
  if (m[5] != kMergeTag + plan_rows_word(D)) return;  // (in the entry: the header is a load more to wait for)
  const int lane = threadIdx.x & 63, c = lane % CH;
  const int rl0 = blockIdx.y * (64 / CH);
  if (row0 + rl0 >= rows) return;
  const int R = min(row0 + rl0 + lane / CH, rows - 1);  // lanes past the last row repeat it
  const int64_t first = ((int64_t)slot * n_kv_heads + kvh) * kPrefillRows + (R - row0);
  const int64_t step = (int64_t)n_kv_heads * kPrefillRows;
  float acc[8], L, M;
  merge_partials<D, 8>(part_o + 8 * c, part_lse, [&](int s) { return first + s * step; }, pieces, pieces, acc, L, M);
  if (threadIdx.x >= 64 || row0 + rl0 + lane / CH >= rows) return;
  const int tok = R / G, hq = kvh * G + (R - tok * G);
  if (M != -INFINITY) L += sink_mass(sinks, hq, M);
  if (lse && c == 0) lse[(int64_t)(q0 + tok) * (G * n_kv_heads) + hq] = row_lse(L, M);
  const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] *= inv;
  st16(out + (int64_t)(q0 + tok) * o_ts + (int64_t)hq * o_hs + 8 * c, pack8(acc));
}

}  // namespace pie

using namespace pie;

// Host: how many splits per request, for per = batch * kv heads work groups a split. A work group
// costs ~4 us before and after its tokens (ranking, page table, first loads, merge), so where per
// fills at most half the CUs a launch aims at the ~2 work groups per CU that run at once, and at more,
// which evens out requests of different lengths, as per grows: 3 per CU below one per CU, 4 from
// there (batches of at most kRankMax, longest requests first; larger batches ~16: request order
// leaves a longer tail). Measured (us, cache cold, Llama-8B heads): 8 x 500-4,000 tokens 8 splits
// 24.0, 16 27.1; 3 x 16-32k 21 splits 80.7, 43 84.9; 24 x 128-4,096 4 splits 53.2, 6 55.1, 2 58.7;
// 32 x 128-4,096 4 splits 73.4, 1 76.7. When the longest context is known (max_kv_len >= 0) no split
// is shorter than kMinChunk tokens. The result depends on the batch only, so one plan serves a
// captured graph.
extern "C" int pie_hip_attention_decode_plan(int64_t batch, int64_t num_kv_heads, int64_t max_kv_len,
                                             int64_t num_cus, int64_t* splits) {
  PIE_REQUIRE(splits && batch >= 0 && num_kv_heads > 0, "decode_plan: bad batch %lld / num_kv_heads %lld",
              (long long)batch, (long long)num_kv_heads);
  const int64_t cus = num_cus > 0 ? num_cus : 256;
  const int64_t per = std::max<int64_t>(1, batch * num_kv_heads);
  int64_t s = batch > kRankMax ? (16 * cus + per - 1) / per
              : per >= cus     ? (4 * cus + per - 1) / per
              : 2 * per > cus  ? 3 * cus / per
                               : 2 * cus / per;
  if (max_kv_len >= 0) s = std::min<int64_t>(s, std::max<int64_t>(1, (max_kv_len + kMinChunk - 1) / kMinChunk));
  *splits = std::max<int64_t>(1, std::min<int64_t>(s, 64));
  return PIE_HIP_OK;
}

int pie::paged_kv_desc(PagedKV* kv, const uint16_t* k_cache, const uint16_t* v_cache,
                         int64_t page_stride, int64_t slot_stride, int64_t head_stride,
                         int64_t num_pages, const int32_t* kv_indptr, const int32_t* kv_indices,
                         const int32_t* kv_last_page_len, int64_t page_size, int64_t D,
                         const char* what) {
  PIE_REQUIRE(k_cache && v_cache && kv_indptr && kv_indices && kv_last_page_len, "%s: null cache or page table", what);
  PIE_REQUIRE(page_size > 0 && page_size <= 65536 && num_pages > 0 && num_pages < (1ll << 31),
              "%s: bad page_size %lld / num_pages %lld", what, (long long)page_size, (long long)num_pages);
  PIE_REQUIRE(aligned16(k_cache) && aligned16(v_cache) && page_stride % 8 == 0 && slot_stride % 8 == 0 &&
                  head_stride % 8 == 0,
              "%s: cache pointers and strides must be 16-byte aligned", what);
  (void)D;
  kv->k = k_cache;
  kv->v = v_cache;
  kv->page_stride = page_stride;
  kv->slot_stride = slot_stride;
  kv->head_stride = head_stride;
  kv->indptr = kv_indptr;
  kv->indices = kv_indices;
  kv->last_len = kv_last_page_len;
  kv->num_pages = (int32_t)num_pages;
  kv->page_size = (int32_t)page_size;
  kv->pdiv = FastDiv::make((uint32_t)page_size);
  return PIE_HIP_OK;
}

template <int D>
static void launch_decode(hipStream_t st, const uint16_t* q, int64_t q_ts, int64_t q_hs,
                          const PagedKV& kv, int G, int Hq, int Hkv, float sl2, int B, int splits,
                          int window_left, int first, uint16_t* out, int64_t o_ts, int64_t o_hs, float* po,
                          float* pl, const float* sinks, float* lse) {
  hipLaunchKernelGGL((first ? attn_decode_kernel<D, true> : attn_decode_kernel<D, false>), dim3(B * splits * Hkv),
                     dim3(256), 0, st, q, q_ts, q_hs, kv, B, G, Hq, sl2, splits, window_left, first, out, o_ts, o_hs,
                     po, pl, sinks, lse);
  if (splits > 1)
    hipLaunchKernelGGL((splits <= 4 ? attn_merge_kernel<D, 1> : attn_merge_kernel<D, 8>),
                       dim3(B, (Hq + 64 / (D / 8) - 1) / (64 / (D / 8))), dim3(256), 0, st, kv, window_left, first, Hq, splits,
                       po, pl, out, o_ts, o_hs, sinks, lse);
}

// The kernels' first tokens: none where no window hides anything.
static int first_within(int window_left, int64_t first_tokens) {
  return window_left < 0 ? 0 : (int)std::min<int64_t>(first_tokens, 0x7fffffff);
}

static int attention_decode_impl(
    const pie_bf16* q, int64_t q_tok_stride, int64_t q_head_stride, const pie_bf16* k_cache,
    const pie_bf16* v_cache, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
    int64_t num_pages, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t batch, int64_t num_qo_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t page_size, float sm_scale, int64_t window_left, int64_t first_tokens, const float* sinks,
    int64_t splits, void* workspace, int64_t workspace_bytes, pie_bf16* out, int64_t o_tok_stride,
    int64_t o_head_stride, float* lse, void* stream, const char* what) {
  PagedKV kv;
  int rc = paged_kv_desc(&kv, k_cache, v_cache, page_stride, slot_stride, head_stride, num_pages,
                         kv_indptr, kv_indices, kv_last_page_len, page_size, head_dim,
                         what);
  if (rc) return rc;
  PIE_REQUIRE(q && out, "attention_decode: null q or out");
  PIE_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256,
              "attention_decode: head_dim %lld not in {64, 128, 256}", (long long)head_dim);
  PIE_REQUIRE(num_kv_heads > 0 && num_qo_heads % num_kv_heads == 0 && num_qo_heads / num_kv_heads <= 16 &&
                  num_kv_heads <= 65535,
              "attention_decode: need num_qo_heads = G * num_kv_heads with G <= 16 (got %lld / %lld)",
              (long long)num_qo_heads, (long long)num_kv_heads);
  PIE_REQUIRE(batch >= 0 && splits >= 1 && splits <= 64 && batch * splits * num_kv_heads < (1ll << 31),
              "attention_decode: bad batch %lld / splits %lld", (long long)batch, (long long)splits);
  PIE_REQUIRE(aligned16(q) && aligned16(out) && q_tok_stride % 8 == 0 && q_head_stride % 8 == 0 &&
                  o_tok_stride % 8 == 0 && o_head_stride % 8 == 0,
              "attention_decode: q/out pointers and strides must be 16-byte aligned");
  PIE_REQUIRE(first_tokens >= 0, "%s: first_tokens %lld is negative", what, (long long)first_tokens);
  PIE_REQUIRE(!lse || !sinks, "%s: no log-sum-exp of attention with sinks", what);
  const int64_t slots = splits > 1 ? batch * splits : 0;
  const int64_t need = slots * num_qo_heads * (head_dim + 1) * 4;
  PIE_REQUIRE(slots == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
              "%s: workspace of %lld bytes < %lld needed for %lld splits", what,
              (long long)workspace_bytes, (long long)need, (long long)splits);
  if (batch == 0) return PIE_HIP_OK;
  float* po = static_cast<float*>(workspace);
  float* pl = po ? po + slots * num_qo_heads * head_dim : nullptr;
  const int G = (int)(num_qo_heads / num_kv_heads);
  const float sl2 = sm_scale * 1.4426950408889634f;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int B = (int)batch, S = (int)splits, Hq = (int)num_qo_heads, Hkv = (int)num_kv_heads;
  const int W = window_left < 0 ? -1 : (int)std::min<int64_t>(window_left, 1 << 30);
  const int F = first_within(W, first_tokens);
  switch (head_dim) {
    case 64: launch_decode<64>(st, q, q_tok_stride, q_head_stride, kv, G, Hq, Hkv, sl2, B, S, W, F, out,
                               o_tok_stride, o_head_stride, po, pl, sinks, lse); break;
    case 128: launch_decode<128>(st, q, q_tok_stride, q_head_stride, kv, G, Hq, Hkv, sl2, B, S, W, F, out,
                                 o_tok_stride, o_head_stride, po, pl, sinks, lse); break;
    default: launch_decode<256>(st, q, q_tok_stride, q_head_stride, kv, G, Hq, Hkv, sl2, B, S, W, F, out,
                                o_tok_stride, o_head_stride, po, pl, sinks, lse); break;
  }
  return check_launch(what);
}

extern "C" int pie_hip_attention_decode(
    const pie_bf16* q, int64_t q_tok_stride, int64_t q_head_stride, const pie_bf16* k_cache,
    const pie_bf16* v_cache, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
    int64_t num_pages, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t batch, int64_t num_qo_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t page_size, float sm_scale, int64_t window_left, const float* sinks, int64_t splits,
    void* workspace, int64_t workspace_bytes, pie_bf16* out, int64_t o_tok_stride,
    int64_t o_head_stride, void* stream) {
  return attention_decode_impl(q, q_tok_stride, q_head_stride, k_cache, v_cache, page_stride,
                               slot_stride, head_stride, num_pages, kv_indptr, kv_indices,
                               kv_last_page_len, batch, num_qo_heads, num_kv_heads, head_dim,
                               page_size, sm_scale, window_left, 0, sinks, splits, workspace, workspace_bytes,
                               out, o_tok_stride, o_head_stride, nullptr, stream, "attention_decode");
}

extern "C" int pie_hip_attention_decode_lse(
    const pie_bf16* q, int64_t q_tok_stride, int64_t q_head_stride, const pie_bf16* k_cache,
    const pie_bf16* v_cache, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
    int64_t num_pages, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t batch, int64_t num_qo_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t page_size, float sm_scale, int64_t window_left, int64_t first_tokens, const float* sinks,
    int64_t splits, void* workspace, int64_t workspace_bytes, pie_bf16* out, int64_t o_tok_stride,
    int64_t o_head_stride, float* lse, void* stream) {
  return attention_decode_impl(q, q_tok_stride, q_head_stride, k_cache, v_cache, page_stride,
                               slot_stride, head_stride, num_pages, kv_indptr, kv_indices,
                               kv_last_page_len, batch, num_qo_heads, num_kv_heads, head_dim,
                               page_size, sm_scale, window_left, first_tokens, sinks, splits, workspace,
                               workspace_bytes, out, o_tok_stride, o_head_stride, lse, stream, "attention_decode_lse");
}

// ---------------------------------------------------------------- decode without allocation
// The split partials (fp32 outputs + log2-sum-exp per (slot, head)) live in a file-scope device
// array instead of a caller workspace, for callers that cannot allocate. Each device holds its
// own copy; host code uses only the address hipGetSymbolAddress returns for the current device
// (the array's name is a host-side stand-in, never a device address). Every partial a run
// reads is written earlier in the same run (empty splits write nothing and are not read), so the
// array needs no clearing between calls; calls that overlap on one device race on it.
constexpr int64_t kDecodeScratchBytes = 32ll << 20;
static __device__ __align__(256) char scratch[kDecodeScratchBytes];

static std::mutex g_scratch_mu;
static void* g_scratch_dev[64] = {nullptr};

static int decode_scratch(void** out) {
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess || dev < 0 || dev >= 64)
    return set_error(PIE_HIP_ELAUNCH, "attention_decode_noalloc: no current device (%s)", hipGetErrorString(e));
  std::lock_guard<std::mutex> lk(g_scratch_mu);
  if (!g_scratch_dev[dev]) {
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !p)
      return set_error(PIE_HIP_ELAUNCH, "attention_decode_noalloc: hipGetSymbolAddress failed on device %d: %s",
                       dev, hipGetErrorString(e));
    g_scratch_dev[dev] = p;
  }
  *out = g_scratch_dev[dev];
  return PIE_HIP_OK;
}

extern "C" int pie_hip_attention_decode_noalloc(
    const pie_bf16* q, int64_t q_tok_stride, int64_t q_head_stride, const pie_bf16* k_cache,
    const pie_bf16* v_cache, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
    int64_t num_pages, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t batch, int64_t num_qo_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t page_size, float sm_scale, int64_t window_left, const float* sinks, int64_t splits,
    pie_bf16* out, int64_t o_tok_stride, int64_t o_head_stride, void* stream) {
  const char* what = "attention_decode_noalloc";
  PIE_REQUIRE(batch >= 0 && splits >= 1 && splits <= 64 && num_qo_heads > 0 && head_dim > 0,
              "%s: bad batch %lld / splits %lld", what, (long long)batch, (long long)splits);
  const int64_t need = splits > 1 ? batch * splits * num_qo_heads * (head_dim + 1) * 4 : 0;
  PIE_REQUIRE(need <= kDecodeScratchBytes,
              "%s: %lld bytes of split partials exceed the %lld-byte static scratch (use fewer splits "
              "or pie_hip_attention_decode with a workspace)",
              what, (long long)need, (long long)kDecodeScratchBytes);
  void* ws = nullptr;
  InflightClaim claim;
  if (need > 0) {
    const int rc = decode_scratch(&ws);
    if (rc) return rc;
    if (claim.take(ws, stream) == InflightClaim::kBusy) return inflight_busy(what);
  }
  return attention_decode_impl(q, q_tok_stride, q_head_stride, k_cache, v_cache, page_stride,
                               slot_stride, head_stride, num_pages, kv_indptr, kv_indices,
                               kv_last_page_len, batch, num_qo_heads, num_kv_heads, head_dim,
                               page_size, sm_scale, window_left, 0, sinks, splits, ws, kDecodeScratchBytes,
                               out, o_tok_stride, o_head_stride, nullptr, stream, what);
}

// Host: the prefill work list. Reads host copies of qo_indptr, kv_indptr and kv_last_page_len
// (as flashinfer's plan does); lists (request, first row) items of kPrefillRows packed rows,
// those that see the most kv positions first, and for mode 2 the byte offset of every
// request's [qo_len, kv_len] mask block (int64, 8-byte aligned in the plan). With `split`, a second
// list after them cuts the items that would outlast the rest of the launch over their kv range.
struct PrefillSplit {
  int64_t window_left, first, num_cus, workspace_bytes;
  int64_t items_word = 0, num_items = 0, merges_word = 0, num_merges = 0, scratch_bytes = 0;
};

// The rule of the split list. Without it a request's rows walk its whole context in one work group:
// 13 drafted tokens each over 4 contexts of 1-9k tokens took 253 us on 32 work groups and take 32 us
// in 256-to-320-token pieces; one 700-token prompt 100 us, and 30 us. A launch is counted as
// num_cus * prefill_groups work groups (head dim 64 as 128, two per CU, although three fit); their mean
// share of the kv tokens (over all items and kv heads) is the length a piece aims at, at least
// kSplitMinChunk, below which a piece is mostly set-up. A custom mask is not looked at: its items count
// their whole context, also where the mask is causal and the kernel stops sooner. Items are cut only
// when the longest exceeds its pieces by kSplitMinGain tokens: less than that the merge launch costs
// more than the cut saves.
constexpr int64_t kSplitMinChunk = 256, kSplitMinGain = 512;

// Bytes of the partial results of `pieces` pieces: kPrefillRows rows of D outputs and a log-sum-exp each.
static int64_t prefill_scratch_bytes(int64_t pieces, int64_t num_kv_heads, int64_t head_dim) {
  return pieces * num_kv_heads * kPrefillRows * (head_dim + 1) * 4;
}

static int prefill_plan_impl(const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_last_page_len,
                             int64_t batch, int64_t page_size, int64_t num_qo_heads, int64_t num_kv_heads,
                             int64_t head_dim, int32_t mode, int32_t* plan, int64_t plan_capacity,
                             int64_t* plan_words, int64_t* num_items, int64_t* mask_bytes, int64_t* mask_words,
                             PrefillSplit* split) {
  PIE_REQUIRE(qo_indptr && kv_indptr && kv_last_page_len && plan && plan_words && num_items && mask_bytes &&
                  mask_words,
              "prefill_plan: null argument");
  PIE_REQUIRE(batch >= 0 && batch < (1 << 24) && page_size > 0 && num_kv_heads > 0 &&
                  num_qo_heads % num_kv_heads == 0 && mode >= 0 && mode <= 2,
              "prefill_plan: bad batch %lld / page_size %lld / heads %lld,%lld / mode %d",
              (long long)batch, (long long)page_size, (long long)num_qo_heads,
              (long long)num_kv_heads, mode);
  PIE_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256,
              "prefill_plan: head_dim %lld not in {64, 128, 256}", (long long)head_dim);
  const int64_t G = num_qo_heads / num_kv_heads;
  struct Item { int32_t b, row0, q0, qo, kv, page0; int64_t work, req_work, span; };
  std::vector<Item> items;
  std::vector<int64_t> moff((size_t)batch + 1, 0), woff((size_t)batch + 1, 0);
  int64_t mtotal = 0, wtotal = 0;
  for (int64_t b = 0; b < batch; ++b) {
    const int64_t qo = (int64_t)qo_indptr[b + 1] - qo_indptr[b];
    const int64_t np = (int64_t)kv_indptr[b + 1] - kv_indptr[b];
    PIE_REQUIRE(qo >= 0 && np >= 0, "prefill_plan: indptr decreases at request %lld", (long long)b);
    const int64_t kv = np > 0 ? (np - 1) * page_size + kv_last_page_len[b] : 0;
    PIE_REQUIRE(kv >= 0 && kv < (mode == 2 ? kExtentCausal : (1ll << 31)) && qo * G < (1ll << 31),
                "prefill_plan: request %lld too long", (long long)b);
    moff[(size_t)b] = mtotal;
    woff[(size_t)b] = wtotal;
    mtotal += qo * kv;
    wtotal += qo * ((kv + 31) / 32);
    for (int64_t r0 = 0; r0 < qo * G; r0 += kPrefillRows) {
      const int64_t last = std::min(qo * G, r0 + kPrefillRows) - 1;
      const int64_t seen = mode == 1 ? std::max<int64_t>(0, std::min(kv, kv - qo + last / G + 1)) : kv;
      // the kernel's kv range: from the first row's window start, 32-aligned
      const int64_t wl = split ? split->window_left : -1;
      const int64_t begin = wl >= 0 ? std::max<int64_t>(0, kv - qo + r0 / G - wl) / 32 * 32 : 0;
      // and the kept first tokens before it, in whole tiles, or from 0 where they reach it
      const int64_t first = split && wl >= 0 ? split->first : 0, kept = std::min(first, seen);
      const int64_t span = begin > 0 && first < begin ? (kept + 63) / 64 * 64 + std::max<int64_t>(0, seen - begin)
                           : first > 0                ? seen
                                                      : std::max<int64_t>(0, seen - begin);
      items.push_back(Item{(int32_t)b, (int32_t)r0, qo_indptr[b], (int32_t)qo, (int32_t)kv, kv_indptr[b],
                           seen, kv * qo, span});
    }
  }
  // Each request's items stay together (they share its K/V prefix, which the kernels' XCD-aware
  // order keeps in one L2): longest requests first, and in each request the items that see the
  // most K/V first, so the shortest work comes last.
  std::stable_sort(items.begin(), items.end(), [](const Item& x, const Item& y) {
    if (x.req_work != y.req_work) return x.req_work > y.req_work;
    if (x.b != y.b) return x.b < y.b;
    return x.work > y.work;
  });
  int64_t words = kPlanHeader + kPlanItemWords * (int64_t)items.size();
  words = (words + 1) / 2 * 2;  // int64 mask offsets start 8-byte aligned
  moff[(size_t)batch] = mtotal;
  woff[(size_t)batch] = wtotal;
  const int64_t moff_word = words, woff_word = words + 2 * (batch + 1);
  if (mode == 2) words += 4 * (batch + 1);
  *num_items = (int64_t)items.size();
  *mask_bytes = mtotal;
  *mask_words = wtotal;
  int64_t chunk = 0;
  if (split && !items.empty()) {
    int64_t total = 0, longest = 0;
    for (const Item& it : items) {
      total += it.span;
      longest = std::max(longest, it.span);
    }
    const int64_t groups = (head_dim == 256 ? prefill_groups<256>() : prefill_groups<128>()) *
                           (split->num_cus > 0 ? split->num_cus : 256);
    chunk = std::max(kSplitMinChunk, (total * num_kv_heads + groups - 1) / groups);
    chunk = (chunk + 63) / 64 * 64;
    for (; longest >= chunk + kSplitMinGain; chunk *= 2) {  // longer pieces where the scratch is short
      int64_t pieces = 0, cut = 0, whole = 0;
      for (const Item& it : items) {
        const int64_t n = (it.span + chunk - 1) / chunk;
        if (n > 1) { pieces += n; ++cut; } else ++whole;
      }
      const int64_t all = words + kPlanItemWords * (pieces + whole) + kPlanMergeWords * cut;
      const int64_t scratch = prefill_scratch_bytes(pieces, num_kv_heads, head_dim);
      const int64_t masks = mode == 2 ? (wtotal * 4 + 15) / 16 * 16 + qo_indptr[batch] * 4ll : 0;
      if (all <= plan_capacity && (all * 4 + 15) / 16 * 16 + (masks + 15) / 16 * 16 + scratch <= split->workspace_bytes &&
          (pieces + whole) * num_kv_heads < (1ll << 31)) {
        split->items_word = words;
        split->num_items = pieces + whole;
        split->merges_word = words + kPlanItemWords * (pieces + whole);
        split->num_merges = cut;
        split->scratch_bytes = scratch;
        words = all;
        break;
      }
    }
  }
  *plan_words = words;
  PIE_REQUIRE(words <= plan_capacity, "prefill_plan: needs %lld words, capacity %lld",
              (long long)words, (long long)plan_capacity);
  for (int i = 0; i < kPlanHeader; ++i) plan[i] = 0;
  plan[0] = (int32_t)items.size();
  plan[1] = (int32_t)batch;
  plan[2] = plan_rows_word(head_dim);
  plan[3] = (int32_t)moff_word;  // mode 2: int64 byte offsets of the mask blocks [batch + 1]
  plan[4] = (int32_t)woff_word;  // mode 2: int64 offsets of the packed mask words [batch + 1]
  plan[kPlanChunkWord] = split && split->num_items ? (int32_t)chunk : 0;
  // [7] and [8, 16): the persistent kernel's work counters (zero between launches)
  const auto put = [](int32_t* p, const Item& it, int32_t piece, int32_t slot1) {
    const int32_t w8[kPlanItemWords] = {it.b, it.row0, it.q0, it.qo, it.kv, it.page0, piece, slot1};
    memcpy(p, w8, sizeof(w8));
  };
  int32_t* p = plan + kPlanHeader;
  for (const Item& it : items) { put(p, it, 0, 0); p += kPlanItemWords; }
  if (mode == 2) {
    memcpy(plan + moff_word, moff.data(), sizeof(int64_t) * (size_t)(batch + 1));
    memcpy(plan + woff_word, woff.data(), sizeof(int64_t) * (size_t)(batch + 1));
  }
  if (split && split->num_items) {
    int32_t slot = 0;
    int32_t* m = plan + split->merges_word;
    p = plan + split->items_word;
    for (const Item& it : items) {
      const int32_t n = (int32_t)((it.span + chunk - 1) / chunk);
      if (n <= 1) { put(p, it, 0, 0); p += kPlanItemWords; continue; }
      const int32_t w8[kPlanMergeWords] = {it.row0, it.q0, it.qo, slot, n, kMergeTag + plan_rows_word(head_dim), 0, 0};
      memcpy(m, w8, sizeof(w8));
      m += kPlanMergeWords;
      for (int32_t i = 0; i < n; ++i) { put(p, it, i, ++slot); p += kPlanItemWords; }
    }
  }
  return PIE_HIP_OK;
}

extern "C" int pie_hip_attention_prefill_plan(const int32_t* qo_indptr, const int32_t* kv_indptr,
                                              const int32_t* kv_last_page_len, int64_t batch,
                                              int64_t page_size, int64_t num_qo_heads,
                                              int64_t num_kv_heads, int64_t head_dim, int32_t mode,
                                              int32_t* plan,
                                              int64_t plan_capacity, int64_t* plan_words,
                                              int64_t* num_items, int64_t* mask_bytes,
                                              int64_t* mask_words) {
  return prefill_plan_impl(qo_indptr, kv_indptr, kv_last_page_len, batch, page_size, num_qo_heads, num_kv_heads,
                           head_dim, mode, plan, plan_capacity, plan_words, num_items, mask_bytes, mask_words,
                           nullptr);
}

// split[6]: the window a plan's pieces are cut for, and its first tokens.
static int64_t window_key(int64_t window_left, int64_t first_tokens) {
  const int64_t first = first_within(window_left < 0 ? -1 : 0, first_tokens);
  return first ? (1ll << 62) + (first << 31) + std::min<int64_t>(window_left, 1 << 30) : std::max<int64_t>(window_left, -1);
}

static int prefill_split_plan_impl(
    const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_last_page_len, int64_t batch,
    int64_t page_size, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim, int32_t mode,
    int64_t window_left, int64_t first_tokens, int64_t num_cus, int64_t workspace_bytes, int32_t* plan,
    int64_t plan_capacity, int64_t* plan_words, int64_t* num_items, int64_t* mask_bytes, int64_t* mask_words,
    int64_t* split) {
  PIE_REQUIRE(split, "prefill_split_plan: null argument");
  PIE_REQUIRE(first_tokens >= 0, "prefill_split_plan: first_tokens %lld is negative", (long long)first_tokens);
  PrefillSplit sp{window_left, std::min<int64_t>(first_tokens, 0x7fffffff), num_cus, workspace_bytes};
  const int rc = prefill_plan_impl(qo_indptr, kv_indptr, kv_last_page_len, batch, page_size, num_qo_heads,
                                   num_kv_heads, head_dim, mode, plan, plan_capacity, plan_words, num_items,
                                   mask_bytes, mask_words, &sp);
  if (rc) return rc;
  split[0] = sp.items_word;
  split[1] = sp.num_items;
  split[2] = sp.merges_word;
  split[3] = sp.num_merges;
  split[4] = sp.scratch_bytes;
  split[5] = mode;
  split[6] = window_key(window_left, first_tokens);
  return PIE_HIP_OK;
}

extern "C" int pie_hip_attention_prefill_split_plan(
    const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_last_page_len, int64_t batch,
    int64_t page_size, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim, int32_t mode,
    int64_t window_left, int64_t num_cus, int64_t workspace_bytes, int32_t* plan, int64_t plan_capacity,
    int64_t* plan_words, int64_t* num_items, int64_t* mask_bytes, int64_t* mask_words, int64_t* split) {
  return prefill_split_plan_impl(qo_indptr, kv_indptr, kv_last_page_len, batch, page_size, num_qo_heads, num_kv_heads,
                                 head_dim, mode, window_left, 0, num_cus, workspace_bytes, plan, plan_capacity,
                                 plan_words, num_items, mask_bytes, mask_words, split);
}

extern "C" int pie_hip_attention_prefill_first_plan(
    const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_last_page_len, int64_t batch,
    int64_t page_size, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim, int32_t mode,
    int64_t window_left, int64_t first_tokens, int64_t num_cus, int64_t workspace_bytes, int32_t* plan,
    int64_t plan_capacity, int64_t* plan_words, int64_t* num_items, int64_t* mask_bytes, int64_t* mask_words,
    int64_t* split) {
  return prefill_split_plan_impl(qo_indptr, kv_indptr, kv_last_page_len, batch, page_size, num_qo_heads, num_kv_heads,
                                 head_dim, mode, window_left, first_tokens, num_cus, workspace_bytes, plan,
                                 plan_capacity, plan_words, num_items, mask_bytes, mask_words, split);
}

struct PrefillLaunch {
  hipStream_t st;
  const uint16_t* q;
  int64_t q_ts, q_hs;
  PagedKV kv;
  const int32_t* qo_indptr;
  int G, Hkv;
  float sl2;
  const int32_t* plan;
  int items_word, n_items, mode, window_left;
  const uint32_t* packed;
  const int64_t* woff;
  const int32_t* extent;
  uint16_t* out;
  int64_t o_ts, o_hs;
  const float* sinks;
  int first;
  float* lse;
  int merges_word, n_merges;
  float *part_o, *part_lse;
};

template <int D>
static void launch_prefill(const PrefillLaunch& a) {
  // the kernel scales raw scores inside the exponent, where a zero scale would turn a hidden
  // (-inf) score into NaN; 1e-30 gives the same result (every exponent rounds to 2^0)
  const float sl2 = a.sl2 == 0.f ? 1e-30f : a.sl2;
  const int64_t units = (int64_t)a.n_items * a.Hkv;
  if constexpr (D == 128) {
    const int fit = 8 * ((prefill_groups<D>() * num_cus() + 7) / 8);  // work groups the chip runs at once
    if (!a.n_merges && !a.first && units > fit) {
      hipLaunchKernelGGL(attn_prefill32_kernel<D>, dim3(fit), dim3(256), 0, a.st, a.q, a.q_ts, a.q_hs, a.kv,
                         a.qo_indptr, a.G, sl2, a.plan, a.n_items, a.Hkv, a.mode, a.window_left, a.packed, a.woff,
                         a.extent, a.out, a.o_ts, a.o_hs, a.sinks, a.lse);
      return;
    }
  }
  const unsigned grid = (unsigned)(8 * ((units + 7) / 8));  // one work group per unit, padded to 8 XCDs
  hipLaunchKernelGGL((a.first ? attn_prefill_kernel<D, true> : attn_prefill_kernel<D, false>), dim3(grid), dim3(256), 0,
                     a.st, a.q, a.q_ts, a.q_hs, a.kv, a.qo_indptr, a.G, sl2, a.plan, a.items_word, a.n_items, a.Hkv,
                     a.mode, a.window_left, a.first, a.packed, a.woff, a.extent, a.out, a.o_ts, a.o_hs, a.sinks,
                     a.part_o, a.part_lse, a.lse);
  if (a.n_merges)
    hipLaunchKernelGGL(attn_prefill_merge_kernel<D>, dim3(a.n_merges * a.Hkv, kPrefillRows / (512 / D)), dim3(256), 0,
                       a.st, a.plan, a.merges_word, a.Hkv, a.G, a.part_o, a.part_lse, a.out, a.o_ts, a.o_hs, a.sinks,
                       a.lse);
}

// Packs the custom mask and finds every query token's visible extent: one work group per query token
// j (token i of request b), whose mask row of kv_len bytes its four waves read 64 positions at a time
// (a lane a byte, a ballot gives two words; bit n of word w = position 32w+n, 0 past kv_len). The
// extent is 1 + the last visible position (0 if none), with kExtentCausal set when the row is
// exactly causal: the causal extent, and as many visible positions. Bound: load latency, kMaskBatch
// loads in flight per wave. Against a thread per packed word and another per row before: 52 tokens
// over 1-9k positions 49.0 -> 8.9 us, 3.4k tokens over 0.2-1.5k 20.9 -> 7.5 us.
constexpr int kMaskBatch = 8;
__global__ __launch_bounds__(256) void attn_mask_kernel(const uint8_t* __restrict__ mask,
                                                        const int32_t* __restrict__ plan,
                                                        const int32_t* __restrict__ qo_indptr, PagedKV kv, int B,
                                                        uint32_t* __restrict__ packed,
                                                        int32_t* __restrict__ extent) {
  __shared__ int32_t s_ext[4], s_cnt[4];
  const int j = blockIdx.x;
  int lo = 0, hi = B - 1;  // the request holding query token j
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (qo_indptr[mid] <= j) lo = mid; else hi = mid - 1;
  }
  const int b = lo, q0 = qo_indptr[b], i = j - q0, qo_len = qo_indptr[b + 1] - q0;
  if (i < 0 || i >= qo_len) {  // a token outside the batch (qo_indptr may start past 0): no mask row
    if (threadIdx.x == 0) extent[j] = 0;
    return;
  }
  const int kv_len = kv_length(kv, b), nw = (kv_len + 31) / 32;
  const uint8_t* src = mask + reinterpret_cast<const int64_t*>(plan + plan[3])[b] + (int64_t)i * kv_len;
  uint32_t* dst = packed + reinterpret_cast<const int64_t*>(plan + plan[4])[b] + (int64_t)i * nw;
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  const int n64 = (kv_len + 63) / 64;  // 64-position groups; wave w takes w, w + 4, ...
  int ext = 0, cnt = 0;
  for (int g0 = w; g0 < n64; g0 += 4 * kMaskBatch) {
    uint8_t v[kMaskBatch];
#pragma unroll
    for (int k = 0; k < kMaskBatch; ++k) v[k] = src[min(64 * (g0 + 4 * k) + lane, kv_len - 1)];
#pragma unroll
    for (int k = 0; k < kMaskBatch; ++k) {
      const int g = g0 + 4 * k;
      const uint64_t bits = __builtin_amdgcn_ballot_w64(v[k] != 0 && 64 * g + lane < kv_len);
      if (g >= n64) break;
      if (bits) ext = 64 * g + 64 - __builtin_clzll(bits);
      cnt += __builtin_popcountll(bits);
      if (lane < 2 && 2 * g + lane < nw) dst[2 * g + lane] = (uint32_t)(bits >> (32 * lane));
    }
  }
  if (lane == 0) { s_ext[w] = ext; s_cnt[w] = cnt; }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int e = max(max(s_ext[0], s_ext[1]), max(s_ext[2], s_ext[3]));
    const bool causal = e > 0 && e == kv_len - qo_len + i + 1 && s_cnt[0] + s_cnt[1] + s_cnt[2] + s_cnt[3] == e;
    extent[j] = e | (causal ? kExtentCausal : 0);
  }
}

static int attention_prefill_impl(
    const pie_bf16* q, int64_t q_tok_stride, int64_t q_head_stride, const pie_bf16* k_cache,
    const pie_bf16* v_cache, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
    int64_t num_pages, const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim,
    int64_t page_size, float sm_scale, int32_t mode, int64_t window_left, int64_t first_tokens, const float* sinks,
    const uint32_t* packed_mask, const int32_t* mask_extent, const int32_t* plan, int64_t num_items,
    int64_t mask_offsets_word, const int64_t* split, void* scratch, int64_t scratch_bytes, pie_bf16* out,
    int64_t o_tok_stride, int64_t o_head_stride, float* lse, void* stream) {
  PagedKV kv;
  int rc = paged_kv_desc(&kv, k_cache, v_cache, page_stride, slot_stride, head_stride, num_pages,
                         kv_indptr, kv_indices, kv_last_page_len, page_size, head_dim,
                         "attention_prefill");
  if (rc) return rc;
  PIE_REQUIRE(q && out && plan && qo_indptr, "attention_prefill: null q, out, plan or qo_indptr");
  PIE_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256,
              "attention_prefill: head_dim %lld not in {64, 128, 256}", (long long)head_dim);
  PIE_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65535 && num_qo_heads % num_kv_heads == 0,
              "attention_prefill: num_qo_heads %lld not a multiple of num_kv_heads %lld",
              (long long)num_qo_heads, (long long)num_kv_heads);
  PIE_REQUIRE(mode >= 0 && mode <= 2 && (mode != 2 || (packed_mask && mask_extent && mask_offsets_word > 0 &&
                                                       mask_offsets_word % 2 == 0)),
              "attention_prefill: mode %d needs the packed mask and its plan offsets", mode);
  PIE_REQUIRE(num_items >= 0 && num_items * num_kv_heads < (1ll << 31), "attention_prefill: bad item count");
  PIE_REQUIRE(aligned16(q) && aligned16(out) && q_tok_stride % 8 == 0 && q_head_stride % 8 == 0 &&
                  o_tok_stride % 8 == 0 && o_head_stride % 8 == 0,
              "attention_prefill: q/out pointers and strides must be 16-byte aligned");
  PIE_REQUIRE(first_tokens >= 0, "attention_prefill: first_tokens %lld is negative", (long long)first_tokens);
  PIE_REQUIRE(!lse || !sinks, "attention_prefill: no log-sum-exp of attention with sinks");
  bool cut = split && split[1] > 0;
  if (cut) {
    PIE_REQUIRE(split[0] > 0 && split[2] > split[0] && split[3] > 0 && split[1] * num_kv_heads < (1ll << 31) &&
                    scratch && aligned16(scratch) && split[4] > 0 && scratch_bytes >= split[4],
                "attention_prefill: a split plan needs %lld bytes of 16-byte-aligned scratch, got %lld",
                (long long)split[4], (long long)scratch_bytes);
    // the pieces: the cut list without the items that stayed whole
    PIE_REQUIRE(split[4] == prefill_scratch_bytes(split[1] - (num_items - split[3]), num_kv_heads, head_dim),
                "attention_prefill: the split plan is for another head_dim or num_kv_heads than %lld, %lld",
                (long long)head_dim, (long long)num_kv_heads);
    // the pieces cover the kv range of the plan's mode and window; at others the uncut items run
    cut = split[5] == mode && split[6] == window_key(window_left, first_tokens);
  }
  if (num_items == 0) return PIE_HIP_OK;
  // The head-dim-128 kernel counts its work in the plan's header words, so runs of one plan must not
  // overlap. The other head dims' runs may: one that overlaps another stream's (or is captured,
  // when that cannot be seen) leaves the scratch alone and runs the plan's uncut items. So does, at
  // any head dim, one whose launches would fall between those of another thread's run on its stream.
  const bool counters = head_dim == 128;
  InflightClaim claim;
  if (counters || cut) {
    const InflightClaim::State got = claim.take(plan, stream);
    if (counters && got == InflightClaim::kBusy) return inflight_busy("attention_prefill");
    cut = cut && (got == InflightClaim::kOwn || (counters && got == InflightClaim::kCapture));
  }
  PrefillLaunch a{};
  a.st = static_cast<hipStream_t>(stream);
  a.q = q; a.q_ts = q_tok_stride; a.q_hs = q_head_stride;
  a.kv = kv;
  a.qo_indptr = qo_indptr;
  a.G = (int)(num_qo_heads / num_kv_heads); a.Hkv = (int)num_kv_heads;
  a.sl2 = sm_scale * 1.4426950408889634f;
  a.plan = plan;
  a.items_word = cut ? (int)split[0] : kPlanHeader;
  a.n_items = (int)(cut ? split[1] : num_items);
  a.mode = mode;
  a.window_left = window_left < 0 ? -1 : (int)std::min<int64_t>(window_left, 1 << 30);
  a.packed = packed_mask;
  a.woff = mode == 2 ? reinterpret_cast<const int64_t*>(plan + mask_offsets_word) : nullptr;
  a.extent = mask_extent;
  a.out = out; a.o_ts = o_tok_stride; a.o_hs = o_head_stride;
  a.sinks = sinks;
  a.first = first_within(a.window_left, first_tokens);
  a.lse = lse;
  if (cut) {
    a.merges_word = (int)split[2];
    a.n_merges = (int)split[3];
    a.part_o = static_cast<float*>(scratch);
    a.part_lse = a.part_o + split[4] / 4 / (head_dim + 1) * head_dim;
  }
  switch (head_dim) {
    case 64: launch_prefill<64>(a); break;
    case 128: launch_prefill<128>(a); break;
    default: launch_prefill<256>(a); break;
  }
  return check_launch("attention_prefill");
}

extern "C" int pie_hip_attention_prefill(
    const pie_bf16* q, int64_t q_tok_stride, int64_t q_head_stride, const pie_bf16* k_cache,
    const pie_bf16* v_cache, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
    int64_t num_pages, const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim,
    int64_t page_size, float sm_scale, int32_t mode, int64_t window_left, const float* sinks,
    const uint32_t* packed_mask, const int32_t* mask_extent, const int32_t* plan, int64_t num_items,
    int64_t mask_offsets_word, pie_bf16* out,
    int64_t o_tok_stride, int64_t o_head_stride, void* stream) {
  return attention_prefill_impl(q, q_tok_stride, q_head_stride, k_cache, v_cache, page_stride, slot_stride,
                                head_stride, num_pages, qo_indptr, kv_indptr, kv_indices, kv_last_page_len,
                                num_qo_heads, num_kv_heads, head_dim, page_size, sm_scale, mode, window_left, 0, sinks,
                                packed_mask, mask_extent, plan, num_items, mask_offsets_word, nullptr, nullptr, 0,
                                out, o_tok_stride, o_head_stride, nullptr, stream);
}

extern "C" int pie_hip_attention_prefill_split(
    const pie_bf16* q, int64_t q_tok_stride, int64_t q_head_stride, const pie_bf16* k_cache,
    const pie_bf16* v_cache, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
    int64_t num_pages, const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim,
    int64_t page_size, float sm_scale, int32_t mode, int64_t window_left, const float* sinks,
    const uint32_t* packed_mask, const int32_t* mask_extent, const int32_t* plan, int64_t num_items,
    int64_t mask_offsets_word, const int64_t* split, void* scratch, int64_t scratch_bytes, pie_bf16* out,
    int64_t o_tok_stride, int64_t o_head_stride, void* stream) {
  PIE_REQUIRE(split, "attention_prefill_split: null split");
  return attention_prefill_impl(q, q_tok_stride, q_head_stride, k_cache, v_cache, page_stride, slot_stride,
                                head_stride, num_pages, qo_indptr, kv_indptr, kv_indices, kv_last_page_len,
                                num_qo_heads, num_kv_heads, head_dim, page_size, sm_scale, mode, window_left, 0, sinks,
                                packed_mask, mask_extent, plan, num_items, mask_offsets_word, split, scratch,
                                scratch_bytes, out, o_tok_stride, o_head_stride, nullptr, stream);
}

extern "C" int pie_hip_attention_prefill_lse(
    const pie_bf16* q, int64_t q_tok_stride, int64_t q_head_stride, const pie_bf16* k_cache,
    const pie_bf16* v_cache, int64_t page_stride, int64_t slot_stride, int64_t head_stride,
    int64_t num_pages, const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
    const int32_t* kv_last_page_len, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim,
    int64_t page_size, float sm_scale, int32_t mode, int64_t window_left, int64_t first_tokens, const float* sinks,
    const uint32_t* packed_mask, const int32_t* mask_extent, const int32_t* plan, int64_t num_items,
    int64_t mask_offsets_word, const int64_t* split, void* scratch, int64_t scratch_bytes, pie_bf16* out,
    int64_t o_tok_stride, int64_t o_head_stride, float* lse, void* stream) {
  return attention_prefill_impl(q, q_tok_stride, q_head_stride, k_cache, v_cache, page_stride, slot_stride,
                                head_stride, num_pages, qo_indptr, kv_indptr, kv_indices, kv_last_page_len,
                                num_qo_heads, num_kv_heads, head_dim, page_size, sm_scale, mode, window_left,
                                first_tokens, sinks, packed_mask, mask_extent, plan, num_items, mask_offsets_word, split,
                                scratch, scratch_bytes, out, o_tok_stride, o_head_stride, lse, stream);
}

extern "C" int pie_hip_attention_pack_mask(const uint8_t* custom_mask, const int32_t* plan,
                                           const int32_t* qo_indptr, const int32_t* kv_indptr,
                                           const int32_t* kv_last_page_len, int64_t batch,
                                           int64_t page_size, int64_t mask_words, int64_t num_tokens,
                                           uint32_t* packed_mask, int32_t* mask_extent, void* stream) {
  PIE_REQUIRE(custom_mask && plan && qo_indptr && kv_indptr && kv_last_page_len && packed_mask && mask_extent,
              "attention_pack_mask: null argument");
  PIE_REQUIRE(num_tokens >= 0 && num_tokens < (1ll << 31), "attention_pack_mask: bad token count");
  PIE_REQUIRE(batch > 0 && batch < (1 << 24) && page_size > 0 && mask_words >= 0,
              "attention_pack_mask: bad batch %lld / page_size %lld / words %lld", (long long)batch,
              (long long)page_size, (long long)mask_words);
  PagedKV kv{};
  kv.indptr = kv_indptr;
  kv.last_len = kv_last_page_len;
  kv.page_size = (int32_t)page_size;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (num_tokens > 0)
    hipLaunchKernelGGL(attn_mask_kernel, dim3((unsigned)num_tokens), dim3(256), 0, st, custom_mask, plan, qo_indptr,
                       kv, (int)batch, packed_mask, mask_extent);
  return check_launch("attention_pack_mask");
}
