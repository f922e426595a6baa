// Attention over parts of a cache, built for the host by the emulator in include/hip/hip_runtime.h: first
// tokens kept beside a window, log-sum-exps, shared prefixes and joined states, on exact-size heap buffers
// under AddressSanitizer against the CPU oracle (oracle/oracle.c). TEST INFRASTRUCTURE.
//
//   emu_states <case>    case = decode | prefill | shared | merge | plan | all
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <random>
#include <string>
#include <vector>

#include "../../include/pie_hip.h"

extern "C" void oracle_attention(const uint16_t*, int64_t, int64_t, const uint16_t*, const uint16_t*, int64_t, int64_t,
                                 int64_t, const int32_t*, const int32_t*, const int32_t*, const int32_t*, const uint8_t*,
                                 const int64_t*, int, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, double,
                                 uint16_t*, int64_t, int64_t, double*, const float*);

static std::mt19937 rng(4321);
static int failures = 0;

template <typename T>
struct Buf {  // exact-size heap allocation: any access past the end trips ASan
  T* p;
  size_t n;
  explicit Buf(size_t n_) : p((T*)malloc(n_ ? n_ * sizeof(T) : 1)), n(n_) {}
  explicit Buf(const std::vector<T>& v) : Buf(v.size()) { std::copy(v.begin(), v.end(), p); }
  ~Buf() { free(p); }
  Buf(const Buf&) = delete;
  T& operator[](size_t i) { return p[i]; }
};

static uint16_t f2bf(float f) {
  uint32_t u;
  memcpy(&u, &f, 4);
  u += 0x7fffu + ((u >> 16) & 1u);
  return (uint16_t)(u >> 16);
}
static float bf2f(uint16_t h) {
  uint32_t u = (uint32_t)h << 16;
  float f;
  memcpy(&f, &u, 4);
  return f;
}
static void fill_normal(Buf<uint16_t>& b) {
  std::normal_distribution<float> d(0.f, 1.f);
  for (size_t i = 0; i < b.n; ++i) b[i] = f2bf(d(rng));
}
static int pick(int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); }
static void rc_is(int rc, int want, const char* what) {
  if (rc != want) {
    printf("  FAIL: %s returned %d, not %d: %s\n", what, rc, want, pie_hip_last_error());
    ++failures;
  }
}

// Outputs are averages of N(0, 1) values: the weights' and the output's roundings to bf16 (each half a
// step, 2^-8 relative, of terms whose absolute sum stays below 1 here) against 64 bits.
static void check(const char* what, const Buf<uint16_t>& got, const Buf<uint16_t>& want, const Buf<float>* lse,
                  const std::vector<double>& want_lse) {
  float worst = 0.f;
  for (size_t i = 0; i < want.n; ++i) {
    const float g = bf2f(got.p[i]), w = bf2f(want.p[i]), off = fabsf(g - w) / (1.f / 256 + fabsf(w) / 128);
    worst = off <= worst ? worst : off;  // (a NaN counts)
  }
  double far = 0;
  if (lse)
    for (size_t i = 0; i < lse->n; ++i) {
      const double w = want_lse[i] / log(2.0), g = lse->p[i];
      const double off = w == -INFINITY || g == -INFINITY ? (w == g ? 0 : INFINITY) : fabs(g - w) / (1e-4 + 1e-5 * fabs(w));
      far = off <= far ? far : off;
    }
  const bool ok = worst <= 1.f && far <= 1;
  printf("  %-36s %s (worst %.3f, lse %.3f of the tolerance)\n", what, ok ? "ok" : "FAIL", worst, far);
  failures += !ok;
}

// A pool of pages handed out in random order, as runs of tokens (NHD cache [pages, 2, P, Hkv, D]).
struct Pool {
  int64_t P, Hkv, D;
  std::vector<int32_t> order;
  size_t used = 0;
  Pool(int64_t pages, int64_t P_, int64_t Hkv_, int64_t D_) : P(P_), Hkv(Hkv_), D(D_), order(pages) {
    for (int64_t i = 0; i < pages; ++i) order[i] = (int32_t)i;
    std::shuffle(order.begin(), order.end(), rng);
  }
  int64_t page_elems() const { return 2 * P * Hkv * D; }
};
struct Runs {
  std::vector<int32_t> len, indptr{0}, indices, last;
  void add(Pool& pool, int n) {
    const int np = (int)((n + pool.P - 1) / pool.P);
    for (int i = 0; i < np; ++i) indices.push_back(pool.order.at(pool.used++));
    len.push_back(n);
    indptr.push_back((int32_t)indices.size());
    last.push_back(np ? n - (np - 1) * (int)pool.P : 0);
  }
  // token t of run i as a page of one token: page * 2P + slot, rows Hkv * D apart
  int32_t token(const Pool& pool, int i, int t) const {
    return (int32_t)(indices[indptr[i] + t / pool.P] * 2 * pool.P + t % pool.P);
  }
};
static int64_t pages_of(const std::vector<int>& lens, int64_t P) {
  int64_t n = 0;
  for (int l : lens) n += (l + P - 1) / P;
  return std::max<int64_t>(1, n);
}

// The oracle over explicit token lists and masks.
static void want_attention(const Pool& pool, const Buf<uint16_t>& q, const Buf<uint16_t>& cache,
                           const std::vector<std::vector<int32_t>>& tokens, const std::vector<int32_t>& qo,
                           const std::vector<uint8_t>& mask, int64_t Hq, Buf<uint16_t>& out, std::vector<double>& lse) {
  const int64_t B = (int64_t)tokens.size(), D = pool.D, Hkv = pool.Hkv;
  std::vector<int32_t> indptr{0}, ids, last(B, 1);
  std::vector<int64_t> off;
  int64_t at = 0;
  for (int64_t b = 0; b < B; ++b) {
    ids.insert(ids.end(), tokens[b].begin(), tokens[b].end());
    indptr.push_back((int32_t)ids.size());
    off.push_back(at);
    at += (int64_t)(qo[b + 1] - qo[b]) * (int64_t)tokens[b].size();
  }
  ids.push_back(0);
  lse.assign((size_t)qo[B] * Hq, -INFINITY);
  oracle_attention(q.p, Hq * D, D, cache.p, cache.p + pool.P * Hkv * D, Hkv * D, Hkv * D, D, qo.data(), indptr.data(),
                   ids.data(), last.data(), mask.data(), off.data(), 0, -1, B, Hq, Hkv, D, 1, 1.0 / sqrt((double)D), out.p,
                   Hq * D, D, lse.data(), nullptr);
}

// Positions no query sees become NaN in the cache: they must not reach any output.
static void poison(Pool& pool, const Runs& runs, int b, int t, Buf<uint16_t>& cache) {
  const int64_t row = pool.Hkv * pool.D, at = (int64_t)runs.token(pool, b, t) * row;
  for (int64_t e = 0; e < row; ++e) cache[at + e] = cache[at + pool.P * row + e] = 0x7fc0;
}

// ---------------------------------------------------------------------------- window with first tokens
static void case_decode(std::vector<int> lens, int64_t Hq, int64_t Hkv, int64_t D, int64_t P, int64_t window,
                        int64_t first, int64_t splits) {
  printf("decode B=%zu Hq=%lld Hkv=%lld D=%lld P=%lld window=%lld first=%lld splits=%lld\n", lens.size(), (long long)Hq,
         (long long)Hkv, (long long)D, (long long)P, (long long)window, (long long)first, (long long)splits);
  const int64_t B = (int64_t)lens.size(), pages = pages_of(lens, P);
  Pool pool(pages, P, Hkv, D);
  Runs runs;
  for (int n : lens) runs.add(pool, n);
  Buf<uint16_t> cache(pages * pool.page_elems()), q(B * Hq * D), out(B * Hq * D), want(B * Hq * D);
  fill_normal(cache);
  fill_normal(q);
  std::vector<std::vector<int32_t>> tokens(B);
  std::vector<int32_t> qo(B + 1);
  std::vector<uint8_t> mask;
  for (int b = 0; b < B; ++b) {
    qo[b + 1] = b + 1;
    for (int t = 0; t < lens[b]; ++t) {
      const bool see = window < 0 || t >= lens[b] - 1 - window || t < first;
      tokens[b].push_back(runs.token(pool, b, t));
      mask.push_back(see);
      if (!see) poison(pool, runs, b, t, cache);
    }
  }
  std::vector<double> want_lse;
  want_attention(pool, q, cache, tokens, qo, mask, Hq, want, want_lse);
  Buf<int32_t> ip(runs.indptr), ix(runs.indices), ll(runs.last);
  Buf<float> ws(splits > 1 ? B * splits * Hq * (D + 1) : 1), lse(B * Hq);
  rc_is(pie_hip_attention_decode_lse(q.p, Hq * D, D, cache.p, cache.p + P * Hkv * D, pool.page_elems(), Hkv * D, D, pages,
                                     ip.p, ix.p, ll.p, B, Hq, Hkv, D, P, 1.f / sqrtf((float)D), window, first, nullptr,
                                     splits, ws.p, (int64_t)ws.n * 4, out.p, Hq * D, D, lse.p, nullptr),
        0, "decode_lse");
  check("decode", out, want, &lse, want_lse);
}

static void case_prefill(std::vector<int> lens, std::vector<int> news, int64_t Hq, int64_t Hkv, int64_t D, int64_t P,
                         int mode, int64_t window, int64_t first, int cut_cus) {
  printf("prefill B=%zu Hq=%lld Hkv=%lld D=%lld P=%lld mode=%d window=%lld first=%lld cut=%d\n", lens.size(), (long long)Hq,
         (long long)Hkv, (long long)D, (long long)P, mode, (long long)window, (long long)first, cut_cus);
  const int64_t B = (int64_t)lens.size(), pages = pages_of(lens, P);
  Pool pool(pages, P, Hkv, D);
  Runs runs;
  for (int n : lens) runs.add(pool, n);
  std::vector<int32_t> qo{0};
  for (int n : news) qo.push_back(qo.back() + n);
  const int64_t T = qo[B];
  Buf<uint16_t> cache(pages * pool.page_elems()), q(T * Hq * D), out(T * Hq * D), want(T * Hq * D);
  fill_normal(cache);
  fill_normal(q);
  std::vector<std::vector<int32_t>> tokens(B);
  std::vector<uint8_t> mask, custom;
  for (int b = 0; b < B; ++b) {
    std::vector<bool> seen(lens[b], false);
    for (int t = 0; t < lens[b]; ++t) tokens[b].push_back(runs.token(pool, b, t));
    for (int i = 0; i < news[b]; ++i)
      for (int t = 0; t < lens[b]; ++t) {
        const int p = lens[b] - news[b] + i;
        custom.push_back(pick(0, 9) < 7);
        bool see = mode == 2 ? custom.back() : mode == 0 || t <= p;
        see = see && (window < 0 || t >= p - window || t < first);
        mask.push_back(see);
        if (see || window < 0 || t >= lens[b] - news[b] - window) seen[t] = true;  // (kept finite: some row's range)
      }
    for (int t = 0; t < lens[b]; ++t)
      if (!seen[t] && t >= first) poison(pool, runs, b, t, cache);
  }
  std::vector<double> want_lse;
  want_attention(pool, q, cache, tokens, qo, mask, Hq, want, want_lse);
  Buf<int32_t> qi(qo), ip(runs.indptr), ix(runs.indices), ll(runs.last);
  const int64_t cap = 16384;
  Buf<int32_t> plan(cap);
  int64_t words = 0, items = 0, mb = 0, mw = 0, split[7] = {};
  rc_is(pie_hip_attention_prefill_first_plan(qi.p, ip.p, ll.p, B, P, Hq, Hkv, D, mode, window, first,
                                             cut_cus ? cut_cus : 1, cut_cus ? 1ll << 30 : 0, plan.p, cap, &words, &items,
                                             &mb, &mw, split),
        0, "prefill_first_plan");
  if (cut_cus && !split[1]) { printf("  FAIL: nothing was cut\n"); ++failures; }
  Buf<uint8_t> cm(custom);
  Buf<uint32_t> packed(std::max<int64_t>(mw, 1));
  Buf<int32_t> extent(T);
  if (mode == 2)
    rc_is(pie_hip_attention_pack_mask(cm.p, plan.p, qi.p, ip.p, ll.p, B, P, mw, T, packed.p, extent.p, nullptr), 0, "pack");
  Buf<float> scratch(std::max<int64_t>(split[4] / 4, 4)), lse(T * Hq);
  rc_is(pie_hip_attention_prefill_lse(q.p, Hq * D, D, cache.p, cache.p + P * Hkv * D, pool.page_elems(), Hkv * D, D, pages,
                                      qi.p, ip.p, ix.p, ll.p, Hq, Hkv, D, P, 1.f / sqrtf((float)D), mode, window, first,
                                      nullptr, mode == 2 ? packed.p : nullptr, mode == 2 ? extent.p : nullptr, plan.p, items,
                                      plan[4], split, scratch.p, split[4], out.p, Hq * D, D, lse.p, nullptr),
        0, "prefill_lse");
  check("prefill", out, want, &lse, want_lse);
}

// ---------------------------------------------------------------------------- shared prefixes
// sizes: requests per group; news empty: one query token per request.
static void case_shared(std::vector<int> sizes, std::vector<int> prefixes, std::vector<int> suffixes, std::vector<int> news,
                        int64_t Hq, int64_t Hkv, int64_t D, int64_t P, int cus, bool bad_page = false,
                        int64_t scratch_max = 1ll << 30) {
  printf("shared groups=%zu B=%zu Hq=%lld Hkv=%lld D=%lld P=%lld cus=%d%s%s\n", sizes.size(), suffixes.size(), (long long)Hq,
         (long long)Hkv, (long long)D, (long long)P, cus, news.empty() ? "" : " ragged", bad_page ? " bad page" : "");
  const int64_t B = (int64_t)suffixes.size(), Gp = (int64_t)sizes.size();
  const int64_t pages = pages_of(prefixes, P) + pages_of(suffixes, P);
  Pool pool(pages, P, Hkv, D);
  Runs pre, suf;
  for (int n : prefixes) pre.add(pool, n);
  for (int n : suffixes) suf.add(pool, n);
  std::vector<int32_t> gi{0}, qo{0};
  for (int n : sizes) gi.push_back(gi.back() + n);
  for (int b = 0; b < B; ++b) qo.push_back(qo.back() + (news.empty() ? 1 : news[b]));
  const int64_t T = qo[B];
  Buf<uint16_t> cache(pages * pool.page_elems()), q(T * Hq * D), out(T * Hq * D), want(T * Hq * D);
  fill_normal(cache);
  fill_normal(q);
  std::vector<std::vector<int32_t>> tokens(B);
  std::vector<uint8_t> mask;
  for (int g = 0; g < Gp; ++g)
    for (int b = gi[g]; b < gi[g + 1]; ++b) {
      const int n = qo[b + 1] - qo[b];
      for (int t = 0; t < prefixes[g]; ++t) tokens[b].push_back(pre.token(pool, g, t));
      for (int t = 0; t < suffixes[b]; ++t) tokens[b].push_back(suf.token(pool, b, t));
      for (int i = 0; i < n; ++i) {
        for (int t = 0; t < prefixes[g]; ++t) mask.push_back(!(bad_page && g == 0 && t / P == 0));
        for (int t = 0; t < suffixes[b]; ++t) mask.push_back(news.empty() || t <= suffixes[b] - n + i);
      }
    }
  std::vector<double> want_lse;
  want_attention(pool, q, cache, tokens, qo, mask, Hq, want, want_lse);
  if (bad_page) pre.indices[0] = (int32_t)pages;  // outside the pool: its positions are masked
  if (pre.indices.empty()) pre.indices.push_back(0);
  Buf<int32_t> gb(gi), pb(pre.indptr), px(pre.indices), pl(pre.last), sb(suf.indptr), sx(suf.indices), sl(suf.last), qb(qo);

  const int32_t* qp = news.empty() ? nullptr : qb.p;
  int64_t info[17];
  rc_is(pie_hip_attention_shared_plan(gb.p, Gp, pb.p, pl.p, qp, sb.p, sl.p, B, P, Hq, Hkv, D, cus, scratch_max, nullptr, 0, info),
        0, "shared_plan");
  Buf<int32_t> plan(info[0]);
  rc_is(pie_hip_attention_shared_plan(gb.p, Gp, pb.p, pl.p, qp, sb.p, sl.p, B, P, Hq, Hkv, D, cus, scratch_max, plan.p,
                                      (int64_t)plan.n, info),
        0, "shared_plan");
  Buf<float> scratch(info[1] / 4), lse(T * Hq);
  rc_is(pie_hip_attention_shared(q.p, Hq * D, D, cache.p, cache.p + P * Hkv * D, pool.page_elems(), Hkv * D, D, pages, px.p,
                                 sb.p, sx.p, sl.p, T, Hq, Hkv, D, P, 1.f / sqrtf((float)D), plan.p, info, scratch.p, info[1],
                                 out.p, Hq * D, D, lse.p, nullptr),
        0, "shared");
  printf("  prefix items %lld + %lld streamed, suffix items %lld, splits %lld, parts <= %lld\n", (long long)info[2],
         (long long)info[4], (long long)info[3], (long long)info[6], (long long)info[8]);
  check("shared", out, want, &lse, want_lse);
}

// ---------------------------------------------------------------------------- joined states
static void case_merge(int64_t S, int64_t T, int64_t H, int64_t D, bool bf16) {
  printf("merge parts=%lld tokens=%lld heads=%lld D=%lld %s\n", (long long)S, (long long)T, (long long)H, (long long)D,
         bf16 ? "bf16" : "fp32");
  const int64_t N = T * H * D;
  Buf<uint16_t> pb(bf16 ? S * N : 0), ob(bf16 ? N : 0);
  Buf<float> pf(bf16 ? 0 : S * N), of(bf16 ? 0 : N), l(S * T * H), lse(T * H);
  std::normal_distribution<float> d(0.f, 1.f);
  for (int64_t i = 0; i < S * T * H; ++i) {
    const bool none = pick(0, 4) == 0;
    l[i] = none ? -INFINITY : 3 * d(rng) + 8;
    for (int64_t e = 0; e < D; ++e) {
      const float v = none ? NAN : d(rng);  // whatever a part that saw nothing holds
      if (bf16) pb[i * D + e] = none ? 0x7fc0 : f2bf(v); else pf[i * D + e] = v;
    }
  }
  rc_is(pie_hip_attention_merge_states(bf16 ? (void*)pb.p : (void*)pf.p, bf16, N, H * D, D, l.p, T * H, H, 1, S, T, H, D,
                                       bf16 ? (void*)ob.p : (void*)of.p, H * D, D, lse.p, H, 1, nullptr),
        0, "merge_states");
  double far = 0;
  for (int64_t r = 0; r < T * H; ++r) {
    double M = -INFINITY, L = 0;
    for (int64_t s = 0; s < S; ++s) M = std::max(M, (double)l[s * T * H + r]);
    for (int64_t s = 0; s < S; ++s) L += M == -INFINITY ? 0 : exp2((double)l[s * T * H + r] - M);
    const double want_lse = L > 0 ? M + log2(L) : -INFINITY;
    const double off = want_lse == -INFINITY ? (lse[r] == want_lse ? 0 : INFINITY) : fabs(lse[r] - want_lse) / 1e-5;
    far = off <= far ? far : off;
    for (int64_t e = 0; e < D; ++e) {
      double o = 0, mag = 0;
      for (int64_t s = 0; s < S; ++s) {
        const float li = l[s * T * H + r];
        if (li == -INFINITY) continue;
        const double v = bf16 ? bf2f(pb[(s * T * H + r) * D + e]) : pf[(s * T * H + r) * D + e], w = exp2((double)li - M) / L;
        o += w * v;
        mag += w * fabs(v);
      }
      const double got = bf16 ? bf2f(ob[r * D + e]) : of[r * D + e];
      const double o2 = fabs(got - o) / (1e-30 + mag * 1e-6 * (double)(S + 4) + (bf16 ? fabs(o) / 256 : 0));
      far = o2 <= far ? far : o2;
    }
  }
  printf("  %-36s %s (worst %.3f of the tolerance)\n", "merge", far <= 1 ? "ok" : "FAIL", far);
  failures += !(far <= 1);
}

// Refusals of the plans and entry points, before any launch.
static void case_plan() {
  printf("refusals\n");
  int32_t gi[] = {0, 2}, pi[] = {0, 3}, pl[] = {5}, ki[] = {0, 1, 2}, kl[] = {1, 16}, qo[] = {0, 1, 3};
  int64_t info[17];
  const auto plan = [&](int64_t Hq = 8, int64_t Hkv = 2, int64_t D = 128, const int32_t* q = nullptr, int64_t scratch = 1 << 30,
                        int32_t* words = nullptr, int64_t cap = 0) {
    return pie_hip_attention_shared_plan(gi, 1, pi, pl, q, ki, kl, 2, 16, Hq, Hkv, D, 256, scratch, words, cap, info);
  };
  rc_is(plan(), 0, "a plan");
  rc_is(plan(8, 2, 128, qo), 0, "a ragged plan");
  rc_is(plan(8, 3), 1, "heads that do not divide");
  rc_is(plan(64, 2), 1, "32 query heads per kv head, one query token");
  rc_is(plan(64, 2, 128, qo), 0, "32 query heads per kv head, ragged");
  rc_is(plan(8, 2, 96), 1, "head dim 96");
  rc_is(plan(8, 2, 128, nullptr, 64), 1, "64 bytes of scratch");
  int32_t words[4];
  rc_is(plan(8, 2, 128, nullptr, 1 << 30, words, 4), 1, "four words");
  pl[0] = 17;
  rc_is(plan(), 1, "17 tokens on a page of 16");
  pl[0] = 5;
  pi[1] = -1;
  rc_is(plan(), 1, "a negative page count");
  pi[1] = 3;
  gi[1] = 1;
  rc_is(plan(), 1, "a request outside every group");
  gi[1] = 2;
  ki[1] = 3;
  rc_is(plan(), 1, "a decreasing table");
  ki[1] = 1;
  qo[0] = 1;
  rc_is(plan(8, 2, 128, qo), 1, "query tokens from 1");
  qo[0] = 0;
  rc_is(plan(), 0, "the plan again");
  alignas(16) static char mem[64];
  uint16_t* p = (uint16_t*)mem;
  const auto run = [&](int64_t T, int64_t D, int64_t P, void* scratch, int64_t bytes) {
    return pie_hip_attention_shared(p, 8 * D, D, p, p, 16, 16, 16, 1, ki, ki, ki, kl, T, 8, 2, D, P, 1.f, pi, info, scratch,
                                    bytes, p, 8 * D, D, nullptr, nullptr);
  };
  rc_is(run(3, 128, 16, mem, 1 << 30), 1, "a run of another token count");
  rc_is(run(2, 64, 16, mem, 1 << 30), 1, "a run of another head dim");
  rc_is(run(2, 128, 8, mem, 1 << 30), 1, "a run of another page size");
  rc_is(run(2, 128, 16, nullptr, 1 << 30), 1, "a run without scratch");
  rc_is(run(2, 128, 16, mem, 64), 1, "a run with too little scratch");
  const auto merge = [&](int64_t S, int64_t D, int64_t stride) {
    return pie_hip_attention_merge_states(p, 1, stride, stride, D, (float*)mem, 1, 1, 1, S, 1, 1, D, p, D, D, (float*)mem, 1, 1,
                                          nullptr);
  };
  rc_is(merge(0, 128, 128), 1, "a merge of nothing");
  rc_is(merge(2, 96, 96), 1, "a merge of head dim 96");
  rc_is(merge(2, 128, 132), 1, "rows off a 16-byte boundary");
  const float sinks[8] = {};
  const auto decode = [&](int64_t first, const float* sk, float* lse) {
    return pie_hip_attention_decode_lse(p, 1024, 128, p, p, 16, 16, 16, 1, ki, ki, kl, 2, 8, 2, 128, 16, 1.f, 5, first, sk, 1,
                                        nullptr, 0, p, 1024, 128, lse, nullptr);
  };
  rc_is(decode(-1, nullptr, nullptr), 1, "negative first tokens");
  rc_is(decode(1, sinks, (float*)mem), 1, "log-sum-exps with sinks");
}

int main(int argc, char** argv) {
  const std::string c = argc > 1 ? argv[1] : "all";
  const bool all = c == "all";
  if (all || c == "plan") case_plan();
  if (all || c == "merge") {
    case_merge(1, 3, 2, 128, true);
    case_merge(2, 3, 5, 64, false);
    case_merge(11, 2, 3, 256, true);
    case_merge(19, 2, 3, 128, false);
  }
  if (all || c == "decode") {
    case_decode({1, 40, 300, 0}, 8, 2, 128, 16, 63, 4, 1);  // shorter than the window, empty, hidden tokens between
    case_decode({700, 130, 65}, 8, 2, 128, 16, 100, 21, 3);  // the seam inside a split, a page and a tile
    case_decode({500, 90}, 4, 4, 64, 5, 0, 1, 1);            // the query alone and one first token
    case_decode({900}, 6, 1, 256, 8, 40, 600, 5);            // more first tokens than window; several splits
    case_decode({1400}, 4, 2, 64, 1, 700, 650, 1);           // page size 1: page windows on both sides of the seam
    case_decode({1400}, 4, 2, 64, 1, 300, 520, 2);
    case_decode({200, 33}, 8, 2, 128, 16, -1, 7, 2);         // no window: first tokens change nothing
    case_decode({50}, 8, 2, 128, 16, 20, 29, 1);             // first tokens reach the window exactly
    case_decode({50}, 8, 2, 128, 16, 20, 1000, 1);           // and past it
  }
  if (all || c == "prefill") {
    case_prefill({300, 40, 0}, {60, 40, 0}, 8, 2, 128, 16, 1, 63, 4, 0);
    case_prefill({400}, {33}, 8, 2, 128, 5, 1, 50, 70, 0);       // first tokens over a tile, rows on several pages
    case_prefill({300, 150}, {20, 90}, 4, 2, 64, 16, 2, 40, 9, 0);  // custom mask
    case_prefill({260}, {40}, 2, 1, 256, 16, 1, 31, 5, 0);
    case_prefill({200}, {20}, 2, 1, 256, 3, 0, 45, 140, 0);       // full visibility; first tokens reach the window
    case_prefill({700}, {10}, 4, 1, 64, 1, 1, 90, 33, 0);         // page size 1
    case_prefill({1500}, {9}, 4, 2, 128, 16, 1, 1100, 130, 64);   // cut, pieces over the seam
    case_prefill({1500}, {9}, 4, 2, 128, 16, 2, 1100, 40, 64);
    case_prefill({1400}, {7}, 8, 2, 64, 8, 1, 900, 400, 64);
    case_prefill({1300}, {5}, 4, 2, 256, 16, 1, 1000, 1, 64);
    case_prefill({1300}, {5}, 4, 2, 128, 16, 1, 600, 900, 64);    // cut, first tokens past the window's start
    case_prefill({90, 200}, {90, 31}, 8, 2, 128, 16, 1, -1, 3, 0);  // no window (persistent kernel), log-sum-exps
  }
  if (all || c == "shared") {
    case_shared({4}, {200}, {1, 33, 0, 60}, {}, 8, 2, 128, 16, 4);
    case_shared({3, 0, 2, 1}, {70, 500, 0, 129}, {5, 0, 90, 300, 1, 0}, {}, 8, 2, 128, 16, 4);  // empty group, prefix, suffix
    case_shared({2, 1}, {0, 0}, {0, 0, 7}, {}, 4, 2, 128, 16, 4);                               // rows that see nothing
    case_shared({19}, {330}, std::vector<int>(19, 3), {}, 14, 2, 128, 5, 1);                    // 133 rows, 7 heads, page 5
    case_shared({5}, {400}, {40, 2, 9, 700, 1}, {}, 16, 2, 64, 16, 64);
    case_shared({3, 2}, {290, 31}, {4, 40, 1, 2, 300}, {}, 8, 2, 256, 16, 64);
    case_shared({6}, {700}, {1, 1, 1, 1, 1, 1}, {}, 4, 1, 64, 1, 256);                          // page size 1, six pieces
    case_shared({2}, {200}, {20, 5}, {}, 8, 2, 128, 16, 4, true);                               // a page id out of range
    case_shared({3}, {900}, {5, 600, 4}, {}, 4, 2, 128, 16, 256, false, 30000);                 // fewer, longer pieces
    case_shared({3, 2}, {150, 40}, {9, 30, 4, 12, 60}, {9, 5, 1, 0, 3}, 8, 2, 128, 16, 4);
    case_shared({2}, {600}, {70, 300}, {40, 2}, 4, 2, 64, 5, 64);
    case_shared({1, 2}, {0, 270}, {3, 20, 8}, {3, 6, 8}, 4, 2, 256, 16, 64);
    case_shared({2}, {64}, {3, 0}, {5, 2}, 20, 1, 128, 16, 4);  // more query tokens than the suffix holds
  }
  printf(failures ? "%d FAILURES\n" : "all ok\n", failures);
  return failures != 0;
}
