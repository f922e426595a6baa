// The join of attention results over disjoint parts of a context. Part i of a row holds its normalised
// output o_i and the base-2 logarithm l_i of its softmax mass; the whole row's are
//   M = max_i l_i,  w_i = 2^(l_i - M),  out = sum w_i o_i / sum w_i,  lse = M + log2 sum w_i.
// A part that saw nothing (l_i = -inf) counts for nothing, whatever its o_i holds; a row that no part saw
// is 0 with lse -inf. Statistics and sums are fp32, the output is rounded once.
#include "attn_dev.h"

namespace pie {

// One element type's 8 consecutive values, and their load and store.
struct Bf16 {
  typedef uint16_t elem;
  static constexpr int kAlign = 8;  // elements in 16 bytes
  typedef uint4 raw;
  static __device__ __forceinline__ raw load(const elem* p) { return ld16(p); }
  static __device__ __forceinline__ void unpack(const raw& r, float (&f)[8]) { unpack8(r, f); }
  static __device__ __forceinline__ void store(elem* p, const float (&f)[8]) { st16(p, pack8(f)); }
};
struct Fp32 {
  typedef float elem;
  static constexpr int kAlign = 4;
  struct raw { float4 a, b; };
  static __device__ __forceinline__ raw load(const elem* p) {
    return raw{*reinterpret_cast<const float4*>(p), *reinterpret_cast<const float4*>(p + 4)};
  }
  static __device__ __forceinline__ void unpack(const raw& r, float (&f)[8]) {
    f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w;
    f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
  }
  static __device__ __forceinline__ void store(elem* p, const float (&f)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  }
};

struct StatesArgs {
  const void* parts;
  int64_t p_s, p_t, p_h;  // strides of the part, token and head, elements
  const float* lses;
  int64_t l_s, l_t, l_h;
  int S;
  int64_t rows;  // tokens * heads
  FastDiv heads;
  void* out;
  int64_t o_t, o_h;
  float* lse;
  int64_t e_t, e_h;
};

// D / 8 lanes a row, 8 dims a lane; KB parts are loaded before the first is used: 8, or 2 where there are no
// more (the loads past the last part repeat it: 2 parts of 8190 x 32 rows of 128 in bf16 take 30.5 us at 2
// and 38.3 at 8). HBM bounds it: 4 such parts, 341 MB, in 60 us (5.7 TB/s, mostly reads; a large copy's rate
// is 4.9); 17 parts of 300 x 16 rows of 256 in fp32, 89 MB, in 16 us; a few rows in a launch's 3 us.
template <typename T, int D, int KB>
__global__ __launch_bounds__(256) void attn_states_kernel(StatesArgs a) {
  constexpr int CH = D / 8;
  const int64_t r = (int64_t)blockIdx.x * (256 / CH) + threadIdx.x / CH;
  const int c = threadIdx.x % CH;
  if (r >= a.rows) return;
  const uint32_t t = a.heads.div((uint32_t)r), h = (uint32_t)r - t * a.heads.d;
  const typename T::elem* p = static_cast<const typename T::elem*>(a.parts) + t * a.p_t + h * a.p_h + 8 * c;
  const float* l = a.lses + t * a.l_t + h * a.l_h;
  float M = -INFINITY, L = 0.f, acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  for (int s0 = 0; s0 < a.S; s0 += KB) {
    float ls[KB];
    typename T::raw v[KB];
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const int64_t s = min(s0 + k, a.S - 1);
      ls[k] = l[s * a.l_s];
      v[k] = T::load(p + s * a.p_s);
    }
    float mx = M;
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      if (s0 + k >= a.S) ls[k] = -INFINITY;
      mx = fmaxf(mx, ls[k]);
    }
    const float ref = mx == -INFINITY ? 0.f : mx;
    const float f0 = fast_exp2(M - ref);
    L *= f0;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= f0;
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const float w = fast_exp2(ls[k] - ref);
      float f[8];
      T::unpack(v[k], f);
      L += w;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(ls[k] == -INFINITY ? 0.f : f[e], w, acc[e]);
    }
    M = mx;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= inv;
  T::store(static_cast<typename T::elem*>(a.out) + t * a.o_t + h * a.o_h + 8 * c, acc);
  if (c == 0) a.lse[t * a.e_t + h * a.e_h] = row_lse(L, M);
}

template <typename T, int D>
static void launch_states(hipStream_t st, const StatesArgs& a) {
  const unsigned grid = (unsigned)((a.rows + 2048 / D - 1) / (2048 / D));
  hipLaunchKernelGGL((a.S <= 2 ? attn_states_kernel<T, D, 2> : attn_states_kernel<T, D, 8>), dim3(grid), dim3(256), 0, st, a);
}
template <typename T>
static void launch_states(hipStream_t st, const StatesArgs& a, int64_t D) {
  switch (D) {
    case 64: launch_states<T, 64>(st, a); break;
    case 128: launch_states<T, 128>(st, a); break;
    default: launch_states<T, 256>(st, a); break;
  }
}

}  // namespace pie

using namespace pie;

extern "C" int pie_hip_attention_merge_states(const void* parts, int32_t is_bf16, int64_t part_stride,
                                              int64_t part_tok_stride, int64_t part_head_stride, const float* lses,
                                              int64_t lse_part_stride, int64_t lse_tok_stride, int64_t lse_head_stride,
                                              int64_t num_parts, int64_t num_tokens, int64_t num_heads,
                                              int64_t head_dim, void* out, int64_t o_tok_stride, int64_t o_head_stride,
                                              float* lse, int64_t e_tok_stride, int64_t e_head_stride, void* stream) {
  const char* what = "attention_merge_states";
  PIE_REQUIRE(num_parts >= 1 && num_parts < (1ll << 31) && num_tokens >= 0 && num_heads >= 0 && num_heads < (1ll << 31) &&
                  (num_heads == 0 || num_tokens < (1ll << 31) / num_heads),
              "%s: bad parts %lld / tokens %lld / heads %lld", what, (long long)num_parts, (long long)num_tokens,
              (long long)num_heads);
  PIE_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s: head_dim %lld not in {64, 128, 256}", what,
              (long long)head_dim);
  if (num_tokens == 0 || num_heads == 0) return PIE_HIP_OK;
  const int64_t al = is_bf16 ? Bf16::kAlign : Fp32::kAlign;
  PIE_REQUIRE(parts && lses && out && lse, "%s: null argument", what);
  PIE_REQUIRE(aligned16(parts) && aligned16(out) && part_stride % al == 0 && part_tok_stride % al == 0 &&
                  part_head_stride % al == 0 && o_tok_stride % al == 0 && o_head_stride % al == 0,
              "%s: parts and out must be 16-byte aligned, rows included", what);
  const StatesArgs a = {parts, part_stride, part_tok_stride, part_head_stride, lses, lse_part_stride, lse_tok_stride,
                        lse_head_stride, (int)num_parts, num_tokens * num_heads, FastDiv::make((uint32_t)num_heads), out,
                        o_tok_stride, o_head_stride, lse, e_tok_stride, e_head_stride};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (is_bf16) launch_states<Bf16>(st, a, head_dim);
  else launch_states<Fp32>(st, a, head_dim);
  return check_launch(what);
}
