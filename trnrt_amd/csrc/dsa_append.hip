// Appends to the paged caches for gfx950: each new token's rows (its latent row, its indexer key) normed, rotated,
// quantised and written to the slot that its place in its sequence has in the page table, in one launch:
//   y = x, its first n columns normed: x / sqrt(mean x^2 + eps) w, or (x - mean) / sqrt(var + eps) w + b;
//   2R of y's columns rotated by the token's positions (dsa_rope.h);
//   s = max(absmax(y), 1e-30) / 448, cache[slot] = e4m3(clamp(y / s)), scale[slot] = s.
// Everything between the row's load and its store is in fp32 and is rounded once.
#include "dsa_append.h"

namespace dsa {

constexpr int AP_WAVES = 4;
constexpr int AP_GROUPS = AP_MAX_WIDTH / (8 * WAVE);  // of 8 columns that a lane holds
constexpr float AP_FP8_MAX = 448.0f;

__device__ __forceinline__ void ap_load8(const void* p, int fp32, long at, float (&v)[8]) {
  if (fp32) {
    const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
    const f32x4 a = q[0], b = q[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  } else {
    const u32x4 u = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(u[e] << 16);
      v[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
    }
  }
}

// The number of sequences that end by row t (cu ascends), the same in every lane.
__device__ __forceinline__ int ap_sequence(const int* __restrict__ cu, int B, int t) {
  const int lane = threadIdx.x & (WAVE - 1);
  int lo = 0, hi = B;  // the answer is in [lo, hi]
  while (hi > lo) {
    const int step = (hi - lo + WAVE - 1) / WAVE, at = min(lo + (lane + 1) * step, hi);
    const int n = __popcll(__ballot(lo + (lane + 1) * step <= hi && cu[at] <= t));
    const int to = lo + n * step;  // (cu[to] <= t)
    hi = min(hi, to + step - 1);
    lo = to;
  }
  return lo;
}

// One wave per token and kind of rows.
__global__ __launch_bounds__(AP_WAVES* WAVE) void cache_append_kernel(AppendSet set, RopeAngles a,
                                                                      const int* __restrict__ table,
                                                                      const int* __restrict__ ctx_len,
                                                                      const int* __restrict__ cu, int T, int B,
                                                                      int max_pages, int page_size, int num_pages) {
  __shared__ float stage[AP_WAVES][2 * RP_MAX_R];
  const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const long unit = (long)blockIdx.x * AP_WAVES + wave;
  const int t = (int)(unit / set.n), kind = (int)(unit - (long)t * set.n);
  if (t >= T) return;
  const AppendRows& r = set.rows[kind];
  const int G = r.width / 8;
  float v[AP_GROUPS][8];
#pragma unroll
  for (int i = 0; i < AP_GROUPS; ++i)  // (lanes past the row load its last columns)
    ap_load8(r.x, r.fp32, (long)t * r.x_row + 8 * min(lane + WAVE * i, G - 1), v[i]);

  // the token's place and slot
  int b, j, n;
  if (cu) {
    if (t < cu[0]) return;
    b = ap_sequence(cu, B, t);
    if (b >= B) return;  // (rows past the last sequence)
    j = t - cu[b], n = cu[b + 1] - cu[b];
  } else {
    n = T / B, b = t / n, j = t - b * n;
  }
  const long place = (long)ctx_len[b] - n + j;
  if (place < 0 || place >= (long)max_pages * page_size) return;
  const int page = table[(size_t)b * max_pages + place / page_size];
  if (page < 1 || page >= num_pages) return;
  const long slot = (long)page * page_size + place % page_size;

  if (r.weight) {
    const int NG = r.norm_width / 8;
    float sum = 0.0f, mean = 0.0f;
    if (r.bias) {
#pragma unroll
      for (int i = 0; i < AP_GROUPS; ++i)
        if (lane + WAVE * i < NG)
#pragma unroll
          for (int e = 0; e < 8; ++e) sum += v[i][e];
      mean = wave_sum(sum) / (float)r.norm_width;
    }
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < AP_GROUPS; ++i)
      if (lane + WAVE * i < NG)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(v[i][e] - mean, v[i][e] - mean, sum);
    const float inv = 1.0f / sqrtf(wave_sum(sum) / (float)r.norm_width + r.eps);
#pragma unroll
    for (int i = 0; i < AP_GROUPS; ++i) {
      const int g = lane + WAVE * i;
      if (g >= NG) break;
      float w[8], c[8] = {};
      ap_load8(r.weight, r.norm_fp32, 8 * g, w);
      if (r.bias) ap_load8(r.bias, r.norm_fp32, 8 * g, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = fmaf((v[i][e] - mean) * inv, w[e], c[e]);
    }
  }

  if (r.rope_at >= 0) {  // the rotated columns through LDS, a pair a lane
    float* const st = stage[wave];
    const int g0 = r.rope_at / 8, ng = a.R / 4;
#pragma unroll
    for (int i = 0; i < AP_GROUPS; ++i) {
      const int g = lane + WAVE * i - g0;
      if (g >= 0 && g < ng)
#pragma unroll
        for (int e = 0; e < 8; ++e) st[8 * g + e] = v[i][e];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int f = lane; f < a.R; f += WAVE) {
      const int pos = a.positions ? a.positions[(size_t)rope_axis(a, f) * T + t] : (int)place;
      const float2 cs = rope_angle(a, pos, f);
      const int p = r.half ? f : 2 * f, q = r.half ? f + a.R : 2 * f + 1;
      float x = st[p], y = st[q];
      turn_pair(x, y, cs);
      st[p] = x, st[q] = y;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < AP_GROUPS; ++i) {
      const int g = lane + WAVE * i - g0;
      if (g >= 0 && g < ng)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = st[8 * g + e];
    }
  }

  if (r.cache_bf16) {
    uint16_t* const row = static_cast<uint16_t*>(r.cache) + (size_t)slot * r.width;
#pragma unroll
    for (int i = 0; i < AP_GROUPS; ++i) {
      const int g = lane + WAVE * i;
      if (g < G)
        *reinterpret_cast<u32x4*>(row + 8 * g) = u32x4{bf16_pack(v[i][0], v[i][1]), bf16_pack(v[i][2], v[i][3]),
                                                       bf16_pack(v[i][4], v[i][5]), bf16_pack(v[i][6], v[i][7])};
    }
    return;
  }
  float s = 1.0f;
  if (r.scale) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < AP_GROUPS; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = lane + WAVE * i < G ? fmaxf(amax, fabsf(v[i][e])) : amax;
    s = fmaxf(wave_max(amax), 1e-30f) / AP_FP8_MAX;
    if (lane == 0) r.scale[slot] = s;
  }
  uint8_t* const row = static_cast<uint8_t*>(r.cache) + (size_t)slot * r.width;
#pragma unroll
  for (int i = 0; i < AP_GROUPS; ++i) {
    const int g = lane + WAVE * i;
    if (g >= G) break;
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = fminf(fmaxf(v[i][e] / s, -r.fp8_max), r.fp8_max);
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    *reinterpret_cast<uint2*>(row + 8 * g) = make_uint2((uint32_t)lo, (uint32_t)hi);
  }
}

hipError_t launch_cache_append(const AppendSet& set, const RopeAngles& a, const int* table, const int* ctx_len,
                               const int* cu, int T, int B, int max_pages, int page_size, int num_pages, hipStream_t s) {
  const long units = (long)T * set.n;
  return launch("cache_append_kernel", cache_append_kernel, dim3((unsigned)((units + AP_WAVES - 1) / AP_WAVES)),
                dim3(AP_WAVES * WAVE), s, set, a, table, ctx_len, cu, T, B, max_pages, page_size, num_pages);
}

}  // namespace dsa
