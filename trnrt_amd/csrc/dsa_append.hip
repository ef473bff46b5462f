// Appends to the paged caches for gfx950: each new token's rows (its latent row, its indexer key) normed, rotated,
// quantised and written to the slot that its place in its sequence has in the page table, in one launch:
//   y = x, its first n columns normed: x / sqrt(mean x^2 + eps) w, or (x - mean) / sqrt(var + eps) w + b;
//   2R of y's columns rotated by the token's positions (dsa_rope.h);
//   s = max(absmax(y), 1e-30) / 448, cache[slot] = e4m3(clamp(y / s)), scale[slot] = s.
// Everything between the row's load and its store is in fp32 and is rounded once.
//
// 16 lanes have a row (a row of the DPP network: its sums and maxima never leave it), 8 of its columns at a time each, so that
// rows of 576 and of 128 columns both leave few lanes idle; a wave has the rows of one kind of 4 tokens. What bounds it is
// vector issue (13 of the 23 us of 21,456 tokens with norms and three axes, whose 46 MB a copy would move in 9), then loads
// that one wave's four tokens do not cover; 8 tokens 4.4 us: a launch and three dependent reads (lengths, page, row). Not
// kept, of those 23 us: every kind's rows in one wave 23.2; registers for 5 or 6 waves a SIMD 22.8 and 32; workgroups of 1
// and 2 waves 27 and 24; a wave a row, which
// divides by s, 40.
#include "dsa_append.h"

namespace dsa {

constexpr int AP_WAVES = 4;
constexpr int AP_LANES = 16;                            // of a row
constexpr int AP_TOKENS = WAVE / AP_LANES;              // of a wave
constexpr float AP_FP8_MAX = 448.0f;

template <int R>
struct ApWave {  // LDS of a wave: its tokens' (cos, sin), and the rotated columns where pairs lie apart
  float2 cs[AP_TOKENS][R];
  float x[AP_TOKENS][2 * R];
};

// Eight values of type T from p + n on; p is a lane's own address, n the same in every lane.
template <typename T>
__device__ __forceinline__ void ap_load8(const T* p, int n, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4* q = reinterpret_cast<const f32x4*>(p + n);
    const f32x4 a = q[0], b = q[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  } else {
    const u32x4 u = *reinterpret_cast<const u32x4*>(p + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(u[e] << 16);
      v[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ void ap_wave_sync() {  // (LDS accesses of a wave are in order; so must the compiler's be)
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The number of sequences that end by token t (cu ascends), each row of 16 lanes its own t.
__device__ __forceinline__ int ap_sequence(const int* __restrict__ cu, int B, int t) {
  const int lane = threadIdx.x & (WAVE - 1), j = lane & (AP_LANES - 1);
  int lo = 0, hi = B;  // the answer is in [lo, hi]
  while (__ballot(hi > lo)) {
    const int step = max((hi - lo + AP_LANES - 1) / AP_LANES, 1), at = lo + (j + 1) * step;
    const uint64_t below = __ballot(at <= hi && cu[min(at, hi)] <= t);
    const int to = lo + step * __popc((uint32_t)(below >> (lane & ~(AP_LANES - 1))) & 0xffffu);
    hi = min(hi, to + step - 1);
    lo = to;
  }
  return lo;
}

// A token's slot, -1 where it is not written; place: where it stands in its sequence.
__device__ __forceinline__ long ap_slot(const int* __restrict__ table, const int* __restrict__ ctx_len,
                                        const int* __restrict__ cu, int t, int T, int B, int max_pages, int page_size,
                                        int num_pages, int& place) {
  int b, j, n;
  if (cu) {
    b = ap_sequence(cu, B, t);
    if (b >= B || t < cu[0]) return -1;  // (in no sequence)
    j = t - cu[b], n = cu[b + 1] - cu[b];
  } else {
    n = T / B, b = t / n, j = t - b * n;
  }
  const long at = (long)ctx_len[b] - n + j;
  if (at < 0 || at >= (long)max_pages * page_size) return -1;
  place = (int)at;
  const uint32_t col = (uint32_t)place / (uint32_t)page_size;
  const int page = table[(size_t)b * max_pages + col];
  return page < 1 || page >= num_pages ? -1 : (long)page * page_size + (place - (int)col * page_size);
}

// Rows of up to 128 NG columns: group i of a lane is columns 8 (16 i + j) .. + 7.
template <int NG, int R>
__device__ __forceinline__ void ap_rows(const AppendRows& r, const RopeAngles& a, const int* __restrict__ table,
                                        const int* __restrict__ ctx_len, const int* __restrict__ cu, int t0, int T, int B,
                                        int max_pages, int page_size, int num_pages, ApWave<R>& sh) {
  const int lane = threadIdx.x & (WAVE - 1), j = lane & (AP_LANES - 1), tok = lane / AP_LANES;
  const int t = min(t0 + tok, T - 1), G = r.width / 8;
  const int full = G / AP_LANES, rest = G % AP_LANES;  // groups of every lane, and lanes with one more
  float v[NG][8];
  const auto load = [&](auto* x) {
    x += (long)t * r.x_row + 8 * j;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      if (i < full) ap_load8(x, 8 * AP_LANES * i, v[i]);
      if (i == full) {  // (the other lanes' are 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
        if (j < rest) ap_load8(x, 8 * AP_LANES * i, v[i]);
      }
    }
  };
  if (r.fp32) load(static_cast<const float*>(r.x));
  else load(static_cast<const uint16_t*>(r.x));
  int place = 0;
  long slot = ap_slot(table, ctx_len, cu, t, T, B, max_pages, page_size, num_pages, place);
  if (t0 + tok >= T) slot = -1;

  if (r.weight) {
    const int N = r.norm_width / 8;
    const float count = 1.0f / (float)r.norm_width;
    if (r.bias) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < NG; ++i)
        if (j + AP_LANES * i < N)
#pragma unroll
          for (int e = 0; e < 8; ++e) sum += v[i][e];
      const float mean = row_sum(sum) * count;
#pragma unroll
      for (int i = 0; i < NG; ++i)
        if (j + AP_LANES * i < N)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] -= mean;
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NG; ++i)
      if (j + AP_LANES * i < N)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(v[i][e], v[i][e], sum);
    const float inv = 1.0f / sqrtf(fmaf(row_sum(sum), count, r.eps));
    const auto apply = [&](auto* w, auto* c) {
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        if (j + AP_LANES * i >= N) continue;
        float x[8];
        ap_load8(w + 8 * j, 8 * AP_LANES * i, x);
        if (c) {
          float y[8];
          ap_load8(c + 8 * j, 8 * AP_LANES * i, y);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = fmaf(v[i][e] * inv, x[e], y[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * inv * x[e];
        }
      }
    };
    if (r.norm_fp32) apply(static_cast<const float*>(r.weight), static_cast<const float*>(r.bias));
    else apply(static_cast<const uint16_t*>(r.weight), static_cast<const uint16_t*>(r.bias));
  }

  if (r.rope_at >= 0) {
    const int g0 = r.rope_at / 8, ng = a.R / 4;
    for (int f = j, n = 0; f < a.R; f += AP_LANES, ++n) {
      static_assert(AP_LANES == 16, "frequencies whose axes one word holds");
      const uint32_t axis = (a.axis[n] >> (2 * j)) & 3;
      sh.cs[tok][f] = rope_angle(a, a.positions ? a.positions[axis * (uint32_t)T + (uint32_t)t] : place, f);
    }
    if (r.half) {
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const int g = j + AP_LANES * i - g0;
        if (g >= 0 && g < ng)
#pragma unroll
          for (int e = 0; e < 8; ++e) sh.x[tok][8 * g + e] = v[i][e];
      }
    }
    ap_wave_sync();
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int g = j + AP_LANES * i - g0;
      if (g < 0 || g >= ng) continue;
      if (r.half) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // (column c: of pair c, or c - R)
          const int c = 8 * g + e;
          float x = c < a.R ? v[i][e] : sh.x[tok][c - a.R], y = c < a.R ? sh.x[tok][c + a.R] : v[i][e];
          turn_pair(x, y, sh.cs[tok][c < a.R ? c : c - a.R]);
          v[i][e] = c < a.R ? x : y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2) turn_pair(v[i][e], v[i][e + 1], sh.cs[tok][4 * g + e / 2]);
      }
    }
  }

  if (r.cache_bf16) {
    if (slot < 0) return;
    uint16_t* const row = static_cast<uint16_t*>(r.cache) + (size_t)slot * r.width;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int g = j + AP_LANES * i;
      if (g < G)
        *reinterpret_cast<u32x4*>(row + 8 * g) = u32x4{bf16_pack(v[i][0], v[i][1]), bf16_pack(v[i][2], v[i][3]),
                                                       bf16_pack(v[i][4], v[i][5]), bf16_pack(v[i][6], v[i][7])};
    }
    return;
  }
  // The quotient by s, correctly rounded as store's is: the product with the (correctly rounded) reciprocal, corrected by the
  // remainder, which is exact; only a divisor whose mantissa is all ones needs the division itself, and an infinite one no
  // correction. Without a scale nothing is divided (an infinity's remainder by 1 would be NaN, which is clamped to -).
  float s = 1.0f;
  if (r.scale) {
    float amax = 0.0f;  // (columns past the row are 0)
#pragma unroll
    for (int i = 0; i < NG; ++i)
      if (AP_LANES * i < G)
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[i][e]));
    s = fmaxf(row_max(amax), 1e-30f) / AP_FP8_MAX;
    if (slot >= 0 && j == 0) r.scale[slot] = s;
  }
  if (slot < 0) return;
  const float inv = 1.0f / s;
  const bool ones = (__float_as_uint(s) & 0x7fffffu) == 0x7fffffu;
  const float by = s < INFINITY ? s : 0.0f;
  uint8_t* const row = static_cast<uint8_t*>(r.cache) + (size_t)slot * r.width + 8 * j;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int g = j + AP_LANES * i;
    if (g >= G) continue;
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = v[i][e] * inv;
      q[e] = fmaf(fmaf(-p, by, v[i][e]), inv, p);
    }
    if (ones) {
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = v[i][e] / s;
    }
    if (!r.scale) {
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = v[i][e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = __builtin_amdgcn_fmed3f(q[e], -r.fp8_max, r.fp8_max);  // (NaN: -)
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    *reinterpret_cast<uint2*>(row + 8 * AP_LANES * i) = make_uint2((uint32_t)lo, (uint32_t)hi);
  }
}

// For rows of up to 128 NG columns and R frequencies.
template <int NG, int R>
__global__ __launch_bounds__(AP_WAVES* WAVE) void cache_append_kernel(AppendSet set, RopeAngles a,
                                                                      const int* __restrict__ table,
                                                                      const int* __restrict__ ctx_len,
                                                                      const int* __restrict__ cu, int T, int B,
                                                                      int max_pages, int page_size, int num_pages) {
  __shared__ ApWave<R> sh[AP_WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int unit = blockIdx.x * AP_WAVES + wave, four = unit / set.n, t0 = four * AP_TOKENS;
  if (t0 >= T) return;
  const AppendRows& r = set.rows[unit - four * set.n];
  if (r.width <= 128)
    ap_rows<1>(r, a, table, ctx_len, cu, t0, T, B, max_pages, page_size, num_pages, sh[wave]);
  else
    ap_rows<NG>(r, a, table, ctx_len, cu, t0, T, B, max_pages, page_size, num_pages, sh[wave]);
}

hipError_t launch_cache_append(const AppendSet& set, const RopeAngles& a, const int* table, const int* ctx_len,
                               const int* cu, int T, int B, int max_pages, int page_size, int num_pages, hipStream_t s) {
  const long units = ((long)T + AP_TOKENS - 1) / AP_TOKENS * set.n;
  int width = 0;
  for (int i = 0; i < set.n; ++i) width = width > set.rows[i].width ? width : set.rows[i].width;
  const auto go = [&](auto kernel) {
    return launch("cache_append_kernel", kernel, dim3((unsigned)((units + AP_WAVES - 1) / AP_WAVES)), dim3(AP_WAVES * WAVE), s,
                  set, a, table, ctx_len, cu, T, B, max_pages, page_size, num_pages);
  };
  // (the wider one for the same rows: 39 us for 23)
  return width <= 640 && a.R <= 64 ? go(cache_append_kernel<5, 64>) : go(cache_append_kernel<AP_MAX_WIDTH / 128, RP_MAX_R>);
}

}  // namespace dsa
