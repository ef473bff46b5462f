// Rotary positions for gfx950: x [T, H, 2R] rotated by each token's positions on up to four axes (time, height, width, ..),
// pair i by the angle p[axis(i)] inv_freq[i]:
//   (y0, y1) = factor (x0 cos - x1 sin, x1 cos + x0 sin),  pairs (2i, 2i + 1), or (i, i + R).
//
// A copy's bytes bound it (6 operations a pair): 8,192 tokens of 64 heads, the 64 last of 192 columns in bf16, 134 MB in and
// out, take 33 us, 4.1 TB/s where a large copy of whole rows reaches 5.1; 8 tokens 3.2 us, a launch and two round trips to
// memory. So a thread's values are 16 bytes, four of its items are on the way before the angles are computed, and those (a
// 64-bit product and two series) are a workgroup's, for all heads of its tokens, instead of each item's.
#include "dsa_rope.h"

namespace dsa {

constexpr int RT_THREADS = 256;
constexpr int RT_AT_ONCE = 4;

template <typename T>
struct RopeVec;  // 16 bytes of values

template <>
struct RopeVec<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const uint16_t* p, float (&v)[8]) {
    const u32x4 u = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(uint16_t* p, const float (&v)[8]) {
    *reinterpret_cast<u32x4*>(p) =
        u32x4{bf16_pack(v[0], v[1]), bf16_pack(v[2], v[3]), bf16_pack(v[4], v[5]), bf16_pack(v[6], v[7])};
  }
  static __device__ __forceinline__ float get(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
  static __device__ __forceinline__ void put(uint16_t* p, float v) { *p = (uint16_t)bf16_pack(v, 0.0f); }
};

template <>
struct RopeVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
    const f32x4 u = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = u[i];
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};

// A workgroup has `tokens` tokens and `heads` heads of them. Its angles are computed once, into LDS. VEC: 16 bytes of a row
// at a time (from both halves of it, where the pairs are (i, i + R)); else a pair at a time.
template <typename T, bool HALF, bool VEC>
__global__ __launch_bounds__(RT_THREADS) void rope_rotate_kernel(const T* x, long x_row, long x_head, T* out, long out_row,
                                                                 long out_head, RopeAngles a, int n_tokens, int H,
                                                                 int tokens, int heads, int head_groups) {
  __shared__ float2 cs[RT_THREADS];
  constexpr int N = RopeVec<T>::N;
  const int R = a.R, tid = threadIdx.x;
  const int tg = blockIdx.x / head_groups, hg = blockIdx.x - tg * head_groups;
  const int t0 = tg * tokens, h0 = hg * heads;
  const int nt = min(tokens, n_tokens - t0), nh = min(heads, H - h0);
  // A thread has the same item of every `step`-th row (token t, head h). RT_AT_ONCE rows' loads go out before the first store
  // (which may be to the same memory), the first of them before the angles are computed.
  const int per = VEC ? (HALF ? R / N : 2 * R / N) : R;  // items of a row
  const int step = RT_THREADS / per, row0 = tid / per, c = tid - row0 * per;
  const int dt = step / nh, dh = step - dt * nh;
  int t = row0 / nh, h = row0 - t * nh;
  if (row0 >= step) t = nt;  // (no item)
  constexpr int V = VEC ? N : 1;
  T* yr[RT_AT_ONCE];
  int tok[RT_AT_ONCE];
  float u[RT_AT_ONCE][V], v[RT_AT_ONCE][V];
  const auto load = [&]() {
#pragma unroll
    for (int k = 0; k < RT_AT_ONCE; ++k) {
      tok[k] = t;
      if (t < nt) {
        const T* const xr = x + (size_t)(t0 + t) * x_row + (size_t)(h0 + h) * x_head;
        yr[k] = out + (size_t)(t0 + t) * out_row + (size_t)(h0 + h) * out_head;
        if constexpr (VEC) {
          RopeVec<T>::load(xr + N * c, u[k]);
          if (HALF) RopeVec<T>::load(xr + R + N * c, v[k]);
        } else {
          u[k][0] = RopeVec<T>::get(xr + (HALF ? c : 2 * c));
          v[k][0] = RopeVec<T>::get(xr + (HALF ? c + R : 2 * c + 1));
        }
      }
      t += dt, h += dh;
      if (h >= nh) h -= nh, ++t;
    }
  };
  load();
  for (int i = tid; i < nt * R; i += RT_THREADS) {
    const int y = i / R, f = i - y * R;
    cs[i] = rope_angle(a, a.positions[(size_t)rope_axis(a, f) * n_tokens + t0 + y], f);
  }
  __syncthreads();
  for (;;) {
#pragma unroll
    for (int k = 0; k < RT_AT_ONCE; ++k) {
      if (tok[k] >= nt) return;
      const float2* const w = cs + tok[k] * R;
      if constexpr (!VEC) {
        turn_pair(u[k][0], v[k][0], w[c]);
        RopeVec<T>::put(yr[k] + (HALF ? c : 2 * c), u[k][0]);
        RopeVec<T>::put(yr[k] + (HALF ? c + R : 2 * c + 1), v[k][0]);
      } else if constexpr (HALF) {
#pragma unroll
        for (int e = 0; e < N; ++e) turn_pair(u[k][e], v[k][e], w[N * c + e]);
        RopeVec<T>::store(yr[k] + N * c, u[k]);
        RopeVec<T>::store(yr[k] + R + N * c, v[k]);
      } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) turn_pair(u[k][e], u[k][e + 1], w[(N * c + e) / 2]);
        RopeVec<T>::store(yr[k] + N * c, u[k]);
      }
    }
    load();
  }
}

template <typename T>
static hipError_t rotate(const T* x, long x_row, long x_head, T* out, long out_row, long out_head, const RopeAngles& a,
                         int n_tokens, int H, int half, int num_cu, hipStream_t s) {
  constexpr int N = RopeVec<T>::N;
  const auto bytes16 = [](const void* p, long u, long v) {
    return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(u * (long)sizeof(T)) | (uintptr_t)(v * (long)sizeof(T))) & 15) == 0;
  };
  const bool vec = bytes16(x, x_row, x_head) && bytes16(out, out_row, out_head) && (half ? a.R : 2 * a.R) % N == 0;
  // As many tokens a workgroup as it has threads for their angles while that leaves 4 workgroups a CU (16,384 tokens of one
  // head 4.6 us, 6.1 with 16 a CU; 2,000 of 128 heads 12.8, 13.5 with one), all heads while there is a workgroup a CU (with 4
  // asked for 200 tokens of 64 heads 3.2 -> 4.0 us: the angles again for each group of heads).
  int tokens = RT_THREADS / a.R, heads = H;
  while (tokens > 1 && (n_tokens + tokens - 1) / tokens < 4 * num_cu) tokens /= 2;
  if (tokens < 1) tokens = 1;
  const long groups = (n_tokens + tokens - 1) / tokens;
  while (heads > 1 && groups * ((H + heads - 1) / heads) < num_cu) heads = (heads + 1) / 2;
  const int head_groups = (H + heads - 1) / heads;
  const dim3 grid((unsigned)(groups * head_groups));
  const auto go = [&](auto kernel) {
    return launch("rope_rotate_kernel", kernel, grid, dim3(RT_THREADS), s, x, x_row, x_head, out, out_row, out_head, a,
                  n_tokens, H, tokens, heads, head_groups);
  };
  if (half) return vec ? go(rope_rotate_kernel<T, true, true>) : go(rope_rotate_kernel<T, true, false>);
  return vec ? go(rope_rotate_kernel<T, false, true>) : go(rope_rotate_kernel<T, false, false>);
}

hipError_t launch_rope_rotate(const void* x, int fp32, long x_row, long x_head, void* out, long out_row, long out_head,
                              const RopeAngles& a, int n_tokens, int H, int half, int num_cu, hipStream_t s) {
  if (fp32)
    return rotate(static_cast<const float*>(x), x_row, x_head, static_cast<float*>(out), out_row, out_head, a, n_tokens,
                  H, half, num_cu, s);
  return rotate(static_cast<const uint16_t*>(x), x_row, x_head, static_cast<uint16_t*>(out), out_row, out_head, a,
                n_tokens, H, half, num_cu, s);
}

}  // namespace dsa
