// Verification of drafted tokens for gfx950. Sequence b's rows of logits are cu[b] .. cu[b + 1] - 1; row j's probabilities
// are p_j = softmax(l_j / T_b), and all rows but the last have a drafted token x_j, drawn from the draft's q_j:
//   x_j is taken iff u_j q_j(x_j) < p_j(x_j), up to the first that is not;
//   then one token from that row, the stop row: the first i with sum_{k <= i} r(k) > v_b sum r, r = max(p - q, 0), or r = p
//   after the last row's drafts were all taken (and where r is 0 everywhere).
// At T_b = 0 a token is taken iff it is the first of the largest logits, and that one comes next.
//
// Which token comes does not depend on roundings in 32 bits, though nearly all rows are only summed in 32: a row's sum of
// exp((l - max) / T) is taken in 32 bits (off by VF_NEAR of itself at most), and only where that decides nothing, with u q
// and p that close, again in 64. The stop row's sums are in 64 bits: with w the weights and z the 32-bit sum, a pass over it
// sums w, and w - q z and q where that is above 0. r's sum at the 64-bit sum z' of w is then theirs plus (z - z') times q's,
// which is summed in 32 bits, off by 2^-20 of itself at most; tokens on either side of w = q z by less than VF_NEAR are too near
// to say, their r is off by q |z' - z| each. Where the sum of those bounds could move the token (or where r would be 0) the row
// is gone through once more with z'.
//
// Two launches, or three. verify_rows_kernel: a workgroup of 16 waves takes up to 32,768 logits of a row to (maximum, sum,
// place of the maximum), so that a row has few parts. verify_pick_kernel: every workgroup of a sequence finds its stop row
// alike, 8 lanes a row (in large batches verify_stop_kernel has found them), and sums a chunk of that; the last of them to be
// done (a count that the first launch cleared) looks for the token.
//
// The first launch is bound by the logits' bytes, where a wave's logits are not all masked (its sum is then NaN, and it goes
// through them twice more: with all but 50 of 131,072 at -infinity 56 us for 22). The others are bound by their chains of
// dependent reads (lengths, parts, the draft's logit, a chunk, the count, the sums, the chunk again) in short workgroups; vector
// instructions, a good part of them the stop row's 30 64-bit operations a logit, issue in half of the pick's time. 64 sequences
// of 5 rows of 131,072 logits (bf16) 45 to 46 us: 22 (3.8 TB/s) + 5 + 20; 13 ragged ones of up to 8 rows of 100,003 (fp32) 17.9
// to 18.4: 7.2 to 8.3 + 11.8; one of 4 rows of 32,768 13.7 to 14.8: 3.3 + 9.5.
#include "dsa_async.h"

namespace dsa {

constexpr int VF_THREADS = 256;
constexpr int VF_WAVES = VF_THREADS / WAVE;
constexpr int VF_VEC = 8;  // logits of a load
constexpr int VF_MAX_V = 1 << 30;
// Bound of a row's sum's error: exponents (l - max) k with three roundings, 1.5 2^-23 of themselves, which are 25 in the weights'
// mean at most (2^30 logits: their entropy less that of the largest alone; 13 for 2^17): 3.1e-6; two times exp2 2^-23; 16
// roundings of a term on its way into the sum, 1e-6; its product with a wave's weight and the part's sum in 32 bits 2^-24 each:
// 4.4e-6.
constexpr double VF_NEAR = 5e-6;

struct VerifyArgs {
  const void* logits;  // [N, V], rows l_row values apart, bf16 or fp32
  const void* probs;   // [N, V] or null: the drafts are certain
  const int* draft;    // [N]
  const int* cu;       // [B + 1]
  const float* u;      // [N]
  const float* v;      // [B]
  const float* temperature;  // [B]
  int* tokens;         // [N]
  int* accepted;       // [B]
  float* logp;         // [N]
  long l_row, q_row;
  int l_fp32, q_fp32;
  int N, V, B;
  int parts, chunks;   // of a row, for the two launches
};

struct VerifyPart {
  float max;
  float sum;  // of exp((l - max) / T)
  int first;  // the first place of the maximum (T = 0 alone)
  int pad;
};

// The count of a sequence's chunks that are summed, in a cache line of its own: the adds to a line wait for each other (32
// sequences a line: the pick of 64 rows of 131,072 34 us for 19).
struct VerifyCount {
  int n, pad[31];
};

struct VerifyChunk {  // sums over a chunk of the stop row
  double all;         // w
  double rest, q;     // w - q z, and q, where that is above 0
  double near;        // bound of what is too near to say
};

template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) VerifyVec {
  T x[N];
};

__device__ __forceinline__ float vf_value(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
__device__ __forceinline__ float vf_value(float x) { return x; }

// Values i .. i + 7 of a row, `none` past its end.
template <typename T>
__device__ __forceinline__ void vf_load(const T* row, int i, int V, float none, float (&x)[VF_VEC]) {
  if (i + VF_VEC <= V) {
    const VerifyVec<T, VF_VEC> u = *reinterpret_cast<const VerifyVec<T, VF_VEC>*>(row + i);
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) x[e] = vf_value(u.x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) {
      const float y = vf_value(row[min(i + e, V - 1)]);
      x[e] = i + e < V ? y : none;
    }
  }
}

// Logits i .. i + 7; a NaN is a token that cannot come.
__device__ __forceinline__ void vf_logits(const VerifyArgs& a, int row, int i, float (&x)[VF_VEC]) {
  if (a.l_fp32)
    vf_load(static_cast<const float*>(a.logits) + (size_t)row * a.l_row, i, a.V, -INFINITY, x);
  else
    vf_load(static_cast<const uint16_t*>(a.logits) + (size_t)row * a.l_row, i, a.V, -INFINITY, x);
#pragma unroll
  for (int e = 0; e < VF_VEC; ++e) x[e] = x[e] > -INFINITY ? x[e] : -INFINITY;
}

__device__ __forceinline__ float vf_logit(const VerifyArgs& a, int row, int i) {
  const float x = a.l_fp32 ? static_cast<const float*>(a.logits)[(size_t)row * a.l_row + i]
                           : vf_value(static_cast<const uint16_t*>(a.logits)[(size_t)row * a.l_row + i]);
  return x > -INFINITY ? x : -INFINITY;
}

// (l - m) / T in base 2, with k = log2 e / T; a maximum of infinity leaves 0 to its own tokens, -infinity to all others.
__device__ __forceinline__ double vf_exponent(float l, float m, double k) {
  const double x = l == m ? 0.0 : ((double)l - (double)m) * k;
  return x <= 0.0 && l > -INFINITY ? x : -INFINITY;
}

// 2^x for x <= 0 (x < -1022: 2^-1022), by the series of e^(f ln 2) about the nearest whole number; the first term left out is
// 2e-16 of it at most. (With two terms less, 2e-13, tokens moved where a draft's probabilities were the target's own.) The
// whole number is found, and put into the exponent, through the low bits of x + 1.5 2^52.
__device__ __forceinline__ double vf_exp2(double x) {
  x = fmax(x, -1022.0);
  const double big = 6755399441055744.0, n = x + big, f = x - (n - big);
  // (ln 2)^k / k!, in scalar registers: as literals each would be moved into the accumulator's first
  double c[13] = {1.0, 6.9314718055994530942e-1, 2.4022650695910071233e-1, 5.5504108664821579953e-2,
                  9.6181291076284771619e-3, 1.3333558146428443423e-3, 1.5403530393381609954e-4, 1.5252733804059840280e-5,
                  1.3215486790144309488e-6, 1.0178086009239699728e-7, 7.0549116208011233299e-9, 4.4455382718708114976e-10,
                  2.5678435993488205142e-11};
#pragma unroll
  for (int i = 0; i <= 12; ++i) asm("" : "+s"(c[i]));
  double p = c[12];
#pragma unroll
  for (int i = 11; i >= 0; --i) p = fma(p, f, c[i]);
  const long long u = __builtin_bit_cast(long long, p);
  const int hi = (int)(u >> 32) + ((int)__builtin_bit_cast(long long, n) << 20);
  return __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)u);
}

__device__ __forceinline__ double vf_weight(float l, float m, double k) {
  const double x = vf_exponent(l, m, k);
  return x > -1022.0 ? vf_exp2(x) : 0.0;
}

__device__ __forceinline__ double vf_rate(float temperature) {
  return 1.4426950408889634074 / (temperature > 0.0f ? (double)temperature : 1.0);
}

// The sum over the wave, in every lane.
__device__ __forceinline__ double vf_swap(double x, int ctrl) {
  const long long u = __builtin_bit_cast(long long, x);
  int lo = (int)u, hi = (int)(u >> 32);
  switch (ctrl) {
    case 0: lo = dpp<0xb1>(lo), hi = dpp<0xb1>(hi); break;
    case 1: lo = dpp<0x4e>(lo), hi = dpp<0x4e>(hi); break;
    case 2: lo = dpp<0x141>(lo), hi = dpp<0x141>(hi); break;
    default: lo = dpp<0x140>(lo), hi = dpp<0x140>(hi); break;
  }
  return __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
}

__device__ __forceinline__ double vf_lane(double x, int lane) {
  const long long u = __builtin_bit_cast(long long, x);
  const int lo = __builtin_amdgcn_readlane((int)u, lane), hi = __builtin_amdgcn_readlane((int)(u >> 32), lane);
  return __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
}

__device__ __forceinline__ double vf_wave_sum(double x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x += vf_swap(x, i);
  return (vf_lane(x, 0) + vf_lane(x, 16)) + (vf_lane(x, 32) + vf_lane(x, 48));
}

// The number of sequences that end by `row` (cu ascends), the same in every lane of the wave; B: past the last.
__device__ __forceinline__ int vf_sequence(const int* __restrict__ cu, int B, int row) {
  const int lane = threadIdx.x & (WAVE - 1);
  int lo = 0, hi = B;
  while (hi > lo) {
    const int step = (hi - lo + WAVE - 1) / WAVE, at = lo + (lane + 1) * step;
    const int n = __popcll(__ballot(at <= hi && cu[min(at, hi)] <= row));
    const int to = lo + n * step;
    hi = min(hi, to + step - 1);
    lo = to;
  }
  return lo;
}

// vf_weight in 32 bits. (In 64, though few lanes come to it, 320 rows of 131,072 took 28.4 us for 21.6.)
__device__ __forceinline__ float vf_weight32(float l, float m, float k) {
  const float x = l == m ? 0.0f : (l - m) * k;
  return x <= 0.0f && l > -INFINITY ? __builtin_amdgcn_exp2f(x) : 0.0f;
}

constexpr int VF_ROW_THREADS = 1024;
constexpr int VF_ROW_WAVES = VF_ROW_THREADS / WAVE;

// A workgroup's part of a row: LOADS x 8,192 logits, a wave's side by side. Not even a comparison is spent on NaN or
// infinities: they (and a wave whose logits are all -infinity) make a wave's sum NaN, and its logits are then gone through again
// with care.
template <typename T, int LOADS>
__global__ __launch_bounds__(VF_ROW_THREADS) void verify_rows_kernel(VerifyArgs a, VerifyPart* __restrict__ parts,
                                                                     VerifyCount* __restrict__ done) {
  __shared__ VerifyPart wave_part[VF_ROW_WAVES];
  const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  for (int b = blockIdx.x * VF_ROW_THREADS + threadIdx.x; b < a.B; b += gridDim.x * VF_ROW_THREADS) done[b].n = 0;
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  const int from = (part * VF_ROW_WAVES + wave) * LOADS * WAVE * VF_VEC, i0 = from + lane * VF_VEC;
  // (the sequences' ends are on their way before the logits, and the temperature while those are)
  const int end = a.cu[min(lane + 1, a.B)];
  float x[LOADS][VF_VEC];
#pragma unroll
  for (int i = 0; i < LOADS; ++i)
    vf_load(static_cast<const T*>(a.logits) + (size_t)row * a.l_row, i0 + i * WAVE * VF_VEC, a.V, -INFINITY, x[i]);
  int b = __popcll(__ballot(lane < a.B && end <= row));
  if (b == WAVE) b = vf_sequence(a.cu, a.B, row);
  if (b >= a.B || row < a.cu[0]) return;
  const float temperature = a.temperature[b];
  const float rate = (float)vf_rate(temperature);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < LOADS; ++i)
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) m = max_nonan(m, x[i][e]);  // (a NaN: as it was)
  m = wave_max(m);
  float s[4] = {};
#pragma unroll
  for (int i = 0; i < LOADS; ++i)
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) s[e & 3] += __builtin_amdgcn_exp2f((x[i][e] - m) * rate);
  float sum = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
  if (__builtin_expect(!(sum >= 0.0f), 0)) {
    const int to = min(from + LOADS * WAVE * VF_VEC, a.V);
    m = -INFINITY;
    for (int i = from + lane; i < to; i += WAVE) m = fmaxf(m, vf_logit(a, row, i));
    m = wave_max(m);
    double t = 0.0;
    for (int i = from + lane; i < to; i += WAVE) t += (double)vf_weight32(vf_logit(a, row, i), m, rate);
    sum = (float)vf_wave_sum(t);
  }
  uint32_t first = 0x7fffffffu;
  if (!(temperature > 0.0f)) {
#pragma unroll
    for (int i = LOADS - 1; i >= 0; --i)
#pragma unroll
      for (int e = VF_VEC - 1; e >= 0; --e) first = x[i][e] == m ? (uint32_t)(i0 + i * WAVE * VF_VEC + e) : first;
    first = wave_min_u32(first);
  }
  if (lane == 0) wave_part[wave] = VerifyPart{m, sum, (int)first, 0};
  __syncthreads();
  if (wave) return;
  VerifyPart w{-INFINITY, 0.0f, 0x7fffffff, 0};
  if (lane < VF_ROW_WAVES) w = wave_part[lane];
  m = wave_max(w.max);
  const double all = vf_wave_sum((double)(w.sum * vf_weight32(w.max, m, rate)));
  first = wave_min_u32(w.max == m ? (uint32_t)w.first : 0x7fffffffu);
  if (lane == 0) parts[blockIdx.x] = VerifyPart{m, (float)all, (int)first, 0};
}

__device__ __forceinline__ float vf_logp(float l, float m, double sum, double k) {
  return (float)(vf_exponent(l, m, k) * 0.69314718055994530942 - log(sum));
}

// A row's sum in 64 bits is asked for by the workgroup's first wave, which has found that it needs it (one row in 100,000),
// and computed by all: the others wait for questions (vf_answer) until there are no more (vf_no_more).
struct VerifyAsk {
  int row;  // -1: no more
  float m;
  double part[16];
};

__device__ __forceinline__ void vf_exact_part(const VerifyArgs& a, VerifyAsk& ask, double k) {
  double s = 0.0;
  for (int i = threadIdx.x * VF_VEC; i < a.V; i += blockDim.x * VF_VEC) {
    float x[VF_VEC];
    vf_logits(a, ask.row, i, x);
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) s += vf_weight(x[e], ask.m, k);
  }
  s = vf_wave_sum(s);
  if ((threadIdx.x & (WAVE - 1)) == 0) ask.part[threadIdx.x / WAVE] = s;
  __syncthreads();
}

__device__ __forceinline__ double vf_exact_sum(const VerifyArgs& a, VerifyAsk& ask, int row, float m, double k) {
  if (threadIdx.x == 0) ask.row = row, ask.m = m;
  __syncthreads();
  vf_exact_part(a, ask, k);
  double s = 0.0;
  for (int w = 0; w < (int)blockDim.x / WAVE; ++w) s += ask.part[w];
  return s;
}

__device__ __forceinline__ void vf_no_more(VerifyAsk& ask) {
  if (threadIdx.x == 0) ask.row = -1;
  __syncthreads();
}

__device__ __forceinline__ void vf_answer(const VerifyArgs& a, VerifyAsk& ask, double k) {
  for (;;) {
    __syncthreads();
    if (__builtin_expect(ask.row < 0, 1)) return;
    vf_exact_part(a, ask, k);
  }
}

struct VerifyStop {  // a sequence's stop row
  double sum;
  float max;
  int row;  // -1: nothing is drawn from it
};

// The stop row of rows r0 .. r1 - 1, by a wave, 8 lanes a row, a lane a part (or every 8th); `write`: and all that is written
// but the token drawn from it.
constexpr int VF_ROW_LANES = 8;
constexpr int VF_STOP_ROWS = WAVE / VF_ROW_LANES;

__device__ __forceinline__ VerifyStop vf_stop(const VerifyArgs& a, const VerifyPart* __restrict__ parts, int b, int r0, int r1,
                                              bool warm, double k, bool write, VerifyAsk& ask) {
  const int lane = threadIdx.x & (WAVE - 1), j = lane & (VF_ROW_LANES - 1);
#pragma unroll 1
  for (int row0 = r0;; row0 += VF_STOP_ROWS) {
    const int mine = row0 + lane / VF_ROW_LANES, row = min(mine, r1 - 1);
    const bool last = row == r1 - 1;
    const VerifyPart* const p = parts + (size_t)row * a.parts;
    VerifyPart part{-INFINITY, 0.0f, 0x7fffffff, 0};
    if (j < a.parts) part = p[j];
    const int x = a.draft[row], i = min(max(x, 0), a.V - 1);
    const float u = a.u[row], l = vf_logit(a, row, i);
    double q = 1.0;
    if (warm && a.probs)
      q = a.q_fp32 ? (double)static_cast<const float*>(a.probs)[(size_t)row * a.q_row + i]
                   : (double)vf_value(static_cast<const uint16_t*>(a.probs)[(size_t)row * a.q_row + i]);
    float m = part.max;
    for (int c = j + VF_ROW_LANES; c < a.parts; c += VF_ROW_LANES) m = fmaxf(m, p[c].max);
    m = fmaxf(m, __int_as_float(dpp<0xb1>(__float_as_int(m))));
    m = fmaxf(m, __int_as_float(dpp<0x4e>(__float_as_int(m))));
    m = fmaxf(m, __int_as_float(dpp<0x141>(__float_as_int(m))));
    double sum = 0.0;
    uint32_t first = 0x7fffffffu;  // (the parts' first places ascend)
    for (int c = j;;) {
      sum += (double)part.sum * vf_weight(part.max, m, k);
      if (part.max == m) first = min(first, (uint32_t)part.first);
      if ((c += VF_ROW_LANES) >= a.parts) break;
      part = p[c];
    }
    sum += vf_swap(sum, 0);
    sum += vf_swap(sum, 1);
    sum += vf_swap(sum, 2);
    first = min(first, (uint32_t)dpp<0xb1>((int)first));
    first = min(first, (uint32_t)dpp<0x4e>((int)first));
    first = min(first, (uint32_t)dpp<0x141>((int)first));
    const bool none = !(m > -INFINITY);
    bool taken = !last && x == i && !none;
    if (warm) {
      const double uq = (double)u * q, w = vf_weight(l, m, k);
      double s = sum;
      uint64_t todo = __ballot(taken && fabs(uq * sum - w) <= VF_NEAR * w);
      while (__builtin_expect(todo != 0, 0)) {
        const int who = __builtin_ctzll(todo) & ~(VF_ROW_LANES - 1);
        todo &= ~(0xffull << who);
        const double e = vf_exact_sum(a, ask, __builtin_amdgcn_readlane(row, who),
                                      __int_as_float(__builtin_amdgcn_readlane(__float_as_int(m), who)), k);
        if ((lane & ~(VF_ROW_LANES - 1)) == who) s = e;
      }
      taken = taken && uq * s < w;  // (not for a u q that is NaN)
    } else {
      taken = taken && x == (int)first;
    }
    const uint64_t refused = __ballot(!taken);  // (at the last row at the latest)
    const int at = refused ? __builtin_ctzll(refused) : WAVE, stop = row0 + at / VF_ROW_LANES;
    const bool drawn = warm && !none;
    if (write && mine < r1 && j == 0 && (row != stop || !drawn)) {
      const int y = row < stop ? x : row > stop || none ? -1 : (int)first;
      a.tokens[row] = y;
      a.logp[row] = y < 0 ? 0.0f : vf_logp(row < stop ? l : m, m, sum, k);
    }
    if (at == WAVE) continue;
    if (write) {
      if (lane == 0) a.accepted[b] = stop - r0;
      for (int r = row0 + VF_STOP_ROWS + lane; r < r1; r += WAVE) a.tokens[r] = -1, a.logp[r] = 0.0f;
    }
    return VerifyStop{vf_lane(sum, at), __int_as_float(__builtin_amdgcn_readlane(__float_as_int(m), at)),
                      __builtin_amdgcn_readlane((int)drawn, at) ? stop : -1};
  }
}

// Logits x and the draft's probabilities q (0 where there are none) of tokens i .. i + 7 of the stop row. A draft that is
// certain, d, cannot come (-1: there is no such draft).
__device__ __forceinline__ void vf_stop_row(const VerifyArgs& a, int row, bool with_q, int d, bool infinite, int i,
                                            float (&x)[VF_VEC], float (&q)[VF_VEC]) {
  if (a.l_fp32)
    vf_load(static_cast<const float*>(a.logits) + (size_t)row * a.l_row, i, a.V, -INFINITY, x);
  else
    vf_load(static_cast<const uint16_t*>(a.logits) + (size_t)row * a.l_row, i, a.V, -INFINITY, x);
  if (d >= i && d < i + VF_VEC) {
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) x[e] = i + e == d ? -INFINITY : x[e];
  }
  if (infinite) {  // (one of several: as many times 0)
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) x[e] = x[e] == INFINITY ? 0.0f : -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < VF_VEC; ++e) q[e] = 0.0f;
  if (with_q) {
    if (a.q_fp32)
      vf_load(static_cast<const float*>(a.probs) + (size_t)row * a.q_row, i, a.V, 0.0f, q);
    else
      vf_load(static_cast<const uint16_t*>(a.probs) + (size_t)row * a.q_row, i, a.V, 0.0f, q);
  }
}

// A weight of the stop row (m is finite there): 0 where vf_weight's is, so that no token comes whose probability is 0.
// (-infinity: exponent -infinity, or NaN at an infinite temperature)
__device__ __forceinline__ double vf_stop_weight(float x, float m, double k) {
  const double e = ((double)x - (double)m) * k, w = vf_exp2(e);
  return e > -1022.0 ? w : 0.0;
}

// v's inclusive prefix sum over the wave.
__device__ __forceinline__ double vf_wave_scan(double v) {
  const auto step = [&](auto lo, auto hi) { v += __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo); };
#define VF_STEP(...)                                                       \
  {                                                                        \
    const long long u = __builtin_bit_cast(long long, v);                  \
    step(dpp<__VA_ARGS__>((int)u), dpp<__VA_ARGS__>((int)(u >> 32)));      \
  }
  VF_STEP(0x111) VF_STEP(0x112) VF_STEP(0x114) VF_STEP(0x118) VF_STEP(0x142, 0xa, false) VF_STEP(0x143, 0xc, false)
#undef VF_STEP
  return v;
}

// The stop rows in a launch of their own, a workgroup a sequence (for its first wave).
constexpr int VF_STOP_THREADS = 1024;

__global__ __launch_bounds__(VF_STOP_THREADS) void verify_stop_kernel(VerifyArgs a, const VerifyPart* __restrict__ parts,
                                                                      VerifyStop* __restrict__ stops) {
  __shared__ VerifyAsk ask;
  const int b = blockIdx.x, r0 = min(max(a.cu[b], 0), a.N), r1 = min(max(a.cu[b + 1], 0), a.N);
  const float temperature = a.temperature[b];
  const double k = vf_rate(temperature);
  VerifyStop s{0.0, 0.0f, -1};
  if (r1 <= r0) {
    if (threadIdx.x == 0) a.accepted[b] = 0;
  } else if (threadIdx.x >= WAVE) {
    vf_answer(a, ask, k);
  } else {
    s = vf_stop(a, parts, b, r0, r1, temperature > 0.0f, k, true, ask);
    vf_no_more(ask);
  }
  if (threadIdx.x == 0) stops[b] = s;
}

// A sequence's workgroups sum a chunk of its stop row each; the last of them looks for the token. (Two or four chunks a
// workgroup, with all workgroups on the CUs at once: 64 rows of 131,072 20.0 and 22.8 us for 20.2.) FOUND: the stop rows are
// in stops, else the first wave finds its sequence's.
constexpr int VF_CHUNK = VF_THREADS * VF_VEC;

template <bool FOUND>
__global__ __launch_bounds__(VF_THREADS) void verify_pick_kernel(VerifyArgs a, const VerifyPart* __restrict__ parts,
                                                                 const VerifyStop* __restrict__ stops,
                                                                 VerifyChunk* __restrict__ sums,
                                                                 VerifyCount* __restrict__ done) {
  __shared__ VerifyStop stop_row;
  __shared__ VerifyAsk ask;
  __shared__ VerifyChunk part[VF_WAVES];
  __shared__ double tot[VF_WAVES], found_at, found_r;
  __shared__ float found_x;
  __shared__ int is_last, found, first[VF_WAVES], end[VF_WAVES];
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks, tid = threadIdx.x;
  const int lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int r0 = min(max(a.cu[b], 0), a.N), r1 = min(max(a.cu[b + 1], 0), a.N);
  const float temperature = a.temperature[b];
  const double k = vf_rate(temperature);
  VerifyStop at_stop;
  if (FOUND) {
    at_stop = stops[b];
  } else {
    if (r1 <= r0 || (chunk > 0 && !(temperature > 0.0f))) {
      if (r1 <= r0 && chunk == 0 && tid == 0) a.accepted[b] = 0;
      return;
    }
    if (wave == 0) {
      const VerifyStop s = vf_stop(a, parts, b, r0, r1, temperature > 0.0f, k, chunk == 0, ask);
      if (lane == 0) stop_row = s;
      vf_no_more(ask);
    } else {
      vf_answer(a, ask, k);
    }
    at_stop = stop_row;
  }
  const int stop = __builtin_amdgcn_readfirstlane(at_stop.row);
  if (stop < 0) return;
  const bool last = stop == r1 - 1, infinite = at_stop.max == INFINITY;
  const float m = infinite ? 0.0f : at_stop.max;
  const double z0 = at_stop.sum;
  const float zf = (float)z0;
  const int d = last || a.probs ? -1 : a.draft[stop];
  VerifyChunk* const row_sums = sums + (size_t)b * a.chunks;
  float xd = -INFINITY;  // a certain draft's logit
  {
    float x[VF_VEC], q[VF_VEC];
    vf_stop_row(a, stop, !last && a.probs, d, infinite, chunk * VF_CHUNK + VF_VEC * tid, x, q);
    if (d >= 0 && d < a.V) {
      xd = vf_logit(a, stop, d);
      if (infinite) xd = xd == INFINITY ? 0.0f : -INFINITY;
    }
    double all = 0.0, rest = 0.0;
    float taken = 0.0f, near = 0.0f;
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) {
      const double w = vf_stop_weight(x[e], m, k), r = fma(-(double)q[e], z0, w);
      const float edge = (float)VF_NEAR * q[e] * zf;
      all += w, rest += fmax(r, 0.0);
      taken += r > 0.0 ? q[e] : 0.0f;
      near += fabsf((float)r) <= edge ? edge : 0.0f;
    }
    all = vf_wave_sum(all), rest = vf_wave_sum(rest);
    taken = wave_sum(taken), near = wave_sum(near);
    if (lane == 0) part[wave] = VerifyChunk{all, rest, (double)taken, 1.01 * (double)near};
  }
  __syncthreads();
  if (wave == 0) {
    if (lane < 4) {  // (a number each)
      const double* const from = &part[0].all + lane;
      double t = from[0];
      for (int w = 1; w < VF_WAVES; ++w) t += from[4 * w];
      __hip_atomic_store(&row_sums[chunk].all + lane, t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // The sums are stored and loaded past the L2s, and are there before the count rises: no cache has to be written back or
    // emptied for them (a release and acquire here, which do that, made the launch 108 us for 29).
    wait_loads<0>();
    if (lane == 0)
      is_last = __hip_atomic_fetch_add(&done[b].n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.chunks - 1;
  }
  __syncthreads();
  if (!is_last) return;

  // The whole row's sums, every wave alike, 64 chunks at a time (the first of them stay in registers).
  const auto load = [&](int c) {
    VerifyChunk t{0.0, 0.0, 0.0, 0.0};
    if (c < a.chunks) {
      const double* const from = &row_sums[c].all;
      t.all = __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      t.rest = __hip_atomic_load(from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      t.q = __hip_atomic_load(from + 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      t.near = __hip_atomic_load(from + 3, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    return t;
  };
  const VerifyChunk front = load(lane);
  double z = front.all, near = front.near;
  for (int c0 = WAVE; c0 < a.chunks; c0 += WAVE) {
    const VerifyChunk t = load(c0 + lane);
    z += t.all, near += t.near;
  }
  // (a certain draft's own weight is not in `all`)
  z = vf_wave_sum(z) + vf_stop_weight(xd, m, k);
  // r's sum at z: it moves by q for every one that z does
  const auto rest_of = [&](const VerifyChunk& t) { return fmax(fma(z0 - z, t.q, t.rest), 0.0); };
  double rest = rest_of(front), taken = front.q;
  for (int c0 = WAVE; c0 < a.chunks; c0 += WAVE) {
    const VerifyChunk t = load(c0 + lane);
    rest += rest_of(t), taken += t.q;
  }
  rest = vf_wave_sum(rest);
  // The bounds were for a z off by VF_NEAR of itself; by now it is known by how much. And the chunks' q are sums in 32 bits,
  // 14 roundings of 2^-24 on a term's way into them.
  near = fabs(z - z0) * (vf_wave_sum(near) / (VF_NEAR * z0) + 0x1p-20 * vf_wave_sum(taken));
  // The chunk in which the sum passes the target (if rounding has it pass nowhere: the last that has anything).
  const double v = (double)a.v[b];
  double target = v * rest, before = 0.0;
  int c = -1;
  {
    double at = 0.0;
    VerifyChunk t = front;
    for (int c0 = 0;;) {
      const double y = rest_of(t), upto = at + vf_wave_scan(y);
      const uint64_t some = __ballot(y > 0.0), hit = __ballot(y > 0.0 && upto > target);
      const int l = hit ? __builtin_ctzll(hit) : some ? 63 - __builtin_clzll(some) : -1;
      if (l >= 0) c = c0 + l, before = vf_lane(upto - y, l);
      if (hit || (c0 += WAVE) >= a.chunks) break;
      at = vf_lane(upto, WAVE - 1);
      t = load(c0 + lane);
    }
  }
  // The token in it, first from these sums; where the tokens that were too near to say might move it, or r is 0 throughout,
  // chunk after chunk: r's sum, then its place, of max(w - q z, 0) and if that is 0 of w.
  enum { QUICK, SUM, PLACE } way = c >= 0 ? QUICK : SUM;
  if (way == SUM) c = 0, before = 0.0, target = INFINITY;
  bool from_p = false;
  int token = -1;
  for (;;) {
    const int i0 = c * VF_CHUNK + VF_VEC * tid;
    double w[VF_VEC], mine = 0.0;
    float x[VF_VEC], q[VF_VEC];
    vf_stop_row(a, stop, !last && !from_p && a.probs, from_p ? -1 : d, infinite, i0, x, q);
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) mine += w[e] = fmax(fma(-(double)q[e], z, vf_stop_weight(x[e], m, k)), 0.0);
    double upto = vf_wave_scan(mine);
    if (lane == WAVE - 1) tot[wave] = upto;
    __syncthreads();
    double sum = 0.0;
    for (int y = 0; y < VF_WAVES; ++y) {
      if (y == wave) upto += before + sum;
      sum += tot[y];
    }
    const uint64_t some = __ballot(mine > 0.0), hit = __ballot(mine > 0.0 && upto > target);
    if (lane == 0) {
      first[wave] = hit ? tid + __builtin_ctzll(hit) : VF_THREADS;
      end[wave] = some ? tid + 63 - __builtin_clzll(some) : -1;
    }
    __syncthreads();
    int passed = VF_THREADS, who = -1;
    for (int y = VF_WAVES - 1; y >= 0; --y) passed = min(passed, first[y]), who = max(who, end[y]);
    if (passed < VF_THREADS) who = passed;
    if (tid == who) {
      double at = upto - mine, at_y = at, r = 0.0;
      float xy = 0.0f;
      int y = -1;
      bool open = true;
#pragma unroll
      for (int e = 0; e < VF_VEC; ++e) {
        if (open && w[e] > 0.0) y = i0 + e, at_y = at, r = w[e], xy = x[e];
        at += w[e];
        open = open && !(w[e] > 0.0 && at > target);
      }
      found = y, found_at = at_y, found_r = r, found_x = xy;
    }
    __syncthreads();
    if (who >= 0) token = found;
    if (way == QUICK) {
      // (the chunks' sums, and with them the target, are off by `near` at most: 0 where there is no q)
      if (who >= 0 && (near == 0.0 || (target - found_at > 2.0 * near && found_at + found_r - target > 2.0 * near))) break;
      way = SUM, c = 0, before = 0.0, target = INFINITY, token = -1;
      continue;
    }
    if (way == PLACE && passed < VF_THREADS) break;
    before += sum;
    if (++c < a.chunks) continue;
    if (way == PLACE) break;
    if (before > 0.0) way = PLACE, target = v * before, token = -1;
    else if (from_p) break;
    else from_p = true;
    c = 0, before = 0.0;
  }
  if (tid == 0) {
    a.tokens[stop] = token;
    a.logp[stop] = token < 0 ? 0.0f : vf_logp(found_x, m, z, k);
  }
}

// Loads of a thread of the first launch: few, so that a small vocabulary is spread out, as long as a row has at most 8 parts
// (4 for 52 rows of 100,003 11.6 us for 9.0 then; 1 for 320 of 131,072 29.4 for 23.9 then).
static int verify_loads(int V) { return V > 16 * VF_ROW_THREADS * VF_VEC ? 4 : V > 8 * VF_ROW_THREADS * VF_VEC ? 2 : 1; }
static int verify_units(int V, int per) { return (V + per - 1) / per; }

// (a row's tiles end less than 2^16 logits past it: their indices are ints)
bool verify_grid_ok(int N, int V) {
  return V <= VF_MAX_V && (long)N * verify_units(V, VF_CHUNK) <= 0xffffffL && (long)N * verify_units(V, VF_ROW_THREADS * VF_VEC) <= 0x3fffffL;
}

size_t verify_workspace_bytes(int N, int V, int B) {
  if (V > VF_MAX_V) return 0;
  const int parts = verify_units(V, VF_ROW_THREADS * VF_VEC * verify_loads(V)), chunks = verify_units(V, VF_CHUNK);
  return (size_t)B * sizeof(VerifyCount) + (size_t)N * parts * sizeof(VerifyPart) +
         (size_t)B * (chunks * sizeof(VerifyChunk) + sizeof(VerifyStop));
}

hipError_t launch_verify(const void* logits, int l_fp32, long l_row, const int* draft, const void* probs, int q_fp32,
                         long q_row, const int* cu, const float* u, const float* v, const float* temperature, int* tokens,
                         int* accepted, float* logp, void* ws, int N, int V, int B, int num_cu, hipStream_t s) {
  const int loads = verify_loads(V);
  const VerifyArgs a{logits, probs, draft, cu, u, v, temperature, tokens, accepted, logp, l_row, q_row, l_fp32, q_fp32,
                     N, V, B, verify_units(V, VF_ROW_THREADS * VF_VEC * loads), verify_units(V, VF_CHUNK)};
  VerifyCount* const done = static_cast<VerifyCount*>(ws);
  VerifyPart* const parts = reinterpret_cast<VerifyPart*>(done + B);
  VerifyChunk* const sums = reinterpret_cast<VerifyChunk*>(parts + (size_t)N * a.parts);
  VerifyStop* const stops = reinterpret_cast<VerifyStop*>(sums + (size_t)B * a.chunks);
  const auto rows = [&](auto kernel) {
    return launch("verify_rows_kernel", kernel, dim3((unsigned)(N * a.parts)), dim3(VF_ROW_THREADS), s, a, parts, done);
  };
  hipError_t e = hipSuccess;
  if (N > 0 && l_fp32)
    e = loads == 4   ? rows(verify_rows_kernel<float, 4>)
        : loads == 2 ? rows(verify_rows_kernel<float, 2>)
                     : rows(verify_rows_kernel<float, 1>);
  else if (N > 0)
    e = loads == 4   ? rows(verify_rows_kernel<uint16_t, 4>)
        : loads == 2 ? rows(verify_rows_kernel<uint16_t, 2>)
                     : rows(verify_rows_kernel<uint16_t, 1>);
  if (e != hipSuccess) return e;
  const auto pick = [&](auto kernel) {
    return launch("verify_pick_kernel", kernel, dim3((unsigned)(B * a.chunks)), dim3(VF_THREADS), s, a, parts, stops, sums,
                  done);
  };
  // Where the workgroups do not all run at once (5 a CU), each finding its stop row costs more than a launch that does: 64
  // sequences of 131,072 42 us for 5 + 20, 13 of 100,003 13.6 for 5 + 9.6.
  if ((long)B * a.chunks <= 5L * num_cu) return pick(verify_pick_kernel<false>);
  e = launch("verify_stop_kernel", verify_stop_kernel, dim3(B), dim3(VF_STOP_THREADS), s, a, parts, stops);
  return e == hipSuccess ? pick(verify_pick_kernel<true>) : e;
}

}  // namespace dsa
