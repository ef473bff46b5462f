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
// sums w, and w and q where w > q z. r's sum is then the latter two's difference at the 64-bit sum; tokens on either side of
// w = q z by less than VF_NEAR are too near to say, their r is at most VF_NEAR q z each, and where the sum of those bounds
// could move the token (or where r would be 0) the row is gone through once more with the 64-bit sum.
//
// Two launches. verify_rows_kernel: a wave takes 512 to 2,048 logits of a row to (maximum, sum, place of the maximum),
// without LDS. verify_pick_kernel: every workgroup of a sequence finds the stop row from those alike; each sums a chunk of it,
// and the last to be done (a count per sequence, cleared by the first launch) looks for the token.
#include "dsa_common.h"

namespace dsa {

constexpr int VF_THREADS = 256;
constexpr int VF_WAVES = VF_THREADS / WAVE;
constexpr int VF_VEC = 8;  // logits of a load
// Bound of a row's sum's error: exponents (l - max) k in two terms, 2^-23 of themselves, 20 at the weights' mean (2^17 logits)
// at most: 1.7e-6; exp2 2^-23; 16 roundings of a term on its way into the sum, 1e-6; the part's sum in 32 bits 2^-24.
constexpr double VF_NEAR = 1e-5;

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

struct VerifyChunk {  // of the stop row
  double all;         // w
  double over, q;     // w and q where w > q z
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
    for (int e = 0; e < VF_VEC; ++e) x[e] = i + e < V ? vf_value(row[i + e]) : none;
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

__device__ __forceinline__ double vf_weight(float l, float m, double k) { return exp2(vf_exponent(l, m, k)); }

__device__ __forceinline__ double vf_rate(float temperature) {
  return 1.4426950408889634074 / (temperature > 0.0f ? (double)temperature : 1.0);
}

__device__ __forceinline__ int vf_row(const VerifyArgs& a, int b) { return min(max(a.cu[b], 0), a.N); }

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

// 2^x for x <= 0, by the series of e^(x ln 2) about the nearest whole number: the first term left out is 6e-15 of it.
__device__ __forceinline__ double vf_exp2(double x) {
  x = fmax(x, -1100.0);  // (2^-1100 is 0)
  const double n = rint(x), t = (x - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = fma(p, t, 1.0 / 3628800.0);
  p = fma(p, t, 1.0 / 362880.0);
  p = fma(p, t, 1.0 / 40320.0);
  p = fma(p, t, 1.0 / 5040.0);
  p = fma(p, t, 1.0 / 720.0);
  p = fma(p, t, 1.0 / 120.0);
  p = fma(p, t, 1.0 / 24.0);
  p = fma(p, t, 1.0 / 6.0);
  p = fma(p, t, 0.5);
  p = fma(p, t, 1.0);
  p = fma(p, t, 1.0);
  return ldexp(p, (int)n);
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

// A wave per unit: LOADS x 512 logits of a row. Not even a comparison is spent on NaN or infinities: they make the sum NaN,
// and the unit is then done again with care.
template <typename T, int LOADS>
__global__ __launch_bounds__(VF_THREADS) void verify_rows_kernel(VerifyArgs a, VerifyPart* __restrict__ parts,
                                                                 int* __restrict__ done) {
  const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int unit = blockIdx.x * VF_WAVES + wave;
  for (int b = blockIdx.x * VF_THREADS + threadIdx.x; b < a.B; b += gridDim.x * VF_THREADS) done[b] = 0;
  const int row = unit / a.parts, part = unit - row * a.parts;
  if (row >= a.N) return;
  const int i0 = (part * LOADS * WAVE + lane) * VF_VEC;
  float x[LOADS][VF_VEC];
#pragma unroll
  for (int i = 0; i < LOADS; ++i)
    vf_load(static_cast<const T*>(a.logits) + (size_t)row * a.l_row, i0 + i * WAVE * VF_VEC, a.V, -INFINITY, x[i]);
  if (row < a.cu[0]) return;
  const int b = vf_sequence(a.cu, a.B, row);
  if (b >= a.B) return;
  const float temperature = a.temperature[b];
  const double k = vf_rate(temperature);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < LOADS; ++i)
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) m = fmaxf(m, x[i][e]);
  m = wave_max(m);
  const float kh = (float)k, kl = (float)(k - (double)kh);
  float s[4] = {};
#pragma unroll
  for (int i = 0; i < LOADS; ++i)
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) {
      const float d = x[i][e] - m;
      s[e & 3] += __builtin_amdgcn_exp2f(fmaf(d, kh, d * kl));
    }
  float sum = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
  if (!(sum >= 0.0f)) {
    m = -INFINITY;
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
#pragma unroll
      for (int e = 0; e < VF_VEC; ++e) {
        x[i][e] = x[i][e] > -INFINITY ? x[i][e] : -INFINITY;
        m = fmaxf(m, x[i][e]);
      }
    m = wave_max(m);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
#pragma unroll
      for (int e = 0; e < VF_VEC; ++e) t += vf_weight(x[i][e], m, k);
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
  if (lane == 0) parts[unit] = VerifyPart{m, sum, (int)first, 0};
}

struct VerifyRow {
  double sum;
  float max;
  int first;
};

// A row from its parts, in every lane of the wave.
__device__ __forceinline__ VerifyRow vf_join(const VerifyArgs& a, const VerifyPart* __restrict__ parts, int row, double k) {
  const int lane = threadIdx.x & (WAVE - 1);
  const VerifyPart* const p = parts + (size_t)row * a.parts;
  VerifyRow r{0.0, -INFINITY, 0};
  uint32_t first = 0x7fffffffu;
  for (int c = lane; c < a.parts; c += WAVE) {
    const VerifyPart x = p[c];
    if (x.max > r.max) {
      r.sum = r.sum * vf_weight(r.max, x.max, k) + (double)x.sum;
      r.max = x.max, first = (uint32_t)x.first;
    } else {
      r.sum += (double)x.sum * vf_weight(x.max, r.max, k);
    }
  }
  const float m = wave_max(r.max);
  r.sum = vf_wave_sum(r.sum * vf_weight(r.max, m, k));
  r.first = (int)wave_min_u32(r.max == m ? first : 0x7fffffffu);
  r.max = m;
  return r;
}

// The row's sum in 64 bits, by the wave alone.
__device__ __forceinline__ double vf_exact_sum(const VerifyArgs& a, int row, float m, double k) {
  double s = 0.0;
  for (int i = (threadIdx.x & (WAVE - 1)) * VF_VEC; i < a.V; i += WAVE * VF_VEC) {
    float x[VF_VEC];
    vf_logits(a, row, i, x);
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) s += vf_weight(x[e], m, k);
  }
  return vf_wave_sum(s);
}

// Whether row's drafted token is taken.
__device__ __forceinline__ bool vf_taken(const VerifyArgs& a, const VerifyPart* __restrict__ parts, int row, bool warm,
                                         double k) {
  const int x = a.draft[row];
  if ((unsigned)x >= (unsigned)a.V) return false;
  const double q = !warm || !a.probs ? 1.0
                   : a.q_fp32 ? (double)static_cast<const float*>(a.probs)[(size_t)row * a.q_row + x]
                              : (double)vf_value(static_cast<const uint16_t*>(a.probs)[(size_t)row * a.q_row + x]);
  const float l = vf_logit(a, row, x);
  const VerifyRow r = vf_join(a, parts, row, k);
  if (!warm) return r.max > -INFINITY && x == r.first;
  const double uq = (double)a.u[row] * q, w = vf_weight(l, r.max, k);
  if (fabs(uq * r.sum - w) > VF_NEAR * w) return uq * r.sum < w;  // (false for a q that is NaN)
  return uq * vf_exact_sum(a, row, r.max, k) < w;
}

// The row that sequence b's next token comes from (the first whose draft is not taken, or the last), by the workgroup.
__device__ __forceinline__ int vf_stop(const VerifyArgs& a, const VerifyPart* __restrict__ parts, int r0, int r1, bool warm,
                                       double k, int* found) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  if (threadIdx.x == 0) *found = r1 - 1;
  __syncthreads();
  for (int row = r0 + wave; row < r1 - 1; row += VF_WAVES)
    if (!vf_taken(a, parts, row, warm, k)) {
      if ((threadIdx.x & (WAVE - 1)) == 0) atomicMin(found, row);
      break;
    }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*found);
}

// Weights w and draft's probabilities q of tokens i .. i + 7 of the stop row, 0 past the last: r = max(w - q sum, 0). (A
// draft that is certain takes its token's weight out.)
__device__ __forceinline__ void vf_stop_row(const VerifyArgs& a, int row, bool last, float m, double k, int i,
                                            double (&w)[VF_VEC], float (&q)[VF_VEC]) {
  float x[VF_VEC];
  vf_logits(a, row, i, x);
#pragma unroll
  for (int e = 0; e < VF_VEC; ++e) q[e] = 0.0f;
  if (!last && a.probs) {
    if (a.q_fp32)
      vf_load(static_cast<const float*>(a.probs) + (size_t)row * a.q_row, i, a.V, 0.0f, q);
    else
      vf_load(static_cast<const uint16_t*>(a.probs) + (size_t)row * a.q_row, i, a.V, 0.0f, q);
  }
  if (m < INFINITY) {
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) w[e] = vf_exp2(((double)x[e] - (double)m) * k);
  } else {
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) w[e] = vf_weight(x[e], m, k);
  }
  if (!last && !a.probs) {
    const int d = a.draft[row];
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) w[e] = i + e == d ? 0.0 : w[e];
  }
}

// v's inclusive prefix sum over the workgroup; tot: VF_WAVES doubles of LDS.
__device__ __forceinline__ double vf_scan(double v, double* tot) {
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
#pragma unroll
  for (int d = 1; d < WAVE; d *= 2) {
    const long long u = __builtin_bit_cast(long long, v);
    const int lo = __shfl_up((int)u, d, WAVE), hi = __shfl_up((int)(u >> 32), d, WAVE);
    if (lane >= d) v += __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
  }
  __syncthreads();
  if (lane == WAVE - 1) tot[wave] = v;
  __syncthreads();
  double before = 0.0;
  for (int w = 0; w < wave; ++w) before += tot[w];
  return before + v;
}

__device__ __forceinline__ float vf_logp(float l, float m, double sum, double k) {
  return (float)(vf_exponent(l, m, k) * 0.69314718055994530942 - log(sum));
}

// What a workgroup sums of the stop row: chunk's tokens, those of one thread side by side where `inner` (for the search).
struct VerifySearch {
  double tot[VF_WAVES];
  int found, passed, positive, pick;
  int last;
  double at, r;  // (of the token that was found: the sum before it, and its r)
  VerifyChunk part[VF_WAVES];
};

// Looks for the target in a chunk whose tokens come after a sum of `before`; the whole workgroup. pick: the token, -1: r is 0
// throughout.
template <int LOADS>
__device__ __forceinline__ void vf_search(const VerifyArgs& a, VerifySearch& sh, int stop, bool last, float m, double z,
                                          double k, int chunk, double before, double target) {
  constexpr int PER = LOADS * VF_VEC;
  const int tid = threadIdx.x, i0 = (chunk * VF_THREADS + tid) * PER;
  __syncthreads();
  if (tid == 0) sh.passed = VF_THREADS, sh.positive = -1, sh.pick = -1;
  double w[PER], mine = 0.0;
#pragma unroll
  for (int i = 0; i < PER; i += VF_VEC) {
    double x[VF_VEC];
    float q[VF_VEC];
    vf_stop_row(a, stop, last, m, k, i0 + i, x, q);
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) mine += w[i + e] = fmax(x[e] - (double)q[e] * z, 0.0);
  }
  const double upto = before + vf_scan(mine, sh.tot);
  if (mine > 0.0) {
    atomicMax(&sh.positive, tid);
    if (upto > target) atomicMin(&sh.passed, tid);
  }
  __syncthreads();
  if (tid == (sh.passed < VF_THREADS ? sh.passed : sh.positive)) {  // (where rounding has it pass nowhere: the last token)
    double x = upto - mine, at = x, r = 0.0;
    int y = -1;
    bool open = true;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (open && w[e] > 0.0) y = i0 + e, at = x, r = w[e];
      x += w[e];
      open = open && !(w[e] > 0.0 && x > target);
    }
    sh.pick = y, sh.at = at, sh.r = r;
  }
  __syncthreads();
}

// Workgroups 0 .. chunks - 1 of a sequence sum a chunk of its stop row each, the last of them looks for the token; workgroup
// `chunks` writes what the rows before and behind it get (and, at T = 0, the stop row).
template <int LOADS>
__global__ __launch_bounds__(VF_THREADS) void verify_pick_kernel(VerifyArgs a, const VerifyPart* __restrict__ parts,
                                                                 VerifyChunk* __restrict__ sums, int* __restrict__ done) {
  __shared__ VerifySearch sh;
  const int b = blockIdx.x / (a.chunks + 1), chunk = blockIdx.x - b * (a.chunks + 1), tid = threadIdx.x;
  const int lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int r0 = vf_row(a, b), r1 = vf_row(a, b + 1);
  const float temperature = a.temperature[b];
  const bool warm = temperature > 0.0f;
  if (r1 <= r0) {
    if (chunk == a.chunks && tid == 0) a.accepted[b] = 0;
    return;
  }
  if (!warm && chunk < a.chunks) return;
  const double k = vf_rate(temperature);
  const int stop = vf_stop(a, parts, r0, r1, warm, k, &sh.found);
  if (chunk == a.chunks) {
    if (tid == 0) a.accepted[b] = stop - r0;
    for (int row = r0 + wave; row < r1; row += VF_WAVES) {
      if (row > stop) {
        if (lane == 0) a.tokens[row] = -1, a.logp[row] = 0.0f;
        continue;
      }
      const VerifyRow r = vf_join(a, parts, row, k);
      const bool none = !(r.max > -INFINITY);
      if (lane || (row == stop && warm && !none)) continue;
      const int y = row < stop ? a.draft[row] : none ? -1 : r.first;
      a.tokens[row] = y;
      a.logp[row] = y < 0 ? 0.0f : vf_logp(vf_logit(a, row, y), r.max, r.sum, k);
    }
    return;
  }
  const VerifyRow r = vf_join(a, parts, stop, k);
  if (!(r.max > -INFINITY)) return;
  const bool last = stop == r1 - 1;
  VerifyChunk mine{0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    double w[VF_VEC];
    float q[VF_VEC];
    vf_stop_row(a, stop, last, r.max, k, ((chunk * LOADS + i) * VF_THREADS + tid) * VF_VEC, w, q);
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) {
      const double qz = (double)q[e] * r.sum;
      mine.all += w[e];
      if (w[e] > qz) mine.over += w[e], mine.q += (double)q[e];
      if (fabs(w[e] - qz) <= VF_NEAR * qz) mine.near += VF_NEAR * qz;
    }
  }
  mine.all = vf_wave_sum(mine.all), mine.over = vf_wave_sum(mine.over);
  mine.q = vf_wave_sum(mine.q), mine.near = vf_wave_sum(mine.near);
  if (lane == 0) sh.part[wave] = mine;
  __syncthreads();
  VerifyChunk* const row_sums = sums + (size_t)b * a.chunks;
  if (tid == 0) {
    VerifyChunk t = sh.part[0];
    for (int w = 1; w < VF_WAVES; ++w)
      t.all += sh.part[w].all, t.over += sh.part[w].over, t.q += sh.part[w].q, t.near += sh.part[w].near;
    double* const to = &row_sums[chunk].all;
    __hip_atomic_store(to, t.all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(to + 1, t.over, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(to + 2, t.q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(to + 3, t.near, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh.last = __hip_atomic_fetch_add(&done[b], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == a.chunks - 1;
  }
  __syncthreads();
  if (!sh.last) return;

  // the whole row's sums, every wave alike, 64 chunks at a time
  const auto sum_of = [&](int c) {
    VerifyChunk t{0.0, 0.0, 0.0, 0.0};
    if (c < a.chunks) {
      const double* const from = &row_sums[c].all;
      t.all = __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      t.over = __hip_atomic_load(from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      t.q = __hip_atomic_load(from + 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      t.near = __hip_atomic_load(from + 3, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    return t;
  };
  VerifyChunk whole{0.0, 0.0, 0.0, 0.0};
  for (int c0 = 0; c0 < a.chunks; c0 += WAVE) {
    const VerifyChunk t = sum_of(c0 + lane);
    whole.all += t.all, whole.over += t.over, whole.q += t.q, whole.near += t.near;
  }
  whole.all = vf_wave_sum(whole.all), whole.over = vf_wave_sum(whole.over);
  whole.q = vf_wave_sum(whole.q), whole.near = vf_wave_sum(whole.near);
  // (a certain draft's own weight is not in `all`: the row's sum has it)
  double z = whole.all;
  if (!last && !a.probs && (unsigned)a.draft[stop] < (unsigned)a.V) z += vf_weight(vf_logit(a, stop, a.draft[stop]), r.max, k);
  const double v = (double)a.v[b];
  double rest = whole.over - whole.q * z;
  bool sure = whole.near == 0.0 ? true : rest > 0.0;
  int token = -1;
  if (sure && rest > 0.0) {
    const double target = v * rest;
    double before = 0.0, at = 0.0;
    int in = 0;
    for (int c0 = 0, go = 1; go && c0 < a.chunks; c0 += WAVE) {
      const VerifyChunk t = sum_of(c0 + lane);
      const double x = t.over - t.q * z;
      for (int c = 0; c < WAVE && c0 + c < a.chunks; ++c) {
        const double y = vf_lane(x, c);
        if (y > 0.0) {
          in = c0 + c, before = at;
          if (at + y > target) {
            go = 0;
            break;
          }
        }
        at += y;
      }
    }
    vf_search<LOADS>(a, sh, stop, last, r.max, z, k, in, before, target);
    token = sh.pick;
    // r's sums up to either side of the token are off by less than `near` from what the 64-bit sum gives
    sure = whole.near == 0.0 || (token >= 0 && target - sh.at > 2.0 * whole.near && sh.at + sh.r - target > 2.0 * whole.near);
  }
  if (!sure || token < 0) {  // once more, chunk after chunk; from p where r is 0
    bool from_p = false;
    for (int pass = 0; pass < 2; ++pass) {
      double total = 0.0;
      for (int c = 0; c < a.chunks; ++c) {
        vf_search<LOADS>(a, sh, stop, last || from_p, r.max, z, k, c, 0.0, INFINITY);
        double s = 0.0;
        for (int w = 0; w < VF_WAVES; ++w) s += sh.tot[w];
        total += s;
      }
      if (total > 0.0) {
        const double target = v * total;
        double before = 0.0;
        for (int c = 0; c < a.chunks; ++c) {
          vf_search<LOADS>(a, sh, stop, last || from_p, r.max, z, k, c, before, target);
          if (sh.pick >= 0) token = sh.pick;
          if (sh.passed < VF_THREADS) break;
          double s = 0.0;
          for (int w = 0; w < VF_WAVES; ++w) s += sh.tot[w];
          before += s;
        }
        break;
      }
      from_p = true;
    }
  }
  if (tid == 0) {
    a.tokens[stop] = token;
    a.logp[stop] = token < 0 ? 0.0f : vf_logp(vf_logit(a, stop, token), r.max, z, k);
  }
}

static int verify_loads(long n, int num_cu) {  // loads of a thread: 4 where enough of them are left to fill the CUs
  const long at_once = 8L * VF_WAVES * num_cu * WAVE * VF_VEC;
  return n >= 4 * at_once ? 4 : n >= 2 * at_once ? 2 : 1;
}
static int verify_units(int V, int per) { return (V + per - 1) / per; }

bool verify_grid_ok(int N, int V) { return (long)N * (verify_units(V, WAVE * VF_VEC) + 1L) <= 0xffffffL; }

size_t verify_workspace_bytes(int N, int V, int B, int num_cu) {
  const int parts = verify_units(V, WAVE * VF_VEC * verify_loads((long)N * V, num_cu));
  const int chunks = verify_units(V, VF_THREADS * VF_VEC * verify_loads((long)B * V, num_cu));
  return (size_t)N * parts * sizeof(VerifyPart) + (size_t)B * chunks * sizeof(VerifyChunk) + (size_t)B * sizeof(int);
}

hipError_t launch_verify(const void* logits, int l_fp32, long l_row, const int* draft, const void* probs, int q_fp32,
                         long q_row, const int* cu, const float* u, const float* v, const float* temperature, int* tokens,
                         int* accepted, float* logp, void* ws, int N, int V, int B, int num_cu, hipStream_t s) {
  const int rows = verify_loads((long)N * V, num_cu), pick = verify_loads((long)B * V, num_cu);
  VerifyArgs a{logits, probs, draft, cu, u, v, temperature, tokens, accepted, logp, l_row, q_row, l_fp32, q_fp32,
               N, V, B, verify_units(V, WAVE * VF_VEC * rows), verify_units(V, VF_THREADS * VF_VEC * pick)};
  VerifyPart* const parts = static_cast<VerifyPart*>(ws);
  VerifyChunk* const sums = reinterpret_cast<VerifyChunk*>(parts + (size_t)N * a.parts);
  int* const done = reinterpret_cast<int*>(sums + (size_t)B * a.chunks);
  const unsigned groups = (unsigned)(((long)N * a.parts + VF_WAVES - 1) / VF_WAVES);
  const auto first = [&](auto kernel) {
    return launch("verify_rows_kernel", kernel, dim3(groups), dim3(VF_THREADS), s, a, parts, done);
  };
  const auto second = [&](auto kernel) {
    return launch("verify_pick_kernel", kernel, dim3((unsigned)B * (a.chunks + 1)), dim3(VF_THREADS), s, a, parts, sums, done);
  };
  hipError_t e = hipSuccess;
  if (N > 0 && l_fp32)
    e = rows == 4   ? first(verify_rows_kernel<float, 4>)
        : rows == 2 ? first(verify_rows_kernel<float, 2>)
                    : first(verify_rows_kernel<float, 1>);
  else if (N > 0)
    e = rows == 4   ? first(verify_rows_kernel<uint16_t, 4>)
        : rows == 2 ? first(verify_rows_kernel<uint16_t, 2>)
                    : first(verify_rows_kernel<uint16_t, 1>);
  if (e != hipSuccess) return e;
  return pick == 4 ? second(verify_pick_kernel<4>) : pick == 2 ? second(verify_pick_kernel<2>) : second(verify_pick_kernel<1>);
}

}  // namespace dsa
