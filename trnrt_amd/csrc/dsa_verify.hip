// Verification of drafted tokens for gfx950. Sequence b's rows of logits are cu[b] .. cu[b + 1] - 1; row j's probabilities
// are p_j = softmax(l_j / T_b), and all rows but the last have a drafted token x_j, drawn from the draft's q_j:
//   x_j is taken iff u_j q_j(x_j) < p_j(x_j), up to the first that is not;
//   then one token from that row: the first i with sum_{k <= i} r(k) > v_b sum r, r = max(p - q, 0), or r = p after the last
//   row's drafts were all taken (and where r is 0 everywhere).
// At T_b = 0 a token is taken iff it is the first of the largest logits, and that one comes next.
//
// Three launches: each row's chunks to (maximum, sum of exponentials, place of the maximum); each sequence's stop row,
// found by every workgroup of it alike, to the chunks' sums of r; the chunk that the sum passes v in, and the token in it.
// Sums and the exponentials that they are of are in 64 bits, so that a token does not depend on how they were split.
#include "dsa_common.h"

namespace dsa {

constexpr int VF_THREADS = 256;
constexpr int VF_VEC = 8;                        // logits of a load
constexpr int VF_LOADS = 4;                      // of a thread
constexpr int VF_CHUNK = VF_THREADS * VF_VEC * VF_LOADS;

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
  int N, V, B, chunks;
};

struct VerifyPart {  // of a row's chunk
  double sum;        // of exp((l - max) / T)
  float max;
  int first;         // the first place of the maximum
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

__device__ __forceinline__ double vf_shfl(double x, int m) {
  const long long u = __builtin_bit_cast(long long, x);
  const int lo = __shfl_xor((int)u, m, WAVE), hi = __shfl_xor((int)(u >> 32), m, WAVE);
  return __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
}

__device__ __forceinline__ double vf_wave_sum(double x) {
#pragma unroll
  for (int m = 1; m < WAVE; m *= 2) x += vf_shfl(x, m);
  return x;
}

// The sum over the workgroup, in every thread.
__device__ __forceinline__ double vf_sum(double x, double* tot) {
  x = vf_wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & (WAVE - 1)) == 0) tot[threadIdx.x / WAVE] = x;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < (int)blockDim.x / WAVE; ++w) s += tot[w];
  return s;
}

// The sequence that row is in, -1: none.
__device__ __forceinline__ int vf_sequence(const VerifyArgs& a, int row) {
  if (row < a.cu[0] || row >= a.cu[a.B]) return -1;
  int lo = 0, hi = a.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__global__ __launch_bounds__(VF_THREADS) void verify_rows_kernel(VerifyArgs a, VerifyPart* __restrict__ parts) {
  __shared__ double tot[VF_THREADS / WAVE];
  __shared__ float top[VF_THREADS / WAVE];
  __shared__ uint32_t at[VF_THREADS / WAVE];
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, tid = threadIdx.x;
  const int lane = tid & (WAVE - 1), wave = tid / WAVE;
  const int b = vf_sequence(a, row);
  if (b < 0) return;
  float x[VF_LOADS][VF_VEC];
#pragma unroll
  for (int i = 0; i < VF_LOADS; ++i) vf_logits(a, row, chunk * VF_CHUNK + VF_VEC * (tid + VF_THREADS * i), x[i]);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < VF_LOADS; ++i)
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) m = fmaxf(m, x[i][e]);
  m = wave_max(m);
  if (lane == 0) top[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  const double k = vf_rate(a.temperature[b]);
  double s = 0.0;
  uint32_t first = 0x7fffffffu;
#pragma unroll
  for (int i = 0; i < VF_LOADS; ++i)
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) {
      s += vf_weight(x[i][e], m, k);
      const uint32_t p = chunk * VF_CHUNK + VF_VEC * (tid + VF_THREADS * i) + e;
      if (x[i][e] == m && m > -INFINITY) first = min(first, p);
    }
  first = wave_min_u32(first);
  if (lane == 0) at[wave] = first;
  s = vf_sum(s, tot);
  if (tid == 0) parts[blockIdx.x] = VerifyPart{s, m, (int)min(min(at[0], at[1]), min(at[2], at[3]))};
}

struct VerifyRow {
  double sum;
  float max;
  int first;  // -1: no token can come
};

// A row from its chunks, in every lane of the wave.
__device__ __forceinline__ VerifyRow vf_join(const VerifyArgs& a, const VerifyPart* __restrict__ parts, int row, double k) {
  const int lane = threadIdx.x & (WAVE - 1);
  const VerifyPart* const p = parts + (size_t)row * a.chunks;
  VerifyRow r{0.0, -INFINITY, -1};
  for (int c = lane; c < a.chunks; c += WAVE) r.max = fmaxf(r.max, p[c].max);
  r.max = wave_max(r.max);
  uint32_t first = 0x7fffffffu;
  for (int c = lane; c < a.chunks; c += WAVE) {
    if (p[c].max == r.max) first = min(first, (uint32_t)p[c].first);
    r.sum += p[c].sum * vf_weight(p[c].max, r.max, k);
  }
  r.sum = vf_wave_sum(r.sum);
  first = wave_min_u32(first);
  r.first = r.max > -INFINITY ? (int)first : -1;
  return r;
}

// Whether row's drafted token is taken.
__device__ __forceinline__ bool vf_taken(const VerifyArgs& a, const VerifyRow& r, int row, bool warm, double k) {
  const int x = a.draft[row];
  if ((unsigned)x >= (unsigned)a.V) return false;
  if (!warm) return x == r.first;
  const double q = !a.probs     ? 1.0
                   : a.q_fp32 ? (double)static_cast<const float*>(a.probs)[(size_t)row * a.q_row + x]
                              : (double)vf_value(static_cast<const uint16_t*>(a.probs)[(size_t)row * a.q_row + x]);
  return (double)a.u[row] * q * r.sum < vf_weight(vf_logit(a, row, x), r.max, k);
}

// The row that sequence b's next token comes from (the first whose draft is not taken, or the last), by the workgroup.
__device__ __forceinline__ int vf_stop(const VerifyArgs& a, const VerifyPart* __restrict__ parts, int r0, int r1, bool warm,
                                       double k, int* found) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), waves = blockDim.x / WAVE;
  if (threadIdx.x == 0) *found = r1 - 1;
  __syncthreads();
  for (int row = r0 + wave; row < r1 - 1; row += waves)
    if (!vf_taken(a, vf_join(a, parts, row, k), row, warm, k)) {
      if ((threadIdx.x & (WAVE - 1)) == 0) atomicMin(found, row);
      break;
    }
  __syncthreads();
  return *found;
}

// r (times the sum of the weights) of tokens i .. i + 7, 0 past the last.
__device__ __forceinline__ void vf_rest(const VerifyArgs& a, int row, bool last, const VerifyRow& r, double k, int i,
                                        double (&w)[VF_VEC]) {
  float x[VF_VEC];
  vf_logits(a, row, i, x);
#pragma unroll
  for (int e = 0; e < VF_VEC; ++e) w[e] = i + e < a.V ? vf_weight(x[e], r.max, k) : 0.0;
  if (last) return;
  if (a.probs) {
    float q[VF_VEC];
    if (a.q_fp32)
      vf_load(static_cast<const float*>(a.probs) + (size_t)row * a.q_row, i, a.V, 0.0f, q);
    else
      vf_load(static_cast<const uint16_t*>(a.probs) + (size_t)row * a.q_row, i, a.V, 0.0f, q);
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) w[e] = fmax(w[e] - (double)q[e] * r.sum, 0.0);
  } else {
    const int d = a.draft[row];
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) w[e] = i + e == d ? 0.0 : w[e];
  }
}

__global__ __launch_bounds__(VF_THREADS) void verify_rest_kernel(VerifyArgs a, const VerifyPart* __restrict__ parts,
                                                                 double* __restrict__ rest) {
  __shared__ double tot[VF_THREADS / WAVE];
  __shared__ int found;
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  const int r0 = vf_row(a, b), r1 = vf_row(a, b + 1);
  const float temperature = a.temperature[b];
  if (r1 <= r0 || !(temperature > 0.0f)) return;
  const double k = vf_rate(temperature);
  const int stop = vf_stop(a, parts, r0, r1, true, k, &found);
  const VerifyRow r = vf_join(a, parts, stop, k);
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < VF_LOADS; ++i) {
    double w[VF_VEC];
    vf_rest(a, stop, stop == r1 - 1, r, k, chunk * VF_CHUNK + VF_VEC * ((int)threadIdx.x + VF_THREADS * i), w);
#pragma unroll
    for (int e = 0; e < VF_VEC; ++e) s += w[e];
  }
  s = vf_sum(s, tot);
  if (threadIdx.x == 0) rest[blockIdx.x] = s;
}

// v's inclusive prefix sum over the workgroup.
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

// One workgroup a sequence.
__global__ __launch_bounds__(VF_THREADS) void verify_pick_kernel(VerifyArgs a, const VerifyPart* __restrict__ parts,
                                                                 const double* __restrict__ rest) {
  constexpr int PER = VF_CHUNK / VF_THREADS;  // tokens of a thread, one after another
  __shared__ double tot[VF_THREADS / WAVE];
  __shared__ int found, passed, positive, pick;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & (WAVE - 1);
  const int r0 = vf_row(a, b), r1 = vf_row(a, b + 1);
  if (r1 <= r0) {
    if (tid == 0) a.accepted[b] = 0;
    return;
  }
  const float temperature = a.temperature[b];
  const bool warm = temperature > 0.0f;
  const double k = vf_rate(temperature);
  const int stop = vf_stop(a, parts, r0, r1, warm, k, &found);
  const VerifyRow r = vf_join(a, parts, stop, k);
  int token = r.first;
  if (warm && token >= 0) {
    const double* const s = rest + (size_t)b * a.chunks;
    double whole = 0.0;
    for (int c = 0; c < a.chunks; ++c) whole += s[c];
    const bool all = !(whole > 0.0);  // (the draft leaves nothing: from p)
    if (all) whole = r.sum;
    const double target = (double)a.v[b] * whole;
    // the chunk in which the sum passes the target (if rounding has it pass nowhere, the last one with anything in it)
    double sum = 0.0, before = 0.0;
    int chunk = 0;
    for (int c = 0; c < a.chunks; ++c) {
      const VerifyPart p = parts[(size_t)stop * a.chunks + c];
      const double mine = all ? p.sum * vf_weight(p.max, r.max, k) : s[c];
      if (mine > 0.0) {
        chunk = c;
        before = sum;
        if (sum + mine > target) break;
      }
      sum += mine;
    }
    // and the token, the same way
    if (tid == 0) passed = VF_THREADS, positive = -1, pick = -1;
    const int i0 = chunk * VF_CHUNK + PER * tid;
    double w[PER], mine = 0.0;
#pragma unroll
    for (int i = 0; i < PER; i += VF_VEC) {
      double x[VF_VEC];
      vf_rest(a, stop, all || stop == r1 - 1, r, k, i0 + i, x);
#pragma unroll
      for (int e = 0; e < VF_VEC; ++e) mine += w[i + e] = x[e];
    }
    const double upto = before + vf_scan(mine, tot);
    if (mine > 0.0) {
      atomicMax(&positive, tid);
      if (upto > target) atomicMin(&passed, tid);
    }
    __syncthreads();
    if (tid == (passed < VF_THREADS ? passed : positive)) {
      double x = upto - mine;
      int y = -1;
      bool open = true;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        if (open && w[e] > 0.0) y = i0 + e;
        x += w[e];
        open = open && !(w[e] > 0.0 && x > target);
      }
      pick = y;
    }
    __syncthreads();
    token = pick;
  }
  if (tid == 0) a.accepted[b] = stop - r0;
  for (int row = r0 + tid / WAVE; row < r1; row += VF_THREADS / WAVE) {
    const VerifyRow x = vf_join(a, parts, row, k);
    if (lane) continue;
    const int y = row < stop ? a.draft[row] : row == stop ? token : -1;
    a.tokens[row] = y;
    a.logp[row] =
        y < 0 ? 0.0f : (float)(vf_exponent(vf_logit(a, row, y), x.max, k) * 0.69314718055994530942 - log(x.sum));
  }
}

static int verify_chunks(int V) { return (V + VF_CHUNK - 1) / VF_CHUNK; }

bool verify_grid_ok(int N, int V) { return (long)N * verify_chunks(V) <= 0xffffffL; }

size_t verify_workspace_bytes(int N, int V, int B) {
  return (size_t)verify_chunks(V) * ((size_t)N * sizeof(VerifyPart) + (size_t)B * sizeof(double));
}

hipError_t launch_verify(const void* logits, int l_fp32, long l_row, const int* draft, const void* probs, int q_fp32,
                         long q_row, const int* cu, const float* u, const float* v, const float* temperature, int* tokens,
                         int* accepted, float* logp, void* ws, int N, int V, int B, hipStream_t s) {
  const VerifyArgs a{logits, probs, draft, cu, u, v, temperature, tokens, accepted, logp, l_row, q_row, l_fp32, q_fp32,
                     N, V, B, verify_chunks(V)};
  VerifyPart* const parts = static_cast<VerifyPart*>(ws);
  double* const rest = reinterpret_cast<double*>(parts + (size_t)N * a.chunks);
  hipError_t e = hipSuccess;
  if (N > 0)
    e = launch("verify_rows_kernel", verify_rows_kernel, dim3((unsigned)(N * a.chunks)), dim3(VF_THREADS), s, a, parts);
  if (e == hipSuccess && N > 0)
    e = launch("verify_rest_kernel", verify_rest_kernel, dim3((unsigned)(B * a.chunks)), dim3(VF_THREADS), s, a, parts, rest);
  if (e == hipSuccess)
    e = launch("verify_pick_kernel", verify_pick_kernel, dim3(B), dim3(VF_THREADS), s, a, parts, rest);
  return e;
}

}  // namespace dsa
