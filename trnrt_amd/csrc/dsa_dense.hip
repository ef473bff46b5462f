// Absorbed latent attention over every cached token of a paged FP8 latent cache for gfx950: decode rows and the S new
// tokens of a speculative step, with no selection (the arithmetic of dsa_attention.hip, whose slots are chosen).
//
//   s[r, t] = scale x sigma_t x (q_r . c_t),  p = softmax_t(s),  out_r = sum_t p sigma_t c_t[:512],  lse
//
// for the M = S x H rows r (query, head) of a sequence over its tokens t: e4m3 rows c_t with a scale sigma_t.
//
// What bounds it: a token is 580 bytes for 2 x M x 1,088 FLOP, so up to about 64 rows the cache's stream is the bound,
// above it the matrix units and the conversions beside them. One workgroup a CU has a tile of 32 or 64 rows of one
// sequence and a range of its chunks of 64 tokens; its 8 waves have two kinds of work, one of each on every SIMD, a
// chunk apart, with one barrier a chunk (products of one kind run under the other's conversions and exponentials):
//   - scoring waves 0-3, interval c: chunk c's scores S^T = K . Q^T, 32 tokens x 32 rows a wave (16 x 32 where there are
//     32 rows), the queries in registers, then P = 2^(s - m) x the tokens' scales in bf16 into LDS;
//   - value waves 4-7, interval c: chunk c - 1's O^T += V^T . P, 128 dims of all rows a wave, in registers; and the
//     rows of chunk c + 1 from their registers into LDS and chunk c + 2's loads into the same registers, piece by piece
//     between the products. (Loads straight into LDS cost their wave 150 to 200 cycles each beside the other waves' LDS
//     reads.)
// Both products are v_mfma_f32_32x32x16_bf16 (16x16x32 in the scores of 32 rows) with the e4m3 operand converted on the
// way (exact). The chunks of all sequences and row tiles form one list that the workgroups share evenly, whatever the
// lengths: each takes a stretch of it and writes a row tile's outputs where it holds all its chunks, else a partial
// (the rows x 512 in fp32, their maxima and sums) that dense_combine_kernel joins. Neighbouring stretches lie on one
// XCD, so that the row tiles of a sequence read its cache through the same L2.
//
// Measured (the attention alone, the joining beside it): 8 x 32k tokens, 64 heads 44 + 8 us, of which the loop is 27 at
// 5.6 TB/s of cache rows, the rest the list's search, the first loads and the partials; 13 x 4 new tokens of 128 heads
// (2k to 12k tokens, 512 wide) 106 + 11, 920 TFLOP/s over the call; 16 heads: 8 x 32k tokens 34 + 5, 1 x 4k 9.6 + 4.8,
// latency.
//
// The online softmax rescales lazily without waiting for the chunk's maximum: P is taken against the running maximum as
// it stands; a wave that meets a score past its slack raises a flag, and before the chunk's values are multiplied every
// wave sees the flags and, when one is up, the maxima are exchanged, P is taken again and O rescaled (a stretch's chunk
// 0 always does, with O still zero).
#include "dsa_async.h"
#include "dsa_scan.h"

namespace dsa {

constexpr int DN_DV = 512;
constexpr int DN_CHUNK = 64;
constexpr int DN_THREADS = 512;
// Lazy rescaling (base 2): p = 2^(s - m) <= 2^60 between moves of m. (bf16 and fp32 keep their precision at that size,
// and 2^31 such weights sum to less than fp32's end. With 2^11.5 m moved so often that 8 x 32k tokens took 50.0 us for
// 45.5.)
constexpr float DN_SLACK = 60.0f;
constexpr float DN_LOG2E = 1.44269504088896341f;
constexpr float DN_LOG2E_LO = (float)(1.44269504088896341 - (double)DN_LOG2E);
constexpr int DN_PROW = DN_CHUNK + 8;  // P row stride (bf16)
constexpr int DN_KAHEAD = 3;           // score steps whose key reads are in flight
constexpr int DN_VAHEAD = 3;           // value steps whose operand reads are in flight
constexpr int DN_STORE = 5;            // the value step that begins storing the next chunk's rows

typedef int dn_v2i __attribute__((ext_vector_type(2)));

// A chunk's LDS layout: row r (token) at r x DN_KROW, its 16-byte piece p at p ^ dn_swizzle(r). With it the stores of
// 16 lanes (4 rows x 4 pieces), the key operand's reads (16 lanes: a piece of 16 rows) and the value operand's,
// transposed (32 lanes: two pieces of 8 rows), cover the 64 banks once.
__device__ __forceinline__ int dn_swizzle(int r) { return (r >> 2 & 1) << 1 | (r >> 3 & 1); }
constexpr int DN_KROW = 576;

// The same of the staged queries, rows of 2 DQK bytes: one piece of 16 rows covers the 64 banks once.
template <int DQK>
__device__ __forceinline__ int dn_q_swizzle(int r) {
  return DQK == 576 ? r >> 1 & 7 : r & 15;
}
constexpr int DN_BUFS = 3;  // chunk c being scored, c - 1 whose values are multiplied, c + 1 being stored

// RB: blocks of 32 rows in a tile.
template <int RB>
struct DnShared {
  alignas(1024) uint8_t tile[DN_BUFS][DN_CHUNK * DN_KROW];  // (the queries in the last two before)
  alignas(16) uint16_t p[2][64 * DN_PROW];  // P[row][token] of two chunks (32 rows: their second terms after them)
  alignas(16) float ksc[DN_BUFS][DN_CHUNK];       // the chunks' token scales
  alignas(16) float kfac[DN_BUFS][DN_CHUNK];      // x softmax scale x log2 e
  alignas(16) float klog[RB == 2 ? DN_CHUNK : 4];  // chunk 0's dn_log2_mantissa
  // [part][row], of the halves of a chunk's tokens (with 32 rows its quarters): a chunk's maxima when one moves, and a
  // stretch's sums
  float cmax[4 / RB][32 * RB];
  float lsum[4 / RB][32 * RB];
  float al[32 * RB];                              // and its rescale factors
  alignas(16) int flag[2][4];                     // per chunk parity and wave: a score past the running maximum's slack
  float mfin[32 * RB];                            // and its maxima (base 2)
  int tot[DN_THREADS / WAVE];
  int found[4];
};

// t / page_size for 0 <= t < 2^31: t x mul >> shift (mul = ceil(2^shift / page_size), shift = 31 + ceil(log2
// page_size)).
struct DnPage {
  uint32_t mul;
  int shift;
  int size;
};

// A sequence's tokens and chunks of them.
__device__ __forceinline__ int dn_len(int ctx_len, int max_pages, int page_size) {
  const long cap = (long)max_pages * page_size;
  return (int)min(max((long)ctx_len, 0L), min(cap, 0x7fffff00L));
}
__device__ __forceinline__ int dn_chunks(int len) { return (len + DN_CHUNK - 1) / DN_CHUNK; }

// How a sequence's row tiles go to workgroups: `span` neighbours on one XCD are a team, with the same stretch of chunks
// and a tile each, so that they read the cache through one L2 at one time; more tiles than that are `sets` of span
// tiles, one after another in the list. `teams` of them share the list.
struct DnTeams {
  int rows;   // of a tile
  int tiles;
  int span;
  int sets;
  int teams;
};

// The list of units (sequence, set of row tiles, chunk of tokens), in equal shares (one unit more for the first
// `more`).
struct DnList {
  int teams;  // that have a share
  int share;
  int more;
};
__device__ __forceinline__ DnList dn_list(int units, int teams) {
  DnList x;
  x.teams = min(teams, units);
  x.share = units > 0 ? units / x.teams : 0;
  x.more = units - x.share * x.teams;
  return x;
}
// The first unit of team w, and the team that has unit u.
__device__ __forceinline__ int dn_start(int w, const DnList& x) { return w * x.share + min(w, x.more); }
__device__ __forceinline__ int dn_owner(int u, const DnList& x) {
  const int big = x.more * (x.share + 1);
  return u < big ? u / (x.share + 1) : x.more + (u - big) / x.share;
}

// Where a partial's piece lies: dims 128 w + 32 d + 8 g + 4 h .. + 3 of row 32 i + j of a tile, at 4 (32 h + j) from
// there, as the value waves' lanes hold it.
__device__ __forceinline__ constexpr int dn_partial(int w, int i, int d, int g, int blocks) {
  return (((w * blocks + i) * 4 + d) * 4 + g) * 4 * WAVE;
}

// Four weights into P: bf16, off by 2^-8 of each at most, as everywhere in this library (the sums take them unrounded).
// With two TERMS what that left follows 32 rows on, bf16 again (2^-16): for a tile of 32 rows, whose bound is the cache's
// stream.
template <int TERMS>
__device__ __forceinline__ void dn_store_weights(uint16_t* to, const float (&p)[4]) {
  uint32_t w[2] = {bf16_pack(p[0], p[1]), bf16_pack(p[2], p[3])};
  *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  if (TERMS == 2) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      w[e] = bf16_pack(p[2 * e] - __uint_as_float(w[e] << 16), p[2 * e + 1] - __uint_as_float(w[e] & 0xffff0000u));
    *reinterpret_cast<uint2*>(to + 32 * DN_PROW) = make_uint2(w[0], w[1]);
  }
}

// log2 of a token scale without its whole part, -1/2 .. 1/2 (any of them for 0, which adds nothing). The one bf16 term of
// a tile of 64 rows is off by up to 2^-8 of the weight p sigma, and by nothing where that is a power of two. One token often
// has most of a row's weight, so a stretch's first chunk puts m at the largest score + this of its token's scale: that
// token's p sigma = 2^(s - m) sigma is such a power then. Over 120 calls of 1 to 41k tokens a sequence the bf16 outputs'
// error is 1.09 times that of their own rounding, at most 1.42 (m at the largest score: 1.40 and 1.80); 48 ragged rows of 64
// heads take 136.9 us for 135.7.
__device__ __forceinline__ float dn_log2_mantissa(float sigma) {
  const float x = __builtin_amdgcn_logf(fabsf(sigma));
  return __builtin_amdgcn_fmed3f(x - rintf(x), -0.5f, 0.5f);  // (NaN, of a scale 0: -1/2)
}

template <int DQK, int RB>
__global__ __launch_bounds__(DN_THREADS, 1) void dense_mla_kernel(
    const uint16_t* __restrict__ q, const uint8_t* __restrict__ kv, const float* __restrict__ kvs,
    const int* __restrict__ table, const int* __restrict__ ctx_len, uint16_t* __restrict__ out,
    float* __restrict__ out_f32, float* __restrict__ lse_out, float* __restrict__ ws_o, float* __restrict__ ws_ml,
    int B, int S, int H, int max_pages, DnPage pg, int num_pages, float scale, DnTeams tm) {
  constexpr int ROWS = 32 * RB, BUFS = DN_BUFS;
  constexpr int STEPS = DQK / 32;           // 32 dims: one 16-byte read of a key row per lane, two products
  constexpr int PIECES = DQK / 64;  // 16-byte pieces of a chunk per loading thread (4 threads a row)
  __shared__ DnShared<RB> sh;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int M = S * H;

  // the list, and the sequence of this team's first unit
  int chunks = 0, len = 0, n = 0, incl = 0;
  for (int b0 = 0; b0 < B; b0 += DN_THREADS) {
    const int x = b0 + tid;
    int total;
    len = x < B ? dn_len(ctx_len[x], max_pages, pg.size) : 0;
    n = dn_chunks(len);
    incl = group_incl_scan<DN_THREADS>(n, sh.tot, total);
    chunks += total;
  }
  const DnList list = dn_list(chunks * tm.sets, tm.teams);
  // (workgroup x runs on XCD x % 8: neighbours in the list on one XCD, and all XCDs at work however few the teams)
  const int per_xcd = (list.teams + 7) >> 3, place = blockIdx.x >> 3;
  const int team = (blockIdx.x & 7) * per_xcd + place / tm.span, member = place % tm.span;
  if (place / tm.span >= per_xcd || team >= list.teams) return;
  const int u0 = dn_start(team, list), u1 = dn_start(team + 1, list);
  for (int b0 = 0, before = 0; b0 < B && before <= u0; b0 += DN_THREADS) {
    const int x = b0 + tid;
    int total = 0;
    if (B > DN_THREADS) {  // (else they are still at hand)
      len = x < B ? dn_len(ctx_len[x], max_pages, pg.size) : 0;
      n = dn_chunks(len);
      incl = group_incl_scan<DN_THREADS>(n, sh.tot, total);
    }
    const int lo = before + (incl - n) * tm.sets;
    if (lo <= u0 && u0 < lo + n * tm.sets) {
      sh.found[0] = x;
      sh.found[1] = (u0 - lo) / n;
      sh.found[2] = (u0 - lo) % n;
      sh.found[3] = len;
    }
    before += total * tm.sets;
  }
  if (tid < 8) sh.flag[tid >> 2][tid & 3] = 0;
  __syncthreads();

  // scale x log2 e to twice fp32's digits: rounded, its error would be the same for every score, and so the lse's
  auto uniform = [](float x) __attribute__((always_inline)) {
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
  };
  const float sl2 = uniform(scale * DN_LOG2E);
  const float sl2_lo = uniform(fmaf(scale, DN_LOG2E, -sl2) + scale * DN_LOG2E_LO);
  // the stretch at hand: chunks c0 .. of set `set` of sequence b
  int b = __builtin_amdgcn_readfirstlane(sh.found[0]);
  int set = __builtin_amdgcn_readfirstlane(sh.found[1]);
  int c0 = __builtin_amdgcn_readfirstlane(sh.found[2]);
  len = __builtin_amdgcn_readfirstlane(sh.found[3]);
  __syncthreads();  // every wave has them: a workgroup without a tile in this set goes straight to the next search

  for (int u = u0; u < u1;) {
    const int all = dn_chunks(len);
    const int nch = min(all - c0, u1 - u);  // this stretch's chunks
    const bool whole = nch == all;
    const int t0 = c0 * DN_CHUNK, r0 = (set * tm.span + member) * ROWS;  // its first token, and this workgroup's row
    const int part = (2 * team + (u > u0)) * tm.span + member;            // where its partials go
    if (r0 < M) {  // (else the last set has no tile for this member)
      auto row_sum = [&](int r) __attribute__((always_inline)) {
        float l = sh.lsum[0][r] + sh.lsum[1][r];
        if constexpr (RB == 1) l += sh.lsum[2][r] + sh.lsum[3][r];
        return l;
      };
      // A whole row tile's outputs go through LDS, 256 dims at a time: dims 4 x .. + 3 of row r at place 64 x + (r ^ (x
      // & 7)), so that a row's pieces in order and a piece's rows in order both cover the banks once; a wave writes
      // whole rows.
      f32x4* const area = reinterpret_cast<f32x4*>(&sh.tile[0][0]);
      auto write = [&](int half) __attribute__((always_inline)) {
        const int lane = fresh_lane(), dim = 256 * half + 4 * lane;
#pragma unroll 4
        for (int i = 0; i < ROWS / 8; ++i) {
          const int r = wave + 8 * i;
          if (r0 + r >= M) break;
          f32x4 v = area[64 * lane + (r ^ (lane & 7))];
          const float m = sh.mfin[r], l = row_sum(r);
          const float inv = inverse_or_0(l);  // (a row that sees nothing: 0)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= inv;
          const size_t at = (size_t)b * M + r0 + r;
          if (out)
            *reinterpret_cast<uint2*>(out + at * DN_DV + dim) = make_uint2(bf16_pack(v[0], v[1]), bf16_pack(v[2], v[3]));
          if (out_f32) *reinterpret_cast<f32x4*>(out_f32 + at * DN_DV + dim) = v;
          if (lse_out && half == 0 && lane == 0) lse_out[at] = lse_or_none(m, l);
        }
      };
      // The end of a stretch in every wave, after the barrier behind which the tiles are free and the sums in LDS; the
      // value waves bring store(half).
      auto finish = [&](auto store) __attribute__((always_inline)) {
        if (whole) {
          store(0);
          lds_barrier();
          write(0);
          lds_barrier();
          store(1);
          lds_barrier();
          write(1);
        } else if (tid < ROWS && r0 + tid < M) {
          float2* const ml = reinterpret_cast<float2*>(ws_ml) + (size_t)part * ROWS + tid;
          *ml = make_float2(sh.mfin[tid], row_sum(tid));
        }
      };

      if (wave < 4) {
        // -- the scores: of 64 rows wave (th, hh) takes tokens 32 th .. + 31 of a chunk for rows 32 hh .. + 31 --
        const int th = wave >> 1, hh = wave & 1;
        const int lane = fresh_lane(), j = lane & 31, h = lane >> 5;
        // the queries through LDS, into the buffers that the first chunks leave: row r at r x 2 DQK, its 16-byte piece
        // p at p ^ dn_q_swizzle(r)
        {
          constexpr int QP = DQK / 8, PER = ROWS * QP / (4 * WAVE);
          static_assert(ROWS * QP * 16 <= 2 * DN_CHUNK * DN_KROW, "the staged queries");
          const uint32_t q_lds = lds_address(sh.tile[1]) + 1024 * PER * wave;
          const int r_max = M - 1 - r0;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int x = WAVE * (PER * wave + i) + lane, r = x / QP, p = x - r * QP;
            load_lds16(q + ((size_t)b * M + r0 + min(r, r_max)) * DQK + 8 * (p ^ dn_q_swizzle<DQK>(r)), q_lds + 1024 * i);
          }
          wait_loads<0>();
        }
        lds_barrier();  // the queries and chunk 0 are in place
        if constexpr (RB == 1) {
          // of 32 rows wave w takes tokens 16 w .. + 15 of a chunk, by products of 16 x 16, so that no SIMD has more of
          // them (8 x 32k tokens, 16 heads: 33.9 us, where two waves of 32 tokens took 38.2)
          const int j = lane & 15, kq = lane >> 4;
          int seen[2];  // tokens that this lane's rows 16 x + j see
#pragma unroll
          for (int x = 0; x < 2; ++x) seen[x] = len - S + min(r0 + 16 * x + j, M - 1) / H + 1;
          const int seen0 = len - S + r0 / H + 1;  // and the tile's first row, the fewest
          bf16x8 qb[2][2 * PIECES];  // rows 16 x + j: step s holds dims 64 (s / 2) + 16 kq + 8 (s % 2) .. + 7
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int s = 0; s < 2 * PIECES; ++s)
              qb[x][s] = as_bf16x8(*reinterpret_cast<const uint4*>(
                  sh.tile[1] + (16 * x + j) * 2 * DQK +
                  16 * ((8 * (s >> 1) + 2 * kq + (s & 1)) ^ dn_q_swizzle<DQK>(16 * x + j))));
          lds_barrier();  // the queries are read
          float m_run[2] = {}, l_run[2] = {}, psum[2] = {};  // as in the other form, of each of its two rows
          f32x4 sv[2] = {};  // the last chunk's scores - m_run: rows 16 x + j, tokens 16 w + 4 kq + r
          const int koff = (16 * wave + j) * DN_KROW + 16 * (kq ^ dn_swizzle(16 * wave + j));
          uint16_t* const pw = &sh.p[0][j * DN_PROW + 16 * wave + 4 * kq];
          int buf = 0, last = 0;  // chunk c's buffer and chunk c - 1's
          auto four = [&](const float* a) __attribute__((always_inline)) {
            return *reinterpret_cast<const f32x4*>(a + 16 * wave + 4 * kq);
          };
          auto weights = [&](int c, const f32x4& ks) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float pv[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) pv[e] = __builtin_amdgcn_exp2f(sv[x][e]);
              psum[x] += (pv[0] + pv[1]) + (pv[2] + pv[3]);
#pragma unroll
              for (int e = 0; e < 4; ++e) pv[e] *= ks[e];
              dn_store_weights<2>(pw + (c & 1) * 64 * DN_PROW + 16 * x * DN_PROW, pv);
            }
          };
          auto settle = [&](int c, const int4& fl) __attribute__((always_inline)) {
            if (__builtin_amdgcn_readfirstlane(fl.x | fl.y | fl.z | fl.w)) {
              float cm[2];
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                cm[x] = max_nonan(max_nonan(sv[x][0], sv[x][1]), max_nonan(sv[x][2], sv[x][3]));
                cm[x] = max_nonan(cm[x], __shfl_xor(cm[x], 16, WAVE));
                cm[x] = max_nonan(cm[x], __shfl_xor(cm[x], 32, WAVE));
                if (kq == 0) sh.cmax[wave][16 * x + j] = cm[x];
              }
              lds_barrier();
#pragma unroll
              for (int x = 0; x < 2; ++x) {
#pragma unroll
                for (int w = 0; w < 4; ++w) cm[x] = max_nonan(cm[x], sh.cmax[w][16 * x + j]);
                const float up = c == 0 ? max_nonan(cm[x], -1e30f) : cm[x] > DN_SLACK ? cm[x] : 0.0f;
                const float alpha = c == 0 ? 0.0f : __builtin_amdgcn_exp2f(-up);
                m_run[x] += up;
                l_run[x] *= alpha;
                psum[x] = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) sv[x][e] -= up;
                if (wave == 0 && kq == 0) sh.al[16 * x + j] = alpha;
              }
              weights(c, four(sh.ksc[last]));
              lds_barrier();
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              l_run[x] += psum[x];
              psum[x] = 0.0f;
            }
          };
          auto flags = [&](int c) __attribute__((always_inline)) {
            return *reinterpret_cast<const int4*>(sh.flag[c & 1]);
          };
          __builtin_amdgcn_s_setprio(1);
          for (int c = 0; c < nch; ++c) {
            const uint8_t* tile = sh.tile[buf];
            auto k_read = [&](int m) __attribute__((always_inline)) {
              return *reinterpret_cast<const u32x4*>(tile + koff + 64 * m);
            };
            int4 fl = make_int4(0, 0, 0, 0);
            if (c > 0) fl = flags(c - 1);
            f32x4 sa[2] = {};
            u32x4 kk[DN_KAHEAD + 1];
            bf16x8 ka[2], kb[2];
#pragma unroll
            for (int m = 0; m < DN_KAHEAD; ++m) kk[m] = k_read(m);
            __builtin_amdgcn_sched_barrier(0);
            settle(c - 1, fl);
            ka[0] = fp8x8_to_bf16x8(kk[0][0], kk[0][1]);
            kb[0] = fp8x8_to_bf16x8(kk[0][2], kk[0][3]);
#pragma unroll
            for (int m = 0; m < PIECES; ++m) {
              if (m + DN_KAHEAD < PIECES) kk[(m + DN_KAHEAD) % (DN_KAHEAD + 1)] = k_read(m + DN_KAHEAD);
#pragma unroll
              for (int x = 0; x < 2; ++x)
                sa[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[m & 1], qb[x][2 * m], sa[x], 0, 0, 0);
#pragma unroll
              for (int x = 0; x < 2; ++x)
                sa[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kb[m & 1], qb[x][2 * m + 1], sa[x], 0, 0, 0);
              if (m + 1 < PIECES) {
                const u32x4 k1 = kk[(m + 1) % (DN_KAHEAD + 1)];
                ka[(m + 1) & 1] = fp8x8_to_bf16x8(k1[0], k1[1]);
                kb[(m + 1) & 1] = fp8x8_to_bf16x8(k1[2], k1[3]);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
            const f32x4 kx = four(sh.kfac[buf]), ks = four(sh.ksc[buf]);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int e = 0; e < 4; ++e) sv[x][e] = fmaf(sa[x][e], kx[e], -m_run[x]);
            if (t0 + (c + 1) * DN_CHUNK > seen0) {  // tokens that a row does not see
              const int at = t0 + c * DN_CHUNK + 16 * wave + 4 * kq;
#pragma unroll
              for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) sv[x][e] = at + e < seen[x] ? sv[x][e] : -INFINITY;
            }
            float cm = sv[0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) cm = max_nonan(cm, sv[e >> 2][e & 3]);
            weights(c, ks);
            const bool any = c == 0 || __ballot(cm > DN_SLACK) != 0;
            if (lane == 0) sh.flag[c & 1][wave] = any;
            last = buf;
            buf = buf == BUFS - 1 ? 0 : buf + 1;
            lds_barrier();
          }
          __builtin_amdgcn_s_setprio(0);
          settle(nch - 1, flags(nch - 1));
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float lw = l_run[x] + __shfl_xor(l_run[x], 16, WAVE);
            lw += __shfl_xor(lw, 32, WAVE);
            if (kq == 0) sh.lsum[wave][16 * x + j] = lw;
            if (wave == 0 && kq == 0) sh.mfin[16 * x + j] = m_run[x];
          }
          lds_barrier();
          finish([](int) {});
        } else {
          const int row = min(r0 + 32 * hh + j, M - 1);
          const int seen = len - S + row / H + 1;  // tokens that this lane's row sees
          const int seen0 = len - S + r0 / H + 1;  // and the tile's first row, the fewest
          bf16x8 qb[2 * STEPS];  // row 32 hh + j: step s holds dims 32 s + 16 h .. + 15
          {
            const uint8_t* const qr = sh.tile[1] + (32 * hh + j) * 2 * DQK;
#pragma unroll
            for (int s = 0; s < 2 * STEPS; ++s)
              qb[s] = as_bf16x8(*reinterpret_cast<const uint4*>(
                  qr + 16 * ((4 * (s >> 1) + 2 * h + (s & 1)) ^ dn_q_swizzle<DQK>(j))));
          }
          lds_barrier();  // the queries are read
          float m_run = 0.0f;  // running max (base 2) of row 32 hh + j; chunk 0's scores are taken against 0, its flags are
                               // always up
          float l_run = 0.0f;  // this lane's share of its running sum
          float psum = 0.0f;   // and of the last chunk's, not yet in l_run
          f32x16 sv = {};      // the last chunk's scores - m_run: row 32 hh + j, tokens 32 th + 8 (r / 4) + 4 h + r % 4
          const int kr = 32 * th + j;
          const int kf = dn_swizzle(kr);  // byte offsets of a row's pieces at even and odd steps of 32 dims
          const int koff[2] = {kr * DN_KROW + 16 * (h ^ kf), kr * DN_KROW + 16 * ((2 | h) ^ kf)};
          uint16_t* const pw = &sh.p[0][(32 * hh + j) * DN_PROW + 32 * th + 4 * h];
          int buf = 0, last = 0;  // chunk c's buffer and chunk c - 1's
          auto four = [&](const float* a, int g) __attribute__((always_inline)) {
            return *reinterpret_cast<const f32x4*>(a + 32 * th + 8 * g + 4 * h);
          };
          // four tokens (group g of the lane's 16) of P from their scores and scales
          auto p_group = [&](int c, int g, const f32x4& ks) __attribute__((always_inline)) {
            float pv[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) pv[e] = __builtin_amdgcn_exp2f(sv[4 * g + e]);
            psum += (pv[0] + pv[1]) + (pv[2] + pv[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) pv[e] *= ks[e];
            dn_store_weights<1>(pw + (c & 1) * 64 * DN_PROW + 8 * g, pv);
          };
          // a chunk whose flags (fl) are up: its maxima over both token halves, the moved running maxima, P again
          auto settle = [&](int c, const int4& fl) __attribute__((always_inline)) {
            if (__builtin_amdgcn_readfirstlane(fl.x | fl.y | fl.z | fl.w)) {
              float cm = sv[0];
              if (c == 0) {  // m's start: see dn_log2_mantissa
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                  const f32x4 kl = four(sh.klog, g);
#pragma unroll
                  for (int e = 0; e < 4; ++e) cm = g + e == 0 ? sv[0] + kl[0] : max_nonan(cm, sv[4 * g + e] + kl[e]);
                }
              } else {
#pragma unroll
                for (int r = 1; r < 16; ++r) cm = max_nonan(cm, sv[r]);
              }
              cm = max_nonan(cm, __shfl_xor(cm, 32, WAVE));
              if (h == 0) sh.cmax[th][32 * hh + j] = cm;
              lds_barrier();
              cm = max_nonan(cm, sh.cmax[th ^ 1][32 * hh + j]);
              // a row that sees none of chunk 0 sees none of the stretch: its maximum stays finite
              const float up = c == 0 ? max_nonan(cm, -1e30f) : cm > DN_SLACK ? cm : 0.0f;
              // chunk 0 has nothing to rescale, and its factor would be infinite where every score is at or below -128
              const float alpha = c == 0 ? 0.0f : __builtin_amdgcn_exp2f(-up);
              m_run += up;
              l_run *= alpha;
              psum = 0.0f;
#pragma unroll
              for (int r = 0; r < 16; ++r) sv[r] -= up;
#pragma unroll
              for (int g = 0; g < 4; ++g) p_group(c, g, four(sh.ksc[last], g));
              if (th == 0 && h == 0) sh.al[32 * hh + j] = alpha;
              lds_barrier();
            }
            l_run += psum;
            psum = 0.0f;
          };
          auto flags = [&](int c) __attribute__((always_inline)) { return *reinterpret_cast<const int4*>(sh.flag[c & 1]); };
          __builtin_amdgcn_s_setprio(1);  // these waves bound the interval: their products go before the value products
          for (int c = 0; c < nch; ++c) {
            const uint8_t* tile = sh.tile[buf];
            auto k_read = [&](int s) __attribute__((always_inline)) {
              return *reinterpret_cast<const u32x4*>(tile + koff[s & 1] + 64 * (s >> 1));
            };
            int4 fl = make_int4(0, 0, 0, 0);
            if (c > 0) fl = flags(c - 1);
            f32x16 sa = {};
            u32x4 kk[DN_KAHEAD + 1];
            bf16x8 ka[2], kb[2];
            f32x4 ks[2], kx[2];
#pragma unroll
            for (int s = 0; s < DN_KAHEAD; ++s) kk[s] = k_read(s);
            __builtin_amdgcn_sched_barrier(0);
            settle(c - 1, fl);
            ka[0] = fp8x8_to_bf16x8(kk[0][0], kk[0][1]);
            kb[0] = fp8x8_to_bf16x8(kk[0][2], kk[0][3]);
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
              if (s + DN_KAHEAD < STEPS) kk[(s + DN_KAHEAD) % (DN_KAHEAD + 1)] = k_read(s + DN_KAHEAD);
              sa = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[s & 1], qb[2 * s], sa, 0, 0, 0);
              sa = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kb[s & 1], qb[2 * s + 1], sa, 0, 0, 0);
              if (s + 1 < STEPS) {
                const u32x4 k1 = kk[(s + 1) % (DN_KAHEAD + 1)];
                ka[(s + 1) & 1] = fp8x8_to_bf16x8(k1[0], k1[1]);
                kb[(s + 1) & 1] = fp8x8_to_bf16x8(k1[2], k1[3]);
              }
              if (s == STEPS - 2) {
                ks[0] = four(sh.ksc[buf], 0);
                kx[0] = four(sh.kfac[buf], 0);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              if (g < 3) kx[(g + 1) & 1] = four(sh.kfac[buf], g + 1);
#pragma unroll
              for (int e = 0; e < 4; ++e) sv[4 * g + e] = fmaf(sa[4 * g + e], kx[g & 1][e], -m_run);
            }
            if (t0 + (c + 1) * DN_CHUNK > seen0) {  // tokens that a row does not see
              const int lim = seen - t0 - c * DN_CHUNK - 32 * th - 4 * h;
#pragma unroll
              for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) sv[4 * g + e] = 8 * g + e < lim ? sv[4 * g + e] : -INFINITY;
            }
            float cm = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              if (g < 3) ks[(g + 1) & 1] = four(sh.ksc[buf], g + 1);
#pragma unroll
              for (int e = 0; e < 4; ++e) cm = max_nonan(cm, sv[4 * g + e]);
              p_group(c, g, ks[g & 1]);
            }
            const bool any = c == 0 || __ballot(cm > DN_SLACK) != 0;
            if (lane == 0) sh.flag[c & 1][wave] = any;
            last = buf;
            buf = buf == BUFS - 1 ? 0 : buf + 1;
            lds_barrier();
          }
          __builtin_amdgcn_s_setprio(0);
          settle(nch - 1, flags(nch - 1));
          const float lw = l_run + __shfl_xor(l_run, 32, WAVE);
          if (h == 0) sh.lsum[th][32 * hh + j] = lw;
          if (th == 0 && h == 0) sh.mfin[32 * hh + j] = m_run;
          lds_barrier();
          finish([](int) {});
        }
      } else {
        // -- the loads and the values: thread 4 r + e of the value waves brings row r of a chunk, pieces e + 4 i; wave w
        // takes dims 128 w .. + 127 of all rows --
        const int w = wave - 4;
        const int lane = fresh_lane(), j = lane & 31, h = lane >> 5;
        const int* trow = table + (size_t)b * max_pages;
        const int gr = 16 * w + (lane >> 2);  // this thread's row
        // its token in chunk c, the stretch's last one past its end (a slot behind the sequence may never have been
        // written, and its NaN x weight 0 is NaN)
        const int t_last = min(t0 + nch * DN_CHUNK, len) - 1;
        auto token = [&](int c) __attribute__((always_inline)) { return min(t0 + c * DN_CHUNK + gr, t_last); };
        auto page_of = [&](int t) __attribute__((always_inline)) { return (int)((uint64_t)t * pg.mul >> pg.shift); };
        auto slot_of = [&](int c, int page) __attribute__((always_inline)) {
          const int t = token(c);
          return safe_page(page, num_pages) * pg.size + (t - page_of(t) * pg.size);
        };
        const int gs = gr * DN_KROW + 16 * ((lane & 3) ^ dn_swizzle(gr));  // where its pieces go in a tile
        u32x4 held[PIECES];  // the pieces in flight, of the chunk after the one being stored
        float sc;          // and its token's scale
        auto row_of = [&](int slot) __attribute__((always_inline)) { return kv + (size_t)slot * DQK + 16 * (lane & 3); };
        auto store_scale = [&](int to) __attribute__((always_inline)) {
          if ((lane & 3) == 0) {
            sh.ksc[to][gr] = sc;
            sh.kfac[to][gr] = fmaf(sc, sl2, sc * sl2_lo);
          }
        };
        f32x16 o[4][RB];  // [dim block][row block]: row 32 i + j, dims 128 w + 32 d + 8 (r / 4) + 4 h + r % 4
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i = 0; i < RB; ++i) o[d][i] = f32x16{};
        // (the value operand's reads)
        const int vr = 8 * h + ((lane & 15) >> 1), vf = dn_swizzle(vr), vb0 = (lane >> 4) & 1;
        const int vrow = vr * DN_KROW + 128 * w + 8 * (lane & 1);
        const int voff[2] = {vrow + 16 * (vb0 ^ vf), vrow + 16 * ((2 | vb0) ^ vf)};
        const uint16_t* const pr = &sh.p[0][j * DN_PROW + 8 * h];
        // the value operand of step i (tokens 16 (i / 4) .. + 15, dims 128 w + 32 (i % 4) .. + 31), read transposed
        auto v_read = [&](const uint8_t* kt, int i) __attribute__((always_inline)) {
          return __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (__attribute__((address_space(3))) dn_v2i*)(kt + voff[i & 1] + 16 * (i >> 2) * DN_KROW +
                                                          64 * ((i & 3) >> 1)));
        };
        auto p_read = [&](int pb, int t, int i) __attribute__((always_inline)) {
          return as_bf16x8(*reinterpret_cast<const uint4*>(pr + pb * 64 * DN_PROW + 32 * i * DN_PROW + 16 * t));
        };
        // Interval c: chunk c - 1's weights are final (and O on their maxima) once its flags are seen; then its value
        // product, 16 steps of two products, the next steps' operands read and converted ahead, side(i) beside step i.
        auto interval = [&](int c, const uint8_t* kt, auto side) __attribute__((always_inline)) {
          const int pb = (c - 1) & 1;
          const int4 fl = *reinterpret_cast<const int4*>(sh.flag[pb]);
          dn_v2i vv[DN_VAHEAD + 1];
          bf16x8 pa[2][2], vb[2];
#pragma unroll
          for (int i = 0; i < DN_VAHEAD; ++i) vv[i] = v_read(kt, i);
          if (__builtin_amdgcn_readfirstlane(fl.x | fl.y | fl.z | fl.w)) {
            lds_barrier();
            lds_barrier();
            if (c > 1) {  // O is zero before
#pragma unroll
              for (int i = 0; i < RB; ++i) {
                const float a = sh.al[32 * i + j];
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                  for (int r = 0; r < 16; ++r) o[d][i][r] *= a;
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) pa[0][i] = p_read(pb, 0, i);
          vb[0] = fp8x8_to_bf16x8((uint32_t)vv[0].x, (uint32_t)vv[0].y);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int t = i >> 2, d = i & 3;
            if (i + DN_VAHEAD < 16) vv[(i + DN_VAHEAD) % (DN_VAHEAD + 1)] = v_read(kt, i + DN_VAHEAD);
            if (d < 2 && t < 3) pa[(t + 1) & 1][d] = p_read(pb, t + 1, d);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              f32x16& sum = o[d][RB == 1 ? 0 : x];
              sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb[i & 1], pa[t & 1][x], sum, 0, 0, 0);
            }
            if (i < 15) {
              const dn_v2i r = vv[(i + 1) % (DN_VAHEAD + 1)];
              vb[(i + 1) & 1] = fp8x8_to_bf16x8((uint32_t)r.x, (uint32_t)r.y);
            }
            side(i);
            __builtin_amdgcn_sched_barrier(0);
          }
        };
        int page = trow[page_of(token(2))];  // of this thread's token two chunks on
        const int page0 = trow[page_of(token(0))], page1 = trow[page_of(token(1))];
        {  // chunks 0 and 1 together: the first into LDS, the second stays in flight
          const int slot0 = slot_of(0, page0), slot1 = slot_of(1, page1);
          const uint8_t *src0 = row_of(slot0), *src1 = row_of(slot1);
          u32x4 first[PIECES];
#pragma unroll
          for (int i = 0; i < PIECES; ++i) first[i] = *reinterpret_cast<const u32x4*>(src0 + 64 * i);
          const float sc0 = kvs ? kvs[slot0] : 1.0f;
#pragma unroll
          for (int i = 0; i < PIECES; ++i) held[i] = *reinterpret_cast<const u32x4*>(src1 + 64 * i);
          const float sc1 = kvs ? kvs[slot1] : 1.0f;
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < PIECES; ++i) *reinterpret_cast<u32x4*>(sh.tile[0] + gs + 64 * i) = first[i];
          sc = sc0;
          store_scale(0);
          if (RB == 2 && (lane & 3) == 0) sh.klog[gr] = dn_log2_mantissa(sc0);
          sc = sc1;
        }
        lds_barrier();  // the queries and chunk 0 are in place
        lds_barrier();  // the queries are read
        // Interval c stores chunk c + 1 into the buffer that chunk c - 2 left and loads chunk c + 2, piece by piece, in
        // the last intervals too (the stretch's last row then, into buffers that nobody reads).
        const uint8_t* src = nullptr;
        float sc_next = 1.0f;
        auto ahead = [&](int c) __attribute__((always_inline)) {
          const int slot = slot_of(c + 2, page);
          page = trow[page_of(token(c + 3))];
          src = row_of(slot);
          if (kvs) sc_next = kvs[slot];
        };
        auto piece = [&](int i, uint8_t* to) __attribute__((always_inline)) {
          *reinterpret_cast<u32x4*>(to + gs + 64 * i) = held[i];
          held[i] = *reinterpret_cast<const u32x4*>(src + 64 * i);
        };
        ahead(0);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) piece(i, sh.tile[1]);
        store_scale(1);
        sc = sc_next;
        lds_barrier();
        int buf = 1;  // chunk c's buffer
#pragma unroll 1
        for (int c = 1; c <= nch; ++c) {
          const int prev = buf == 0 ? BUFS - 1 : buf - 1, next = buf == BUFS - 1 ? 0 : buf + 1;
          ahead(c);
          interval(c, sh.tile[prev], [&](int i) __attribute__((always_inline)) {
            if (i >= DN_STORE && i < DN_STORE + PIECES) piece(i - DN_STORE, sh.tile[next]);
          });
          store_scale(next);
          sc = sc_next;
          buf = next;
          lds_barrier();
        }
        if (!whole) {  // as they lie in the registers: see dn_partial
          float* const to = ws_o + (size_t)part * ROWS * DN_DV + dn_partial(w, 0, 0, 0, RB) + 4 * lane;
#pragma unroll
          for (int i = 0; i < RB; ++i)
            if (32 * i + j < M - r0)
#pragma unroll
              for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                  *reinterpret_cast<f32x4*>(to + dn_partial(0, i, d, g, RB)) =
                      f32x4{o[d][i][4 * g], o[d][i][4 * g + 1], o[d][i][4 * g + 2], o[d][i][4 * g + 3]};
        }
        finish([&](int half) __attribute__((always_inline)) {
          if ((w >> 1) != half) return;
#pragma unroll
          for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const int x = 32 * (w & 1) + 8 * d + 2 * g + h;
                area[64 * x + ((32 * i + j) ^ (x & 7))] =
                    f32x4{o[d][i][4 * g], o[d][i][4 * g + 1], o[d][i][4 * g + 2], o[d][i][4 * g + 3]};
              }
        });
      }
      lds_barrier();  // (the area's readers, before the next stretch's loads)
    }
    u += nch;
    c0 = 0;
    if (u < u1 && ++set == tm.sets) {  // the next sequence with tokens
      set = 0;
      if (++b >= B) return;
      len = dn_len(ctx_len[b], max_pages, pg.size);
      while (len == 0) {  // (a padded batch may have many without: the next of them looked for side by side)
        if (tid == 0) sh.found[0] = B;
        __syncthreads();
        const int x = b + 1 + tid;
        if (x < B && ctx_len[x] > 0) atomicMin(&sh.found[0], x);
        __syncthreads();
        const int next = __builtin_amdgcn_readfirstlane(sh.found[0]);
        __syncthreads();
        if (next >= B && b + DN_THREADS >= B - 1) return;
        b = min(next, b + DN_THREADS);
        len = dn_len(ctx_len[b], max_pages, pg.size);
      }
    }
  }
}

// Joins the partials of a row tile where teams shared it: out = sum 2^(m - max) O / sum 2^(m - max) l; and writes the
// rows of sequences without tokens. A wave has a block of 32 rows x 8 G dims, in the partials' own order; WPR waves of
// a workgroup share a block's partials, each taking every WPR-th, DEEP of them in flight.
constexpr int DC_WAVES = 8;
constexpr int DC_THREADS = DC_WAVES * WAVE;

template <int RB, int WPR, int G>
__global__ __launch_bounds__(DC_THREADS) void dense_combine_kernel(
    const float* __restrict__ ws_o, const float* __restrict__ ws_ml, const int* __restrict__ ctx_len,
    uint16_t* __restrict__ out, float* __restrict__ out_f32, float* __restrict__ lse_out, int B, int S, int H,
    int max_pages, int page_size, DnTeams tm) {
  constexpr int ROWS = 32 * RB, BLOCKS = 64 / G * RB, DEEP = G == 1 ? 8 : 4;
  __shared__ int tot[DC_WAVES];
  __shared__ int chunks_before[2];
  __shared__ float wm[DC_WAVES][32], wl[DC_WAVES][32];
  __shared__ f32x4 acc[WPR > 1 ? DC_WAVES : 1][G][WAVE];
  const int M = S * H, tid = threadIdx.x;
  const int lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int j = lane & 31, h = lane >> 5;
  // this wave's block (the last one again past the end, not written)
  const int blocks = B * tm.tiles * BLOCKS, first_at = blockIdx.x * (DC_WAVES / WPR), at = first_at + wave / WPR;
  const int block = min(at, blocks - 1) % BLOCKS, tile = min(at, blocks - 1) / BLOCKS;
  const int b = tile / tm.tiles, mt = tile - b * tm.tiles;
  const int first_b = first_at / BLOCKS / tm.tiles;  // (8 blocks are of two tiles at most)
  int chunks = 0;
  for (int b0 = 0; b0 < B; b0 += DC_THREADS) {
    const int x = b0 + tid;
    const int n = x < B ? dn_chunks(dn_len(ctx_len[x], max_pages, page_size)) : 0;
    int total;
    const int incl = chunks + group_incl_scan<DC_THREADS>(n, tot, total);
    if (x >= first_b && x < first_b + 2) chunks_before[x - first_b] = incl - n;
    chunks += total;
  }
  __syncthreads();
  const DnList list = dn_list(chunks * tm.sets, tm.teams);
  const int nch = dn_chunks(dn_len(ctx_len[b], max_pages, page_size));
  // the row tile's units: first .. first + nch - 1
  const int first = chunks_before[b - first_b] * tm.sets + mt / tm.span * nch;
  const int w0 = nch ? dn_owner(first, list) : 0, w1 = nch ? dn_owner(first + nch - 1, list) : -1;
  if (at >= blocks || w0 == w1) return;  // (one team's: its workgroup wrote them; the same for all of a block's waves)
  const int block32 = block * G / 4, w = block32 / (4 * RB), i = block32 / 4 % RB, d = block32 & 3;
  const int g0 = G == 1 ? block & 3 : 0;
  const int r = 32 * i + j, row = mt * ROWS + r;  // this lane's row of the tile, and of the sequence
  float m = -INFINITY, l = 0.0f;
  f32x4 a[G] = {};
  if (nch > 0 && row < M) {
    const float* const from = ws_o + dn_partial(w, i, d, g0, RB) + 4 * lane;
    // team w0's stretch is not its first where it started before the tile, the others' is
    const int slot0 = 2 * w0 + (dn_start(w0, list) < first);
    for (int t = w0 + wave % WPR; t <= w1; t += DEEP * WPR) {
      const int n = (w1 - t) / WPR + 1;  // this round's, up to DEEP
      float2 ml[DEEP];
      f32x4 v[DEEP][G];
#pragma unroll
      for (int x = 0; x < DEEP; ++x) {
        ml[x] = make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int g = 0; g < G; ++g) v[x][g] = f32x4{};
        if (x < n) {
          const int u = t + WPR * x;
          const size_t part = ((size_t)(u == w0 ? slot0 : 2 * u) * tm.span + mt % tm.span) * ROWS;
          ml[x] = reinterpret_cast<const float2*>(ws_ml)[part + r];
#pragma unroll
          for (int g = 0; g < G; ++g) v[x][g] = *reinterpret_cast<const f32x4*>(from + part * DN_DV + 4 * WAVE * g);
        }
      }
      float mx = m;
#pragma unroll
      for (int x = 0; x < DEEP; ++x) mx = max_nonan(mx, ml[x].x);
      const float f = __builtin_amdgcn_exp2f(m - mx);
      m = mx;
      l *= f;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) a[g][e] *= f;
#pragma unroll
      for (int x = 0; x < DEEP; ++x) {
        const float c = __builtin_amdgcn_exp2f(ml[x].x - m);
        l = fmaf(c, ml[x].y, l);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) a[g][e] = fmaf(c, v[x][g][e], a[g][e]);
      }
    }
  }
  const size_t out_row = (size_t)b * M + row;
  if constexpr (WPR == 1) {
    const float inv = inverse_or_0(l);
    uint2 pk[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
#pragma unroll
      for (int e = 0; e < 4; ++e) a[g][e] *= inv;
      pk[g] = make_uint2(bf16_pack(a[g][0], a[g][1]), bf16_pack(a[g][2], a[g][3]));
    }
    // lanes j and 32 + j have a row's 64 bytes by eights in turn: each takes a half of them
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const uint2 give = h ? pk[g] : pk[g + 2];
      const uint2 got = make_uint2(__shfl_xor((int)give.x, 32, WAVE), __shfl_xor((int)give.y, 32, WAVE));
      const uint2 own = h ? pk[g + 2] : pk[g];
      if (out && row < M)
        *reinterpret_cast<uint4*>(out + out_row * DN_DV + 128 * w + 32 * d + 16 * h + 8 * g) =
            h ? make_uint4(got.x, got.y, own.x, own.y) : make_uint4(own.x, own.y, got.x, got.y);
    }
    if (row >= M) return;
    if (out_f32)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(out_f32 + out_row * DN_DV + 128 * w + 32 * d + 8 * g + 4 * h) = a[g];
    if (lse_out && w == 0 && d == 0 && h == 0) lse_out[out_row] = lse_or_none(m, l);
    return;
  }
  if (h == 0) {
    wm[wave][j] = m;
    wl[wave][j] = l;
  }
#pragma unroll
  for (int g = 0; g < G; ++g) acc[WPR > 1 ? wave : 0][g][lane] = a[g];
  __syncthreads();
  if (wave >= G || row >= M) return;  // wave g joins group g
  float mm = wm[0][j], ll = 0.0f;
  f32x4 o = {};
#pragma unroll
  for (int x = 1; x < DC_WAVES; ++x) mm = max_nonan(mm, wm[x][j]);
#pragma unroll
  for (int x = 0; x < DC_WAVES; ++x) {
    const float f = mm > -INFINITY ? __builtin_amdgcn_exp2f(wm[x][j] - mm) : 0.0f;  // (0 for a wave without partials)
    ll = fmaf(f, wl[x][j], ll);
    const f32x4 v = acc[WPR > 1 ? x : 0][wave][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(f, v[e], o[e]);
  }
  const size_t to = out_row * DN_DV + 128 * w + 32 * d + 8 * (g0 + wave) + 4 * h;
  const float inv = inverse_or_0(ll);
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= inv;
  if (out) *reinterpret_cast<uint2*>(out + to) = make_uint2(bf16_pack(o[0], o[1]), bf16_pack(o[2], o[3]));
  if (out_f32) *reinterpret_cast<f32x4*>(out_f32 + to) = o;
  if (lse_out && w == 0 && d == 0 && g0 + wave == 0 && h == 0) lse_out[out_row] = lse_or_none(mm, ll);
}

// Workgroups: one a CU, a multiple of the 8 XCDs.
static int dense_grid(int num_cu) { return num_cu < 8 ? 8 : num_cu / 8 * 8; }

static int dense_rows(int M) { return M <= 32 ? 32 : 64; }

// The teams of M rows: of the spans that divide the tiles and an XCD's CUs with the least left idle, the widest.
static DnTeams dense_teams(int M, int num_cu) {
  const int per_xcd = dense_grid(num_cu) / 8;
  DnTeams t;
  t.rows = dense_rows(M);
  t.tiles = (int)(((long)M + t.rows - 1) / t.rows);
  double best = 0.0;
  for (int span = 1; span <= t.tiles && span <= per_xcd; ++span) {
    if (span == 1 && t.tiles > 1 && per_xcd > 1) continue;  // (two tiles at least read the cache together)
    const int sets = (t.tiles + span - 1) / span, teams = per_xcd / span;
    const double used = (double)t.tiles / ((double)sets * span) * (teams * span) / per_xcd;
    if (used >= best) {
      best = used;
      t.span = span;
      t.sets = sets;
      t.teams = 8 * teams;
    }
  }
  return t;
}

size_t dense_workspace_bytes(int M, int num_cu) {
  const DnTeams t = dense_teams(M, num_cu);
  return (size_t)2 * t.teams * t.span * t.rows * (DN_DV + 2) * sizeof(float);
}

hipError_t launch_dense_mla(const uint16_t* q, const uint8_t* kv, const float* kvs, const int* table,
                            const int* ctx_len, uint16_t* out, float* out_f32, float* lse, void* ws, int B, int S,
                            int H, int Dqk, int max_pages, int page_size, int num_pages, float scale, int num_cu,
                            hipStream_t s) {
  const DnTeams tm = dense_teams(S * H, num_cu);
  const int G = dense_grid(num_cu);
  int log2 = 0;
  while ((1L << log2) < page_size) ++log2;
  const DnPage pg = {(uint32_t)(((1ull << (31 + log2)) + page_size - 1) / page_size), 31 + log2, page_size};
  float* ws_o = static_cast<float*>(ws);
  float* ws_ml = ws_o + (size_t)2 * tm.teams * tm.span * tm.rows * DN_DV;
  const auto kernel = tm.rows == 32 ? Dqk == 512 ? dense_mla_kernel<512, 1> : dense_mla_kernel<576, 1>
                                    : Dqk == 512 ? dense_mla_kernel<512, 2> : dense_mla_kernel<576, 2>;
  const hipError_t e = launch("dense_mla_kernel", kernel, dim3(G), dim3(DN_THREADS), s, q, kv, kvs, table, ctx_len,
                              out, out_f32, lse, ws_o, ws_ml, B, S, H, max_pages, pg, num_pages, scale, tm);
  if (e != hipSuccess) return e;
  // How a block of 32 rows x 32 dims is joined, by how many there are: from 3 blocks a CU on by one wave, a partial after
  // another (4 in flight); fewer by a workgroup, whose 8 waves share its partials; and where there are no more than a
  // quarter of the CUs, each quarter of its dims by a workgroup. Measured, us in turn with quarters, shared, one wave:
  // 1 x 4k tokens, 16 heads (16 blocks) 4.0, 5.5, 21; 1 x 128k, 128 heads (64) 8.0, 9.5, 45; 8 x 32k, 64 heads (256) 9.6,
  // 8.1, 14.6; 16 x 32k (512) 14.7, 8.7, 10.0; 30 x 4k (960) 27, 12.2, 9.3; 4 x 4 new tokens after 1k, 128 heads (1,024)
  // 22, 10.4, 7.8.
  const long blocks = (long)B * tm.tiles * (tm.rows / 2);
  const bool one = tm.rows == 32;
  auto join = [&](auto kernel, long groups) {
    return launch("dense_combine_kernel", kernel, dim3((unsigned)groups), dim3(DC_THREADS), s, ws_o, ws_ml, ctx_len, out,
                  out_f32, lse, B, S, H, max_pages, page_size, tm);
  };
  if (blocks >= 3L * num_cu)
    return join(one ? dense_combine_kernel<1, 1, 4> : dense_combine_kernel<2, 1, 4>, (blocks + DC_WAVES - 1) / DC_WAVES);
  if (4 * blocks > num_cu)
    return join(one ? dense_combine_kernel<1, DC_WAVES, 4> : dense_combine_kernel<2, DC_WAVES, 4>, blocks);
  return join(one ? dense_combine_kernel<1, DC_WAVES, 1> : dense_combine_kernel<2, DC_WAVES, 1>, 4 * blocks);
}

// Whether the list of units fits 32 bits, whatever the lengths, and the rows a launch.
bool dense_list_ok(int B, int S, int H, int max_pages, int page_size) {
  const long M = (long)S * H, tiles = (M + 31) / 32, cap = (long)max_pages * page_size;
  const long tokens = cap < 0x7fffffffL ? cap : 0x7fffffffL;
  return M <= 0x7fffffffL && (long)B * tiles <= 0x3fffffL && (double)B * tiles * (tokens / DN_CHUNK + 1) < 2e9;
}

}  // namespace dsa
