// Expanded latent attention for gfx950, the form of a prefill: the keys and values of every head from the cached latent
// rows (expand_latent_kernel), and attention over them (expanded_attend_kernel). Per pair of tokens and head it costs
// 192 + 128 multiply-adds where the absorbed form's latent products cost 576 + 512.
#include "dsa_async.h"
#include "dsa_expand.h"
#include "dsa_scan.h"

namespace dsa {

constexpr int EX_D = 128;   // a head's key width without rope, and its value width
constexpr int EX_R = 64;    // the rope width, shared by the heads
constexpr int EX_C = 512;   // the latent width

// -- keys and values ------------------------------------------------------------------------------------------------
// k[t, h, :] = sigma_t c_t[:512] . W[h, :128, :]^T, v[t, h, :] the same with W[h, 128:, :]: a product of P x 512 x 256
// H whose left side is e4m3 rows gathered through the page table (the scale is applied to the sums), and k_rope[t] =
// sigma_t c_t[512:].
//
// What bounds it: the matrix units, then the stores. A share is of units (tile of 256 tokens, one head's 128 keys or
// values), a workgroup a CU. The rows of a tile stay in registers, e4m3 until they are operands
// (exact in bf16), while one part's weights after another run through LDS, 64 of the 512 columns a step, by
// asynchronous loads 7 steps ahead that cross the parts: a unit reads 128 KiB instead of the 256 of rows and weights
// through LDS, and stores from registers under the next unit's products (that form with two workgroups a CU: 336 us
// where this took 256 on the same card). The shares of one XCD are 8 tiles' and run through the same weights together,
// out of its L2. 16,384 tokens x 64 heads: 257 to 273 us from card to card, 1.01 to 1.07 PFLOP/s; 8,192 tokens, whose
// outputs the last-level cache holds: 112 us, 1.23.
constexpr int EL_THREADS = 512;
constexpr int EL_TOK = 256;  // (or half of it)
constexpr int EL_K = 64;
constexpr int EL_STEPS = EX_C / EL_K;
constexpr int EL_STAGES = 8;

struct ElShared {
  // a step's weights: 128 bytes a row, 16-byte piece p at p ^ ((row >> 1) & 3 | (row >> 5 & 1) << 2). Before a token
  // tile's first step the rows lie here, 512 bytes each, piece p at p ^ (row & 15).
  alignas(1024) uint16_t b[EL_STAGES][EX_D * EL_K];
  int slot[EL_TOK];
  int seq;
};
static_assert(sizeof(ElShared::b) >= EL_TOK * EX_C, "the rows");

// Lane 4 t + c holds pieces i = 0 .. 3 of row 4 t + c; after this, piece c of rows 4 t + i.
__device__ __forceinline__ void quad_transpose(uint32_t (&o)[4][4]) {
  const int c = threadIdx.x & 3;
#pragma unroll
  for (int d = 1; d < 4; d *= 2)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & d) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // the lane whose bit d is clear gives its piece i + d for the other's i
        const uint32_t lo = o[i][e], hi = o[i + d][e];
        const uint32_t give = c & d ? lo : hi;
        const uint32_t got = d == 1 ? __builtin_amdgcn_mov_dpp(give, 0xb1, 0xf, 0xf, true)
                                    : __builtin_amdgcn_mov_dpp(give, 0x4e, 0xf, 0xf, true);
        o[i][e] = c & d ? got : lo;
        o[i + d][e] = c & d ? hi : got;
      }
    }
}

// X groups of 32 tokens a wave: tiles of 128 X tokens
template <int X>
__global__ __launch_bounds__(EL_THREADS, 1) void expand_latent_kernel(
    const uint8_t* __restrict__ kv, const float* __restrict__ kvs, const int* __restrict__ table,
    const int* __restrict__ cu, const uint16_t* __restrict__ wkv, uint16_t* __restrict__ k_out,
    uint16_t* __restrict__ v_out, uint16_t* __restrict__ r_out, int B, int total, int H, int D, int max_pages,
    int page_size, int num_pages, int units) {
  constexpr int TOK = 128 * X, FIRST = EL_STAGES - TOK / 32;  // (stages that the rows do not take)
  __shared__ ElShared sh;
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int j = lane & 31, h = lane >> 5;
  const int parts = 2 * H, end = min(total, cu[B]);
  // this workgroup's share of the units (token tile, part), parts fastest; an XCD's (workgroup x runs on XCD x % 8) lie
  // next to each other
  const int xcd = blockIdx.x & 7, G = gridDim.x;
  const int g = xcd * (G >> 3) + min(xcd, G & 7) + (blockIdx.x >> 3);
  const int u0 = (int)((long)units * g / G), u1 = (int)((long)units * (g + 1) / G);
  // wave: tokens 32 X wm .. + 63 x columns 64 wn .. + 63; the columns are the products' rows, taken in an order that
  // leaves a lane 32 columns of one token in a row (32 h + 16 y + r)
  const int wm = wave >> 1, wn = wave & 1;
  const uint32_t b_lds = lds_address(sh.b[0] + 1024 * wave);
  const int bcol = 8 * ((lane & 7) ^ (((lane >> 4) & 3) | ((wave >> 1) & 1) << 2));
  const int brow = 64 * wn + 32 * ((j >> 2) & 1) + 4 * (j >> 3) + (j & 3);  // (+ 16 y)
  const int bsw = ((j >> 1) & 1) | ((j >> 3) & 1) << 1 | ((j >> 2) & 1) << 2;

#pragma unroll 1
  for (int u = u0; u < u1;) {
    const int tile = u / parts, part0 = u - tile * parts, n = min(parts - part0, u1 - u), t0 = tile * TOK;
    u += n;
    wait_loads<0>();
    if (t0 >= end) return;  // (rows past the last sequence are left as they were)
    if (tid == 0) sh.seq = 0;
    __syncthreads();  // (the last tile's stages are free)
    // step s of part p0 + p: weights 64 s .. + 63 of the part's 128 rows, this wave's 16 in eights
    const uint16_t* const bp = wkv + ((size_t)part0 * EX_D + 16 * wave + (lane >> 3)) * EX_C + bcol;
    const int last = n * EL_STEPS - 1;
    auto issue = [&](int st) __attribute__((always_inline)) {  // (past the end: the last step again, into a free stage)
      const int f = min(st, last);
      const uint16_t* from = bp + (size_t)(f / EL_STEPS) * EX_D * EX_C + (f % EL_STEPS) * EL_K;
      const uint32_t to = b_lds + 2 * EX_D * EL_K * (st % EL_STAGES);
      load_lds16(from, to);
      load_lds16(from + 8 * EX_C, to + 1024);
    };
#pragma unroll
    for (int i = 0; i < FIRST; ++i) issue(i);
    // the slots of the tile's tokens: the sequence of the first one by counting, the others' from there
    int c = 0;
    for (int b = tid; b < B; b += EL_THREADS) c += cu[b + 1] <= t0;
    if (c) atomicAdd(&sh.seq, c);
    __syncthreads();
    if (tid < TOK) {
      const int t = min(t0 + tid, end - 1);
      int b = min(sh.seq, B - 1), step = 1;  // the last sequence that starts by t, in doubling steps and halving ones
      for (; b + step < B && cu[b + step] <= t; step *= 2) b += step;
      for (step /= 2; step > 0; step /= 2)
        if (b + step < B && cu[b + step] <= t) b += step;
      const int pos = max(t - cu[b], 0), pi = pos / page_size;
      const int page = pi < max_pages ? safe_page(table[(size_t)b * max_pages + pi], num_pages) : 0;
      sh.slot[tid] = page * page_size + (pos - pi * page_size);
    }
    __syncthreads();
    {  // the rows into LDS: this wave's 16 X, two at a time
      const uint32_t a_lds = lds_address(sh.b[FIRST]) + 16 * X * EX_C * wave;
      const int lane = fresh_lane(), j = lane & 31, h = lane >> 5;
#pragma unroll
      for (int i = 0; i < 8 * X; ++i) {
        const int r = 16 * X * wave + 2 * i + h;
        load_lds16(kv + (size_t)sh.slot[r] * D + 16 * (j ^ (r & 15)), a_lds + 2 * EX_C * i);
      }
    }
    float sc[X];
#pragma unroll
    for (int x = 0; x < X; ++x) sc[x] = kvs ? kvs[sh.slot[32 * X * wm + 32 * x + j]] : 1.0f;
    arrive(sc);
    if (part0 == 0 && r_out) {
      const int tid = WAVE * wave + fresh_lane();
#pragma unroll
      for (int i = 0; i < TOK * 8 / EL_THREADS; ++i) {  // 8 rope columns of a token
        const int x = tid + EL_THREADS * i, r = x >> 3, p = x & 7;
        if (t0 + r < end) {
          const int slot = sh.slot[r];
          const uint2 c8 = *reinterpret_cast<const uint2*>(kv + (size_t)slot * D + EX_C + 8 * p);
          const float f = kvs ? kvs[slot] : 1.0f;
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t two = (e & 2 ? c8.y : c8.x) >> (16 * (e & 1));
            const auto v = __builtin_amdgcn_cvt_pk_f32_fp8(two, false);
            o[e] = bf16_pack(v[0] * f, v[1] * f);
          }
          *reinterpret_cast<uint4*>(r_out + (size_t)(t0 + r) * EX_R + 8 * p) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
    }
    wait_loads<0>();
    lds_barrier();
    u32x4 a[X][2 * EL_STEPS];  // tokens 32 X wm + 32 x + j: columns 32 g + 16 h .. + 15
#pragma unroll
    for (int x = 0; x < X; ++x) {
      const int lane = fresh_lane(), j = lane & 31, h = lane >> 5;
      const uint8_t* row = reinterpret_cast<const uint8_t*>(sh.b[FIRST]) + EX_C * (32 * X * wm + 32 * x + j);
#pragma unroll
      for (int i = 0; i < 2 * EL_STEPS; ++i)
        a[x][i] = *reinterpret_cast<const u32x4*>(row + 16 * ((2 * i + h) ^ (j & 15)));
    }
    lds_barrier();  // the stages are free

#pragma unroll
    for (int i = FIRST; i < EL_STAGES - 1; ++i) issue(i);
#pragma unroll 1
    for (int p = 0; p < n; ++p) {
      f32x16 acc[X][2];
#pragma unroll
      for (int x = 0; x < X; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[x][y] = f32x16{};
#pragma unroll
      for (int s = 0; s < EL_STEPS; ++s) {
        wait_loads<2 * (EL_STAGES - 2)>();
        lds_barrier();  // the step is in place, and nobody reads the one before it any more
        issue(EL_STEPS * p + s + EL_STAGES - 1);
        const uint16_t* b = sh.b[s % EL_STAGES] + brow * EL_K;
#pragma unroll
        for (int g2 = 0; g2 < 2; ++g2) {
          bf16x8 wf[2][2];
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              wf[y][e] = as_bf16x8(*reinterpret_cast<const uint4*>(b + 16 * EL_K * y + 8 * ((4 * g2 + 2 * h + e) ^ bsw)));
#pragma unroll
          for (int x = 0; x < X; ++x) {
            u32x4& c4 = a[x][2 * s + g2];
            asm volatile("" : "+v"(c4));  // (else every operand would be made once, before the loop, in 256 registers)
            const bf16x8 c0 = fp8x8_to_bf16x8(c4[0], c4[1]), c1 = fp8x8_to_bf16x8(c4[2], c4[3]);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[y][0], c0, acc[x][y], 0, 0, 0);
              acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[y][1], c1, acc[x][y], 0, 0, 0);
            }
          }
        }
      }
      // a lane's 64 bytes of a token, 4 lanes' tokens: transposed among them, so that 4 lanes write one token's 64
      // bytes
      const int part = part0 + p;
      const size_t row0 = (size_t)(t0 + 32 * X * wm + 4 * (j >> 2));
      uint16_t* const out = (part & 1 ? v_out : k_out) + (row0 * H + (part >> 1)) * EX_D + 64 * wn + 32 * h + 8 * (j & 3);
#pragma unroll
      for (int x = 0; x < X; ++x) {
        uint32_t o[4][4];  // piece, dword
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 8 * (i & 1) + 2 * e;
            o[i][e] = bf16_pack(acc[x][i >> 1][r] * sc[x], acc[x][i >> 1][r + 1] * sc[x]);
          }
        quad_transpose(o);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t0 + 32 * X * wm + 32 * x + 4 * (j >> 2) + i < end)
            *reinterpret_cast<u32x4*>(out + (size_t)(32 * x + i) * H * EX_D) = u32x4{o[i][0], o[i][1], o[i][2], o[i][3]};
      }
    }
  }
  wait_loads<0>();
}

// -- attention ------------------------------------------------------------------------------------------------------
// s = scale (q[:128] . k + q[128:] . k_rope), p = softmax(s), out = p . v, lse, for ragged batches of queries and keys,
// causal (the last query sees every key) or full.
//
// What bounds it: the matrix units, then the LDS reads that feed them and the exponentials. One workgroup a CU has 256
// queries of a head, 8 waves of 32, two on each SIMD, the first of them with priority, so that one's softmax runs under
// the other's products. A tile of 64 keys and values comes by
// asynchronous loads straight into LDS two tiles ahead, with one barrier a tile. S^T = K . Q^T and O^T += V^T . P on
// v_mfma_f32_32x32x16_bf16: a lane's scores are of one query, in the value product's operand layout as they stand (the
// values are read transposed in the same order), so P never leaves the registers and the maxima and sums stay in their
// lanes. The longest tiles of a causal batch go first. Where there are few query tiles, their keys are taken in splits
// that expanded_combine_kernel joins.
//
// 8,192 tokens, 64 heads, causal: 1,208 to 1,250 us from card to card, 1.10 to 1.14 PFLOP/s (a large library product:
// 1.29). A grid of one round lasts as long as its longest tile: 4,096 causal tokens of 16 heads, a workgroup a CU, 119 us
// where an even share of the tiles' keys would be half of that.
constexpr int XA_THREADS = 512;
constexpr int XA_Q = 256;
constexpr int XA_K = 64;
constexpr int XA_STAGES = 3;
constexpr int XA_SPLITS = 16;
constexpr float XA_SLACK = 60.0f;  // lazy rescaling (base 2): p = 2^(s - m) <= 2^60 between moves of m
constexpr float XA_LOG2E = 1.44269504088896341f;

typedef short xa_v4s __attribute__((ext_vector_type(4)));

// A stage's keys and values lie in rows of 256 bytes, 16-byte piece p of key row r at p ^ (r & 15), of value row r at
// p ^ 4 (r & 3) (32 lanes read four pieces of 4 rows), of rope row r (128 bytes) at p ^ ((r >> 1) & 7).
template <int DQ>
struct XaShared {
  alignas(1024) uint8_t k[XA_STAGES][XA_K * 256];
  alignas(1024) uint8_t v[XA_STAGES][XA_K * 256];
  alignas(1024) uint8_t r[DQ > EX_D ? XA_STAGES : 1][DQ > EX_D ? XA_K * 128 : 16];
  alignas(16) uint8_t q[DQ > EX_D ? 16384 : 16];  // (the queries' last 64 columns lie over r[1], r[2] and this)
  int tot[XA_THREADS / WAVE];
  int found[2];
};

// A sequence's first query and their number (the offsets clamped to the queries there are).
__device__ __forceinline__ int xa_first(int b, const int* __restrict__ cu_q, int Tq) {
  return min(max(cu_q[b], 0), Tq);
}
__device__ __forceinline__ int xa_queries(int b, const int* __restrict__ cu_q, int Tq) {
  return max(min(cu_q[b + 1], Tq) - xa_first(b, cu_q, Tq), 0);
}
// The sequence of query tile ti and the tile's place in it, into found (-1: past the last one); the whole workgroup.
__device__ __forceinline__ void xa_find(int ti, const int* __restrict__ cu_q, int B, int Tq, int* tot, int* found) {
  if (threadIdx.x == 0) found[0] = -1;
  int before = 0;
  for (int b0 = 0; b0 < B && before <= ti; b0 += XA_THREADS) {
    const int b = b0 + threadIdx.x;
    const int n = b < B ? (xa_queries(b, cu_q, Tq) + XA_Q - 1) / XA_Q : 0;
    int total;
    const int incl = before + group_incl_scan<XA_THREADS>(n, tot, total);
    if (incl - n <= ti && ti < incl) {
      found[0] = b;
      found[1] = ti - (incl - n);
    }
    before += total;
  }
  __syncthreads();
}

// MORE: 1 with the ranges of ExpandedMore, 2 with all that it asks for; its branches are the workgroup's, or a tile's. 8,192
// causal tokens, 32 heads on one card (601 us without): with first = 0 throughout 608 (as 2: 626 for 617 on another), a window
// of 1,000 215, distances 632, caps 702, both 733. What the ranges cost is the tiles of 64 keys and 256 queries that they cut
// (a window of 1,000: 1.3 times the pairs); caps and distances are vector issue beside the products.
template <int DQ, int MORE>
__global__ __launch_bounds__(XA_THREADS, 1) void expanded_attend_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ k, const uint16_t* __restrict__ kr,
    const uint16_t* __restrict__ v, const int* __restrict__ cu_q, const int* __restrict__ cu_k,
    uint16_t* __restrict__ out, float* __restrict__ out_f32, float* __restrict__ lse_out, float* __restrict__ ws, int B,
    int Tq, int Tk, int H, int q_tiles, int splits, int causal, float scale, ExpandedMore more) {
  constexpr int STEPS = DQ / 16;
  constexpr int LOADS = DQ > EX_D ? 10 : 8;  // a tile's asynchronous loads per wave
  __shared__ XaShared<DQ> sh;
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int j = lane & 31, h = lane >> 5;
  // heads of one XCD (workgroup x runs on XCD x % 8) next to each other, query tiles from the last to the first
  const int grid = q_tiles * H, split = blockIdx.x / grid, at_tile = blockIdx.x - split * grid;
  int head, ti;
  if ((H & 7) == 0) {
    const int per = H >> 3, y = at_tile >> 3;
    head = (at_tile & 7) * per + y % per;
    ti = q_tiles - 1 - y / per;
  } else {
    head = at_tile % H;
    ti = q_tiles - 1 - at_tile / H;
  }
  xa_find(ti, cu_q, B, Tq, sh.tot, sh.found);
  const int b = __builtin_amdgcn_readfirstlane(sh.found[0]);
  if (b < 0) return;  // past the last tile
  const int qt = __builtin_amdgcn_readfirstlane(sh.found[1]) * XA_Q;
  const int nq = xa_queries(b, cu_q, Tq), qb = xa_first(b, cu_q, Tq);
  const int kb = min(max(cu_k[b], 0), Tk), nk = max(min(cu_k[b + 1], Tk) - kb, 0);
  // keys that query i sees
  auto seen = [&](int i) __attribute__((always_inline)) { return causal ? min(nk - nq + i + 1, nk) : nk; };
  const int w0 = qt + 32 * wave;  // the wave's first query
  const int qi = min(w0 + j, nq - 1);
  int low_j = 0, seen_j = seen(qi);  // the keys low_j .. seen_j - 1 are this query's
  // the tiles of keys, i0 .. nt - 1 of this split's, of them i0_w .. nt_w - 1 the wave's; the keys from full_lo to full_hi
  // are every query's of the wave
  int i0, nt, i0_w = 0, nt_w, full_lo = 0, full_hi;
  if constexpr (MORE) {
    if (more.first) low_j = min(max(more.first[qb + qi], 0), nk);
    if (more.last) seen_j = min(seen_j, more.last[qb + qi]);
    seen_j = max(seen_j, 0);
    const bool some = low_j < seen_j;  // (a query that sees nothing asks for no tile)
    int lo = some ? low_j : 0x7fffffff, hi = some ? seen_j : 0;
    full_lo = low_j, full_hi = seen_j;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
      lo = min(lo, __shfl_xor(lo, m, WAVE)), hi = max(hi, __shfl_xor(hi, m, WAVE));
      full_lo = max(full_lo, __shfl_xor(full_lo, m, WAVE)), full_hi = min(full_hi, __shfl_xor(full_hi, m, WAVE));
    }
    lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
    full_lo = __builtin_amdgcn_readfirstlane(full_lo), full_hi = __builtin_amdgcn_readfirstlane(full_hi);
    i0_w = lo / XA_K, nt_w = w0 < nq ? (hi + XA_K - 1) / XA_K : 0;
    __shared__ int2 span[XA_THREADS / WAVE];
    if (lane == 0) span[wave] = make_int2(lo, hi);
    __syncthreads();
    lo = 0x7fffffff, hi = 0;
#pragma unroll
    for (int w = 0; w < XA_THREADS / WAVE; ++w) lo = min(lo, span[w].x), hi = max(hi, span[w].y);
    lo = __builtin_amdgcn_readfirstlane(lo) / XA_K, hi = (__builtin_amdgcn_readfirstlane(hi) + XA_K - 1) / XA_K;
    const int all = max(hi - lo, 0);
    if (all == 0) lo = hi = 0;
    i0 = lo + (int)((long)all * split / splits), nt = lo + (int)((long)all * (split + 1) / splits);
  } else {
    const int all = (max(seen(min(qt + XA_Q, nq) - 1), 0) + XA_K - 1) / XA_K;
    i0 = (int)((long)all * split / splits), nt = (int)((long)all * (split + 1) / splits);
    nt_w = w0 < nq ? (max(seen(min(w0 + 32, nq) - 1), 0) + XA_K - 1) / XA_K : 0;
    full_hi = seen(w0);
  }

  // Waves 0 to 3, the ones with priority, bring the tiles, once they are through with theirs: the loads' issue would
  // delay the others, for whom they wait anyway (8k tokens, 64 heads, on one card: 1,194 us; all waves before
  // their tile 1,235, after it 1,207). Key and value rows 16 wave .. + 15 in fours, rope rows in eights.
  const bool brings = wave < 4;
  const size_t head_off = (size_t)kb * H * EX_D + (size_t)head * EX_D;
  const uint16_t* const k_base = k + head_off;
  const uint16_t* const v_base = v + head_off;
  const int l4 = lane >> 4, lw = wave & 3;
  const int vcol = 8 * ((lane & 15) ^ (4 * l4));
  const uint32_t k_lds = lds_address(sh.k[0] + 4096 * lw), v_lds = lds_address(sh.v[0] + 4096 * lw);
  const uint32_t r_lds = lds_address(sh.r[0] + 2048 * lw);
  auto issue = [&](int i, int to) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {  // (rows past the end: the last one, of weight 0)
      const size_t t = (size_t)min(i * XA_K + 16 * lw + 4 * x + l4, nk - 1) * H * EX_D;
      load_lds16(k_base + t + 8 * ((lane & 15) ^ (4 * x | l4)), k_lds + XA_K * 256 * to + 1024 * x);
      load_lds16(v_base + t + vcol, v_lds + XA_K * 256 * to + 1024 * x);
    }
    if (DQ > EX_D)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        load_lds16(kr + (size_t)(kb + min(i * XA_K + 16 * lw + 8 * x + (lane >> 3), nk - 1)) * EX_R +
                       8 * ((lane & 7) ^ ((8 * x + (lane >> 3)) >> 1)),
                   r_lds + XA_K * 128 * to + 1024 * x);
  };
  // The tile that comes n-th. With distances the last one comes first: its scores are the largest, so that the maximum hardly
  // moves after it (8,192 tokens, 32 heads 632 us for 675; 2,048 of 10,240 309 for 339).
  auto tile = [&](int n) __attribute__((always_inline)) { return MORE == 2 ? nt - 1 - (n - i0) : n; };
  if (brings && nt > i0) issue(tile(i0), 0);
  // the queries through LDS, over the stages that tiles 1 and 2 take: columns 64 p .. + 63 of the wave's 32 rows are 4
  // KiB of k, v or r, laid out as rope rows. (Read straight into the operands' layout, 32 bytes of 32 rows at a time,
  // they took 5,000 cycles more.)
  bf16x8 qf[STEPS];  // query qi: step s holds dims 16 s + 8 h .. + 7
  {
    uint8_t* const at[3] = {sh.k[1], sh.v[1], sh.r[DQ > EX_D ? 1 : 0]};
#pragma unroll
    for (int p = 0; p < DQ / 64; ++p)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = 8 * x + (lane >> 3);
        load_lds16(q + ((size_t)(qb + min(w0 + r, nq - 1)) * H + head) * DQ + 64 * p + 8 * ((lane & 7) ^ ((r >> 1) & 7)),
                   lds_address(at[p] + 4096 * wave) + 1024 * x);
      }
    wait_loads<0>();
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
      qf[s] = as_bf16x8(*reinterpret_cast<const uint4*>(at[s >> 2] + 4096 * wave + 128 * j +
                                                        16 * ((2 * (s & 3) + h) ^ ((j >> 1) & 7))));
  }
  lds_barrier();  // the queries are read
  if (brings && nt > i0 + 1) issue(tile(i0 + 1), 1);
  int koff[8], roff[4], voff[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) koff[i] = 256 * j + 16 * ((2 * i | h) ^ (j & 15));
#pragma unroll
  for (int i = 0; i < 4; ++i) roff[i] = 128 * j + 16 * ((2 * i | h) ^ ((j >> 1) & 7));
  {  // the value operand: this lane's address is of row 4 h + (lane & 15) / 4, columns 16 (lane / 16 % 2) + 4 (lane % 4)
    const int r = (lane & 15) >> 2, p = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) voff[i] = 256 * (4 * h + r) + 16 * ((4 * i | p) ^ (4 * r)) + 8 * (lane & 1);
  }
  const float sl2 = scale * XA_LOG2E;
  [[maybe_unused]] bool fresh = true;  // (MORE) no key of this query's so far
  [[maybe_unused]] float cap2 = 0.0f, cap_in = 0.0f, slope2 = 0.0f, near_s = -1.0f, near_c[4];
  if constexpr (MORE == 2) {
    if (more.softcap > 0.0f) {
      cap2 = more.softcap * XA_LOG2E, cap_in = 2.0f * XA_LOG2E * scale / more.softcap;
      // tanh(x) / x for |x| <= 1/2 as a polynomial of x^2 (least largest error, 5.5e-7 of it), here of the score's square
      const float by = scale / more.softcap, y = by * by;
      if (fabsf(by) < 1e4f) near_s = fminf(0.5f / fabsf(by), 1e15f);
      near_c[0] = 0.99999946f * sl2, near_c[1] = -0.33326318f * sl2 * y;
      near_c[2] = 0.13190297f * sl2 * y * y, near_c[3] = -0.044402226f * sl2 * y * y * y;
    }
    if (more.slopes) slope2 = more.slopes[head] * XA_LOG2E;
  }
  float m_run = 0.0f, l_run = 0.0f;  // running maximum (base 2), this lane's share of the sum
  f32x16 o[4];                       // dims 32 d + 8 (r / 4) + 4 h + r % 4
#pragma unroll
  for (int d = 0; d < 4; ++d) o[d] = f32x16{};
  if (wave < 4) __builtin_amdgcn_s_setprio(1);
  int stage = 0;
#pragma unroll 1
  for (int n = i0; n < nt; ++n) {
    const int i = tile(n);
    if (brings) {
      if (n + 1 < nt)
        wait_loads<LOADS>();
      else
        wait_loads<0>();
    }
    lds_barrier();  // tile i is in place, and nobody reads the one before any more
    if (i < nt_w && (!MORE || i >= i0_w)) {
      const uint8_t* const kt = sh.k[stage];
      const uint8_t* const vt = sh.v[stage];
      const uint8_t* const rt = sh.r[DQ > EX_D ? stage : 0];
      f32x16 s2[2] = {f32x16{}, f32x16{}};  // scores: tokens 32 x + 8 (r / 4) + 4 h + r % 4
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint8_t* at = s < 8 ? kt + koff[s] + 32 * 256 * x : rt + roff[s & 3] + 32 * 128 * x;
          s2[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(*reinterpret_cast<const uint4*>(at)), qf[s], s2[x],
                                                          0, 0, 0);
        }
      const float from = MORE == 2 ? (float)(nk - nq + qi - i * XA_K - 4 * h) : 0.0f;  // (|p - t| < 2^24: exact)
      if (MORE == 2 && cap2 > 0.0f) {
        float top = fabsf(s2[0][0]);
#pragma unroll
        for (int r = 1; r < 32; ++r) top = max_nonan(top, fabsf(s2[r >> 4][r & 15]));
        // Where the tile's scores are all below half the cap, as most are, no exponential and reciprocal (8,192 tokens,
        // 32 heads: 705 us for 728; scores of up to the cap 745 for 730). The two differ by the cap's 2^-20 at most, so that a
        // query's bits may depend on its wave's other queries.
        if (__ballot(!(top <= near_s)) == 0) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float s = s2[x][r], y = s * s;
              s2[x][r] = fmaf(s, fmaf(y, fmaf(y, fmaf(y, near_c[3], near_c[2]), near_c[1]), near_c[0]), -m_run);
            }
        } else {  // cap tanh(s / cap) = cap - 2 cap / (1 + e^(2 s / cap)), here in base 2
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float e = __builtin_amdgcn_exp2f(s2[x][r] * cap_in);
              s2[x][r] = fmaf(-2.0f * cap2, __builtin_amdgcn_rcpf(1.0f + e), cap2 - m_run);
            }
        }
        if (more.slopes)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s2[x][r] = fmaf(-slope2, fabsf(from - (float)(32 * x + 8 * (r >> 2) + (r & 3))), s2[x][r]);
      } else if (MORE == 2 && more.slopes && (i + 1) * XA_K - 1 <= nk - nq + w0) {
        // No key of the tile is behind a query of the wave: slope (p - t) is the tile's own, less slope times the key's place in
        // it: off by up to 64 slopes' roundings more than of |p - t| alone (8,192 tokens, 32 heads: 692 us for 702 then).
        const float base = fmaf(-slope2, from, -m_run);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s2[x][r] = fmaf(s2[x][r], sl2, fmaf(slope2, (float)(32 * x + 8 * (r >> 2) + (r & 3)), base));
      } else {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) s2[x][r] = fmaf(s2[x][r], sl2, -m_run);
        if (MORE == 2 && more.slopes)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s2[x][r] = fmaf(-slope2, fabsf(from - (float)(32 * x + 8 * (r >> 2) + (r & 3))), s2[x][r]);
      }
      if ((i + 1) * XA_K > full_hi || (MORE && i * XA_K < full_lo)) {  // keys that a query does not see
        const int lim = seen_j - i * XA_K - 4 * h, low = MORE ? low_j - i * XA_K - 4 * h : 0;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int t = 32 * x + 8 * (r >> 2) + (r & 3);
            s2[x][r] = t < lim && (!MORE || t >= low) ? s2[x][r] : -INFINITY;
          }
      }
      float cm = s2[0][0];
#pragma unroll
      for (int r = 1; r < 32; ++r) cm = max_nonan(cm, s2[r >> 4][r & 15]);
      if (MORE ? __ballot(fresh || cm > XA_SLACK) != 0 : i == i0 || __ballot(cm > XA_SLACK) != 0) {
        cm = max_nonan(cm, __shfl_xor(cm, 32, WAVE));
        float up, alpha;
        if (MORE) {  // the maximum starts at a query's first key, and is 0 until then
          const bool none = cm == -INFINITY;
          up = fresh ? none ? 0.0f : cm : cm > XA_SLACK ? cm : 0.0f;
          alpha = fresh ? 0.0f : __builtin_amdgcn_exp2f(-up);
          fresh = fresh && none;
        } else {  // a query that sees none of the first tile sees nothing: its maximum stays finite
          up = i == i0 ? max_nonan(cm, -1e30f) : cm > XA_SLACK ? cm : 0.0f;
          alpha = i == i0 ? 0.0f : __builtin_amdgcn_exp2f(-up);
        }
        m_run += up;
        l_run *= alpha;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) s2[x][r] -= up;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
      }
      // P in bf16 (each weight off by 2^-8 of it at most, as everywhere in this library; the sums take it unrounded)
      uint32_t pk[16];
#pragma unroll
      for (int r = 0; r < 32; r += 4) {
        float pv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) pv[e] = __builtin_amdgcn_exp2f(s2[r >> 4][(r & 15) + e]);
        l_run += (pv[0] + pv[1]) + (pv[2] + pv[3]);
        pk[r / 2] = bf16_pack(pv[0], pv[1]);
        pk[r / 2 + 1] = bf16_pack(pv[2], pv[3]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {  // tokens 16 t .. + 15
        const bf16x8 pb = as_bf16x8(make_uint4(pk[4 * t], pk[4 * t + 1], pk[4 * t + 2], pk[4 * t + 3]));
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const uint8_t* at = vt + voff[d] + 16 * 256 * t;
          typedef __attribute__((address_space(3))) xa_v4s* lds4;
          const xa_v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at);
          const xa_v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 8 * 256));
          typedef short v8s __attribute__((ext_vector_type(8)));
          const v8s both = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, both), pb, o[d], 0, 0, 0);
        }
      }
    }
    if (brings && n + 2 < nt) issue(tile(n + 2), stage == 0 ? 2 : stage - 1);  // (where the one before was)
    stage = stage == XA_STAGES - 1 ? 0 : stage + 1;
  }
  __syncthreads();  // the stages are free
  const float l = l_run + __shfl_xor(l_run, 32, WAVE);
  if (splits > 1) {  // a partial, as the registers hold it (expanded_combine_kernel reads it so)
    if (w0 >= nq) return;
    const size_t part = ((size_t)ti * H + head) * splits + split;
    float* const to = ws + part * XA_Q * EX_D + 32 * EX_D * wave + 4 * lane;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(to + 4 * WAVE * (4 * d + g)) =
            f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    float2* const ml = reinterpret_cast<float2*>(ws + (size_t)grid * splits * XA_Q * EX_D) + part * XA_Q + 32 * wave;
    if (h == 0) ml[j] = make_float2(l > 0.0f ? m_run : -1e30f, l);
    return;
  }
  const float inv = inverse_or_0(l);  // (a query that sees nothing: 0)
  const int rows = min(32, nq - w0);
  if (rows <= 0) return;
  if (lse_out && h == 0 && j < rows)
    lse_out[(size_t)(qb + w0 + j) * H + head] = lse_or_none(m_run, l);
  const size_t at = ((size_t)(qb + w0) * H + head) * EX_D;
  if (out) {  // through LDS (8 KiB a wave): 256 bytes a row, piece p of row r at p ^ (r & 15), then whole rows
    uint8_t* const st = sh.k[0] + 8192 * wave;
    static_assert(offsetof(XaShared<DQ>, r) >= 8 * 8192, "the staged outputs");
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint2*>(st + 256 * j + 16 * ((4 * d + g) ^ (j & 15)) + 8 * h) =
            make_uint2(bf16_pack(o[d][4 * g] * inv, o[d][4 * g + 1] * inv),
                       bf16_pack(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int r = 4 * x + (lane >> 4), p = lane & 15;
      if (r < rows)
        *reinterpret_cast<u32x4*>(out + at + (size_t)r * H * EX_D + 8 * p) =
            *reinterpret_cast<const u32x4*>(st + 256 * r + 16 * (p ^ (r & 15)));
    }
  }
  if (out_f32 && j < rows) {
    float* p = out_f32 + at + (size_t)j * H * EX_D + 4 * h;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(p + 32 * d + 8 * g) = f32x4{o[d][4 * g] * inv, o[d][4 * g + 1] * inv,
                                                              o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv};
  }
}

hipError_t launch_expand_latent(const uint8_t* kv, const float* kvs, const int* table, const int* cu,
                                const uint16_t* w, uint16_t* k, uint16_t* v, uint16_t* r, int B, int total, int H,
                                int D, int max_pages, int page_size, int num_pages, int num_cu, hipStream_t s) {
  auto run = [&](auto kernel, int tok) {
    const int units = (total + tok - 1) / tok * 2 * H;
    return launch("expand_latent_kernel", kernel, dim3(min(units, num_cu)), dim3(EL_THREADS), s, kv, kvs, table, cu, w,
                  k, v, r, B, total, H, D, max_pages, page_size, num_pages, units);
  };
  // tiles of 128 tokens where all their units run at once (16 heads: 1 token 8.1 us with them, 11.0 with tiles of 256;
  // 1,001 tokens 12.1 and 13.7), else of 256, which read the weights half as often (1,500 tokens 17.9 and 15.7; 64
  // heads, 8k tokens 136 and 112)
  return (long)((total + EL_TOK / 2 - 1) / (EL_TOK / 2)) * 2 * H <= num_cu ? run(expand_latent_kernel<1>, EL_TOK / 2)
                                                                           : run(expand_latent_kernel<2>, EL_TOK);
}

// Query tiles that a batch of Tq queries in B sequences may have.
static int attend_tiles(int B, int Tq) { return (int)((Tq + (XA_Q - 1L) * B) / XA_Q); }

bool expanded_grid_ok(int B, int Tq, int H) {
  return ((long)Tq / XA_Q + B) * H <= 0x7fffffL && (long)Tq + B <= 0x7fffffffL - XA_Q;
}

// Joins a query tile's splits: out = sum 2^(m - max) O / sum 2^(m - max) l. A workgroup has a tile of a head, a wave
// its 32 queries, the lanes as the partials hold them.
__global__ __launch_bounds__(XA_THREADS) void expanded_combine_kernel(
    const float* __restrict__ ws, const int* __restrict__ cu_q, uint16_t* __restrict__ out, float* __restrict__ out_f32,
    float* __restrict__ lse_out, int B, int Tq, int H, int q_tiles, int splits) {
  __shared__ int tot[XA_THREADS / WAVE];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int j = lane & 31, h = lane >> 5;
  const int unit = blockIdx.x >> 2, d = blockIdx.x & 3, ti = unit / H, head = unit - ti * H;  // (d: 32 of the 128 dims)
  xa_find(ti, cu_q, B, Tq, tot, found);
  const int b = __builtin_amdgcn_readfirstlane(found[0]);
  if (b < 0) return;
  const int i = __builtin_amdgcn_readfirstlane(found[1]) * XA_Q + 32 * wave + j;  // this lane's query
  if (i >= xa_queries(b, cu_q, Tq)) return;
  const size_t part0 = (size_t)unit * splits;
  const float2* const ml = reinterpret_cast<const float2*>(ws + (size_t)q_tiles * H * splits * XA_Q * EX_D) +
                           part0 * XA_Q + 32 * wave + j;
  const float* const from = ws + part0 * XA_Q * EX_D + 32 * EX_D * wave + 4 * WAVE * 4 * d + 4 * lane;
  float m = -INFINITY, l = 0.0f;
  f32x4 a[4] = {};
  for (int s0 = 0; s0 < splits; s0 += 4) {
    float2 x[4];
    f32x4 v[4][4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      x[s] = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int g = 0; g < 4; ++g) v[s][g] = f32x4{};
      if (s0 + s < splits) {
        x[s] = ml[(size_t)(s0 + s) * XA_Q];
#pragma unroll
        for (int g = 0; g < 4; ++g)
          v[s][g] = *reinterpret_cast<const f32x4*>(from + (size_t)(s0 + s) * XA_Q * EX_D + 4 * WAVE * g);
      }
    }
    float mx = m;
#pragma unroll
    for (int s = 0; s < 4; ++s) mx = max_nonan(mx, x[s].x);
    const float f = __builtin_amdgcn_exp2f(m - mx);
    m = mx;
    l *= f;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) a[g][e] *= f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const float c = __builtin_amdgcn_exp2f(x[s].x - m);
      l = fmaf(c, x[s].y, l);
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) a[g][e] = fmaf(c, v[s][g][e], a[g][e]);
    }
  }
  const float inv = inverse_or_0(l);  // (a query that sees nothing: 0)
  const size_t row = (size_t)(xa_first(b, cu_q, Tq) + i) * H + head;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 v = {a[g][0] * inv, a[g][1] * inv, a[g][2] * inv, a[g][3] * inv};
    const size_t to = row * EX_D + 32 * d + 8 * g + 4 * h;
    if (out) *reinterpret_cast<uint2*>(out + to) = make_uint2(bf16_pack(v[0], v[1]), bf16_pack(v[2], v[3]));
    if (out_f32) *reinterpret_cast<f32x4*>(out_f32 + to) = v;
  }
  if (lse_out && d == 0 && h == 0) lse_out[row] = lse_or_none(m, l);
}

// In how many splits a tile's keys are taken: as many as leave the CUs a workgroup each where every sequence has
// queries (the fewest tiles that they can be), none of fewer than 4 tiles of keys on average. (16 heads: 256 queries of
// 32k keys 839 us unsplit, 103 in 16; 1,000 of 1,000 33 and 29 in 3.)
static int attend_splits(int B, int Tq, int Tk, int H, int num_cu) {
  const long tiles = ((long)Tq + XA_Q - 1) / XA_Q, least = (tiles > B ? tiles : B) * H;
  const long by_cu = num_cu / least, by_keys = (long)Tk / B / (4 * XA_K), n = by_cu < by_keys ? by_cu : by_keys;
  return n < 1 ? 1 : n > XA_SPLITS ? XA_SPLITS : (int)n;
}

size_t expanded_workspace_bytes(int B, int Tq, int Tk, int H, int num_cu) {
  const int splits = attend_splits(B, Tq, Tk, H, num_cu);
  return splits > 1 ? (size_t)attend_tiles(B, Tq) * H * splits * XA_Q * (EX_D + 2) * sizeof(float) : 0;
}

hipError_t launch_expanded_attend(const uint16_t* q, const uint16_t* k, const uint16_t* kr, const uint16_t* v,
                                  const int* cu_q, const int* cu_k, uint16_t* out, float* out_f32, float* lse, void* ws,
                                  int B, int Tq, int Tk, int H, int causal, float scale, const ExpandedMore* more,
                                  int num_cu, hipStream_t s) {
  const int q_tiles = attend_tiles(B, Tq), splits = attend_splits(B, Tq, Tk, H, num_cu);
  const auto kernel = !more ? kr ? expanded_attend_kernel<EX_D + EX_R, 0> : expanded_attend_kernel<EX_D, 0>
                      : more->softcap == 0.0f && !more->slopes
                          ? kr ? expanded_attend_kernel<EX_D + EX_R, 1> : expanded_attend_kernel<EX_D, 1>
                      : kr ? expanded_attend_kernel<EX_D + EX_R, 2>
                           : expanded_attend_kernel<EX_D, 2>;
  const hipError_t e = launch("expanded_attend_kernel", kernel, dim3((unsigned)q_tiles * H * splits), dim3(XA_THREADS), s,
                              q, k, kr, v, cu_q, cu_k, out, out_f32, lse, static_cast<float*>(ws), B, Tq, Tk, H, q_tiles,
                              splits, causal, scale, more ? *more : ExpandedMore{});
  if (e != hipSuccess || splits == 1) return e;
  return launch("expanded_combine_kernel", expanded_combine_kernel, dim3((unsigned)q_tiles * H * 4), dim3(XA_THREADS), s,
                static_cast<const float*>(ws), cu_q, out, out_f32, lse, B, Tq, H, q_tiles, splits);
}

}  // namespace dsa
