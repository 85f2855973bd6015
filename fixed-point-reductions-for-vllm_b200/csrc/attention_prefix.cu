// Paged attention of a batch whose requests share the pages of a long prefix:
// the bits of the unified attention, with the prefix's keys and values read
// and converted once for a tile of rows of all requests instead of once per
// request.
//
// Four launches behind a memset; each but the first may start while the one
// before still runs, and waits for it before it reads its results.
//
//   clear    row maxima, normalisers and PV sums (one memset)
//   scores   suffix: each request's own keys (chunk kernels, from key0 on)
//            prefix: tiles of 16/32/64 rows x 64 keys
//            both fold into one maximum per row (integer atomicMax, exact)
//   pv       prefix: p = exp2(s - max), integer normaliser and PV sums of the
//            tile's key range, added to the row's integer accumulators
//            suffix: the same for the own keys, then X2F, divide, store
//
// Rows are the (token, query head) pairs of one KV head over the whole batch,
// row = token * group + head. Integer sums and maxima do not depend on their
// order, so no split, tile or launch order shows in the result.
//
// Bound: the FMA and integer pipes. Each of the 2 * head_dim products per
// (row, key) is rounded to the 2^-f grid by itself (FFMA2 + IADD3 a pair in
// q.k; FMUL2 + FFMA2 + IADD3 in p.v, whose product is not exact), which a
// tensor core cannot do. (Twice that where values are too large for it, below.) What the shared rows buy is that the other
// instructions go away: a thread holds 8 rows x 2 keys (or 4 dims), so an
// operand from shared memory feeds up to 8 products and the conversion of K
// and V is shared by the 64 rows of the tile.
#include "attention_common.cuh"

namespace fxpr {
namespace attn {
namespace prefix {

constexpr int KT64 = 64;      // keys per tile of both kernels
constexpr int DC = 64;        // dims staged at a time (scores)
constexpr int K_LD = DC + 4;  // fp32 pitch of the staged keys: 16-byte reads of 8 rows cover all banks
constexpr int P_LD = KT64 + 16;
constexpr int RUN = 8;        // PV tiles per int32 accumulation run: 8 * 64 products below 2^22 stay below 2^31

struct Args {
  Params p;
  int num_requests;
  int tokens;
  int64_t num_blocks;
  float* scores;    // [kv head][row tile of this launch][RT][key0]
  int tile0, tiles;
  int key_tiles;    // key0 / KT64
  int64_t units;    // kv heads * tiles * key_tiles, cut into equal slices over the CTAs
  float score_mul;  // scale_log2 * 2^-f (the scaling by 2^-f is exact: one rounding, as in two steps)
  int q_vec;        // q rows are 16-byte aligned
  int page_even;    // keys 2i and 2i + 1 lie on one page
  int k_sb, k_ss, v_sb, v_ss;  // cache strides of a block and a key (elements; the host checks that they fit)
  int later_pass;   // the scores' memory is still read by the pass before
};

// Rows of a tile: token, head, position and the range of keys [low, high) of
// the prefix that the row sees (the causal and window masks and the sequence's
// end as intervals); token -1 and an empty range for rows behind the batch or
// its last sequence.
template <int RT>
struct Rows {
  int tok[RT], head[RT], pos[RT], low[RT], high[RT];
  int all_low, all_high;  // keys that every row of the batch in the tile sees
};
template <int RT>
__device__ __forceinline__ void tile_rows(const Args& a, int tile, int kvh, Rows<RT>& rows) {
  const Params& p = a.p;
  const int t = threadIdx.x;
  __syncthreads();  // the rows of the slice before are not read any more
  if (t < RT) {
    rows.tok[t] = -1;
    rows.head[t] = rows.pos[t] = rows.low[t] = rows.high[t] = 0;
  }
  if (t == 0) {
    rows.all_low = 0;
    rows.all_high = p.key0;
  }
  __syncthreads();
  const int row0 = tile * RT, row1 = min(row0 + RT, a.tokens * p.group);
  const int tok0 = row0 / p.group, tok1 = (row1 + p.group - 1) / p.group;
  for (int r = t; r < a.num_requests; r += THREADS) {
    const int qs = p.qsl[r], qe = p.qsl[r + 1];
    if (qe <= tok0 || qs >= tok1) continue;
    const int seq = p.seq_lens[r], ctx = seq - (qe - qs);
    for (int tok = max(tok0, qs); tok < min(tok1, qe); ++tok) {
      const int off = tok - qs, pos = ctx + off;
      // the reference walks keys to the end of its 64-row query block
      int high = p.causal ? min(seq, ctx + (off / 64 + 1) * 64) : seq;
      if (p.causal) high = min(high, pos + 1);
      high = min(high, p.key0);
      const int low = p.window > 0 ? max(0, pos - p.window + 1) : 0;
      if (high < p.key0) atomicMin(&rows.all_high, high);
      if (low > 0) atomicMax(&rows.all_low, low);
      for (int g = 0; g < p.group; ++g) {
        const int i = tok * p.group + g - row0;
        if (i < 0 || i >= RT) continue;
        rows.tok[i] = tok;
        rows.head[i] = kvh * p.group + g;
        rows.pos[i] = pos;
        rows.low[i] = low;
        rows.high[i] = high;
      }
    }
  }
  __syncthreads();
}

// The base-2 exponential of the unified attention with subnormal results
// flushed to zero: those round to 0 on the grid, and so do their products with
// any finite V.
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> __device__ __forceinline__ float2 pair_of(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}

// Rounding a product x to the 2^-f grid, by how large the products of a block
// can be (max|a| * max|b| * 2^f, strict):
//   fast  below 2^22: one addition of the magic constant
//   wide  below LIMIT: first to multiples of 2^U (a constant 2^U times larger),
//         then the rest, x - h * 2^U, with the constant again; both are exact
//         but for the one rounding at the end, so h * 2^U + l = RNE(x). Three
//         packed operations and two integer additions a pair instead of one
//         and one; sums of h and of l stay in 32 bits.
//   else  the definition's clamp and convert (saturation, infinities, NaN)
// An outlier channel, a request of large queries and grids finer than 2^-18
// leave the fast range, and are common. 64 requests behind 4096 keys, 32 / 8
// heads x 128, bf16, 32 bits, the whole operator (unified attention): ordinary
// values 237 us (283), a 20-fold channel of K 274 us (783), one request's
// queries 20-fold 283 us (523), a 60-fold channel of V 377 us (584), 20
// fraction bits 466 us (848), 24 bits 514 us (1105). 30 bits, where nearly all
// products saturate, 1186 us (1108).
template <int BITS> struct Wide {
  static constexpr int U = BITS == 64 ? 20 : 10;
  static constexpr float LIMIT = BITS == 64 ? 4398046511104.0f : 2147483136.0f;  // 2^42; 2^31 - 2^9: no saturation
  static constexpr float C = BITS == 64 ? 13194139533312.0f : 12884901888.0f;    // 1.5 * 2^(23 + U)
  static constexpr uint32_t CBITS = (uint32_t)(150 + U) << 23 | 0x400000u;
  static constexpr float K = C + kMagic;
};
// h and l of two products x (their sums of bit patterns, biased by CBITS and
// kMagicBits a product). X: x of the pair plus an addend, rounded once.
template <int BITS, typename X> __device__ __forceinline__ void wide_pair(X x, float2 minus, uint32_t& h, uint32_t& l) {
  const float2 r = x(make_float2(Wide<BITS>::C, Wide<BITS>::C));
  const float2 s = x(fma2(r, minus, make_float2(Wide<BITS>::K, Wide<BITS>::K)));
  h += __float_as_uint(r.x) + __float_as_uint(r.y);
  l += __float_as_uint(s.x) + __float_as_uint(s.y);
}

// element offset of key j, on block blk, from its KV head's first key
__device__ __forceinline__ int64_t key_offset(const Params& p, int j, int blk, int sb, int ss) {
  const int slot = p.page_shift >= 0 ? (j & (p.page - 1)) : j % p.page;
  return (int64_t)blk * sb + (int64_t)slot * ss;
}
// physical block of key j of the first request (whose prefix pages are
// everyone's); -1, which reads zeros, for an id outside the cache
__device__ __forceinline__ int block_of(const Args& a, int j) {
  const int b = a.p.bt[a.p.page_shift >= 0 ? (j >> a.p.page_shift) : j / a.p.page];
  return b >= 0 && b < a.num_blocks ? b : -1;
}

// ---------------------------------------------------------------------------
// scores: RT rows x 64 keys per step, a thread RT/8 rows x 2 keys. q stays in
// shared memory as fp32 (pre-scaled by 2^f) for the CTA's keys of the row
// tile; K comes 64 dims at a time through registers, converted once,
// double-buffered. Every CTA takes an equal slice of the (KV head, row tile,
// key tile) units, key tiles innermost.
// ---------------------------------------------------------------------------
template <int D, int RT>
struct ScoresSmem {
  static constexpr int Q_LD = D + 4;
  static constexpr size_t off_k = (size_t)RT * Q_LD * 4;
  static constexpr size_t bytes = off_k + 2ull * KT64 * K_LD * 4;
};
// 2 CTAs per SM and 4 k-steps unrolled: 64 requests behind 4096 keys, 32 / 8
// heads x 128, bf16 (1.07 G products): 86 us, 12.5 T products/s of the 18.4 that
// this tile's inner loop alone reaches. The rest: 26% more instructions, 5% less
// issued while an SM has work, and 11% of the cycles in which one has none
// (start, tail). 3 CTAs 3 us more (the 2048 units do not divide as well), 16
// k-steps 1 us less here but 3 us more with head_dim 64.
constexpr int SCORES_CTAS = 2;
constexpr int SU = 4;
constexpr int BD = 16;  // dims of a block that is rounded one way

template <int D, int RT, int BITS, typename T, bool PL>
__global__ void __launch_bounds__(THREADS, SCORES_CTAS) prefix_scores_kernel(const __grid_constant__ Args a) {
  constexpr int TM = RT / 8, TN = KT64 / 32, NCH = D / DC;
  using SM = ScoresSmem<D, RT>;
  using W = Wide<BITS>;
  using UAcc = typename std::conditional<BITS == 64, unsigned long long, uint32_t>::type;
  constexpr int Q_LD = SM::Q_LD;
  constexpr int LOADS = KT64 * DC / 8 / THREADS;  // 16-byte loads of K per thread and step
  const Params& p = a.p;
  extern __shared__ __align__(16) unsigned char smem[];
  float* q_s = reinterpret_cast<float*>(smem);
  float* k_s = reinterpret_cast<float*>(smem + SM::off_k);
  __shared__ Rows<RT> rows;
  __shared__ uint32_t q_max;

  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const float scale = ldexpf(1.0f, p.frac), inv_scale = ldexpf(1.0f, -p.frac);
  const float2 C2 = make_float2(kMagic, kMagic), MINUS2 = make_float2(-p.one, -p.one);
  // 64 bits: what the tile's dots have beyond their 32-bit sums, once a block
  // was not fast; in local memory (volatile), for it is rarely touched
  volatile unsigned long long rest[BITS == 64 ? TM * TN : 1];
  // K staging: thread t moves 8 dims of key rows t / 8 + 32 * u of a tile
  const int krow = t / (DC / 8), kcol = (t % (DC / 8)) * 8;
  int64_t u0 = a.units * blockIdx.x / gridDim.x;
  const int64_t u1 = a.units * (blockIdx.x + 1) / gridDim.x;
  launch_dependents();
  if (a.later_pass) wait_dependencies();

  while (u0 < u1) {
    const int combo = (int)(u0 / a.key_tiles), kt0 = (int)(u0 % a.key_tiles);
    const int n = (int)min(u1 - u0, (int64_t)(a.key_tiles - kt0));  // key tiles of this row tile
    u0 += n;
    const int kvh = combo / a.tiles, tile = combo % a.tiles;
    if (t == 0) q_max = 0u;
    tile_rows<RT>(a, a.tile0 + tile, kvh, rows);
    {
      uint32_t qo = 0;
      for (int e = t; e < RT * (D / 8); e += THREADS) {
        const int i = e / (D / 8), d = (e % (D / 8)) * 8;
        float v[8];
        const int64_t at = (int64_t)rows.tok[i] * p.q_st + (int64_t)rows.head[i] * p.q_sh + d;
        if (rows.tok[i] < 0) {
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = 0.0f;
        } else if (a.q_vec) {
          const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + at);
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float2 f = p.q_dtype == FXPR_F16 ? pair_of<__half>(ws[x]) : pair_of<__nv_bfloat16>(ws[x]);
            v[2 * x] = f.x;
            v[2 * x + 1] = f.y;
          }
        } else {
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = load_f32(p.q, p.q_dtype, at + x);
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          qo = max(qo, __float_as_uint(v[x]) & 0x7FFFFFFFu);
          v[x] = __fmul_rn(v[x], scale);
        }
        *reinterpret_cast<float4*>(q_s + i * Q_LD + d) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(q_s + i * Q_LD + d + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
      qo = __reduce_max_sync(0xffffffffu, qo);
      if (lane == 0) atomicMax(&q_max, qo);
    }

    const T* khead = reinterpret_cast<const T*>(p.k) + kvh * p.k_sh;
    const int steps = n * NCH;
    int64_t at[LOADS], at_next[LOADS];  // element offsets of this thread's key rows; -1 outside the cache
    auto addresses = [&](int ti, int64_t (&x)[LOADS]) {
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        x[u] = -1;
        if (ti >= n) continue;
        const int j = (kt0 + ti) * KT64 + krow + (THREADS / (DC / 8)) * u, blk = block_of(a, j);
        if (blk >= 0) x[u] = key_offset(p, j, blk, a.k_sb, a.k_ss);
      }
    };
    uint4 raw[LOADS];
    auto load = [&](int it) {
      const int ch = it % NCH;
      if (ch == 0) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) at[u] = at_next[u];
        addresses(it / NCH + 1, at_next);
      }
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        raw[u] = make_uint4(0, 0, 0, 0);
        if (at[u] >= 0) raw[u] = *reinterpret_cast<const uint4*>(khead + kcol + at[u] + ch * DC);
      }
    };
    auto store = [&](int it) -> float {  // returns the largest |k| that this thread staged
      float* dst = k_s + (it & 1) * KT64 * K_LD;
      uint32_t m = 0;
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        absmax_word<T>(m, raw[u].x);
        absmax_word<T>(m, raw[u].y);
        absmax_word<T>(m, raw[u].z);
        absmax_word<T>(m, raw[u].w);
        float* d = dst + (krow + (THREADS / (DC / 8)) * u) * K_LD + kcol;
        const float2 f0 = pair_of<T>(raw[u].x), f1 = pair_of<T>(raw[u].y), f2 = pair_of<T>(raw[u].z), f3 = pair_of<T>(raw[u].w);
        *reinterpret_cast<float4*>(d) = make_float4(f0.x, f0.y, f1.x, f1.y);
        *reinterpret_cast<float4*>(d + 4) = make_float4(f2.x, f2.y, f3.x, f3.y);
      }
      return absmax_value<T>(m);
    };
    addresses(0, at_next);
    load(0);
    const float first = store(0);
    if (steps > 1) load(1);
    __syncthreads();
    // max|q| * max|k| * 2^f < 2^22 over the tile's rows and a step's keys: the fast rounding
    const double scale_d = ldexp(1.0, p.frac), mq = (double)__uint_as_float(q_max);
    const float kthr = mq * scale_d < 3.0e38 ? __double2float_rd(4194304.0 / (mq * scale_d)) : 0.0f;
    bool large = __syncthreads_or(!(first < kthr));  // of the step to come, uniform over the CTA

    float rmax[TM];
    uint32_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) rmax[i] = -INFINITY;
    float* out = a.scores + (((int64_t)kvh * a.tiles + tile) * RT + warp * TM) * p.key0 + kt0 * KT64 + lane;

    bool high = false;  // 64 bits: the tile's dots have a part in `rest` (uniform over the warp)
    for (int it = 0; it < steps; ++it) {
      const int ti = it / NCH, ch = it % NCH;
      if (ch == 0) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = 0u - (uint32_t)D * (uint32_t)kMagicBits;
        high = false;
      }
      const float* qb = q_s + warp * TM * Q_LD + ch * DC;
      const float* kb_s = k_s + (it & 1) * KT64 * K_LD + lane * K_LD;
      auto fast4 = [&](int kk) {  // dims kk .. kk + 3
        float4 kv[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) kv[j] = *reinterpret_cast<const float4*>(kb_s + j * 32 * K_LD + kk);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const float4 qv = *reinterpret_cast<const float4*>(qb + i * Q_LD + kk);
          const float2 q0 = make_float2(qv.x, qv.y), q1 = make_float2(qv.z, qv.w);
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const float2 r0 = fma2(q0, make_float2(kv[j].x, kv[j].y), C2);
            const float2 r1 = fma2(q1, make_float2(kv[j].z, kv[j].w), C2);
            acc[i][j] += __float_as_uint(r0.x) + __float_as_uint(r0.y);
            acc[i][j] += __float_as_uint(r1.x) + __float_as_uint(r1.y);
          }
        }
      };
      if (!large) {
#pragma unroll SU
        for (int kk = 0; kk < DC; kk += 4) fast4(kk);
      } else {
        // by blocks of BD dims and the warp's own rows, so that an outlier
        // channel, or a request of large queries, costs its own blocks only
#pragma unroll 1
        for (int b = 0; b < DC; b += BD) {
          uint32_t qm = 0, km = 0;
          auto amax = [](uint32_t& m, const float* src) {
            const uint4 v = *reinterpret_cast<const uint4*>(src);
            m = max(m, max(max(v.x & 0x7FFFFFFFu, v.y & 0x7FFFFFFFu), max(v.z & 0x7FFFFFFFu, v.w & 0x7FFFFFFFu)));
          };
          if (lane < TM * (BD / 4)) amax(qm, qb + lane / (BD / 4) * Q_LD + b + lane % (BD / 4) * 4);
#pragma unroll
          for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int kk = 0; kk < BD; kk += 4) amax(km, kb_s + j * 32 * K_LD + b + kk);
          // q is scaled by 2^f; NaN, and infinity times zero, fail both comparisons
          const float bound = __fmul_ru(__uint_as_float(__reduce_max_sync(0xffffffffu, qm)),
                                        __uint_as_float(__reduce_max_sync(0xffffffffu, km)));
          if (bound < 4194304.0f) {
#pragma unroll 1
            for (int kk = b; kk < b + BD; kk += 4) fast4(kk);
            continue;
          }
          auto beyond = [&](int i, int j, unsigned long long v) {  // 64 bits: the part that acc does not hold
            rest[i * TN + j] = high ? rest[i * TN + j] + v : v;
          };
          if (bound < W::LIMIT) {
            uint32_t h[TM][TN];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int j = 0; j < TN; ++j) h[i][j] = 0u - (uint32_t)BD * W::CBITS;
#pragma unroll 1
            for (int kk = b; kk < b + BD; kk += 4) {
              float4 kv[TN];
#pragma unroll
              for (int j = 0; j < TN; ++j) kv[j] = *reinterpret_cast<const float4*>(kb_s + j * 32 * K_LD + kk);
#pragma unroll
              for (int i = 0; i < TM; ++i) {
                const float4 qv = *reinterpret_cast<const float4*>(qb + i * Q_LD + kk);
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                  wide_pair<BITS>([&](float2 c) { return fma2(make_float2(qv.x, qv.y), make_float2(kv[j].x, kv[j].y), c); },
                                  MINUS2, h[i][j], acc[i][j]);
                  wide_pair<BITS>([&](float2 c) { return fma2(make_float2(qv.z, qv.w), make_float2(kv[j].z, kv[j].w), c); },
                                  MINUS2, h[i][j], acc[i][j]);
                }
              }
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int j = 0; j < TN; ++j) {
                if constexpr (BITS == 64) beyond(i, j, (unsigned long long)(long long)(int32_t)h[i][j] << W::U);
                else acc[i][j] += h[i][j] << W::U;
              }
          } else {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
              UAcc s[TN] = {};
#pragma unroll 1
              for (int kk = b; kk < b + BD; kk += 4) {
                float kv[TN][4];
#pragma unroll
                for (int j = 0; j < TN; ++j)
                  *reinterpret_cast<float4*>(kv[j]) = *reinterpret_cast<const float4*>(kb_s + j * 32 * K_LD + kk);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float x = qb[i * Q_LD + kk + e];
                  float qv = __fmul_rn(x, inv_scale);  // q again, unless its scaling left the fp32 range
                  if (fabsf(x) == INFINITY) {
                    const int r = warp * TM + i;
                    qv = load_f32(p.q, p.q_dtype, (int64_t)rows.tok[r] * p.q_st + (int64_t)rows.head[r] * p.q_sh + ch * DC + kk + e);
                  }
#pragma unroll
                  for (int j = 0; j < TN; ++j) s[j] += (UAcc)f2x_f32<BITS>(__fmul_rn(qv, kv[j][e]), scale);
                }
              }
#pragma unroll
              for (int j = 0; j < TN; ++j) {
                acc[i][j] += (uint32_t)BD * (uint32_t)kMagicBits;
                if constexpr (BITS == 64) beyond(i, j, s[j]);
                else acc[i][j] += s[j];
              }
            }
          }
          if constexpr (BITS == 64) high = true;
        }
      }
      if (ch == NCH - 1) {  // the tile's dots are complete: scores, row maxima
        if (BITS == 64 && high) {
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)  // kept as its fp32 value
              acc[i][j] = __float_as_uint(__ll2float_rn((long long)(int32_t)acc[i][j] + (long long)rest[i * TN + j]));
        }
        const bool ints = !(BITS == 64 && high);
        float* dst = out + ti * KT64;
        const int key0 = (kt0 + ti) * KT64;
        if (PL && ints && key0 >= rows.all_low && key0 + KT64 <= rows.all_high) {  // the usual tile: every row sees every key
#pragma unroll
          for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < TN; ++j) {
              const float s = __fmul_rn(__int2float_rn((int32_t)acc[i][j]), a.score_mul);
              dst[32 * j] = s;
              rmax[i] = fmaxf(rmax[i], s);
            }
            dst += p.key0;
          }
        } else {
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            const int r = warp * TM + i, low = rows.low[r], high = rows.high[r];
#pragma unroll
            for (int j = 0; j < TN; ++j) {
              const int key = key0 + lane + 32 * j;
              float qk = __fmul_rn(ints ? __int2float_rn((int32_t)acc[i][j]) : __uint_as_float(acc[i][j]), a.score_mul);
              if constexpr (!PL) {
                if (p.softcap_log2 > 0.0f) qk = __fmul_rn(p.softcap_log2, prim_tanh(__fmul_rn(qk, p.softcap_rcp)));
                if (p.alibi) qk = __fmaf_rn(p.alibi[rows.head[r]], __fsub_rn((float)key, (float)rows.pos[r]), qk);
              }
              const float s = key >= low && key < high ? qk : -INFINITY;
              dst[32 * j] = s;
              rmax[i] = fmaxf(rmax[i], s);
            }
            dst += p.key0;
          }
        }
      }
      float staged = 0.0f;
      if (it + 1 < steps) staged = store(it + 1);
      if (it + 2 < steps) load(it + 2);
      large = __syncthreads_or(!(staged < kthr) && it + 1 < steps);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, ordered(rmax[i]));
      const int r = warp * TM + i;
      if (lane == 0 && rows.tok[r] >= 0) atomicMax(&p.row_max[(int64_t)rows.tok[r] * p.num_heads + rows.head[r]], m);
    }
  }
  wait_dependencies();  // complete only after the suffix scores: who waits for this kernel has both
}

// ---------------------------------------------------------------------------
// pv: RT rows x D dims, 64 keys per step; a thread TM rows x 4 dims. V is
// staged as fp32 pairs of neighbouring keys (after the reference's cast to
// fp16), so that one packed multiply takes two keys of a row and one IADD3
// adds both; a pair's 16-byte pieces are rotated by their dim group, which
// keeps both the staging writes and the reads free of bank conflicts.
// ---------------------------------------------------------------------------
template <int D, int RT>
struct PvSmem {
  static constexpr size_t v_buf = (size_t)KT64 * D * 4;
  static constexpr size_t p_buf = (size_t)RT * P_LD * 4;
  static constexpr size_t off_p = 2 * v_buf;
  static constexpr size_t bytes = off_p + 2 * p_buf;
};
// At the sizes above 125 us, 8.6 T products/s of the 12.5 of the inner loop
// alone (21% more instructions, 4% less issued, 14% of the cycles without work);
// 16 k-steps unrolled 8 us more.
constexpr int VU_UNROLL = 4;

template <int D, int RT, int BITS, typename T>
__global__ void __launch_bounds__(THREADS, 2) prefix_pv_kernel(const __grid_constant__ Args a) {
  using UAcc = typename std::conditional<BITS == 64, unsigned long long, uint32_t>::type;
  constexpr int LD = D / 4;              // lanes across the dims
  constexpr int GROUPS = THREADS / LD;   // row groups
  constexpr int TM = RT / GROUPS;
  constexpr int TPR = THREADS / RT;      // threads per row in the p phase
  constexpr int SV = KT64 / 4 / TPR;     // 16-byte score loads per thread
  constexpr int VU = (KT64 / 2) * (D / 8) / THREADS;  // (key pair, 8 dims) units per thread
  static_assert(TM >= 1 && SV >= 1 && VU >= 1, "tile mapping");
  using SM = PvSmem<D, RT>;
  using W = Wide<BITS>;
  const Params& p = a.p;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Rows<RT> rows;
  __shared__ uint32_t v_max[3];

  const int t = threadIdx.x, lane = t & 31;
  const float scale = ldexpf(1.0f, p.frac);
  // max|v| <= 65504 (finite after the cast) and max|v| * (1 + 2^-10) * 2^f < 2^22, with p <= 1
  const double scale_d = ldexp(1.0, p.frac);
  const float vthr = __double2float_rd(fmin(65504.5, 4194304.0 / (scale_d * (1.0 + 1.0 / 1024))));
  const float2 C2 = make_float2(kMagic, kMagic), ONE2 = make_float2(p.one, p.one), MINUS2 = make_float2(-p.one, -p.one);
  const bool small_frac = p.frac <= 22;  // p * 2^f <= 2^22: the magic constant rounds it
  const int prow = t / TPR;             // p phase: this row, keys 4 * (t % TPR) + 4 * TPR * u
  const int dl = t % LD, grp = t / LD;  // this thread's dims 4 * dl.., rows grp * TM..
  const int vc = dl / 2, vj = (dl & 1) * 2, vx = (vc >> 1) & 3;
  const int v0 = (vc * 4 + (vj ^ vx)) * 16, v1 = (vc * 4 + ((vj + 1) ^ vx)) * 16;
  int64_t u0 = a.units * blockIdx.x / gridDim.x;
  const int64_t u1 = a.units * (blockIdx.x + 1) / gridDim.x;
  bool waited = false;
  launch_dependents();

  while (u0 < u1) {
    const int combo = (int)(u0 / a.key_tiles), kt0 = (int)(u0 % a.key_tiles);
    const int n = (int)min(u1 - u0, (int64_t)(a.key_tiles - kt0));
    u0 += n;
    const int kvh = combo / a.tiles, tile = combo % a.tiles;
    if (t < 3) v_max[t] = 0u;
    tile_rows<RT>(a, a.tile0 + tile, kvh, rows);
    const bool live = rows.tok[prow] >= 0;
    const int64_t row_id = live ? (int64_t)rows.tok[prow] * p.num_heads + rows.head[prow] : 0;
    float m = 0.0f;
    const float* src = a.scores + (((int64_t)kvh * a.tiles + tile) * RT + prow) * p.key0 + kt0 * KT64 + 4 * (t % TPR);
    UAcc den = 0;

    const T* vhead = reinterpret_cast<const T*>(p.v) + kvh * p.v_sh;
    float4 sc[SV];
    uint4 va[VU], vb[VU];
    int64_t at_a[VU], at_b[VU];  // element offsets of the next tile's key pairs; -1 outside the cache
    auto addresses = [&](int ti) {
#pragma unroll
      for (int u = 0; u < VU; ++u) {
        at_a[u] = at_b[u] = -1;
        if (ti >= n) continue;
        const int unit = t + u * THREADS, j = (kt0 + ti) * KT64 + 2 * (unit / (D / 8)), d = (unit % (D / 8)) * 8;
        const int ba = block_of(a, j);
        if (ba >= 0) at_a[u] = key_offset(p, j, ba, a.v_sb, a.v_ss) + d;
        if (a.page_even) {
          if (ba >= 0) at_b[u] = at_a[u] + a.v_ss;
        } else {
          const int bb = block_of(a, j + 1);
          if (bb >= 0) at_b[u] = key_offset(p, j + 1, bb, a.v_sb, a.v_ss) + d;
        }
      }
    };
    auto load_scores = [&](int ti) {
#pragma unroll
      for (int u = 0; u < SV; ++u) sc[u] = *reinterpret_cast<const float4*>(src + ti * KT64 + 4 * TPR * u);
    };
    auto load_v = [&](int ti) {
#pragma unroll
      for (int u = 0; u < VU; ++u) {
        va[u] = vb[u] = make_uint4(0, 0, 0, 0);
        if (at_a[u] >= 0) va[u] = *reinterpret_cast<const uint4*>(vhead + at_a[u]);
        if (at_b[u] >= 0) vb[u] = *reinterpret_cast<const uint4*>(vhead + at_b[u]);
      }
      addresses(ti + 1);
    };
    auto store = [&](int ti) {
      float* pd = reinterpret_cast<float*>(smem + SM::off_p + (ti & 1) * SM::p_buf) + prow * P_LD + 4 * (t % TPR);
#pragma unroll
      for (int u = 0; u < SV; ++u) {
        const float s[4] = {sc[u].x, sc[u].y, sc[u].z, sc[u].w};
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // a masked key (-inf) is -0: no contribution, whatever its V holds
          const float x = s[e] == -INFINITY ? -0.0f : exp2_ftz(__fsub_rn(s[e], m));
          v[e] = __fmul_rn(x, scale);
          if (small_frac) {
            den += (UAcc)(__float_as_uint(__fadd_rn(v[e], kMagic)) - (uint32_t)kMagicBits);
          } else {
            den += (UAcc)f2x_scaled<BITS>(v[e]);
          }
        }
        *reinterpret_cast<float4*>(pd + 4 * TPR * u) = make_float4(v[0], v[1], v[2], v[3]);
      }
      unsigned char* vd = smem + (ti & 1) * SM::v_buf;
      uint32_t mx = 0;
#pragma unroll
      for (int u = 0; u < VU; ++u) {
        const int unit = t + u * THREADS, kp = unit / (D / 8), c = unit % (D / 8);
        const uint32_t wa[4] = {va[u].x, va[u].y, va[u].z, va[u].w}, wb[4] = {vb[u].x, vb[u].y, vb[u].z, vb[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          absmax_word<T>(mx, wa[e]);
          absmax_word<T>(mx, wb[e]);
          const float2 fa = v_pair_f16<T>(reinterpret_cast<const unsigned char*>(&wa[e]));
          const float2 fb = v_pair_f16<T>(reinterpret_cast<const unsigned char*>(&wb[e]));
          *reinterpret_cast<float4*>(vd + ((size_t)kp * (D / 2) + c * 4 + (e ^ ((c >> 1) & 3))) * 16) =
              make_float4(fa.x, fb.x, fa.y, fb.y);
        }
      }
      const uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(absmax_value<T>(mx)));
      if (lane == 0) atomicMax(&v_max[ti % 3], b);
    };

    uint32_t acc[TM][4];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0u;
    uint32_t bias = 0;  // of the tiles since the last flush
    auto flush = [&]() {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int r = grp * TM + i;
        if (rows.tok[r] < 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][e] = 0u;
          continue;
        }
        unsigned long long* dst = p.row_acc + ((int64_t)rows.tok[r] * p.num_heads + rows.head[r]) * D + 4 * dl;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t s = acc[i][e] - bias;
          const unsigned long long v = BITS == 64 ? (unsigned long long)(long long)(int32_t)s : (unsigned long long)s;
          if (v) atomicAdd(dst + e, v);
          acc[i][e] = 0u;
        }
      }
      bias = 0u;
    };

    addresses(0);
    load_v(0);
    if (!waited) wait_dependencies();  // the scores and maxima are those of launches that may still run
    waited = true;
    load_scores(0);
    if (live) m = from_ordered(p.row_max[row_id]);
    store(0);
    if (n > 1) {
      load_scores(1);
      load_v(1);
    }
    __syncthreads();
    for (int ti = 0; ti < n; ++ti) {
      const float vm = __uint_as_float(v_max[ti % 3]);  // uniform over the CTA
      if (t == 0) v_max[(ti + 2) % 3] = 0u;
      const float* pb = reinterpret_cast<const float*>(smem + SM::off_p + (ti & 1) * SM::p_buf) + grp * TM * P_LD;
      const unsigned char* vs = smem + (ti & 1) * SM::v_buf;
      if (vm < vthr) {
#pragma unroll VU_UNROLL
        for (int k = 0; k < KT64; k += 4) {
          float4 w[2][2];  // pairs k/2 and k/2 + 1, dims (0, 1) and (2, 3)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            w[h][0] = *reinterpret_cast<const float4*>(vs + (size_t)(k / 2 + h) * D * 8 + v0);
            w[h][1] = *reinterpret_cast<const float4*>(vs + (size_t)(k / 2 + h) * D * 8 + v1);
          }
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            const float4 pv = *reinterpret_cast<const float4*>(pb + i * P_LD + k);
            const float2 pp[2] = {make_float2(pv.x, pv.y), make_float2(pv.z, pv.w)};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 r0 = fma2(mul2(pp[h], make_float2(w[h][e].x, w[h][e].y)), ONE2, C2);
                const float2 r1 = fma2(mul2(pp[h], make_float2(w[h][e].z, w[h][e].w)), ONE2, C2);
                acc[i][2 * e] += __float_as_uint(r0.x) + __float_as_uint(r0.y);
                acc[i][2 * e + 1] += __float_as_uint(r1.x) + __float_as_uint(r1.y);
              }
          }
        }
        bias += (uint32_t)KT64 * (uint32_t)kMagicBits;
      } else if (vm < __double2float_rd(fmin(65504.5, (double)W::LIMIT / (scale_d * (1.0 + 1.0 / 1024))))) {
        // 32 bits: h * 2^U + l into the sums. 64 bits: l into the sums, h (zero
        // for most) to the row's accumulators, RW rows at a time.
        constexpr int RW = BITS == 32 ? TM : TM < 2 ? 1 : 2;
#pragma unroll
        for (int ig = 0; ig < TM; ig += RW) {
          uint32_t h[RW][4];
#pragma unroll
          for (int i = 0; i < RW; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) h[i][e] = 0u;
#pragma unroll 1
          for (int k = 0; k < KT64; k += 2) {
            const float4 w[2] = {*reinterpret_cast<const float4*>(vs + (size_t)(k / 2) * D * 8 + v0),
                                 *reinterpret_cast<const float4*>(vs + (size_t)(k / 2) * D * 8 + v1)};
#pragma unroll
            for (int i = 0; i < RW; ++i) {
              const float2 pp = *reinterpret_cast<const float2*>(pb + (ig + i) * P_LD + k);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 v = w[e / 2];
                const float2 x = mul2(pp, e % 2 ? make_float2(v.z, v.w) : make_float2(v.x, v.y));
                uint32_t hs = 0;
                wide_pair<BITS>([&](float2 c) { return fma2(x, ONE2, c); }, MINUS2, hs, acc[ig + i][e]);
                if constexpr (BITS == 32) acc[i][e] += hs << W::U;
                else h[i][e] += hs;
              }
            }
          }
          if constexpr (BITS == 64) {
#pragma unroll
            for (int i = 0; i < RW; ++i) {
              const int r = grp * TM + ig + i;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int32_t hv = (int32_t)(h[i][e] - (uint32_t)KT64 * W::CBITS);
                if (hv && rows.tok[r] >= 0)
                  atomicAdd(p.row_acc + ((int64_t)rows.tok[r] * p.num_heads + rows.head[r]) * D + 4 * dl + e,
                            (unsigned long long)(long long)hv << W::U);
              }
            }
          }
        }
        bias += (uint32_t)KT64 * ((uint32_t)kMagicBits + (BITS == 32 ? W::CBITS << W::U : 0u));
      } else {  // the definition's clamp and convert
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int r = grp * TM + i;
          UAcc s[4] = {};
#pragma unroll 1
          for (int k = 0; k < KT64; k += 2) {
            const float2 pp = *reinterpret_cast<const float2*>(pb + i * P_LD + k);
            const float4 va4 = *reinterpret_cast<const float4*>(vs + (size_t)(k / 2) * D * 8 + v0);
            const float4 vb4 = *reinterpret_cast<const float4*>(vs + (size_t)(k / 2) * D * 8 + v1);
            if (__float_as_uint(pp.x) != 0x80000000u) {  // not masked
              s[0] += (UAcc)f2x_scaled<BITS>(__fmul_rn(pp.x, va4.x));
              s[1] += (UAcc)f2x_scaled<BITS>(__fmul_rn(pp.x, va4.z));
              s[2] += (UAcc)f2x_scaled<BITS>(__fmul_rn(pp.x, vb4.x));
              s[3] += (UAcc)f2x_scaled<BITS>(__fmul_rn(pp.x, vb4.z));
            }
            if (__float_as_uint(pp.y) != 0x80000000u) {
              s[0] += (UAcc)f2x_scaled<BITS>(__fmul_rn(pp.y, va4.y));
              s[1] += (UAcc)f2x_scaled<BITS>(__fmul_rn(pp.y, va4.w));
              s[2] += (UAcc)f2x_scaled<BITS>(__fmul_rn(pp.y, vb4.y));
              s[3] += (UAcc)f2x_scaled<BITS>(__fmul_rn(pp.y, vb4.w));
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (BITS == 32) {
              acc[i][e] += s[e];
            } else if (s[e] && rows.tok[r] >= 0) {
              atomicAdd(p.row_acc + ((int64_t)rows.tok[r] * p.num_heads + rows.head[r]) * D + 4 * dl + e, s[e]);
            }
          }
        }
      }
      if (BITS == 64 && (ti + 1) % RUN == 0) {
        flush();
      }
      if (ti + 1 < n) store(ti + 1);
      if (ti + 2 < n) {
        load_scores(ti + 2);
        load_v(ti + 2);
      }
      __syncthreads();
    }
    flush();
#pragma unroll
    for (int o = 1; o < TPR; o <<= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
    if (t % TPR == 0 && live && den) atomicAdd(p.row_den + row_id, (unsigned long long)den);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int configure(const void* k, size_t smem, bool* done) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && done[dev]) return FXPR_OK;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    set_error("shared_prefix_attention_fxp: cannot configure shared memory");
    return FXPR_ERR_CUDA;
  }
  if (dev >= 0 && dev < 64) done[dev] = true;
  return FXPR_OK;
}

template <int D, int RT, int BITS, typename T>
static int launch(Args& a, bool pv, int kv_heads, cudaStream_t st) {
  const bool plain = !(a.p.softcap_log2 > 0.0f) && a.p.alibi == nullptr && a.p.window <= 0;
  a.key_tiles = a.p.key0 / KT64;
  a.units = (int64_t)kv_heads * a.tiles * a.key_tiles;
  const int64_t resident = (int64_t)num_sms() * (pv ? 2 : SCORES_CTAS);
  const unsigned grid = (unsigned)(a.units < resident ? a.units : resident);
  if (pv) {
    static bool done[64] = {false};
    auto k = prefix_pv_kernel<D, RT, BITS, T>;
    const int rc = configure((const void*)k, PvSmem<D, RT>::bytes, done);
    if (rc != FXPR_OK) return rc;
    return launch_overlapped(k, dim3(grid), PvSmem<D, RT>::bytes, st, a, "fxpr_shared_prefix_attention_fxp (prefix pv)");
  }
  static bool done[2][64] = {{false}};
  auto k = plain ? prefix_scores_kernel<D, RT, BITS, T, true> : prefix_scores_kernel<D, RT, BITS, T, false>;
  const int rc = configure((const void*)k, ScoresSmem<D, RT>::bytes, done[plain ? 1 : 0]);
  if (rc != FXPR_OK) return rc;
  return launch_overlapped(k, dim3(grid), ScoresSmem<D, RT>::bytes, st, a, "fxpr_shared_prefix_attention_fxp (prefix scores)");
}

template <int D, int RT>
static int pick(Args& a, bool pv, int bits, int kv_dtype, int kv_heads, cudaStream_t st) {
  if (kv_dtype == FXPR_F16)
    return bits == 64 ? launch<D, RT, 64, __half>(a, pv, kv_heads, st) : launch<D, RT, 32, __half>(a, pv, kv_heads, st);
  return bits == 64 ? launch<D, RT, 64, __nv_bfloat16>(a, pv, kv_heads, st)
                    : launch<D, RT, 32, __nv_bfloat16>(a, pv, kv_heads, st);
}

template <int D>
static int pick_rows(Args& a, bool pv, int row_tile, int bits, int kv_dtype, int kv_heads, cudaStream_t st) {
  if (row_tile == 16) return pick<D, 16>(a, pv, bits, kv_dtype, kv_heads, st);
  if (row_tile == 32) return pick<D, 32>(a, pv, bits, kv_dtype, kv_heads, st);
  return pick<D, 64>(a, pv, bits, kv_dtype, kv_heads, st);
}

}  // namespace prefix

int launch_prefix(const Params& p, bool pv, int D, int row_tile, int bits, int kv_dtype, int num_requests,
                  int64_t num_blocks, int64_t tokens, float* scores, int tile0, int tiles, cudaStream_t st) {
  prefix::Args a = {};
  a.p = p;
  a.num_requests = num_requests;
  a.tokens = (int)tokens;
  a.num_blocks = num_blocks;
  a.scores = scores;
  a.tile0 = tile0;
  a.tiles = tiles;
  a.score_mul = ldexpf(p.scale_log2, -p.frac);
  a.k_sb = (int)p.k_sb;
  a.k_ss = (int)p.k_ss;
  a.v_sb = (int)p.v_sb;
  a.v_ss = (int)p.v_ss;
  a.page_even = p.page % 2 == 0;
  a.later_pass = tile0 > 0;
  a.q_vec = (uintptr_t)p.q % 16 == 0 && p.q_st % 8 == 0 && p.q_sh % 8 == 0;
  if (D == 64) return prefix::pick_rows<64>(a, pv, row_tile, bits, kv_dtype, p.num_kv_heads, st);
  return prefix::pick_rows<128>(a, pv, row_tile, bits, kv_dtype, p.num_kv_heads, st);
}

}  // namespace attn
}  // namespace fxpr
