// Paged attention of a batch whose requests share the pages of a long prefix:
// the bits of the unified attention, with the prefix's keys and values read
// and converted once for a tile of rows of all requests instead of once per
// request.
//
//   clear    row maxima, normalisers and PV sums (one memset)
//   scores   suffix: each request's own keys (chunk kernels, from key0 on)
//            prefix: tiles of 16/32/64 rows x 128 keys
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
// tensor core cannot do. What the shared rows buy is that the other
// instructions go away: a thread holds 8 rows x 4 keys (or dims), so an
// operand from shared memory feeds 4 or 8 products and the conversion of K
// and V is shared by the 64 rows of the tile.
#include "attention_common.cuh"

namespace fxpr {
namespace attn {
namespace prefix {

constexpr int KQ = 128;       // keys per tile of the scores kernel
constexpr int DC = 32;        // dims staged at a time
constexpr int K_LD = DC + 4;  // fp32 pitch of the staged keys: 16-byte reads of 8 rows cover all banks
constexpr int KP = 64;        // keys per tile of the PV kernel
constexpr int P_LD = KP + 16;
constexpr int RUN = 8;        // PV tiles per int32 accumulation run: 8 * 64 products below 2^22 stay below 2^31

struct Args {
  Params p;
  int num_requests;
  int64_t tokens, num_blocks;
  float* scores;   // [kv head][row tile of this launch][RT][key0]
  int tile0, tiles;
  int keys_per_cta;
};

// Rows of a tile: token, head, position and key limit (as unit_rows of the
// chunk kernels); token -1 for rows behind the batch or its last sequence.
template <int RT>
__device__ __forceinline__ void tile_rows(const Args& a, int tile, int kvh, int* tok_s, int* head_s, int* pos_s,
                                          int* kend_s) {
  const Params& p = a.p;
  const int t = threadIdx.x;
  if (t < RT) tok_s[t] = -1, pos_s[t] = 0, kend_s[t] = 0, head_s[t] = 0;
  __syncthreads();
  const int64_t row0 = (int64_t)tile * RT;
  const int64_t tok0 = row0 / p.group, tok1 = min(a.tokens, (row0 + RT - 1) / p.group + 1);
  for (int r = t; r < a.num_requests; r += THREADS) {
    const int qs = p.qsl[r], qe = p.qsl[r + 1];
    if (qe <= tok0 || qs >= tok1) continue;
    const int seq = p.seq_lens[r], ctx = seq - (qe - qs);
    for (int64_t row = max(row0, (int64_t)qs * p.group); row < min(row0 + RT, min((int64_t)qe, a.tokens) * p.group); ++row) {
      const int i = (int)(row - row0), tok = (int)(row / p.group), off = tok - qs;
      tok_s[i] = tok;
      head_s[i] = kvh * p.group + (int)(row % p.group);
      pos_s[i] = ctx + off;
      kend_s[i] = p.causal ? min(seq, ctx + (off / 64 + 1) * 64) : seq;
    }
  }
  __syncthreads();
}

template <typename T> __device__ __forceinline__ float2 pair_of(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}

__device__ __forceinline__ int64_t key_offset(const Params& p, int j, int blk, int64_t sb, int64_t ss, int64_t sh,
                                              int kvh) {
  const int slot = p.page_shift >= 0 ? (j & (p.page - 1)) : j % p.page;
  return (int64_t)blk * sb + (int64_t)slot * ss + (int64_t)kvh * sh;
}
// physical block of key j of the first request (whose prefix pages are
// everyone's); -1, which reads zeros, for an id outside the cache
__device__ __forceinline__ int block_of(const Args& a, int j) {
  const int b = a.p.bt[a.p.page_shift >= 0 ? (j >> a.p.page_shift) : j / a.p.page];
  return b >= 0 && b < a.num_blocks ? b : -1;
}

// ---------------------------------------------------------------------------
// scores: RT rows x 128 keys per step, a thread RT/8 rows x 4 keys. q stays in
// shared memory as fp32 (pre-scaled by 2^f) for the CTA's whole key range; K
// comes 32 dims at a time through registers, converted once, double-buffered.
// ---------------------------------------------------------------------------
template <int D, int RT>
struct ScoresSmem {
  static constexpr int Q_LD = D + 4;
  static constexpr size_t off_k = (size_t)RT * Q_LD * 4;
  static constexpr size_t bytes = off_k + 2ull * KQ * K_LD * 4;
};

template <int D, int RT, int BITS, typename T, bool PL>
__global__ void __launch_bounds__(THREADS, 2) prefix_scores_kernel(const __grid_constant__ Args a) {
  constexpr int TM = RT / 8, TN = KQ / 32, NCH = D / DC;
  static_assert(NCH >= 2, "a barrier lies between the reset of a tile's maximum and its next use");
  constexpr int Q_LD = ScoresSmem<D, RT>::Q_LD;
  const Params& p = a.p;
  extern __shared__ __align__(16) unsigned char smem[];
  float* q_s = reinterpret_cast<float*>(smem);
  float* k_s = reinterpret_cast<float*>(smem + ScoresSmem<D, RT>::off_k);
  __shared__ int tok_s[RT], head_s[RT], pos_s[RT], kend_s[RT];
  __shared__ uint32_t q_max, k_max[2];

  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int tile = a.tile0 + blockIdx.y, kvh = blockIdx.z;
  const int kb = blockIdx.x * a.keys_per_cta, ke = min(kb + a.keys_per_cta, p.key0);
  if (t == 0) q_max = k_max[0] = k_max[1] = 0u;
  tile_rows<RT>(a, tile, kvh, tok_s, head_s, pos_s, kend_s);
  const float scale = ldexpf(1.0f, p.frac), inv_scale = ldexpf(1.0f, -p.frac);
  {
    uint32_t qo = 0;
    for (int e = t; e < RT * D; e += THREADS) {
      const int i = e / D, d = e % D;
      float v = 0.0f;
      if (tok_s[i] >= 0) v = load_f32(p.q, p.q_dtype, (int64_t)tok_s[i] * p.q_st + (int64_t)head_s[i] * p.q_sh + d);
      q_s[i * Q_LD + d] = __fmul_rn(v, scale);
      qo = max(qo, __float_as_uint(v) & 0x7FFFFFFFu);
    }
    qo = __reduce_max_sync(0xffffffffu, qo);
    if (lane == 0) atomicMax(&q_max, qo);
  }

  // K staging: thread t moves 8 dims of key rows t / 4 and t / 4 + 64 of a tile
  const T* kbase = reinterpret_cast<const T*>(p.k);
  const int ntiles = (ke - kb + KQ - 1) / KQ, steps = ntiles * NCH;
  const int krow = t / 4, kcol = (t % 4) * 8;
  int blk[2], blk_next[2];
  auto blocks = [&](int ti, int (&b)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = kb + ti * KQ + krow + 64 * u;
      b[u] = ti < ntiles && j < ke ? block_of(a, j) : -1;
    }
  };
  uint4 raw[2];
  auto load = [&](int it) {
    const int ti = it / NCH, ch = it % NCH;
    if (ch == 0) {
      blk[0] = blk_next[0], blk[1] = blk_next[1];
      blocks(ti + 1, blk_next);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      raw[u] = make_uint4(0, 0, 0, 0);
      const int j = kb + ti * KQ + krow + 64 * u;
      if (blk[u] >= 0)
        raw[u] = *reinterpret_cast<const uint4*>(kbase + key_offset(p, j, blk[u], p.k_sb, p.k_ss, p.k_sh, kvh) + ch * DC + kcol);
    }
  };
  auto store = [&](int it) {
    float* dst = k_s + (it & 1) * KQ * K_LD;
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      absmax_word<T>(m, raw[u].x);
      absmax_word<T>(m, raw[u].y);
      absmax_word<T>(m, raw[u].z);
      absmax_word<T>(m, raw[u].w);
      float* d = dst + (krow + 64 * u) * K_LD + kcol;
      const float2 f0 = pair_of<T>(raw[u].x), f1 = pair_of<T>(raw[u].y), f2 = pair_of<T>(raw[u].z), f3 = pair_of<T>(raw[u].w);
      *reinterpret_cast<float4*>(d) = make_float4(f0.x, f0.y, f1.x, f1.y);
      *reinterpret_cast<float4*>(d + 4) = make_float4(f2.x, f2.y, f3.x, f3.y);
    }
    const uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(absmax_value<T>(m)));
    if (lane == 0) atomicMax(&k_max[(it / NCH) & 1], b);
  };
  blocks(0, blk_next);
  load(0);
  store(0);
  if (steps > 1) load(1);
  __syncthreads();
  // max|q| * max|k| * 2^f < 2^22: no saturation, and the magic constant rounds every product exactly
  const double scale_d = ldexp(1.0, p.frac), mq = (double)__uint_as_float(q_max);
  const float kthr = mq * scale_d < 3.0e38 ? __double2float_rd(4194304.0 / (mq * scale_d)) : 0.0f;

  const float2 C2 = make_float2(kMagic, kMagic);
  float rmax[TM];
  uint32_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) rmax[i] = -INFINITY;
  float* out = a.scores + (((int64_t)kvh * a.tiles + blockIdx.y) * RT + warp * TM) * p.key0;

  for (int it = 0; it < steps; ++it) {
    const int ti = it / NCH, ch = it % NCH;
    if (ch == 0) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = 0u - (uint32_t)D * (uint32_t)kMagicBits;
      if (t == 0) k_max[(ti + 1) & 1] = 0u;  // read in the step before; its next use is staged after a barrier
    }
    const float* qb = q_s + warp * TM * Q_LD + ch * DC;
    const float* kb_s = k_s + (it & 1) * KQ * K_LD + lane * K_LD;
#pragma unroll
    for (int kk = 0; kk < DC; kk += 4) {
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
    }
    if (ch == NCH - 1) {  // the tile's dots are complete: scores, row maxima
      const bool fast = __uint_as_float(k_max[ti & 1]) < kthr;  // uniform over the CTA
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int key = kb + ti * KQ + lane + 32 * j;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int r = warp * TM + i;
          long long dot = (int32_t)acc[i][j];
          if (!fast) {  // values the constant cannot round: the definition's clamp and convert, from the cache
            dot = 0;
            const int kblk = key < ke ? block_of(a, key) : -1;
            if (tok_s[r] >= 0 && kblk >= 0) {
              const T* kr = kbase + key_offset(p, key, kblk, p.k_sb, p.k_ss, p.k_sh, kvh);
              const int64_t qo = (int64_t)tok_s[r] * p.q_st + (int64_t)head_s[r] * p.q_sh;
              typename std::conditional<BITS == 64, unsigned long long, uint32_t>::type s = 0;
              for (int d = 0; d < D; ++d)
                s += (decltype(s))f2x_f32<BITS>(__fmul_rn(load_f32(p.q, p.q_dtype, qo + d), to_f32(kr[d])), scale);
              dot = BITS == 64 ? (long long)s : (long long)(int32_t)s;
            }
          }
          float qk = BITS == 64 ? __ll2float_rn(dot) : __int2float_rn((int)dot);
          qk = __fmul_rn(__fmul_rn(qk, inv_scale), p.scale_log2);
          bool ok = key < kend_s[r];
          if constexpr (!PL) {
            if (p.softcap_log2 > 0.0f) qk = __fmul_rn(p.softcap_log2, prim_tanh(__fmul_rn(qk, p.softcap_rcp)));
            if (p.alibi) qk = __fmaf_rn(p.alibi[head_s[r]], __fsub_rn((float)key, (float)pos_s[r]), qk);
            if (p.window > 0) ok = ok && key > pos_s[r] - p.window;
          }
          if (p.causal) ok = ok && pos_s[r] >= key;
          const float s = ok && key < ke ? qk : -INFINITY;
          if (key < ke) out[(int64_t)i * p.key0 + key] = s;
          rmax[i] = fmaxf(rmax[i], s);
        }
      }
    }
    if (it + 1 < steps) store(it + 1);
    if (it + 2 < steps) load(it + 2);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, ordered(rmax[i]));
    const int r = warp * TM + i;
    if (lane == 0 && tok_s[r] >= 0) atomicMax(&p.row_max[(int64_t)tok_s[r] * p.num_heads + head_s[r]], m);
  }
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
  static constexpr size_t v_buf = (size_t)KP * D * 4;
  static constexpr size_t p_buf = (size_t)RT * P_LD * 4;
  static constexpr size_t off_p = 2 * v_buf;
  static constexpr size_t bytes = off_p + 2 * p_buf;
};

template <int D, int RT, int BITS, typename T>
__global__ void __launch_bounds__(THREADS, 2) prefix_pv_kernel(const __grid_constant__ Args a) {
  using UAcc = typename std::conditional<BITS == 64, unsigned long long, uint32_t>::type;
  constexpr int LD = D / 4;              // lanes across the dims
  constexpr int GROUPS = THREADS / LD;   // row groups
  constexpr int TM = RT / GROUPS;
  constexpr int TPR = THREADS / RT;      // threads per row in the p phase
  constexpr int SV = KP / 4 / TPR;       // 16-byte score loads per thread
  constexpr int VU = (KP / 2) * (D / 8) / THREADS;  // (key pair, 8 dims) units per thread
  static_assert(TM >= 1 && SV >= 1 && VU >= 1, "tile mapping");
  using SM = PvSmem<D, RT>;
  const Params& p = a.p;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int tok_s[RT], head_s[RT], pos_s[RT], kend_s[RT];
  __shared__ uint32_t v_max[3];

  const int t = threadIdx.x, lane = t & 31;
  const int tile = a.tile0 + blockIdx.y, kvh = blockIdx.z;
  const int kb = blockIdx.x * a.keys_per_cta, ke = min(kb + a.keys_per_cta, p.key0);  // multiples of KP
  if (t < 3) v_max[t] = 0u;
  tile_rows<RT>(a, tile, kvh, tok_s, head_s, pos_s, kend_s);
  const float scale = ldexpf(1.0f, p.frac);
  const int ntiles = (ke - kb) / KP;

  // p phase: row prow, keys 4 * (t % TPR) + 4 * TPR * u
  const int prow = t / TPR;
  const bool live = tok_s[prow] >= 0;
  const int64_t row_id = live ? (int64_t)tok_s[prow] * p.num_heads + head_s[prow] : 0;
  const float m = live ? from_ordered(p.row_max[row_id]) : 0.0f;
  const float* src = a.scores + (((int64_t)kvh * a.tiles + blockIdx.y) * RT + prow) * p.key0 + kb + 4 * (t % TPR);
  UAcc den = 0;

  const T* vbase = reinterpret_cast<const T*>(p.v);
  float4 sc[SV];
  uint4 va[VU], vb[VU];
  int blk_a[VU], blk_b[VU];
  auto blocks = [&](int ti) {
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const int j = kb + ti * KP + 2 * ((t + u * THREADS) / (D / 8));
      blk_a[u] = ti < ntiles ? block_of(a, j) : -1;
      blk_b[u] = ti < ntiles ? block_of(a, j + 1) : -1;
    }
  };
  auto load = [&](int ti) {
#pragma unroll
    for (int u = 0; u < SV; ++u) sc[u] = *reinterpret_cast<const float4*>(src + ti * KP + 4 * TPR * u);
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const int unit = t + u * THREADS, j = kb + ti * KP + 2 * (unit / (D / 8)), d = (unit % (D / 8)) * 8;
      va[u] = vb[u] = make_uint4(0, 0, 0, 0);
      if (blk_a[u] >= 0)
        va[u] = *reinterpret_cast<const uint4*>(vbase + key_offset(p, j, blk_a[u], p.v_sb, p.v_ss, p.v_sh, kvh) + d);
      if (blk_b[u] >= 0)
        vb[u] = *reinterpret_cast<const uint4*>(vbase + key_offset(p, j + 1, blk_b[u], p.v_sb, p.v_ss, p.v_sh, kvh) + d);
    }
    blocks(ti + 1);
  };
  auto store = [&](int ti) {
    float* pd = reinterpret_cast<float*>(smem + SM::off_p + (ti & 1) * SM::p_buf) + prow * P_LD + 4 * (t % TPR);
#pragma unroll
    for (int u = 0; u < SV; ++u) {
      const float s[4] = {sc[u].x, sc[u].y, sc[u].z, sc[u].w};
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = -0.0f;  // a masked key: no contribution, whatever its V holds
        if (live && s[e] != -INFINITY) {
          x = prim_exp2(__fsub_rn(s[e], m));
          den += (UAcc)f2x_f32<BITS>(x, scale);
        }
        v[e] = __fmul_rn(x, scale);
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

  const int dl = t % LD, grp = t / LD;  // this thread's dims 4 * dl.., rows grp * TM..
  const int vc = dl / 2, vj = (dl & 1) * 2, vx = (vc >> 1) & 3;
  const int v0 = (vc * 4 + (vj ^ vx)) * 16, v1 = (vc * 4 + ((vj + 1) ^ vx)) * 16;
  uint32_t acc[TM][4];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0u;
  auto flush = [&]() {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int r = grp * TM + i;
      if (tok_s[r] < 0) continue;
      unsigned long long* dst = p.row_acc + ((int64_t)tok_s[r] * p.num_heads + head_s[r]) * D + 4 * dl;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned long long v =
            BITS == 64 ? (unsigned long long)(long long)(int32_t)acc[i][e] : (unsigned long long)acc[i][e];
        if (v) atomicAdd(dst + e, v);
        acc[i][e] = 0u;
      }
    }
  };
  // max|v| <= 65504 (finite after the cast) and max|v| * (1 + 2^-10) * 2^f < 2^22, with p <= 1
  const double scale_d = ldexp(1.0, p.frac);
  const float vthr = __double2float_rd(fmin(65504.5, 4194304.0 / (scale_d * (1.0 + 1.0 / 1024))));
  const float2 C2 = make_float2(kMagic, kMagic), ONE2 = make_float2(p.one, p.one);

  blocks(0);
  if (ntiles > 0) {
    load(0);
    store(0);
  }
  if (ntiles > 1) load(1);
  __syncthreads();
  for (int ti = 0; ti < ntiles; ++ti) {
    const bool fast = __uint_as_float(v_max[ti % 3]) < vthr;  // uniform over the CTA
    if (t == 0) v_max[(ti + 2) % 3] = 0u;
    const float* pb = reinterpret_cast<const float*>(smem + SM::off_p + (ti & 1) * SM::p_buf) + grp * TM * P_LD;
    const unsigned char* vs = smem + (ti & 1) * SM::v_buf;
    if (fast) {
#pragma unroll 4
      for (int k = 0; k < KP; k += 4) {
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
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] -= (uint32_t)KP * (uint32_t)kMagicBits;
    } else {  // values the constant cannot round: the definition's clamp and convert
#pragma unroll 1
      for (int i = 0; i < TM; ++i) {
        const int r = grp * TM + i;
        if (tok_s[r] < 0) continue;
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
          UAcc s = 0;
          for (int k = 0; k < KP; ++k) {
            const float ps = pb[i * P_LD + k];
            if (__float_as_uint(ps) == 0x80000000u) continue;
            const float vv = reinterpret_cast<const float*>(vs + (size_t)(k / 2) * D * 8 + (e < 2 ? v0 : v1))[2 * (e & 1) + (k & 1)];
            s += (UAcc)f2x_scaled<BITS>(__fmul_rn(ps, vv));
          }
          if (s) atomicAdd(p.row_acc + ((int64_t)tok_s[r] * p.num_heads + head_s[r]) * D + 4 * dl + e, (unsigned long long)s);
        }
      }
    }
    if (BITS == 64 && (ti + 1) % RUN == 0) flush();
    if (ti + 1 < ntiles) store(ti + 1);
    if (ti + 2 < ntiles) load(ti + 2);
    __syncthreads();
  }
  flush();
#pragma unroll
  for (int o = 1; o < TPR; o <<= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  if (t % TPR == 0 && live && den) atomicAdd(p.row_den + row_id, (unsigned long long)den);
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

// Keys per CTA (a multiple of `unit`): as many CTAs as fill the GPU twice over
// or, with few tiles, one step per CTA.
static int split_keys(int keys, int64_t tiles, int unit) {
  const int64_t steps = cdiv(keys, unit);
  int64_t splits = cdiv(4 * (int64_t)num_sms(), tiles);
  if (splits > steps) splits = steps;
  return (int)cdiv(steps, splits) * unit;
}

template <int D, int RT, int BITS, typename T>
static int launch(Args& a, bool pv, int kv_heads, cudaStream_t st) {
  const bool plain = !(a.p.softcap_log2 > 0.0f) && a.p.alibi == nullptr && a.p.window <= 0;
  a.keys_per_cta = split_keys(a.p.key0, (int64_t)a.tiles * kv_heads, pv ? KP : KQ);
  const dim3 grid((unsigned)cdiv(a.p.key0, a.keys_per_cta), (unsigned)a.tiles, (unsigned)kv_heads);
  if (pv) {
    static bool done[64] = {false};
    auto k = prefix_pv_kernel<D, RT, BITS, T>;
    const int rc = configure((const void*)k, PvSmem<D, RT>::bytes, done);
    if (rc != FXPR_OK) return rc;
    k<<<grid, THREADS, PvSmem<D, RT>::bytes, st>>>(a);
    return check_launch("fxpr_shared_prefix_attention_fxp (prefix pv)");
  }
  static bool done[2][64] = {{false}};
  auto k = plain ? prefix_scores_kernel<D, RT, BITS, T, true> : prefix_scores_kernel<D, RT, BITS, T, false>;
  const int rc = configure((const void*)k, ScoresSmem<D, RT>::bytes, done[plain ? 1 : 0]);
  if (rc != FXPR_OK) return rc;
  k<<<grid, THREADS, ScoresSmem<D, RT>::bytes, st>>>(a);
  return check_launch("fxpr_shared_prefix_attention_fxp (prefix scores)");
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
  a.tokens = tokens;
  a.num_blocks = num_blocks;
  a.scores = scores;
  a.tile0 = tile0;
  a.tiles = tiles;
  if (D == 64) return prefix::pick_rows<64>(a, pv, row_tile, bits, kv_dtype, p.num_kv_heads, st);
  return prefix::pick_rows<128>(a, pv, row_tile, bits, kv_dtype, p.num_kv_heads, st);
}

}  // namespace attn
}  // namespace fxpr
