// Verification of drafted tokens (speculative decoding) in integers.
//
// With P = F2X(clamp(p, 0, 1)) and Q = F2X(clamp(q, 0, 1)) the probabilities
// on the 2^-f grid, U and R the given random numbers on the 2^-24 grid:
//
//   token x of position i is taken iff U_i * Q_i(x) < P_i(x) * 2^24
//   at the first position that is not: left = max(P - Q, 0) (P itself if that
//   is zero everywhere), T = sum(left), goal = floor(R * T / 2^24), and the
//   token drawn is the smallest v with left_0 + .. + left_v > goal
//   if all are taken: the bonus token
//
// Whole numbers throughout: sums do not depend on their order and the draw is
// the same whatever the split of the vocabulary. Without draft probabilities
// (a deterministic drafter) Q is 1 at the drafted token and 0 elsewhere.
//
// Bound: HBM for a full batch (the one or two vocabulary rows of each
// refusing position are read once; a 128256-token row of fp32 is 513 KB), the
// chain of dependent reads for a few requests. One cluster of CTAs per
// request: every CTA decides on the drafted tokens by itself (one lane per
// position), then sums its slice of the vocabulary; the slices' sums meet in
// distributed shared memory, and the CTA that holds the goal finds the token:
// the warp whose share it lies in, then that share again from L2, a turn per
// warp. Nothing is read for a request whose drafts are all taken.
#include <cooperative_groups.h>

#include "fxp_common.cuh"

namespace cg = cooperative_groups;

namespace fxpr {
namespace verify {

// 256 threads, six CTAs per SM (40 registers), four 16-byte loads per tensor
// of a lane in flight: 128 requests of 128256 fp32 entries, 81 to 94 of them
// refusing (89 MB), 21.5 us (4.2 TB/s, 64% of a copy). In the same batch 3.6 us
// if none refuses (launch and the chain of reads that decides on the drafted
// tokens), 30.9 us if all do (131 MB, 4.3 TB/s); one request that refuses 6.8 us;
// a refusing request more costs 0.2 us (5.1 TB/s). Four or five CTAs 2 to 3 us
// more, 512 threads 3 us. One request, its drafts taken two times in three: 3.9 us.
constexpr int THREADS = 256;
constexpr int MINB = 6;
constexpr int UNROLL = 4;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_DRAFTS = 32;  // one lane per drafted position
constexpr int MAX_CLUSTER = 8;
typedef unsigned long long u64;

struct Params {
  const void* p;
  const void* q;
  int64_t p_stride, q_stride;
  const void* ids;
  int ids64;
  const int32_t* start;
  const void* bonus;
  int bonus64;
  const float* u;
  const float* r;
  int64_t total;  // drafted positions that exist (rows of p)
  int64_t vocab;
  int most;
  int frac;
  int32_t* out;
  int64_t out_stride;
  int32_t* taken;
  int64_t span;  // vocabulary entries per warp (a multiple of 32 * E)
};

// F2X of a probability: 0 for NaN and below 0, 2^f from 1 on; exact scaling, one rounding
__device__ __forceinline__ uint32_t grid_of(float x, float scale) {
  return __float2uint_rn(__fmul_rn(__saturatef(x), scale));
}
// random number in [0, 1) on the 2^-24 grid (truncated; NaN 0)
__device__ __forceinline__ uint32_t draw_of(float x) {
  return (uint32_t)min(max(__float2int_rz(__fmul_rn(x, 16777216.0f)), 0), 16777215);
}
__device__ __forceinline__ int64_t load_id(const void* p, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// what remains of entry v (0 outside the vocabulary): with draft
// probabilities P - Q, else P except at the drafted token; `all`: P
template <typename T, bool Q>
__device__ __forceinline__ uint32_t left_of(T pv, T qv, int64_t v, int64_t token, float scale, bool all) {
  const uint32_t P = grid_of(to_f32(pv), scale);
  if (all) return P;
  if constexpr (Q) {
    const uint32_t D = grid_of(to_f32(qv), scale);
    return max(P, D) - D;
  } else {
    return v == token ? 0u : P;
  }
}

template <typename T, int E> struct alignas(sizeof(T) * E) Vec { T v[E]; };

// A row of the vocabulary seen from the 16-byte boundary at or before its
// first entry: entry v is element v + shift of `base`, and element blocks of
// E are aligned. Blocks that reach outside the row are read entry by entry.
template <typename T, int E> struct Row {
  const T* base;
  __device__ __forceinline__ Vec<T, E> load(int64_t w, int64_t first, int64_t end) const {
    Vec<T, E> x = {};
    if (w >= first && w + E <= end) {
      x = *reinterpret_cast<const Vec<T, E>*>(base + w);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (w + e >= first && w + e < end) x.v[e] = base[w + e];
    }
    return x;
  }
};

// E consecutive entries per load: 16 bytes, or one entry where the rows of the
// two tensors lie differently to 16-byte boundaries
template <typename T, bool Q, int E>
__global__ void __launch_bounds__(THREADS, MINB) verify_kernel(const __grid_constant__ Params p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t req = blockIdx.x / ranks;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const float scale = ldexpf(1.0f, p.frac);
  __shared__ u64 warp_sum[WARPS], turn_sum[WARPS];
  __shared__ u64 cta_sum;  // read by the other CTAs of the cluster
  __shared__ int s_taken;
  __shared__ bool s_refused;
  __shared__ int64_t s_token;

  // ---- the drafted tokens: one lane per position ----
  const u64 R = draw_of(p.r[req]);  // asked for ahead of its use
  const int64_t first = p.start[req];
  const int64_t length = min((int64_t)p.start[req + 1] - first, (int64_t)p.most);
  if (warp == 0) {
    bool ok = false;
    int64_t id = -1;
    const int64_t row = first + lane;
    if (lane < length && row >= 0 && row < p.total) {
      id = load_id(p.ids, p.ids64, row);
      if (id >= 0 && id < p.vocab) {
        const u64 P = grid_of(to_f32(reinterpret_cast<const T*>(p.p)[row * p.p_stride + id]), scale);
        u64 D = 1ull << p.frac;
        if constexpr (Q) D = grid_of(to_f32(reinterpret_cast<const T*>(p.q)[row * p.q_stride + id]), scale);
        ok = (u64)draw_of(p.u[row]) * D < (P << 24);
      }
    }
    const uint32_t refused = __ballot_sync(0xffffffffu, !ok && lane < length);
    const int n = refused ? __ffs(refused) - 1 : (int)max(length, (int64_t)0);
    if (lane == 0) {
      s_taken = n;
      s_refused = refused != 0;
    }
    if (refused && lane == n) s_token = id;
    if (rank == 0) {
      int32_t* o = p.out + req * p.out_stride;
      for (int i = lane; i <= p.most; i += 32) {
        int32_t v = i < n ? (int32_t)id : -1;  // n <= 32: only the first turn has taken tokens
        if (i == n && !refused) v = (int32_t)load_id(p.bonus, p.bonus64, req);
        o[i] = v;
      }
      if (lane == 0) p.taken[req] = n;
    }
  }
  __syncthreads();
  if (!s_refused) return;  // uniform over the cluster
  const int64_t row = first + s_taken;
  const bool exists = row >= 0 && row < p.total;
  const int64_t token = s_token;
  const T* pr = reinterpret_cast<const T*>(p.p) + (exists ? row : 0) * p.p_stride;
  const int shift = E == 1 ? 0 : (int)((uintptr_t)pr % (E * sizeof(T)) / sizeof(T));
  const Row<T, E> prow = {pr - shift};
  const Row<T, E> qrow = {Q ? reinterpret_cast<const T*>(p.q) + (exists ? row : 0) * p.q_stride - shift : nullptr};
  const int64_t end = p.vocab + shift;  // the row's entries are elements [shift, end)
  const int64_t mark = token >= 0 && token < p.vocab ? token + shift : -1;

  // ---- sums of this warp's share of the vocabulary ----
  const int64_t lo = ((int64_t)rank * WARPS + warp) * p.span;
  const int64_t hi = exists ? min(lo + p.span, end) : lo;
  auto entries = [&](int64_t w, bool all, uint32_t (&x)[E]) {
    const Vec<T, E> a = prow.load(w, shift, end);
    Vec<T, E> b = {};
    if constexpr (Q) b = qrow.load(w, shift, end);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = left_of<T, Q>(a.v[e], b.v[e], w + e, mark, scale, all);
  };
  auto sum_of = [&](bool all) -> u64 {
    u64 s = 0;
    auto add = [&](const uint32_t (&x)[E]) {
      // two entries are at most 2^31
#pragma unroll
      for (int e = 0; e + 1 < E; e += 2) s += x[e] + x[e + 1];
      if (E == 1) s += x[0];
    };
    int64_t w = lo + lane * E;
    if (w < shift && w < hi) {  // the row's first block, where it starts inside one
      uint32_t x[E];
      entries(w, all, x);
      add(x);
      w += 32 * E;
    }
    // whole turns: every block lies in the row, and UNROLL of them are in flight
    for (; w + (UNROLL - 1) * 32 * E + E <= hi; w += UNROLL * 32 * E) {
      Vec<T, E> a[UNROLL], b[UNROLL];
#pragma unroll
      for (int g = 0; g < UNROLL; ++g) {
        a[g] = *reinterpret_cast<const Vec<T, E>*>(prow.base + w + g * 32 * E);
        if constexpr (Q) b[g] = *reinterpret_cast<const Vec<T, E>*>(qrow.base + w + g * 32 * E);
      }
#pragma unroll
      for (int g = 0; g < UNROLL; ++g) {
        uint32_t x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = left_of<T, Q>(a[g].v[e], b[g].v[e], w + g * 32 * E + e, mark, scale, all);
        add(x);
      }
    }
    for (; w < hi; w += 32 * E) {
      uint32_t x[E];
      entries(w, all, x);
      add(x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  };
  u64 total = 0, before = 0;  // over the cluster, and over the CTAs in front of this one
  auto meet = [&](u64 mine) {
    if (lane == 0) warp_sum[warp] = mine;
    __syncthreads();
    if (t == 0) {
      u64 s = 0;
      for (int w = 0; w < WARPS; ++w) s += warp_sum[w];
      cta_sum = s;
    }
    cluster.sync();
    total = before = 0;
    for (int c = 0; c < ranks; ++c) {
      const u64 s = *cluster.map_shared_rank(&cta_sum, c);
      if (c < rank) before += s;
      total += s;
    }
    cluster.barrier_arrive();
  };
  // nobody leaves or overwrites its sum while others may read it
  auto part = [&]() { cluster.barrier_wait(); };
  bool all = false;
  meet(sum_of(false));
  if (total == 0) {  // uniform over the cluster: nothing remains, draw from the target itself
    all = true;
    part();
    meet(sum_of(true));
  }
  if (total == 0) {  // no probability at all: -1 stays
    part();
    return;
  }
  const u64 goal = (total >> 24) * R + (((total & 0xFFFFFFull) * R) >> 24);

  // ---- the CTA that holds the goal looks through the share it lies in, one
  // turn of 32 * E entries per warp ----
  int share = -1;
  u64 run = before;
  for (int w = 0; w < WARPS && share < 0; ++w) {  // uniform over the CTA
    if (goal >= run && goal < run + warp_sum[w]) share = w;
    else run += warp_sum[w];
  }
  if (share < 0) {
    part();
    return;
  }
  const int64_t from = ((int64_t)rank * WARPS + share) * p.span;
  const int turns = (int)(p.span / (32 * E));
  for (int t0 = 0; t0 < turns; t0 += WARPS) {
    uint32_t x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0u;
    const int64_t w = from + ((int64_t)(t0 + warp) * 32 + lane) * E;
    if (t0 + warp < turns) entries(w, all, x);  // beyond the row: 0
    u64 mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) mine += x[e];
    u64 upto = mine;  // over the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 s = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += s;
    }
    if (lane == 31) turn_sum[warp] = upto;
    __syncthreads();
    u64 at = run;  // in front of this warp's turn
    for (int i = 0; i < WARPS; ++i) {
      if (i < warp) at += turn_sum[i];
      run += turn_sum[i];
    }
    if (goal >= at + upto - mine && goal < at + upto) {  // one lane of the CTA
      u64 s = at + upto - mine;
      int e = 0;
#pragma unroll
      for (int i = 0; i < E - 1; ++i)
        if (e == i && s + x[i] <= goal) {
          s += x[i];
          ++e;
        }
      p.out[req * p.out_stride + s_taken] = (int32_t)(w + e - shift);
    }
    if (goal < run) break;  // uniform over the CTA
    __syncthreads();  // turn_sum is read
  }
  part();
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <typename T, bool Q, int E>
static int launch(Params p, int64_t requests, cudaStream_t st) {
  // CTAs per request: what is resident at once over the batch, or somewhat
  // more, since requests that refuse nothing leave early (two per SM 44 us,
  // eight 24 us at the batch above, before the whole-turn loop); each with at least one turn of its warps
  int ranks = MAX_CLUSTER;
  while (ranks > 1 && (requests * ranks > 8 * num_sms() || (int64_t)(ranks / 2) * THREADS * E >= p.vocab)) ranks /= 2;
  p.span = cdiv(cdiv(p.vocab + E, (int64_t)ranks * WARPS), 32 * E) * 32 * E;  // the shift is below E
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(requests * ranks));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, verify_kernel<T, Q, E>, p) != cudaSuccess) return check_launch("fxpr_verify_draft_fxp");
  return check_launch("fxpr_verify_draft_fxp");
}

template <typename T>
static int pick(const Params& p, int64_t requests, cudaStream_t st) {
  constexpr int E = 16 / (int)sizeof(T);
  // rows of both tensors at the same offset from a 16-byte boundary
  const bool vec = p.q == nullptr || ((uintptr_t)p.p % 16 == (uintptr_t)p.q % 16 && (p.p_stride - p.q_stride) % E == 0);
  if (p.q != nullptr) return vec ? launch<T, true, E>(p, requests, st) : launch<T, true, 1>(p, requests, st);
  return vec ? launch<T, false, E>(p, requests, st) : launch<T, false, 1>(p, requests, st);
}

}  // namespace verify
}  // namespace fxpr

using namespace fxpr;

extern "C" int fxpr_verify_draft_fxp(const void* target_probs, const void* draft_probs, int probs_dtype,
                                     int64_t target_row_stride, int64_t draft_row_stride, int64_t num_drafts,
                                     int64_t vocab, const void* draft_token_ids, int draft_ids_64,
                                     const int32_t* draft_start_loc, const void* bonus_token_ids, int bonus_ids_64,
                                     const float* accept_uniform, const float* resample_uniform,
                                     int64_t num_requests, int max_draft_len, int frac_bits, int32_t* token_ids,
                                     int64_t out_row_stride, int32_t* num_accepted, void* stream) {
  if (probs_dtype != FXPR_F16 && probs_dtype != FXPR_BF16 && probs_dtype != FXPR_F32) {
    set_error("verify_draft_fxp: probabilities must be float16/bfloat16/float32");
    return FXPR_ERR_INVALID;
  }
  if (frac_bits < 1 || frac_bits > 30) {
    set_error("verify_draft_fxp: frac_bits must be 1..30, got %d", frac_bits);
    return FXPR_ERR_INVALID;
  }
  if (max_draft_len < 0 || max_draft_len > verify::MAX_DRAFTS) {
    set_error("verify_draft_fxp: max_draft_len must be 0..%d, got %d", verify::MAX_DRAFTS, max_draft_len);
    return FXPR_ERR_INVALID;
  }
  if (num_requests < 0 || num_drafts < 0 || vocab < 1 || vocab > (1 << 24) || num_requests > (1 << 27)) {
    set_error("verify_draft_fxp: the vocabulary must have 1..2^24 entries and the batch at most 2^27 requests");
    return FXPR_ERR_INVALID;
  }
  if (num_requests == 0) return FXPR_OK;
  if (!draft_start_loc || !bonus_token_ids || !resample_uniform || !token_ids || !num_accepted ||
      (num_drafts > 0 && (!target_probs || !draft_token_ids || !accept_uniform))) {
    set_error("verify_draft_fxp: null pointer");
    return FXPR_ERR_INVALID;
  }
  verify::Params p = {};
  p.p = target_probs; p.q = num_drafts > 0 ? draft_probs : nullptr;
  p.p_stride = target_row_stride; p.q_stride = draft_row_stride;
  p.ids = draft_token_ids; p.ids64 = draft_ids_64;
  p.start = draft_start_loc; p.bonus = bonus_token_ids; p.bonus64 = bonus_ids_64;
  p.u = accept_uniform; p.r = resample_uniform;
  p.total = num_drafts; p.vocab = vocab; p.most = max_draft_len; p.frac = frac_bits;
  p.out = token_ids; p.out_stride = out_row_stride; p.taken = num_accepted;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (probs_dtype) {
    case FXPR_BF16: return verify::pick<__nv_bfloat16>(p, num_requests, st);
    case FXPR_F16: return verify::pick<__half>(p, num_requests, st);
    default: return verify::pick<float>(p, num_requests, st);
  }
}
