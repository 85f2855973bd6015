// Rotary position of queries and keys, with the per-head fixed-point RMSNorm
// in the same pass and, for the append form, the new keys and values written
// into the paged cache that the attention kernels read.
//
// Per (token, head) row x of head_dim values, all in fp32:
//   S    = sum_i F2X(x_i^2)                    (integer, order-free)
//   rrms = 1 / sqrt(max(X2F(S) / head_dim, 0) + eps)
//   n_i  = (x_i * w_i) * rrms                  (as the RMSNorm kernels; n = x without weights)
//   y_a  = n_a * cos - n_b * sin,  y_b = n_b * cos + n_a * sin
// for the pairs (a, b) of the first rot_dim dims: (i, i + rot_dim/2), or
// (2i, 2i + 1) when interleaved. cos and sin come from a table row
// [cos | sin] of the token's position. Every product and sum is rounded by
// itself (no contraction) and the result is rounded to the output type once:
// norm and rotation as two operators round twice.
//
// Bound: HBM. Each row is read and written once and the arithmetic (about 12
// instructions a value with the norm) hides behind it.
//
// Layout of the vector kernel: a row belongs to a group of LPR lanes and each
// lane holds two 8-value pieces, chosen so that both halves of a rotation pair
// sit in one lane: no exchange but the integer sum of the squares. A lane
// keeps its piece of cos and sin (and of the weights) in registers for HPG
// heads of the token, so the table is read once per HPG heads. The groups of
// a warp are neighbouring tokens at the same heads: q, k and v rows never mix
// in a warp. HPG = 4 keeps eight 16-byte loads of a lane in flight; batches
// of few rows take HPG = 1, where more CTAs shorten the one wave there is.
#include "fxp_common.cuh"

namespace fxpr {
namespace rope {

constexpr int THREADS = 256;

struct Params {
  const void* x[3];  // q, k, v
  int64_t x_st[3], x_sh[3];
  void* y[2];  // rotated q, rotated k (NULL: not stored)
  int64_t y_st[2], y_sh[2];
  const void* w[2];  // norm weights of q and k
  int w_dtype;
  const void* pos;
  int pos64;
  const void* table;
  int t_dtype;
  int64_t t_rows, t_stride;
  int rot, neox;
  void* cache[2];  // k, v (NULL: no append)
  int c_dtype;
  int64_t c_sb[2], c_ss[2], c_sh[2];
  const int64_t* slots;
  int64_t num_slots;  // tokens that have a slot
  int64_t capacity;   // num_blocks * page
  int page;
  int64_t tokens;
  int heads, kv_heads, dim;
  float eps;
  int frac;
};

// what a row is: head h of the sequence q heads, k heads, v heads
struct Row {
  int part, head;  // part 0 q, 1 k, 2 v
};
__device__ __forceinline__ Row row_of(const Params& p, int h) {
  if (h < p.heads) return {0, h};
  if (h < p.heads + p.kv_heads) return {1, h - p.heads};
  return {2, h - p.heads - p.kv_heads};
}

__device__ __forceinline__ int64_t position_of(const Params& p, int64_t tok) {
  return p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[tok]
                 : (int64_t) reinterpret_cast<const int32_t*>(p.pos)[tok];
}

// cache slot of a token, or -1: padding (negative), a slot beyond the cache,
// or a token behind the slot mapping
__device__ __forceinline__ int64_t slot_of(const Params& p, int64_t tok) {
  if (p.cache[0] == nullptr || tok >= p.num_slots) return -1;
  const int64_t s = p.slots[tok];
  return s >= 0 && s < p.capacity ? s : -1;
}

// offset (elements) of a slot's row of one KV head in the k or v cache
__device__ __forceinline__ int64_t cache_offset(const Params& p, int kv, int64_t slot, int head) {
  const int64_t blk = slot / p.page, off = slot % p.page;
  return blk * p.c_sb[kv] + off * p.c_ss[kv] + head * p.c_sh[kv];
}

template <int BITS>
__device__ __forceinline__ float rrms_of(typename Acc<BITS>::T sum, int dim, float eps, int frac) {
  float s;
  if constexpr (BITS == 64) {
    s = x2f_f32<64>(sum, ldexpf(1.0f, -frac));
  } else {
    s = x2f_f32<32>(sum, ldexpf(1.0f, -frac));  // int16 squares sum in int32, as in the RMSNorm
  }
  const float mean = fmaxf(prim_div(s, (float)dim), 0.0f);
  return prim_div(1.0f, prim_sqrt(__fadd_rn(mean, eps)));
}

// ---- 8 consecutive values as fp32 (16-byte aligned) ----
template <typename T> __device__ __forceinline__ void load8(const T* src, float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 w = *reinterpret_cast<const uint4*>(src);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32(e[i]);
  } else {
    const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
}
template <typename T> __device__ __forceinline__ void store8(T* dst, const float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    uint4 w;
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(f[i]);
    *reinterpret_cast<uint4*>(dst) = w;
  } else {
    reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}
__device__ __forceinline__ void load8_any(const void* p, int dtype, int64_t i, float (&f)[8]) {
  if (dtype == FXPR_BF16) load8(reinterpret_cast<const __nv_bfloat16*>(p) + i, f);
  else if (dtype == FXPR_F16) load8(reinterpret_cast<const __half*>(p) + i, f);
  else load8(reinterpret_cast<const float*>(p) + i, f);
}
__device__ __forceinline__ void store8_any(void* p, int dtype, int64_t i, const float (&f)[8]) {
  if (dtype == FXPR_BF16) store8(reinterpret_cast<__nv_bfloat16*>(p) + i, f);
  else if (dtype == FXPR_F16) store8(reinterpret_cast<__half*>(p) + i, f);
  else store8(reinterpret_cast<float*>(p) + i, f);
}

// NORM: accumulator width of the norm, 0 = none
template <typename T, int NORM, int LPR, int HPG>
__global__ void __launch_bounds__(THREADS) rope_vec_kernel(const __grid_constant__ Params p) {
  constexpr int BITS = NORM == 0 ? 32 : NORM;
  using UAcc = typename std::conditional<BITS == 64, unsigned long long, uint32_t>::type;
  const int64_t tok = (int64_t)blockIdx.x * (THREADS / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR;  // this lane's pair of pieces
  const bool active = tok < p.tokens && c < p.dim / 16;
  const int rp = p.rot / 16;        // pairs of pieces that are rotated
  int lo, hi;
  if (c < rp) {
    lo = p.neox ? 8 * c : 16 * c;
    hi = p.neox ? lo + p.rot / 2 : lo + 8;
  } else {
    lo = 16 * c;
    hi = lo + 8;
  }
  const int rows = p.heads + p.kv_heads + (p.cache[0] != nullptr ? p.kv_heads : 0);
  const int h0 = blockIdx.y * HPG;

  float xa[HPG][8], xb[HPG][8];
  if (active) {
#pragma unroll
    for (int u = 0; u < HPG; ++u) {
      if (h0 + u >= rows) break;
      const Row r = row_of(p, h0 + u);
      const T* src = reinterpret_cast<const T*>(p.x[r.part]) + tok * p.x_st[r.part] + r.head * p.x_sh[r.part];
      load8(src + lo, xa[u]);
      load8(src + hi, xb[u]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < HPG; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) xa[u][e] = xb[u][e] = 0.0f;
  }
  const int64_t slot = active ? slot_of(p, tok) : -1;
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) cs[e] = 1.0f, sn[e] = 0.0f;
  const bool turn = active && c < rp;
  if (turn && h0 < p.heads + p.kv_heads) {
    const int64_t pos = position_of(p, tok);
    if (pos >= 0 && pos < p.t_rows) {
      load8_any(p.table, p.t_dtype, pos * p.t_stride + 8 * c, cs);
      load8_any(p.table, p.t_dtype, pos * p.t_stride + p.rot / 2 + 8 * c, sn);
    } else {  // a position outside the table has no angle
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[e] = sn[e] = __int_as_float(0x7FFFFFFF);
    }
  }

#pragma unroll
  for (int u = 0; u < HPG; ++u) {
    if (h0 + u >= rows) break;  // uniform over the CTA
    const Row r = row_of(p, h0 + u);
    if (r.part < 2) {
      if constexpr (NORM != 0) {
        const float scale = ldexpf(1.0f, p.frac);
        UAcc acc = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          acc += (UAcc)f2x_f32<BITS>(__fmul_rn(xa[u][e], xa[u][e]), scale);
          acc += (UAcc)f2x_f32<BITS>(__fmul_rn(xb[u][e], xb[u][e]), scale);
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
        if (active) {
          const float rrms = rrms_of<BITS>((typename Acc<BITS>::T)acc, p.dim, p.eps, p.frac);
          float wa[8], wb[8];
          load8_any(p.w[r.part], p.w_dtype, lo, wa);
          load8_any(p.w[r.part], p.w_dtype, hi, wb);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            xa[u][e] = __fmul_rn(__fmul_rn(xa[u][e], wa[e]), rrms);
            xb[u][e] = __fmul_rn(__fmul_rn(xb[u][e], wb[e]), rrms);
          }
        }
      }
      if (turn) {
        if (p.neox) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = xa[u][e], b = xb[u][e];
            xa[u][e] = __fsub_rn(__fmul_rn(a, cs[e]), __fmul_rn(b, sn[e]));
            xb[u][e] = __fadd_rn(__fmul_rn(b, cs[e]), __fmul_rn(a, sn[e]));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a = xa[u][2 * e], b = xa[u][2 * e + 1];
            xa[u][2 * e] = __fsub_rn(__fmul_rn(a, cs[e]), __fmul_rn(b, sn[e]));
            xa[u][2 * e + 1] = __fadd_rn(__fmul_rn(b, cs[e]), __fmul_rn(a, sn[e]));
            a = xb[u][2 * e], b = xb[u][2 * e + 1];
            xb[u][2 * e] = __fsub_rn(__fmul_rn(a, cs[4 + e]), __fmul_rn(b, sn[4 + e]));
            xb[u][2 * e + 1] = __fadd_rn(__fmul_rn(b, cs[4 + e]), __fmul_rn(a, sn[4 + e]));
          }
        }
      }
      if (active && p.y[r.part] != nullptr) {
        T* dst = reinterpret_cast<T*>(p.y[r.part]) + tok * p.y_st[r.part] + r.head * p.y_sh[r.part];
        store8(dst + lo, xa[u]);
        store8(dst + hi, xb[u]);
      }
    }
    if (r.part > 0 && slot >= 0) {
      const int kv = r.part - 1;
      const int64_t o = cache_offset(p, kv, slot, r.head);
      store8_any(p.cache[kv], p.c_dtype, o + lo, xa[u]);
      store8_any(p.cache[kv], p.c_dtype, o + hi, xb[u]);
    }
  }
}

// Any head_dim, rot_dim, stride and alignment: one warp per row, one lane per
// rotation pair. The sum's reads all precede the first store of the row (the
// shuffles order them), so the result may overwrite the input.
template <typename T, int NORM>
__global__ void __launch_bounds__(THREADS) rope_any_kernel(const __grid_constant__ Params p) {
  constexpr int BITS = NORM == 0 ? 32 : NORM;
  using UAcc = typename std::conditional<BITS == 64, unsigned long long, uint32_t>::type;
  const int lane = threadIdx.x & 31;
  const int rows = p.heads + p.kv_heads + (p.cache[0] != nullptr ? p.kv_heads : 0);
  const int64_t id = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  if (id >= p.tokens * rows) return;  // uniform over the warp
  const int64_t tok = id / rows;
  const Row r = row_of(p, (int)(id % rows));
  const T* src = reinterpret_cast<const T*>(p.x[r.part]) + tok * p.x_st[r.part] + r.head * p.x_sh[r.part];
  const int64_t slot = r.part > 0 ? slot_of(p, tok) : -1;
  T* dst = r.part < 2 && p.y[r.part] != nullptr
               ? reinterpret_cast<T*>(p.y[r.part]) + tok * p.y_st[r.part] + r.head * p.y_sh[r.part]
               : nullptr;
  const int64_t co = slot >= 0 ? cache_offset(p, r.part - 1, slot, r.head) : 0;
  float rrms = 1.0f;
  if constexpr (NORM != 0) {
    if (r.part < 2) {
      const float scale = ldexpf(1.0f, p.frac);
      UAcc acc = 0;
      for (int i = lane; i < p.dim; i += 32) {
        const float x = to_f32(src[i]);
        acc += (UAcc)f2x_f32<BITS>(__fmul_rn(x, x), scale);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      rrms = rrms_of<BITS>((typename Acc<BITS>::T)acc, p.dim, p.eps, p.frac);
    }
  }
  auto value = [&](int i) -> float {
    float x = to_f32(src[i]);
    if constexpr (NORM != 0)
      if (r.part < 2) x = __fmul_rn(__fmul_rn(x, load_f32(p.w[r.part], p.w_dtype, i)), rrms);
    return x;
  };
  auto put = [&](int i, float v) {
    if (dst) dst[i] = from_f32<T>(v);
    if (slot >= 0) store_f32(p.cache[r.part - 1], p.c_dtype, co + i, v);
  };
  const int half = r.part < 2 ? p.rot / 2 : 0;
  int64_t pos = 0;
  if (half > 0) pos = position_of(p, tok);
  const bool known = pos >= 0 && pos < p.t_rows;
  for (int i = lane; i < half; i += 32) {
    float cs = __int_as_float(0x7FFFFFFF), sn = cs;
    if (known) {
      cs = load_f32(p.table, p.t_dtype, pos * p.t_stride + i);
      sn = load_f32(p.table, p.t_dtype, pos * p.t_stride + half + i);
    }
    const int ia = p.neox ? i : 2 * i, ib = p.neox ? i + half : 2 * i + 1;
    const float a = value(ia), b = value(ib);
    put(ia, __fsub_rn(__fmul_rn(a, cs), __fmul_rn(b, sn)));
    put(ib, __fadd_rn(__fmul_rn(b, cs), __fmul_rn(a, sn)));
  }
  for (int i = 2 * half + lane; i < p.dim; i += 32) put(i, value(i));
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <typename T, int NORM, int LPR>
static int launch_vec(const Params& p, int rows, cudaStream_t st) {
  const int64_t bx = cdiv(p.tokens, THREADS / LPR);
  // four heads per group once that still leaves two CTAs for each SM
  if (bx * cdiv(rows, 4) >= 2 * num_sms()) {
    const dim3 grid((unsigned)bx, (unsigned)cdiv(rows, 4));
    rope_vec_kernel<T, NORM, LPR, 4><<<grid, THREADS, 0, st>>>(p);
  } else {
    rope_vec_kernel<T, NORM, LPR, 1><<<dim3((unsigned)bx, (unsigned)rows), THREADS, 0, st>>>(p);
  }
  return check_launch("fxpr rope");
}

template <typename T, int NORM>
static int launch(const Params& p, bool vec, int rows, cudaStream_t st) {
  if (vec) {
    const int pieces = p.dim / 16;
    if (pieces <= 4) return launch_vec<T, NORM, 4>(p, rows, st);
    if (pieces <= 8) return launch_vec<T, NORM, 8>(p, rows, st);
    if (pieces <= 16) return launch_vec<T, NORM, 16>(p, rows, st);
    return launch_vec<T, NORM, 32>(p, rows, st);
  }
  const int64_t blocks = cdiv(p.tokens * rows, THREADS / 32);
  if (blocks > 0x7fffffffLL) {
    set_error("rope: too many rows");
    return FXPR_ERR_INVALID;
  }
  rope_any_kernel<T, NORM><<<(unsigned)blocks, THREADS, 0, st>>>(p);
  return check_launch("fxpr rope");
}

template <typename T>
static int pick_norm(const Params& p, int norm, bool vec, int rows, cudaStream_t st) {
  switch (norm) {
    case 0: return launch<T, 0>(p, vec, rows, st);
    case 16: return launch<T, 16>(p, vec, rows, st);
    case 32: return launch<T, 32>(p, vec, rows, st);
    default: return launch<T, 64>(p, vec, rows, st);
  }
}

static bool al16(const void* ptr) { return (uintptr_t)ptr % 16 == 0; }
static bool stride16(int64_t s, int es) { return (s * es) % 16 == 0; }

static int run(const fxpr_rope_params* a, bool append, const char* what, void* stream) {
  auto ok_f = [](int d) { return d == FXPR_F16 || d == FXPR_BF16 || d == FXPR_F32; };
  if (a == nullptr) {
    set_error("%s: null parameters", what);
    return FXPR_ERR_INVALID;
  }
  const bool norm = a->q_weight != nullptr || a->k_weight != nullptr;
  if (norm && !valid_bits(a->int_bits)) {
    set_error("fxp_int_bits must be 16/32/64, got %d", a->int_bits);
    return FXPR_ERR_INVALID;
  }
  if (norm && (a->frac_bits < 0 || a->frac_bits >= a->int_bits)) {
    set_error("%s: frac_bits must satisfy 0 <= frac_bits < %d, got %d", what, a->int_bits, a->frac_bits);
    return FXPR_ERR_INVALID;
  }
  if (!ok_f(a->dtype) || !ok_f(a->table_dtype) || (norm && !ok_f(a->weight_dtype)) ||
      (append && !ok_f(a->cache_dtype))) {
    set_error("%s: tensors must be float16/bfloat16/float32", what);
    return FXPR_ERR_INVALID;
  }
  if (a->tokens < 0 || a->num_heads < 0 || a->num_kv_heads < 0 || a->head_dim <= 0 || a->head_dim > 1024 ||
      a->num_heads > 16384 || a->num_kv_heads > 16384) {
    set_error("%s: head_dim must be 1..1024 and the head counts at most 16384", what);
    return FXPR_ERR_INVALID;
  }
  if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 2 != 0) {
    set_error("%s: the rotary table's width must be even and at most head_dim, got %d", what, a->rot_dim);
    return FXPR_ERR_INVALID;
  }
  if (norm && (a->q_weight == nullptr || a->k_weight == nullptr)) {
    set_error("%s: give both norm weights or neither", what);
    return FXPR_ERR_INVALID;
  }
  const bool qs = a->tokens > 0 && a->num_heads > 0, ks = a->tokens > 0 && a->num_kv_heads > 0;
  if ((qs && (!a->q || !a->q_out)) || (ks && (!a->k || (!append && !a->k_out) || (append && !a->v))) ||
      (a->tokens > 0 && a->rot_dim > 0 && (!a->positions || !a->table))) {
    set_error("%s: null pointer", what);
    return FXPR_ERR_INVALID;
  }
  if (append && (a->page_size <= 0 || a->num_blocks < 0 || a->num_slots < 0 || a->num_slots > a->tokens ||
                 (a->num_slots > 0 && ks && (!a->slot_mapping || !a->k_cache || !a->v_cache)))) {
    set_error("%s: bad cache or slot mapping", what);
    return FXPR_ERR_INVALID;
  }
  if (!qs && !ks) return FXPR_OK;
  Params p = {};
  p.x[0] = a->q; p.x_st[0] = a->q_stride_tok; p.x_sh[0] = a->q_stride_head;
  p.x[1] = a->k; p.x_st[1] = a->k_stride_tok; p.x_sh[1] = a->k_stride_head;
  p.y[0] = a->q_out; p.y_st[0] = a->qo_stride_tok; p.y_sh[0] = a->qo_stride_head;
  p.y[1] = a->k_out; p.y_st[1] = a->ko_stride_tok; p.y_sh[1] = a->ko_stride_head;
  p.w[0] = a->q_weight; p.w[1] = a->k_weight; p.w_dtype = a->weight_dtype;
  p.pos = a->positions; p.pos64 = a->positions_64;
  p.table = a->table; p.t_dtype = a->table_dtype; p.t_rows = a->table_rows; p.t_stride = a->table_stride;
  p.rot = a->rot_dim; p.neox = a->is_neox;
  p.tokens = a->tokens; p.heads = a->num_heads; p.kv_heads = a->num_kv_heads; p.dim = a->head_dim;
  p.eps = a->eps; p.frac = a->frac_bits;
  const int es = elem_size(a->dtype);
  bool vec = a->head_dim % 16 == 0 && a->head_dim <= 512 && a->rot_dim % 16 == 0;
  if (qs)
    vec = vec && al16(p.x[0]) && stride16(p.x_st[0], es) && stride16(p.x_sh[0], es) && al16(p.y[0]) &&
          stride16(p.y_st[0], es) && stride16(p.y_sh[0], es);
  if (ks)
    vec = vec && al16(p.x[1]) && stride16(p.x_st[1], es) && stride16(p.x_sh[1], es) &&
          (!p.y[1] || (al16(p.y[1]) && stride16(p.y_st[1], es) && stride16(p.y_sh[1], es)));
  if (p.rot > 0) vec = vec && al16(p.table) && stride16(p.t_stride, elem_size(a->table_dtype));
  if (norm) vec = vec && al16(p.w[0]) && al16(p.w[1]);
  if (append && a->num_slots > 0 && a->num_blocks > 0 && ks) {
    const int ec = elem_size(a->cache_dtype);
    p.x[2] = a->v; p.x_st[2] = a->v_stride_tok; p.x_sh[2] = a->v_stride_head;
    p.cache[0] = a->k_cache; p.cache[1] = a->v_cache; p.c_dtype = a->cache_dtype;
    p.c_sb[0] = a->kc_stride_blk; p.c_ss[0] = a->kc_stride_slot; p.c_sh[0] = a->kc_stride_head;
    p.c_sb[1] = a->vc_stride_blk; p.c_ss[1] = a->vc_stride_slot; p.c_sh[1] = a->vc_stride_head;
    p.slots = a->slot_mapping; p.num_slots = a->num_slots;
    p.page = a->page_size; p.capacity = a->num_blocks * a->page_size;
    vec = vec && al16(p.x[2]) && stride16(p.x_st[2], es) && stride16(p.x_sh[2], es);
    for (int i = 0; i < 2; ++i)
      vec = vec && al16(p.cache[i]) && stride16(p.c_sb[i], ec) && stride16(p.c_ss[i], ec) && stride16(p.c_sh[i], ec);
  }
  const int rows = p.heads + p.kv_heads + (p.cache[0] ? p.kv_heads : 0);
  const int n = norm ? a->int_bits : 0;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case FXPR_BF16: return pick_norm<__nv_bfloat16>(p, n, vec, rows, st);
    case FXPR_F16: return pick_norm<__half>(p, n, vec, rows, st);
    default: return pick_norm<float>(p, n, vec, rows, st);
  }
}

}  // namespace rope
}  // namespace fxpr

extern "C" int fxpr_qk_norm_rope_fxp(const fxpr_rope_params* p, void* stream) {
  return fxpr::rope::run(p, false, "qk_norm_rope_fxp", stream);
}

extern "C" int fxpr_rope_append_kv_fxp(const fxpr_rope_params* p, void* stream) {
  return fxpr::rope::run(p, true, "rope_append_kv_fxp", stream);
}
