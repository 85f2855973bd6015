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
// Bound: HBM. Each row is read and written once. 8192 tokens, 32 + 8 heads x
// 128, bf16: rotation and append 35.6 us for 204 MB (5.7 TB/s, 88% of a copy;
// 49% of the issue slots); with the norm 34.1 us for 170 MB (5.0 TB/s, 76%):
// there 250 instructions a lane and row take 70% of the issue slots, and neither
// side is full.
//
// Layout of the vector kernel: a row belongs to a group of LPR lanes and each
// lane holds two 8-value pieces, chosen so that both halves of a rotation pair
// sit in one lane: no exchange but the integer sum of the squares. The groups
// of a CTA are neighbouring tokens and the CTA walks a range of heads of one
// of q, k and v, with its pieces of cos, sin and the weights in registers
// throughout; the next rows come by asynchronous copies into words of shared
// memory that only the copying thread reads, which costs no registers and no
// barrier.
#include "fxp_common.cuh"

namespace fxpr {
namespace rope {

constexpr int THREADS = 256;
// Resident CTAs per SM (64 registers a thread) and rows in flight per lane.
// 8192 tokens, 32 + 8 heads x 128, bf16, with the norm / with the append: 3
// CTAs 34.7 / 35.6 us, 4 CTAs 34.4 / 35.8 us, 5 CTAs (spills) 56.7 / 38.3 us;
// 4 CTAs with 3 instead of 4 rows 35.7 / 37.0 us; two rows in registers
// instead of the ring 41.5 / 38.9 us.
constexpr int MINB = 4;
template <typename T> constexpr int STAGES = sizeof(T) == 2 ? 4 : 2;

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
  // vector kernel: heads per CTA; CTAs of q and of k (and of v) per block of tokens, and of all
  int range, q_ranges, kv_ranges, ranges;
  float one;                         // 1.0f, opaque to the compiler (adds as FMAs that cannot contract)
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

__device__ __forceinline__ float2 lohi(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 lohi(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// 8 consecutive values as loaded (16-byte aligned)
template <typename T> struct Piece {
  static constexpr int N = sizeof(T) / 2;  // 16-byte words
  uint4 w[N];
  __device__ __forceinline__ void load(const T* src) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint4*>(src)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void pairs(float2 (&f)[4]) const {
    if constexpr (sizeof(T) == 2) {
      f[0] = lohi(w[0].x, T()); f[1] = lohi(w[0].y, T());
      f[2] = lohi(w[0].z, T()); f[3] = lohi(w[0].w, T());
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[2 * i] = make_float2(__uint_as_float(w[i].x), __uint_as_float(w[i].y));
        f[2 * i + 1] = make_float2(__uint_as_float(w[i].z), __uint_as_float(w[i].w));
      }
    }
  }
};
template <typename T> __device__ __forceinline__ void load8(const T* src, float2 (&f)[4]) {
  Piece<T> x;
  x.load(src);
  x.pairs(f);
}
template <typename T> __device__ __forceinline__ void store8(T* dst, const float2 (&f)[4]) {
  if constexpr (sizeof(T) == 2) {
    uint4 w;
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[2 * i] = from_f32<T>(f[i].x);
      e[2 * i + 1] = from_f32<T>(f[i].y);
    }
    *reinterpret_cast<uint4*>(dst) = w;
  } else {
    reinterpret_cast<float4*>(dst)[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
    reinterpret_cast<float4*>(dst)[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
  }
}
__device__ __forceinline__ void load8_any(const void* p, int dtype, int64_t i, float2 (&f)[4]) {
  if (dtype == FXPR_BF16) load8(reinterpret_cast<const __nv_bfloat16*>(p) + i, f);
  else if (dtype == FXPR_F16) load8(reinterpret_cast<const __half*>(p) + i, f);
  else load8(reinterpret_cast<const float*>(p) + i, f);
}
__device__ __forceinline__ void store8_any(void* p, int dtype, int64_t i, const float2 (&f)[4]) {
  if (dtype == FXPR_BF16) store8(reinterpret_cast<__nv_bfloat16*>(p) + i, f);
  else if (dtype == FXPR_F16) store8(reinterpret_cast<__half*>(p) + i, f);
  else store8(reinterpret_cast<float*>(p) + i, f);
}

// max |x| of the 16 values of a 16-bit type, as an fp32 value (NaN stays NaN)
template <typename T> __device__ __forceinline__ float absmax(const Piece<T>& a, const Piece<T>& b) {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  const T2* x = reinterpret_cast<const T2*>(a.w);
  const T2* y = reinterpret_cast<const T2*>(b.w);
  T2 m = __hmax2_nan(__habs2(x[0]), __habs2(y[0]));
#pragma unroll
  for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __hmax2_nan(__habs2(x[i]), __habs2(y[i])));
  const float2 f = lohi(*reinterpret_cast<const uint32_t*>(&m), T());
  return f.x < f.y ? f.y : (f.y <= f.x ? f.x : __int_as_float(0x7FFFFFFF));  // NaN in either: NaN
}

// Integer sum of F2X(x^2) over 16 values. For 16-bit types x^2 is exact in
// fp32, so one packed FMA with the scale-absorbing constant 1.5 * 2^(23-f)
// rounds two squares to the 2^-f grid at once (`cf2`), as long as every
// x^2 * 2^f < 2^22 (no saturation and one binade); `thr` is that bound on |x|.
// Else, and for fp32 values, the clamp-and-convert form of the definition.
// 28 instead of 112 instructions, which is most of what the norm costs.
template <int BITS, typename T, typename UAcc>
__device__ __forceinline__ UAcc square_sum(const Piece<T>& a, const Piece<T>& b, const float2 (&xa)[4],
                                           const float2 (&xb)[4], float thr, float2 cf2, float scale) {
  if constexpr (sizeof(T) == 2) {
    if (absmax(a, b) < thr) {
      uint32_t acc = 0u - 16u * __float_as_uint(cf2.x);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 ra = fma2(xa[e], xa[e], cf2), rb = fma2(xb[e], xb[e], cf2);
        acc += __float_as_uint(ra.x) + __float_as_uint(ra.y);
        acc += __float_as_uint(rb.x) + __float_as_uint(rb.y);
      }
      return (UAcc)acc;  // at most 16 * 2^22: not negative
    }
  }
  UAcc acc = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    acc += (UAcc)f2x_f32<BITS>(__fmul_rn(xa[e].x, xa[e].x), scale);
    acc += (UAcc)f2x_f32<BITS>(__fmul_rn(xa[e].y, xa[e].y), scale);
    acc += (UAcc)f2x_f32<BITS>(__fmul_rn(xb[e].x, xb[e].x), scale);
    acc += (UAcc)f2x_f32<BITS>(__fmul_rn(xb[e].y, xb[e].y), scale);
  }
  return acc;
}

// x * c + y * s with each product and the sum rounded by itself: the add is an
// FMA by a runtime 1.0, which the compiler cannot fuse with the products
__device__ __forceinline__ float2 turn2(float2 x, float2 c, float2 y, float2 s, float2 one) {
  return fma2(mul2(x, c), one, mul2(y, s));
}

// The rows of one CTA: heads [0, n) from the pointers on, for this lane's
// token and pieces. SQ: accumulator width of the norm, 0 = none.
template <typename T> using Ring = uint4[STAGES<T>][2 * Piece<T>::N][THREADS];

template <typename T, int SQ, int LPR, bool TURN>
__device__ __forceinline__ void walk(const Params& p, Ring<T>& ring, int part, bool active, bool turn, int lo, int hi, const T* src,
                                     int64_t src_step, T* dst, int64_t dst_step, bool cached, int64_t cache_at,
                                     int64_t cache_step, int n, const float2 (&cs)[4], const float2 (&sn)[4]) {
  constexpr int BITS = SQ == 0 ? 32 : SQ;
  using UAcc = typename std::conditional<BITS == 64, unsigned long long, uint32_t>::type;
  // rows in flight: a ring of 16-byte words that only this thread reads
  constexpr int NW = Piece<T>::N, S = STAGES<T>;
  const int gap = hi - lo;
  const T* next = src + lo;
  auto fetch = [&](int h) {
    if (active && h < n) {
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        cp_async16(&ring[h % S][i][threadIdx.x], reinterpret_cast<const uint4*>(next) + i, 16);
        cp_async16(&ring[h % S][NW + i][threadIdx.x], reinterpret_cast<const uint4*>(next + gap) + i, 16);
      }
    }
    cp_async_commit();
    next += src_step;
  };
#pragma unroll
  for (int h = 0; h < S - 1; ++h) fetch(h);
  const float2 one = make_float2(p.one, p.one);
  float2 wa[4] = {}, wb[4] = {};
  float scale = 0.0f, thr = 0.0f;
  float2 cf2 = {};
  if constexpr (SQ != 0) {
    if (active) {
      load8_any(p.w[part], p.w_dtype, lo, wa);
      load8_any(p.w[part], p.w_dtype, hi, wb);
    }
    scale = ldexpf(1.0f, p.frac);
    const float cf = ldexpf(1.5f, 23 - p.frac);
    cf2 = make_float2(cf, cf);
    // |x| < thr: x^2 * 2^f < 2^22 (int16: < 2^14, no saturation); rounded down
    thr = __fsqrt_rd(ldexpf(1.0f, (BITS == 16 ? 14 : 22) - p.frac));
  }
  T* out = dst + lo;
  int64_t cat = cache_at + lo;
  auto row = [&](const Piece<T>& pa, const Piece<T>& pb) {
    float2 xa[4], xb[4];
    pa.pairs(xa);
    pb.pairs(xb);
    if constexpr (SQ != 0) {
      UAcc acc = square_sum<BITS, T, UAcc>(pa, pb, xa, xb, thr, cf2, scale);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      const float rrms = rrms_of<BITS>((typename Acc<BITS>::T)acc, p.dim, p.eps, p.frac);
      const float2 rr = make_float2(rrms, rrms);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        xa[e] = mul2(mul2(xa[e], wa[e]), rr);
        xb[e] = mul2(mul2(xb[e], wb[e]), rr);
      }
    }
    if (TURN && turn) {
      if (p.neox) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = xa[e], b = xb[e];
          xa[e] = turn2(a, cs[e], b, make_float2(-sn[e].x, -sn[e].y), one);
          xb[e] = turn2(b, cs[e], a, sn[e], one);
        }
      } else {
        // the pairs are (x, y) of one float2; cos and sin of pair i are half i % 2 of cs[i / 2], sn[i / 2]
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float ca = e % 2 ? cs[e / 2].y : cs[e / 2].x, sa = e % 2 ? sn[e / 2].y : sn[e / 2].x;
          const float cb = e % 2 ? cs[2 + e / 2].y : cs[2 + e / 2].x, sb = e % 2 ? sn[2 + e / 2].y : sn[2 + e / 2].x;
          xa[e] = turn2(xa[e], make_float2(ca, ca), make_float2(xa[e].y, xa[e].x), make_float2(-sa, sa), one);
          xb[e] = turn2(xb[e], make_float2(cb, cb), make_float2(xb[e].y, xb[e].x), make_float2(-sb, sb), one);
        }
      }
    }
    if (active && dst != nullptr) {
      store8(out, xa);
      store8(out + gap, xb);
    }
    out += dst_step;
    if (cached) {
      store8_any(p.cache[part - 1], p.c_dtype, cat, xa);
      store8_any(p.cache[part - 1], p.c_dtype, cat + gap, xb);
    }
    cat += cache_step;
  };
  for (int h = 0; h < n; ++h) {  // uniform over the CTA
    cp_async_wait<S - 2>();
    Piece<T> a, b;
    a.zero();
    b.zero();
    if (active) {
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        a.w[i] = ring[h % S][i][threadIdx.x];
        b.w[i] = ring[h % S][NW + i][threadIdx.x];
      }
    }
    fetch(h + S - 1);  // into the words read in the iteration before
    row(a, b);
  }
}

// NORM: accumulator width of the norm, 0 = none
template <typename T, int NORM, int LPR>
__global__ void __launch_bounds__(THREADS, MINB) rope_vec_kernel(const __grid_constant__ Params p) {
  __shared__ Ring<T> ring;
  const int64_t tok = (int64_t)(blockIdx.x / p.ranges) * (THREADS / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR;  // this lane's pair of pieces
  const bool active = tok < p.tokens && c < p.dim / 16;
  const int rp = p.rot / 16;        // pairs of pieces that are rotated
  const int lo = c < rp && p.neox ? 8 * c : 16 * c;
  const int hi = c < rp && p.neox ? lo + p.rot / 2 : lo + 8;
  // this CTA's heads: range blockIdx.x % ranges of q's, then k's, then v's ranges
  int part = 0, range = (int)(blockIdx.x % p.ranges);
  if (range >= p.q_ranges) {
    part = 1;
    range -= p.q_ranges;
    if (range >= p.kv_ranges) {
      part = 2;
      range -= p.kv_ranges;
    }
  }
  const int h0 = range * p.range;
  const int n = min(p.range, (part == 0 ? p.heads : p.kv_heads) - h0);
  const int64_t t = active ? tok : 0;
  const T* src = reinterpret_cast<const T*>(p.x[part]) + t * p.x_st[part] + h0 * p.x_sh[part];
  int64_t cache_at = 0, slot = -1;
  if (part > 0) {
    if (active) slot = slot_of(p, tok);
    if (slot >= 0) cache_at = cache_offset(p, part - 1, slot, h0);
  }
  const int64_t cache_step = part > 0 ? p.c_sh[part - 1] : 0;
  float2 cs[4], sn[4];
  if (part == 2) {
    walk<T, 0, LPR, false>(p, ring, 2, active, false, lo, hi, src, p.x_sh[2], nullptr, 0, slot >= 0, cache_at, cache_step, n, cs, sn);
    return;
  }
  const bool turn = active && c < rp;
#pragma unroll
  for (int e = 0; e < 4; ++e) cs[e] = sn[e] = make_float2(__int_as_float(0x7FFFFFFF), __int_as_float(0x7FFFFFFF));
  if (turn) {
    const int64_t pos = position_of(p, tok);
    if (pos >= 0 && pos < p.t_rows) {  // no angle outside the table
      load8_any(p.table, p.t_dtype, pos * p.t_stride + 8 * c, cs);
      load8_any(p.table, p.t_dtype, pos * p.t_stride + p.rot / 2 + 8 * c, sn);
    }
  }
  T* dst = reinterpret_cast<T*>(p.y[part]);
  if (dst != nullptr) dst += t * p.y_st[part] + h0 * p.y_sh[part];
  walk<T, NORM, LPR, true>(p, ring, part, active, turn, lo, hi, src, p.x_sh[part], dst, p.y_sh[part], slot >= 0, cache_at,
                           cache_step, n, cs, sn);
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
// Heads per CTA, halved while the CTAs do not fill the GPU. At the sizes above
// 16 heads 37.0 / 37.1 us; one token: one head per CTA, 3.1 us in a graph, 2
// of which are the empty launch.
constexpr int RANGE = 8;

template <typename T, int NORM, int LPR>
static int launch_vec(Params p, int rows, cudaStream_t st) {
  const int64_t bx = cdiv(p.tokens, THREADS / LPR);
  p.range = RANGE;
  while (p.range > 1 && bx * cdiv(rows, p.range) < (int64_t)num_sms() * MINB) p.range /= 2;
  p.q_ranges = (int)cdiv(p.heads, p.range);
  p.kv_ranges = (int)cdiv(p.kv_heads, p.range);
  p.ranges = p.q_ranges + p.kv_ranges * (p.cache[0] ? 2 : 1);
  if (bx * p.ranges > 0x7fffffffLL) {
    set_error("rope: too many rows");
    return FXPR_ERR_INVALID;
  }
  rope_vec_kernel<T, NORM, LPR><<<(unsigned)(bx * p.ranges), THREADS, 0, st>>>(p);
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
  p.eps = a->eps; p.frac = a->frac_bits; p.one = 1.0f;
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
