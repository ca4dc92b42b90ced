// Block-scaled KV cache: append (quantize a block when it is complete) and read back; norms of
// queries and keys for each head with the position rotation; and the joined form of a decode
// step, which does both from the fused q|k|v row in one launch. Layout: block_kv.cuh.
#include "block_kv.cuh"

#include <cstring>

namespace lq {
namespace {

constexpr int kThreads = 256;
constexpr int kMostPieces = 8;  // of 8 values that a thread holds of one block: 128 * 128 / 8 / 256

// 8 consecutive values as they lie in memory, moved as 16-byte words
template <typename T>
struct Pack8 {
  uint4 w[sizeof(T) / 2];
};

// `vec` = every row of the tensor starts on a 16-byte boundary
template <typename T>
__device__ __forceinline__ Pack8<T> load8(const T* p, bool vec) {
  Pack8<T> r;
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i];
    memcpy(&r, v, sizeof(r));
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Pack8<T>& r, bool vec) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
  } else {
    T v[8];
    memcpy(v, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = v[i];
  }
}
template <typename T>
__device__ __forceinline__ Pack8<T> zeros8() {
  Pack8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = make_uint4(0u, 0u, 0u, 0u);
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Pack8<T>& r, float (&x)[8]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = pair_of<T>(w[i]);
    x[2 * i] = p.x;
    x[2 * i + 1] = p.y;
  }
}
template <>
__device__ __forceinline__ void unpack8<float>(const Pack8<float>& r, float (&x)[8]) {
  const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
}
template <typename T>
__device__ __forceinline__ Pack8<T> pack8(const float (&x)[8]) {
  Pack8<T> r;
  r.w[0] = make_uint4(pair_to<T>(x[0], x[1]), pair_to<T>(x[2], x[3]), pair_to<T>(x[4], x[5]), pair_to<T>(x[6], x[7]));
  return r;
}
template <>
__device__ __forceinline__ Pack8<float> pack8<float>(const float (&x)[8]) {
  Pack8<float> r;
  r.w[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  r.w[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
  return r;
}

// Two times four consecutive values (at elements a and b of a row)
template <typename T>
__device__ __forceinline__ Pack8<T> load44(const T* row, int a, int b, bool vec) {
  Pack8<T> r;
  if (vec) {
    if (sizeof(T) == 2) {
      const uint2 x = *reinterpret_cast<const uint2*>(row + a), y = *reinterpret_cast<const uint2*>(row + b);
      r.w[0] = make_uint4(x.x, x.y, y.x, y.y);
    } else {
      r.w[0] = *reinterpret_cast<const uint4*>(row + a);
      r.w[sizeof(T) / 2 - 1] = *reinterpret_cast<const uint4*>(row + b);
    }
  } else {
    T v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = row[a + i]; v[4 + i] = row[b + i]; }
    memcpy(&r, v, sizeof(r));
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store44(T* row, int a, int b, const Pack8<T>& r, bool vec) {
  if (vec) {
    if (sizeof(T) == 2) {
      *reinterpret_cast<uint2*>(row + a) = make_uint2(r.w[0].x, r.w[0].y);
      *reinterpret_cast<uint2*>(row + b) = make_uint2(r.w[0].z, r.w[0].w);
    } else {
      *reinterpret_cast<uint4*>(row + a) = r.w[0];
      *reinterpret_cast<uint4*>(row + b) = r.w[sizeof(T) / 2 - 1];
    }
  } else {
    T v[8];
    memcpy(v, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < 4; ++i) { row[a + i] = v[i]; row[b + i] = v[4 + i]; }
  }
}

// ---------------------------------------------------------------- norm + rotation of one head
struct Rope {
  const float* cos;  // [table_len, rot / 2]
  const float* sin;
  int64_t table_len;
  int rot;
  int interleaved;
  float eps;
};

// The 8 values that lane li of a head's lanes holds: four from `a` on and four from `b` on, chosen so
// that it has both values of each of its pairs and the rotation exchanges nothing between lanes.
struct Hold {
  int a, b;
};
__device__ __forceinline__ Hold hold_of(int li, const Rope& rp) {
  const bool halves = !rp.interleaved && li * 8 < rp.rot;
  return halves ? Hold{li * 4, rp.rot / 2 + li * 4} : Hold{li * 8, li * 8 + 4};
}

// Cosines and sines of the lane's four pairs at a position (1 and 0 behind the rotated values).
struct Angles {
  float4 c, s;
};
__device__ __forceinline__ Angles angles_of(const Rope& rp, int64_t pos, int li) {
  Angles a{make_float4(1.f, 1.f, 1.f, 1.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  if (li * 8 < rp.rot) {
    a.c = *reinterpret_cast<const float4*>(rp.cos + pos * (rp.rot / 2) + li * 4);
    a.s = *reinterpret_cast<const float4*>(rp.sin + pos * (rp.rot / 2) + li * 4);
  }
  return a;
}
// (p, q) -> (p cos - q sin, q cos + p sin)
__device__ __forceinline__ void turn(float& p, float& q, float c, float s) {
  const float x = __fmaf_rn(p, c, -__fmul_rn(q, s));
  q = __fmaf_rn(q, c, __fmul_rn(p, s));
  p = x;
}

// y = x * rsqrt(mean(x^2) + eps) * w over a head, then the rotation of its first rp.rot values, a
// pair being (i, i + rot/2) or, interleaved, (2i, 2i + 1). GRP lanes hold a head; all 32 lanes of
// the warp call this together. fp32 throughout, every operation named, so that the joined and the
// separate forms round alike; the caller rounds once.
template <int GRP>
__device__ __forceinline__ void norm_rope8(float (&x)[8], float inv_D, const float* w, const Rope& rp, const Angles& a) {
  if (w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __fmaf_rn(x[i], x[i], ss);
#pragma unroll
    for (int o = GRP / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(__fmaf_rn(ss, inv_D, rp.eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], r), w[i]);
  }
  if (rp.interleaved) {
    turn(x[0], x[1], a.c.x, a.s.x);
    turn(x[2], x[3], a.c.y, a.s.y);
    turn(x[4], x[5], a.c.z, a.s.z);
    turn(x[6], x[7], a.c.w, a.s.w);
  } else {
    turn(x[0], x[4], a.c.x, a.s.x);
    turn(x[1], x[5], a.c.y, a.s.y);
    turn(x[2], x[6], a.c.z, a.s.z);
    turn(x[3], x[7], a.c.w, a.s.w);
  }
}

template <typename T>
struct NormRopeArgs {
  const T *q, *k;
  T *q_out, *k_out;
  int64_t qs[3], ks[3], qos[3], kos[3];  // element strides of (b, t, head)
  const int64_t* positions;
  int64_t ps[2];
  const T *q_weight, *k_weight;
  int B, T_new, Hq, Hk, D, heads_per_item, q_items, k_items;  // items: lane groups for the heads of a token
};

// A group of GRP lanes owns one token and up to heads_per_item of its query heads, or of its key heads:
// the token's angles and the weights are loaded once and stay in registers. Bound by HBM (each
// value read and written once): 688 MB of bf16 heads of 128 in 125 us, 5.5 TB/s, 0.86 of a copy's rate.
// Two heads are worked on while the next two are on their way; four CTAs on an SM (138 us with three and
// four heads at a time, 139 without the requests ahead, 150 with five CTAs, whose registers spill).
template <typename T, int GRP, bool VEC>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 3 : 4)
qk_norm_rope_kernel(const NormRopeArgs<T> p, const Rope rp, int* error_word) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int li = threadIdx.x % GRP, each = p.q_items + p.k_items;
  const int64_t items = (int64_t)p.B * p.T_new * each;
  const int64_t item0 = (int64_t)blockIdx.x * (kThreads / GRP) + threadIdx.x / GRP;
  const bool live = item0 < items;
  const int64_t item = live ? item0 : items - 1;
  const int64_t token = item / each;
  const int chunk = (int)(item - token * each);
  const int b = (int)(token / p.T_new), t = (int)(token - (int64_t)b * p.T_new);
  const bool key = chunk >= p.q_items;
  const int lo = (key ? chunk - p.q_items : chunk) * p.heads_per_item;
  const bool mine = live && li * 8 < p.D;
  const int n = mine ? min(p.heads_per_item, (key ? p.Hk : p.Hq) - lo) : 0;
  const Hold own = mine ? hold_of(li, rp) : Hold{0, 4};
  const int step = (int)(key ? p.ks[2] : p.qs[2]), out_step = (int)(key ? p.kos[2] : p.qos[2]);
  const T* src = (key ? p.k + b * p.ks[0] + t * p.ks[1] + lo * p.ks[2] : p.q + b * p.qs[0] + t * p.qs[1] + lo * p.qs[2]);
  T* dst = (key ? p.k_out + b * p.kos[0] + t * p.kos[1] + lo * p.kos[2] : p.q_out + b * p.qos[0] + t * p.qos[1] + lo * p.qos[2]);
  constexpr int UN = 2;  // heads at a time, as many on their way
  Pack8<T> in[UN], next[UN];
  auto fetch = [&](Pack8<T> (&to)[UN], int h0) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      to[u] = zeros8<T>();
      if (h0 + u < n) to[u] = load44(src + (h0 + u) * step, own.a, own.b, VEC);
    }
  };
  fetch(in, 0);  // (before the position and the angles that wait for it)
  const int64_t at = p.positions[b * p.ps[0] + t * p.ps[1]];
  const bool known = at >= 0 && at < rp.table_len;
  if (!known && live && li == 0) atomicExch(error_word, LQ_BLOCK_BAD_ANGLE);
  const T* weight = key ? p.k_weight : p.q_weight;
  Pack8<T> w = zeros8<T>();
  if (weight != nullptr && mine) w = load44(weight, own.a, own.b, VEC);
  Angles a = angles_of(rp, known ? at : 0, mine ? li : 32);
  if (!known) a.c = a.s = make_float4(NAN, NAN, NAN, NAN);  // no angle: nothing usable
  const float inv_D = 1.f / p.D;
#pragma unroll 1
  for (int h0 = 0; h0 < p.heads_per_item; h0 += UN) {  // (the same trip count for the whole warp)
    fetch(next, h0 + UN);
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (h0 + u >= p.heads_per_item) break;
      float x[8], wf[8];
      unpack8(in[u], x);
      unpack8(w, wf);
      norm_rope8<GRP>(x, inv_D, weight != nullptr ? wf : nullptr, rp, a);
      if (h0 + u < n) store44(dst + (h0 + u) * out_step, own.a, own.b, pack8<T>(x), VEC);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) in[u] = next[u];
  }
}

// ---------------------------------------------------------------- append
// The largest magnitude of what a thread holds, INF if any of it is not finite. 16-bit values are
// compared as pairs (the comparison keeps NaN).
template <typename T>
struct Largest {
  float top = 0.f;
  __device__ __forceinline__ void take(const Pack8<T>& r) {
    float x[8];
    unpack8(r, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float m = fabsf(x[i]);
      top = m <= 3.402823466e38f ? fmaxf(top, m) : INFINITY;
    }
  }
  __device__ __forceinline__ float value() const { return top; }
};
template <typename T2>
struct LargestPair {
  T2 top;
  __device__ __forceinline__ LargestPair() { memset(&top, 0, sizeof(top)); }
  template <typename P>
  __device__ __forceinline__ void take(const P& r) {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const T2*>(&w[i])));
  }
  __device__ __forceinline__ float value(float lo, float hi) const {
    const float m = fmaxf(lo, hi);
    return lo <= 3.402823466e38f && hi <= 3.402823466e38f ? m : INFINITY;
  }
};
template <>
struct Largest<__half> : LargestPair<__half2> {
  __device__ __forceinline__ float value() const { return LargestPair::value(__low2float(top), __high2float(top)); }
};
template <>
struct Largest<__nv_bfloat16> : LargestPair<__nv_bfloat162> {
  __device__ __forceinline__ float value() const { return LargestPair::value(__low2float(top), __high2float(top)); }
};

// Codes of 8 values: rint(x / scale), the quotient rounded as IEEE division rounds it (many values lie on
// a half exactly, so a product with 1 / scale alone would decide wrongly). With inv = 1 / scale
// correctly rounded, one correction of x * inv by its exact remainder is the correctly rounded
// quotient (P. Markstein, IBM J. Res. Dev. 34, 1990, theorem 8.1); where the remainder underflows the
// quotient rounds to zero anyway. Adding 1.5 * 2^23 then rounds to the nearest even integer and
// leaves it in the low byte. |x| <= 127 scale up to rounding, so there is nothing to clamp.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float scale, float inv) {
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float near = __fmul_rn(x[i], inv);
    const float quotient = __fmaf_rn(__fmaf_rn(-near, scale, x[i]), inv, near);
    q[i] = __float_as_uint(__fadd_rn(quotient, 12582912.f));
  }
  const uint32_t lo = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  const uint32_t hi = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
  return make_uint2(lo, hi);
}

template <typename T>
struct AppendArgs {
  const T *k, *v;            // plain form: new rows
  int64_t ks[3], vs[3];      // element strides of (b, h, t)
  int vec;
  // joined form: q heads of the same rows, and where they go ([B, T, Hq, D])
  const T* q;
  int64_t qs[3];             // (b, h, t)
  T* q_out;
  int Hq;
  const T *q_weight, *k_weight;
};

// grid (blocks a call can touch, 2 * Hkv [+ CTAs for the query heads], B). A CTA owns one block
// of one KV head's keys or values: it copies the new rows that belong into the ring, and if the
// block is complete now it takes all P rows (older ones from the ring) into registers, finds
// their maximum and writes the codes. The block that the call begins in may read ring rows that
// a later block of the same parity replaces; its CTA then writes that later block's rows too,
// after its own reads. Every value goes through a maximum and a rounded quotient, about 20
// instructions with all that surrounds them: an SM issues 3.4 of them a cycle while 135 MB of bf16
// (8 prompts of 4111 tokens, 8 heads of 128) become 67 MB of codes in 43 us, 4.7 TB/s, 0.73 of a copy's
// rate. The instructions bound it, not the memory.
template <typename T, int D, bool JOINED, int kMaxVec>  // kMaxVec: pieces of 8 values a thread holds of a block
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : kMaxVec > 4 ? 4 : 5)
block_append_kernel(const lq_block_kv c, const BlockSpan sp, const AppendArgs<T> p, const Rope rp, int* error_word) {
  constexpr int LPR = D / 8;  // lanes that hold a row
  __shared__ float red[kThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int b = blockIdx.z, P = c.block;
  const int tid = threadIdx.x, li = tid % LPR;
  bool bad;
  const SeqSpan s = span_of(c, sp, b, bad);
  if (bad) {
    if (tid == 0 && blockIdx.x == 0) atomicExch(error_word, LQ_BLOCK_BAD_POSITION);
  }
  const int L = s.start + s.n;

  float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const bool query_cta = JOINED && (int)blockIdx.y >= 2 * c.kv_heads;
  const bool is_v = blockIdx.y & 1;
  const T* weight = !JOINED ? nullptr : (query_cta ? p.q_weight : p.k_weight);
  const Hold own = JOINED && (query_cta || !is_v) ? hold_of(li, rp) : Hold{li * 8, li * 8 + 4};
  if (JOINED && weight != nullptr) unpack8(load44(weight, own.a, own.b, p.vec), w);

  if (query_cta) {
    const int rows = sp.tokens * p.Hq;
    const int ctas = (gridDim.y - 2 * c.kv_heads) * gridDim.x;
    const int cta = (blockIdx.y - 2 * c.kv_heads) * gridDim.x + blockIdx.x;
    for (int r0 = cta * (kThreads / LPR); r0 < rows; r0 += ctas * (kThreads / LPR)) {
      const int r = r0 + tid / LPR;
      const bool row = r < rows;
      const int t = row ? r / p.Hq : 0, h = row ? r % p.Hq : 0;
      const bool fresh = row && t < s.n;
      const int64_t pos = s.start + t;
      const bool known = pos < rp.table_len;
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (fresh) unpack8(load44(p.q + b * p.qs[0] + h * p.qs[1] + t * p.qs[2], own.a, own.b, p.vec), x);
      const Angles a = angles_of(rp, fresh && known ? pos : 0, li);
      norm_rope8<LPR>(x, 1.f / D, weight != nullptr ? w : nullptr, rp, a);
      if (fresh && !known) {
        if (li == 0) atomicExch(error_word, LQ_BLOCK_BAD_ANGLE);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __int_as_float(0x7fffffff);
      }
      if (row) {
        if (!fresh) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = 0.f;  // rows behind the sequence's count
        }
        store44(p.q_out + (((int64_t)b * sp.tokens + t) * p.Hq + h) * D, own.a, own.b, pack8<T>(x), true);
      }
    }
    return;
  }

  const int h = blockIdx.y >> 1;
  const int shift = 31 - __clz(P), first = s.start >> shift, last = L >> shift;  // (P is a power of two)
  const int j = first + blockIdx.x;
  if (s.n == 0 || (int64_t)j * P >= L) return;
  const bool complete = (j + 1) * P <= L;
  const bool reads_ring = (s.start & (P - 1)) != 0 && (first + 1) * P <= L;  // the first block, completed by this call
  T* ring = reinterpret_cast<T*>(is_v ? c.v_ring : c.k_ring) + ((int64_t)b * c.kv_heads + h) * 2 * P * D;
  const T* src = is_v ? p.v + b * p.vs[0] + h * p.vs[1] : p.k + b * p.ks[0] + h * p.ks[1];
  const int64_t step = is_v ? p.vs[2] : p.ks[2];
  const bool turned = JOINED && !is_v;

  // this thread's 8 values of a row
  auto row_load = [&](const T* row, bool vec) { return JOINED ? load44(row, own.a, own.b, vec) : load8(row + li * 8, vec); };
  auto row_store = [&](T* row, const Pack8<T>& r) {
    if (JOINED) store44(row, own.a, own.b, r, true);
    else store8(row + li * 8, r, true);
  };
  // the same of a new row; every lane of the warp calls it
  auto fetch = [&](int pos, bool fresh) {
    Pack8<T> r = zeros8<T>();
    if (fresh) r = row_load(src + (int64_t)(pos - s.start) * step, p.vec);
    if (turned) {
      float x[8];
      unpack8(r, x);
      const bool known = pos < rp.table_len;
      const Angles a = angles_of(rp, fresh && known ? pos : 0, li);
      norm_rope8<LPR>(x, 1.f / D, weight != nullptr ? w : nullptr, rp, a);
      if (fresh && !known) {
        if (li == 0) atomicExch(error_word, LQ_BLOCK_BAD_ANGLE);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __int_as_float(0x7fffffff);
      }
      r = pack8<T>(x);
    }
    return r;
  };

  const bool to_ring = j >= last - 1 && !(reads_ring && j != first && ((j ^ first) & 1) == 0);
  const int pieces = P * LPR;
  const int64_t page = complete ? page_of(c, b, j) : 0;  // (on its way while the rows are)
  Pack8<T> val[kMaxVec];
  Largest<T> top;
  constexpr int kStep = kThreads / LPR;  // rows between two pieces of a thread
  const int row0 = tid / LPR;
  if (complete && j * P >= s.start && !to_ring) {  // the inside of a long prompt: nothing but new rows to codes
    const T* row = src + (int64_t)(j * P + row0 - s.start) * step;
#pragma unroll
    for (int v = 0; v < kMaxVec; ++v) {
      if (v * kThreads < pieces) {
        val[v] = turned ? fetch(j * P + row0 + v * kStep, row0 + v * kStep < P)
                        : (row0 + v * kStep < P ? row_load(row, p.vec) : zeros8<T>());
        row += kStep * step;
      }
    }
#pragma unroll
    for (int v = 0; v < kMaxVec; ++v)
      if (v * kThreads < pieces) top.take(val[v]);
  } else {
#pragma unroll
    for (int v = 0; v < kMaxVec; ++v) {
      if (v * kThreads < pieces) {
        const int idx = tid + v * kThreads, pos = j * P + row0 + v * kStep;
        const bool inside = idx < pieces;
        const bool fresh = inside && pos >= s.start && pos < L;
        T* held = ring + (int64_t)(pos & (2 * P - 1)) * D;
        val[v] = fetch(pos, fresh);
        if (inside && complete && pos < s.start) val[v] = row_load(held, true);
        if (fresh && to_ring) row_store(held, val[v]);
        if (complete) top.take(val[v]);
      }
    }
  }
  if (!complete) return;
  float amax = warp_max(top.value());
  if ((tid & 31) == 0) red[tid >> 5] = amax;
  __syncthreads();  // (also: every read of the ring above is done)
  amax = red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) amax = fmaxf(amax, red[i]);
  const bool finite = amax <= 3.402823466e38f;
  const float scale = finite ? scale_of(amax, 127.f) : __int_as_float(0x7fffffff);
  const float inv = finite ? __fdiv_rn(1.f, scale) : 0.f;
  if (page < 0) {
    if (tid == 0) atomicExch(error_word, LQ_BLOCK_BAD_PAGE);
  } else {
    const int64_t ph = page * c.kv_heads + h;
    if (tid == 0) (is_v ? c.v_scales : c.k_scales)[ph] = scale;
    int8_t* codes = (is_v ? c.v_pages : c.k_pages) + ph * P * D;
#pragma unroll
    for (int v = 0; v < kMaxVec; ++v) {
      const int idx = tid + v * kThreads;
      if (idx < pieces) {
        float x[8];
        unpack8(val[v], x);
        const uint2 q = finite ? codes8(x, scale, inv) : make_uint2(0u, 0u);
        if (JOINED) {
          int8_t* row = codes + (int64_t)(idx / LPR) * D;
          *reinterpret_cast<uint32_t*>(row + own.a) = q.x;
          *reinterpret_cast<uint32_t*>(row + own.b) = q.y;
        } else {
          *reinterpret_cast<uint2*>(codes + (int64_t)idx * 8) = q;
        }
      }
    }
  }
  if (j == first && reads_ring) {
    for (int jx = max(last - 1, first + 1); jx <= last; ++jx) {
      if ((jx ^ first) & 1) continue;
      for (int v = 0; v * kThreads < pieces; ++v) {
        const int idx = tid + v * kThreads;
        const int pos = jx * P + idx / LPR;
        const bool fresh = idx < pieces && pos < L;
        const Pack8<T> r = fetch(pos, fresh);
        if (fresh) row_store(ring + (int64_t)(pos & (2 * P - 1)) * D, r);
      }
    }
  }
}

// ---------------------------------------------------------------- read back
// grid (blocks of the output, 2 * Hkv, B): code * scale rounded once, rows of the incomplete block
// as they are, zeros behind the sequence. Bound by HBM: 67 MB of codes to 135 MB of bf16 in 33 us,
// 6.1 TB/s, 0.95 of a copy's rate.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads)
block_read_kernel(const lq_block_kv c, const BlockSpan sp, T* __restrict__ k_out, T* __restrict__ v_out, int length,
                  int* error_word) {
  constexpr int LPR = D / 8;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int b = blockIdx.z, h = blockIdx.y >> 1, j = blockIdx.x, P = c.block, tid = threadIdx.x;
  const bool is_v = blockIdx.y & 1;
  bool bad;
  const SeqSpan s = span_of(c, sp, b, bad);
  if (bad && tid == 0 && j == 0) atomicExch(error_word, LQ_BLOCK_BAD_POSITION);
  const int L = s.start + s.n;
  const int64_t bh = (int64_t)b * c.kv_heads + h;
  T* out = (is_v ? v_out : k_out) + (bh * length + (int64_t)j * P) * D;
  const int rows = min(P, length - j * P);
  const bool complete = (int64_t)(j + 1) * P <= L;
  const int8_t* codes = nullptr;
  float scale = 0.f;
  if (complete) {
    const int64_t page = page_of(c, b, j);
    if (page < 0) {
      if (tid == 0) atomicExch(error_word, LQ_BLOCK_BAD_PAGE);
    } else {
      const int64_t ph = page * c.kv_heads + h;
      codes = (is_v ? c.v_pages : c.k_pages) + ph * P * D;
      scale = (is_v ? c.v_scales : c.k_scales)[ph];
    }
  }
  const T* ring = reinterpret_cast<const T*>(is_v ? c.v_ring : c.k_ring) + bh * 2 * P * D;
  const float nan = __int_as_float(0x7fffffff);
  if (complete) {
    uint2 raw[kMostPieces];
#pragma unroll
    for (int v = 0; v < kMostPieces; ++v) {
      const int idx = tid + v * kThreads;
      raw[v] = make_uint2(0u, 0u);
      if (idx < rows * LPR && codes != nullptr) raw[v] = *reinterpret_cast<const uint2*>(codes + (int64_t)idx * 8);
    }
#pragma unroll
    for (int v = 0; v < kMostPieces; ++v) {
      const int idx = tid + v * kThreads;
      if (idx >= rows * LPR) break;
      const int8_t* q = reinterpret_cast<const int8_t*>(&raw[v]);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = codes != nullptr ? __fmul_rn((float)q[i], scale) : nan;
      store8(out + (int64_t)idx * 8, pack8<T>(x), true);
    }
    return;
  }
  for (int idx = tid; idx < rows * LPR; idx += kThreads) {
    const int pos = j * P + idx / LPR;
    Pack8<T> r = zeros8<T>();
    if (pos < L) r = load8(ring + (int64_t)(pos & (2 * P - 1)) * D + (idx % LPR) * 8, true);
    store8(out + (int64_t)idx * 8, r, true);
  }
}

__device__ int g_block_error = 0;

template <typename Kern, typename... Args>
int launch(Kern kern, dim3 grid, cudaStream_t stream, int pdl, const char* what, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(LQ_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  }
  return LQ_OK;
}

int check_rope(const float* cos, const float* sin, int64_t table_len, int rot, int D) {
  LQ_REQUIRE(cos && sin && table_len > 0, LQ_ERR_ARG, "the angle tables are missing or empty");
  LQ_REQUIRE(rot > 0 && rot <= D && rot % 16 == 0, LQ_ERR_ARG,
             "the rotated part must be a multiple of 16 values of the head (%d), got %d", D, rot);
  LQ_REQUIRE(((uintptr_t)cos | (uintptr_t)sin) % 16 == 0, LQ_ERR_ARG, "the angle tables must be 16-byte aligned");
  return LQ_OK;
}

bool aligned_rows(const void* p, const int64_t* strides, int n, size_t elem) {
  bool ok = (uintptr_t)p % 16 == 0;
  for (int i = 0; i < n; ++i) ok = ok && (strides[i] * (int64_t)elem) % 16 == 0;
  return ok;
}

template <typename T>
int append(const lq_block_kv& c, const BlockSpan& sp, AppendArgs<T>& p, const Rope& rp, bool joined, int pdl,
           void* stream, const char* what) {
  int* error_word = block_error_word();
  if (error_word == nullptr) return LQ_ERR_LAUNCH;
  // the most blocks `tokens` rows can touch, whatever the first one's offset
  const int touched = (int)(((int64_t)c.block + sp.tokens - 2) / c.block) + 1;
  unsigned y = 2u * c.kv_heads;
  if (joined) {
    const int64_t passes = ((int64_t)sp.tokens * p.Hq + kThreads / (c.head_dim / 8) - 1) / (kThreads / (c.head_dim / 8));
    y += (unsigned)((passes + touched - 1) / touched);
  }
  LQ_REQUIRE(y <= 65535, LQ_ERR_ARG, "%s: too many heads or tokens for one launch", what);
  const dim3 grid((unsigned)touched, y, (unsigned)c.batch);
  const cudaStream_t s = (cudaStream_t)stream;
  // blocks of up to 8192 values leave a thread 4 pieces, fewer registers and so more CTAs on an SM
  // (whole prompts, blocks of 64 x 128 and their read: 89 us with four CTAs, 77 with five, 79 with six)
  const bool few = c.block * c.head_dim <= 4 * 8 * kThreads;
#define LQ_APPEND(DD, JJ)                                                                                    \
  return few ? launch(block_append_kernel<T, DD, JJ, 4>, grid, s, pdl, what, c, sp, p, rp, error_word)           \
             : launch(block_append_kernel<T, DD, JJ, kMostPieces>, grid, s, pdl, what, c, sp, p, rp, error_word)
  if (c.head_dim == 64) {
    if (joined) LQ_APPEND(64, true);
    LQ_APPEND(64, false);
  }
  if (joined) LQ_APPEND(128, true);
  LQ_APPEND(128, false);
#undef LQ_APPEND
}

}  // namespace

int* block_error_word() {
  static thread_local int cached_dev = -1;
  static thread_local int* cached = nullptr;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    fail(LQ_ERR_LAUNCH, "no current device");
    return nullptr;
  }
  if (dev != cached_dev) {
    void* ptr = nullptr;
    if (cudaGetSymbolAddress(&ptr, g_block_error) != cudaSuccess) {
      cudaGetLastError();
      fail(LQ_ERR_LAUNCH, "cannot resolve the device error word");
      return nullptr;
    }
    cached = (int*)ptr;
    cached_dev = dev;
  }
  return cached;
}

int check_block_kv(const lq_block_kv* c, const char* what) {
  LQ_REQUIRE(c != nullptr, LQ_ERR_ARG, "%s: no cache given", what);
  LQ_REQUIRE(c->batch > 0 && c->batch <= 65535 && c->kv_heads > 0 && c->num_pages > 0 && c->max_blocks > 0, LQ_ERR_ARG,
             "%s: bad cache shape (batch %d, %d heads, %d blocks)", what, c->batch, c->kv_heads, c->max_blocks);
  LQ_REQUIRE(c->head_dim == 64 || c->head_dim == 128, LQ_ERR_UNSUPPORTED,
             "%s: the block-scaled cache is built for head_dim 64 and 128, got %d", what, c->head_dim);
  LQ_REQUIRE(c->block == 16 || c->block == 32 || c->block == 64 || c->block == 128, LQ_ERR_UNSUPPORTED,
             "%s: a block is 16, 32, 64 or 128 tokens, got %d", what, c->block);
  LQ_REQUIRE(c->num_pages <= 0x7fffffffLL / c->kv_heads, LQ_ERR_ARG, "%s: the pool has too many pages", what);
  LQ_REQUIRE((int64_t)c->max_blocks * c->block <= 0x7fff0000LL, LQ_ERR_ARG, "%s: the table spans too many positions", what);
  LQ_REQUIRE(c->dtype == LQ_F32 || c->dtype == LQ_F16 || c->dtype == LQ_BF16, LQ_ERR_DTYPE,
             "%s: the cache's dtype must be float32, float16 or bfloat16, got dtype id %d", what, c->dtype);
  LQ_REQUIRE(c->k_pages && c->v_pages && c->k_scales && c->v_scales && c->k_ring && c->v_ring && c->table, LQ_ERR_ARG,
             "%s: null cache pointer", what);
  LQ_REQUIRE((((uintptr_t)c->k_pages | (uintptr_t)c->v_pages | (uintptr_t)c->k_ring | (uintptr_t)c->v_ring) & 15) == 0,
             LQ_ERR_ARG, "%s: pages and rings must be 16-byte aligned", what);
  return LQ_OK;
}

}  // namespace lq

using namespace lq;

extern "C" int lq_block_kv_device_error(void) {
  int* ptr = block_error_word();
  if (ptr == nullptr) return -1;
  int value = 0;
  if (cudaMemcpy(&value, ptr, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) { cudaGetLastError(); return -1; }
  if (value != 0) cudaMemset(ptr, 0, sizeof(int));
  return value;
}

extern "C" int lq_qk_norm_rope(const void* q, const void* k, const int64_t* q_strides, const int64_t* k_strides,
                               void* q_out, void* k_out, const int64_t* q_out_strides, const int64_t* k_out_strides,
                               int dtype, int B, int T_new, int Hq, int Hk, int D, const void* q_weight,
                               const void* k_weight, float eps, const float* cos_table, const float* sin_table,
                               int64_t table_len, int rot, int interleaved, const int64_t* positions, int64_t pos_stride_b,
                               int64_t pos_stride_t, int pdl, void* stream) {
  LQ_REQUIRE(B > 0 && T_new > 0 && Hq >= 0 && Hk >= 0 && Hq + Hk > 0, LQ_ERR_ARG, "bad shape");
  LQ_REQUIRE(D % 8 == 0 && D >= 16 && D <= 256, LQ_ERR_UNSUPPORTED,
             "head_dim must be a multiple of 8 in [16, 256], got %d", D);
  LQ_REQUIRE((Hq == 0 || (q && q_out)) && (Hk == 0 || (k && k_out)) && positions, LQ_ERR_ARG, "null tensor pointer");
  LQ_REQUIRE(Hq == 0 || Hk == 0 || (q_weight != nullptr) == (k_weight != nullptr), LQ_ERR_ARG,
             "norm weights are given for both queries and keys or for neither");
  if (const int rc = check_rope(cos_table, sin_table, table_len, rot, D)) return rc;
  int* error_word = nullptr;
  LQ_REQUIRE(dtype == LQ_F32 || dtype == LQ_F16 || dtype == LQ_BF16, LQ_ERR_DTYPE,
             "q and k must be float32, float16 or bfloat16, got dtype id %d", dtype);
  if ((error_word = block_error_word()) == nullptr) return LQ_ERR_LAUNCH;
  const Rope rp{cos_table, sin_table, table_len, rot, interleaved, eps};
  const int grp = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32;
  const int64_t rows = (int64_t)B * T_new * (Hq + Hk);
  // One head to a lane group while that leaves SMs idle; eight once there are rows enough for
  // eight CTAs on every SM: the angles are then loaded once for eight heads.
  const int64_t busy = rows / ((int64_t)sm_count() * 8 * (kThreads / grp));
  int64_t widest = 0;  // (heads of a group are addressed by 32-bit offsets)
  for (const int64_t v : {Hq ? q_strides[2] : 0, Hk ? k_strides[2] : 0, Hq ? q_out_strides[2] : 0, Hk ? k_out_strides[2] : 0})
    widest = v > widest ? v : -v > widest ? -v : widest;
  const int per = widest > 0x7fffffffLL / 8 ? 1 : busy >= 8 ? 8 : busy >= 4 ? 4 : busy >= 2 ? 2 : 1;
  const int q_items = (Hq + per - 1) / per, k_items = (Hk + per - 1) / per;
  const int64_t groups = (int64_t)B * T_new * (q_items + k_items);
  const int64_t ctas = (groups + kThreads / grp - 1) / (kThreads / grp);
  LQ_REQUIRE(ctas <= 0x7fffffffLL, LQ_ERR_ARG, "too many rows for one launch");
#define LQ_GRP(G)                                                                             \
  if (grp == G)                                                                               \
    return vec ? launch(qk_norm_rope_kernel<T, G, true>, grid, s, pdl, what, p, rp, error_word) \
               : launch(qk_norm_rope_kernel<T, G, false>, grid, s, pdl, what, p, rp, error_word);
  LQ_DISPATCH_DTYPE(dtype, T, {
    NormRopeArgs<T> p;
    p.q = (const T*)q; p.k = (const T*)k; p.q_out = (T*)q_out; p.k_out = (T*)k_out;
    bool vec = true;
    for (int i = 0; i < 3; ++i) {
      p.qs[i] = Hq ? q_strides[i] : 0; p.ks[i] = Hk ? k_strides[i] : 0;
      p.qos[i] = Hq ? q_out_strides[i] : 0; p.kos[i] = Hk ? k_out_strides[i] : 0;
    }
    vec = aligned_rows(q, p.qs, 3, sizeof(T)) && aligned_rows(k, p.ks, 3, sizeof(T)) &&
          aligned_rows(q_out, p.qos, 3, sizeof(T)) && aligned_rows(k_out, p.kos, 3, sizeof(T)) &&
          ((uintptr_t)q_weight | (uintptr_t)k_weight) % 16 == 0;
    p.positions = positions; p.ps[0] = pos_stride_b; p.ps[1] = pos_stride_t;
    p.q_weight = (const T*)q_weight; p.k_weight = (const T*)k_weight;
    p.B = B; p.T_new = T_new; p.Hq = Hq; p.Hk = Hk; p.D = D;
    p.heads_per_item = per; p.q_items = q_items; p.k_items = k_items;
    const dim3 grid((unsigned)ctas);
    const cudaStream_t s = (cudaStream_t)stream;
    const char* what = "lq_qk_norm_rope";
    LQ_GRP(4) LQ_GRP(8) LQ_GRP(16) LQ_GRP(32)
  })
#undef LQ_GRP
  return LQ_OK;
}

extern "C" int lq_block_kv_append(const lq_block_kv* cache, const void* k, const void* v, const int64_t* k_strides,
                                  const int64_t* v_strides, int T_new, const int64_t* start_dev, int start_stride,
                                  int64_t start, const int64_t* count_dev, int pdl, void* stream) {
  const char* what = "lq_block_kv_append";
  if (const int rc = check_block_kv(cache, what)) return rc;
  LQ_REQUIRE(T_new > 0 && k && v && k_strides && v_strides, LQ_ERR_ARG, "%s: no tokens or null tensor pointer", what);
  const BlockSpan sp{start_dev, start, count_dev, start_stride, T_new};
  const Rope rp{};
  LQ_DISPATCH_DTYPE(cache->dtype, T, {
    AppendArgs<T> p{};
    p.k = (const T*)k; p.v = (const T*)v;
    for (int i = 0; i < 3; ++i) { p.ks[i] = k_strides[i]; p.vs[i] = v_strides[i]; }
    p.vec = aligned_rows(k, p.ks, 3, sizeof(T)) && aligned_rows(v, p.vs, 3, sizeof(T));
    return append(*cache, sp, p, rp, false, pdl, stream, what);
  })
  return LQ_OK;
}

extern "C" int lq_block_kv_append_qkv(const lq_block_kv* cache, const void* qkv, int64_t stride_b, int64_t stride_t,
                                      void* q_out, int Hq, int T_new, const void* q_weight, const void* k_weight,
                                      float eps, const float* cos_table, const float* sin_table, int64_t table_len,
                                      int rot, int interleaved, const int64_t* start_dev, int start_stride,
                                      int64_t start, const int64_t* count_dev, int pdl, void* stream) {
  const char* what = "lq_block_kv_append_qkv";
  if (const int rc = check_block_kv(cache, what)) return rc;
  const int D = cache->head_dim, Hkv = cache->kv_heads;
  LQ_REQUIRE(T_new > 0 && Hq > 0 && qkv && q_out, LQ_ERR_ARG, "%s: no tokens, no heads or null tensor pointer", what);
  LQ_REQUIRE((q_weight != nullptr) == (k_weight != nullptr), LQ_ERR_ARG,
             "%s: norm weights are given for both queries and keys or for neither", what);
  LQ_REQUIRE((uintptr_t)q_out % 16 == 0, LQ_ERR_ARG, "%s: q_out must be 16-byte aligned", what);
  if (const int rc = check_rope(cos_table, sin_table, table_len, rot, D)) return rc;
  const BlockSpan sp{start_dev, start, count_dev, start_stride, T_new};
  const Rope rp{cos_table, sin_table, table_len, rot, interleaved, eps};
  LQ_DISPATCH_DTYPE(cache->dtype, T, {
    AppendArgs<T> p{};
    const int64_t strides[3] = {stride_b, D, stride_t};
    p.q = (const T*)qkv;
    p.k = p.q + (int64_t)Hq * D;
    p.v = p.k + (int64_t)Hkv * D;
    for (int i = 0; i < 3; ++i) p.qs[i] = p.ks[i] = p.vs[i] = strides[i];
    p.vec = aligned_rows(qkv, strides, 3, sizeof(T)) && ((uintptr_t)q_weight | (uintptr_t)k_weight) % 16 == 0;
    p.q_out = (T*)q_out; p.Hq = Hq; p.q_weight = (const T*)q_weight; p.k_weight = (const T*)k_weight;
    return append(*cache, sp, p, rp, true, pdl, stream, what);
  })
  return LQ_OK;
}

extern "C" int lq_block_kv_read(const lq_block_kv* cache, void* k_out, void* v_out, int length, const int64_t* start_dev,
                                int start_stride, int64_t start, const int64_t* count_dev, int T_new, int pdl, void* stream) {
  const char* what = "lq_block_kv_read";
  if (const int rc = check_block_kv(cache, what)) return rc;
  LQ_REQUIRE(length > 0 && T_new >= 0 && k_out && v_out, LQ_ERR_ARG, "%s: empty output or null tensor pointer", what);
  LQ_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, LQ_ERR_ARG, "%s: outputs must be 16-byte aligned", what);
  int* error_word = block_error_word();
  if (error_word == nullptr) return LQ_ERR_LAUNCH;
  const BlockSpan sp{start_dev, start, count_dev, start_stride, T_new};
  const dim3 grid((unsigned)((length + cache->block - 1) / cache->block), 2u * cache->kv_heads, (unsigned)cache->batch);
  LQ_REQUIRE(grid.y <= 65535, LQ_ERR_ARG, "%s: too many heads for one launch", what);
  LQ_DISPATCH_DTYPE(cache->dtype, T, {
    const cudaStream_t s = (cudaStream_t)stream;
    return cache->head_dim == 64
               ? launch(block_read_kernel<T, 64>, grid, s, pdl, what, *cache, sp, (T*)k_out, (T*)v_out, length, error_word)
               : launch(block_read_kernel<T, 128>, grid, s, pdl, what, *cache, sp, (T*)k_out, (T*)v_out, length, error_word);
  })
  return LQ_OK;
}
