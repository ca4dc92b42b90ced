// Block-scaled KV cache: append (quantize a block when it is complete) and read back; norms of
// queries and keys for each head with the position rotation; and the joined form of a decode
// step, which does both from the fused q|k|v row in one launch. Layout: block_kv.cuh.
#include "block_kv.cuh"

#include <cstring>

namespace lq {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxVec = 8;  // 8-value pieces a thread holds of one block: 128 * 128 / 8 / 256

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
  T v[8];
  memcpy(v, &r, sizeof(r));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = Conv<T>::to_f32(v[i]);
}
template <typename T>
__device__ __forceinline__ Pack8<T> pack8(const float (&x)[8]) {
  T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = Conv<T>::from_f32(x[i]);
  Pack8<T> r;
  memcpy(&r, v, sizeof(r));
  return r;
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

// This lane's 8 values' angles (values d0 .. d0 + 7 of the head), requested early.
struct Angles {
  float c[8], s[8];
};
__device__ __forceinline__ Angles angles_of(const Rope& rp, int64_t pos, int d0) {
  Angles a;
#pragma unroll
  for (int i = 0; i < 8; ++i) { a.c[i] = 1.f; a.s[i] = 0.f; }
  if (d0 >= rp.rot) return a;
  const int half = rp.rot / 2;
  if (rp.interleaved) {
    const float4 c = *reinterpret_cast<const float4*>(rp.cos + pos * half + d0 / 2);
    const float4 s = *reinterpret_cast<const float4*>(rp.sin + pos * half + d0 / 2);
    a.c[0] = a.c[1] = c.x; a.c[2] = a.c[3] = c.y; a.c[4] = a.c[5] = c.z; a.c[6] = a.c[7] = c.w;
    a.s[0] = a.s[1] = s.x; a.s[2] = a.s[3] = s.y; a.s[4] = a.s[5] = s.z; a.s[6] = a.s[7] = s.w;
  } else {
    const int i0 = d0 < half ? d0 : d0 - half;
    const float4* c = reinterpret_cast<const float4*>(rp.cos + pos * half + i0);
    const float4* s = reinterpret_cast<const float4*>(rp.sin + pos * half + i0);
    const float4 c0 = c[0], c1 = c[1], s0 = s[0], s1 = s[1];
    a.c[0] = c0.x; a.c[1] = c0.y; a.c[2] = c0.z; a.c[3] = c0.w;
    a.c[4] = c1.x; a.c[5] = c1.y; a.c[6] = c1.z; a.c[7] = c1.w;
    a.s[0] = s0.x; a.s[1] = s0.y; a.s[2] = s0.z; a.s[3] = s0.w;
    a.s[4] = s1.x; a.s[5] = s1.y; a.s[6] = s1.z; a.s[7] = s1.w;
  }
  return a;
}

// y = x * rsqrt(mean(x^2) + eps) * w over a head, then the rotation of its first rp.rot values:
// pair (a, c) -> (a cos - c sin, c cos + a sin), a pair being (i, i + rot/2) or, interleaved,
// (2i, 2i + 1). GRP lanes hold a head, 8 values each; all 32 lanes of the warp call this
// together. fp32 throughout, every operation named, so that the joined and the separate forms
// round alike; the caller rounds once.
template <int GRP>
__device__ __forceinline__ void norm_rope8(float (&x)[8], int li, int D, const float* w, const Rope& rp,
                                           const Angles& a) {
  if (w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __fmaf_rn(x[i], x[i], ss);
#pragma unroll
    for (int o = GRP / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(__fadd_rn(__fdiv_rn(ss, (float)D), rp.eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], r), w[i]);
  }
  const int d0 = li * 8;
  if (rp.interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float p = x[i], q = x[i + 1];
      x[i] = __fmaf_rn(p, a.c[i], -__fmul_rn(q, a.s[i]));
      x[i + 1] = __fmaf_rn(q, a.c[i], __fmul_rn(p, a.s[i]));
    }
  } else {
    const int step = rp.rot / 16;  // lanes between the two values of a pair
    const bool first = d0 < rp.rot / 2;
    const int lane = threadIdx.x & 31;
    const int src = d0 < rp.rot ? (first ? lane + step : lane - step) : lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_sync(0xffffffffu, x[i], src);
      const float turned = __fmul_rn(other, a.s[i]);  // (a.s is zero behind the rotated values)
      x[i] = __fmaf_rn(x[i], a.c[i], first ? -turned : turned);
    }
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
  int B, T_new, Hq, Hk, D, heads_per_item, items_per_token;
  int vec;
};

// A group of GRP lanes owns one token and up to heads_per_item of its heads: the token's angles
// are loaded once and stay in registers. Bound by HBM (each value read and written once).
template <typename T, int GRP>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const NormRopeArgs<T> p, const Rope rp, int* error_word) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int li = threadIdx.x % GRP;
  const int64_t items = (int64_t)p.B * p.T_new * p.items_per_token;
  const int64_t item0 = (int64_t)blockIdx.x * (kThreads / GRP) + threadIdx.x / GRP;
  const bool live = item0 < items;
  const int64_t item = live ? item0 : items - 1;
  const int64_t token = item / p.items_per_token;
  const int chunk = (int)(item % p.items_per_token);
  const int b = (int)(token / p.T_new), t = (int)(token % p.T_new);
  const int64_t at = p.positions[b * p.ps[0] + t * p.ps[1]];
  const bool known = at >= 0 && at < rp.table_len;
  if (!known && live && li == 0) atomicExch(error_word, LQ_BLOCK_BAD_ANGLE);
  const int heads = p.Hq + p.Hk;
  const int lo = chunk * p.heads_per_item, hi = min(lo + p.heads_per_item, heads);
  const bool mine = live && li * 8 < p.D;
  const int d0 = mine ? li * 8 : 0;
  const Angles a = angles_of(rp, known ? at : 0, li * 8 < p.D ? li * 8 : rp.rot);
  constexpr int UN = 4;
  float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int held = -1;  // whose weights are in w: 0 queries', 1 keys'
  for (int h0 = lo; h0 < lo + p.heads_per_item; h0 += UN) {  // (the same trip count for the whole warp)
    Pack8<T> in[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int h = h0 + u;
      if (mine && h < hi) {
        const T* src = h < p.Hq ? p.q + b * p.qs[0] + t * p.qs[1] + h * p.qs[2]
                                : p.k + b * p.ks[0] + t * p.ks[1] + (h - p.Hq) * p.ks[2];
        in[u] = load8(src + d0, p.vec);
      } else {
        in[u] = zeros8<T>();
      }
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int h = h0 + u;
      if (u > 0 && u >= p.heads_per_item) break;
      const int whose = h < p.Hq ? 0 : 1;
      const T* weight = whose ? p.k_weight : p.q_weight;
      if (p.q_weight != nullptr && whose != held && mine && h < hi) {
        unpack8(load8(weight + d0, p.vec), w);
        held = whose;
      }
      float x[8];
      unpack8(in[u], x);
      norm_rope8<GRP>(x, li, p.D, p.q_weight != nullptr ? w : nullptr, rp, a);
      if (mine && h < hi) {
        if (!known) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = __int_as_float(0x7fffffff);  // no angle: nothing usable
        }
        T* dst = h < p.Hq ? p.q_out + b * p.qos[0] + t * p.qos[1] + h * p.qos[2]
                          : p.k_out + b * p.kos[0] + t * p.kos[1] + (h - p.Hq) * p.kos[2];
        store8(dst + d0, pack8<T>(x), p.vec);
      }
    }
  }
}

// ---------------------------------------------------------------- append
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
// after its own reads.
template <typename T, int D, bool JOINED>
__global__ void __launch_bounds__(kThreads)
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
  if (JOINED && weight != nullptr) unpack8(load8(weight + li * 8, p.vec), w);

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
      if (fresh) unpack8(load8(p.q + b * p.qs[0] + h * p.qs[1] + t * p.qs[2] + li * 8, p.vec), x);
      const Angles a = angles_of(rp, fresh && known ? pos : 0, li * 8);
      norm_rope8<LPR>(x, li, D, weight != nullptr ? w : nullptr, rp, a);
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
        store8(p.q_out + (((int64_t)b * sp.tokens + t) * p.Hq + h) * D + li * 8, pack8<T>(x), true);
      }
    }
    return;
  }

  const int h = blockIdx.y >> 1;
  const int first = s.start / P, last = L / P;
  const int j = first + blockIdx.x;
  if (s.n == 0 || (int64_t)j * P >= L) return;
  const bool complete = (j + 1) * P <= L;
  const bool reads_ring = s.start % P != 0 && (first + 1) * P <= L;  // the first block, completed by this call
  T* ring = reinterpret_cast<T*>(is_v ? c.v_ring : c.k_ring) + ((int64_t)b * c.kv_heads + h) * 2 * P * D;
  const T* src = is_v ? p.v + b * p.vs[0] + h * p.vs[1] : p.k + b * p.ks[0] + h * p.ks[1];
  const int64_t step = is_v ? p.vs[2] : p.ks[2];
  const bool turned = JOINED && !is_v;

  // one 8-value piece of a new row; every lane of the warp calls it
  auto fetch = [&](int pos, bool fresh) {
    Pack8<T> r = zeros8<T>();
    if (fresh) r = load8(src + (int64_t)(pos - s.start) * step + li * 8, p.vec);
    if (turned) {
      float x[8];
      unpack8(r, x);
      const bool known = pos < rp.table_len;
      const Angles a = angles_of(rp, fresh && known ? pos : 0, li * 8);
      norm_rope8<LPR>(x, li, D, weight != nullptr ? w : nullptr, rp, a);
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
  Pack8<T> val[kMaxVec];
  float amax = 0.f;
#pragma unroll
  for (int v = 0; v < kMaxVec; ++v) {
    if (v * kThreads < pieces) {
      const int idx = tid + v * kThreads;
      const int row = idx / LPR, pos = j * P + row;
      const bool inside = idx < pieces;
      const bool fresh = inside && pos >= s.start && pos < L;
      val[v] = fetch(pos, fresh);
      if (inside && complete && pos < s.start) val[v] = load8(ring + (int64_t)(pos % (2 * P)) * D + li * 8, true);
      if (fresh && to_ring) store8(ring + (int64_t)(pos % (2 * P)) * D + li * 8, val[v], true);
      if (complete) {
        float x[8];
        unpack8(val[v], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float m = fabsf(x[i]);
          amax = m <= 3.402823466e38f ? fmaxf(amax, m) : INFINITY;  // INF and NaN both: not finite
        }
      }
    }
  }
  if (!complete) return;
  amax = warp_max(amax);
  if ((tid & 31) == 0) red[tid >> 5] = amax;
  __syncthreads();  // (also: every read of the ring above is done)
  amax = red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) amax = fmaxf(amax, red[i]);
  const bool finite = amax <= 3.402823466e38f;
  const float scale = finite ? scale_of(amax, 127.f) : __int_as_float(0x7fffffff);
  const int64_t page = page_of(c, b, j);
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
        alignas(8) int8_t q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = finite ? (int8_t)code_of(x[i], scale, -128.f, 127.f) : (int8_t)0;
        *reinterpret_cast<uint2*>(codes + (int64_t)idx * 8) = *reinterpret_cast<const uint2*>(q);
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
        if (fresh) store8(ring + (int64_t)(pos % (2 * P)) * D + li * 8, r, true);
      }
    }
  }
}

// ---------------------------------------------------------------- read back
// grid (blocks of the output, 2 * Hkv, B): code * scale rounded once, rows of the incomplete block
// as they are, zeros behind the sequence.
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
    uint2 raw[kMaxVec];
#pragma unroll
    for (int v = 0; v < kMaxVec; ++v) {
      const int idx = tid + v * kThreads;
      raw[v] = make_uint2(0u, 0u);
      if (idx < rows * LPR && codes != nullptr) raw[v] = *reinterpret_cast<const uint2*>(codes + (int64_t)idx * 8);
    }
#pragma unroll
    for (int v = 0; v < kMaxVec; ++v) {
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
    if (pos < L) r = load8(ring + (int64_t)(pos % (2 * P)) * D + (idx % LPR) * 8, true);
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
  if (c.head_dim == 64)
    return joined ? launch(block_append_kernel<T, 64, true>, grid, s, pdl, what, c, sp, p, rp, error_word)
                  : launch(block_append_kernel<T, 64, false>, grid, s, pdl, what, c, sp, p, rp, error_word);
  return joined ? launch(block_append_kernel<T, 128, true>, grid, s, pdl, what, c, sp, p, rp, error_word)
                : launch(block_append_kernel<T, 128, false>, grid, s, pdl, what, c, sp, p, rp, error_word);
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
  const int per = busy >= 8 ? 8 : busy >= 4 ? 4 : busy >= 2 ? 2 : 1;
  const int items_per_token = (Hq + Hk + per - 1) / per;
  const int64_t groups = (int64_t)B * T_new * items_per_token;
  const int64_t ctas = (groups + kThreads / grp - 1) / (kThreads / grp);
  LQ_REQUIRE(ctas <= 0x7fffffffLL, LQ_ERR_ARG, "too many rows for one launch");
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
    p.q_weight = (const T*)(Hq ? q_weight : k_weight); p.k_weight = (const T*)k_weight;
    p.B = B; p.T_new = T_new; p.Hq = Hq; p.Hk = Hk; p.D = D;
    p.heads_per_item = per; p.items_per_token = items_per_token; p.vec = vec;
    const dim3 grid((unsigned)ctas);
    const cudaStream_t s = (cudaStream_t)stream;
    const char* what = "lq_qk_norm_rope";
    switch (grp) {
      case 4: return launch(qk_norm_rope_kernel<T, 4>, grid, s, pdl, what, p, rp, error_word);
      case 8: return launch(qk_norm_rope_kernel<T, 8>, grid, s, pdl, what, p, rp, error_word);
      case 16: return launch(qk_norm_rope_kernel<T, 16>, grid, s, pdl, what, p, rp, error_word);
      default: return launch(qk_norm_rope_kernel<T, 32>, grid, s, pdl, what, p, rp, error_word);
    }
  })
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
