// Attention of the newest tokens over the block-scaled KV cache (layout: block_kv.cuh).
//
//   out[t, h] = sum_p softmax_p(scaling q[t, h] . k[p]) v[p],  p <= start + t
//
// One pass over the cache. The codes go to the tensor cores as fp16 integers (exact); the scales
// never touch an element: with key scale ks and value scale vs of a block,
//   x_p = log2(e) scaling ks (q . code_p) + log2(vs),  M = running maximum of x,
//   w_p = 2^(x_p - M)  (the weight with the value scale folded in),
//   O  += w_p code_p,  sum += (sum of the block's w_p) / vs,   out = O / sum.
//
// A unit of work is 16 tokens of one KV head. The units of all sequences and heads form one line,
// which the CTAs share in equal contiguous runs, so ragged lengths and single long contexts both
// fill the GPU without the host knowing a length. A CTA's warps take the units of its run in
// turn; at the end of a (sequence, head) they merge through shared memory, and where a run ends
// inside one the partial (M, sum, O) goes to scratch and the second kernel joins the parts.
//
// Scores are computed as K q^T (16 tokens x 8 query rows a tile) and outputs as V^T w (16 dims x 8
// query rows), so that the few query rows of a decode step are the narrow side of the MMA: with
// queries as its 16 rows half of every product would be padding. The k index of the first product
// and the row index of the second are mapped onto the head's dims so that each thread's bytes of
// a cached row are contiguous.
#include "block_kv.cuh"

namespace lq {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 16;  // tokens

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
// Bytes (sel) of biased codes (code + 128) under the high byte 0x64 are the halves 1024 + 128 + code.
__device__ __forceinline__ uint32_t codes_h2(uint32_t biased, uint32_t sel) {
  return as_u32(__hsub2(as_h2(__byte_perm(biased, 0x64646464u, sel)), __floats2half2_rn(1152.f, 1152.f)));
}

// 2^e with e the exponent of the largest finite |x| (0 for none), as the power of two that brings
// it to [2^top, 2^(top + 1)), and its reciprocal.
__device__ __forceinline__ float lift_of(float amax, int top, float& unit) {
  int e = (int)(__float_as_uint(amax) >> 23) - 127;
  e = amax > 0.f ? max(e, -100) : top;
  unit = __uint_as_float((unsigned)(127 + e - top) << 23);
  return __uint_as_float((unsigned)(127 - e + top) << 23);
}
__device__ __forceinline__ float finite_abs(float x) {
  const float m = fabsf(x);
  return m <= 3.402823466e38f ? m : 0.f;
}

// ---------------------------------------------------------------- how the line of units is cut
struct Shape {
  int Hq, G, rows, tile;  // query rows per KV head: T_new * G; rows of one pass
};

// Units that row tile rt of sequence b takes per KV head: complete blocks first, then the ring.
__device__ __forceinline__ int units_of(const lq_block_kv& c, const BlockSpan& sp, const Shape& sh, int b, int rt,
                                        SeqSpan& s, bool& bad) {
  s = span_of(c, sp, b, bad);
  const int t_lo = rt * sh.tile / sh.G;
  if (t_lo >= s.n) return 0;
  const int t_hi = min(s.n - 1, (rt * sh.tile + sh.tile - 1) / sh.G);
  const int visible = s.start + t_hi + 1, L = s.start + s.n, held = L - L % c.block;
  return (min(visible, held) + kUnit - 1) / kUnit + (max(0, visible - held) + kUnit - 1) / kUnit;
}

// All units of row tile rt, and the sequence that unit `want(total)` lies in with the units before
// it. One warp calls it.
struct Place {
  int64_t total, before;
  int b;
};
template <typename Want>
__device__ __forceinline__ Place find_place(const lq_block_kv& c, const BlockSpan& sp, const Shape& sh, int rt, int* error_word,
                                            Want want) {
  const int lane = threadIdx.x & 31;
  int64_t total = 0;
  for (int b = lane; b < c.batch; b += 32) {
    SeqSpan s;
    bool bad;
    total += units_of(c, sp, sh, b, rt, s, bad);
    if (bad) atomicExch(error_word, LQ_BLOCK_BAD_POSITION);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  total *= c.kv_heads;
  const int64_t unit = want(total);
  int64_t before = 0;
  for (int b0 = 0; b0 < c.batch; b0 += 32) {
    SeqSpan s;
    bool bad;
    const int64_t mine = b0 + lane < c.batch ? (int64_t)units_of(c, sp, sh, b0 + lane, rt, s, bad) * c.kv_heads : 0;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > unit);
    if (hit != 0) {
      const int at = __ffs(hit) - 1;
      return Place{total, before + __shfl_sync(0xffffffffu, upto - mine, at), b0 + at};
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return Place{total, before, c.batch};
}

template <int D, int NT>
struct Smem {
  static constexpr int kRows = 8 * NT;
  static constexpr int kQ = D + 4;   // halves to a staged query row: rows 8 bytes apart in the banks
  static constexpr int kO = D + 4;   // floats to a partial output row
  static constexpr size_t q_bytes = (size_t)kRows * kQ * 2;
  static constexpr size_t o_bytes = (size_t)kWarps * kRows * kO * 4;
  static constexpr size_t ml_bytes = (size_t)kWarps * kRows * 8;
  static constexpr size_t total = q_bytes + o_bytes + ml_bytes + kRows * 4;
};

// ---------------------------------------------------------------- main kernel
// grid (CTAs that share the line, row tiles). T is the type of q, out and the ring.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads)
block_attn_kernel(const lq_block_kv c, const BlockSpan sp, const Shape sh, const T* __restrict__ q, int64_t qsb, int64_t qst,
                  int64_t qsh, T* __restrict__ out, float* __restrict__ part, float qk_scale, int* error_word) {
  constexpr int ROWS = 8 * NT, KS = D / 16, MT = D / 16, DPT = D / 8;  // DPT: dims of V a thread owns
  using SM = Smem<D, NT>;
  extern __shared__ __align__(16) uint8_t smem[];
  __half* q_s = reinterpret_cast<__half*>(smem);
  float* o_s = reinterpret_cast<float*>(smem + SM::q_bytes);
  float2* ml_s = reinterpret_cast<float2*>(smem + SM::q_bytes + SM::o_bytes);
  float* unit_s = reinterpret_cast<float*>(smem + SM::q_bytes + SM::o_bytes + SM::ml_bytes);
  __shared__ Place place_s;

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gid = lane >> 2, q4 = lane & 3;
  const int rt = blockIdx.y, P = c.block;
  const int ctas = gridDim.x, cta = blockIdx.x;
  if (warp == 0) {
    const Place p = find_place(c, sp, sh, rt, error_word, [&](int64_t total) {
      const int64_t n = total < ctas ? total : ctas;
      return cta < n ? total * cta / n : total;
    });
    if (lane == 0) place_s = p;
  }
  __syncthreads();
  const int64_t total = place_s.total;
  const int64_t n_ctas = total < ctas ? total : ctas;
  if (cta >= n_ctas) return;
  int64_t left = total * (cta + 1) / n_ctas - total * cta / n_ctas;
  int64_t off = total * cta / n_ctas - place_s.before;
  float* my_part = part + (int64_t)rt * (ctas + (int64_t)c.batch * c.kv_heads) * ROWS * (D + 2);

  for (int b = place_s.b; left > 0 && b < c.batch; ++b) {
    SeqSpan s;
    bool bad;
    const int units = units_of(c, sp, sh, b, rt, s, bad);
    if (off >= (int64_t)units * c.kv_heads) {
      off -= (int64_t)units * c.kv_heads;
      continue;
    }
    const int L = s.start + s.n, held = L - L % P;
    const int t_lo = rt * sh.tile / sh.G, t_hi = min(s.n - 1, (rt * sh.tile + sh.tile - 1) / sh.G);
    const int visible = s.start + t_hi + 1;
    const int code_units = (min(visible, held) + kUnit - 1) / kUnit;
    for (int h = (int)(off / units); h < c.kv_heads && left > 0; ++h) {
      const int ua = (int)(off - (int64_t)h * units);
      const int ub = (int)min((int64_t)units, ua + left);
      off += ub - ua;
      left -= ub - ua;

      // ---- the tile's query rows as fp16, each lifted by a power of two
      __syncthreads();  // (the last segment's merge has read the shared memory)
      for (int r = warp; r < ROWS; r += kWarps) {
        const int row = rt * sh.tile + r, t = row / sh.G, g = row % sh.G;
        const bool live = row < sh.rows && t < s.n;
        float x[D / 32], amax = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          x[i] = live ? Conv<T>::to_f32(q[b * qsb + t * qst + (int64_t)(h * sh.G + g) * qsh + lane + 32 * i]) : 0.f;
          amax = fmaxf(amax, finite_abs(x[i]));
        }
        float unit;
        const float lift = lift_of(warp_max(amax), 10, unit);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) q_s[r * SM::kQ + lane + 32 * i] = __float2half_rn(x[i] * lift);
        if (lane == 0) unit_s[r] = unit * qk_scale;
      }
      __syncthreads();

      // this thread's query rows are 8 nt + 2 q4 (+ 1): their units and last visible positions
      float qu[NT][2];
      int seen[NT][2];
      uint32_t qb[NT][KS][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + q4 * 2 + e;
          qu[nt][e] = unit_s[r];
          seen[nt][e] = s.start + (rt * sh.tile + r) / sh.G;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const uint2 v = *reinterpret_cast<const uint2*>(q_s + (nt * 8 + gid) * SM::kQ + (k / 4) * 64 + q4 * 16 + (k % 4) * 4);
          qb[nt][k][0] = v.x;
          qb[nt][k][1] = v.y;
        }
      }
      float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      }
      const T* k_ring = reinterpret_cast<const T*>(c.k_ring) + ((int64_t)b * c.kv_heads + h) * 2 * P * D;
      const T* v_ring = reinterpret_cast<const T*>(c.v_ring) + ((int64_t)b * c.kv_heads + h) * 2 * P * D;

      for (int u = ua + warp; u < ub; u += kWarps) {
        const bool tail = u >= code_units;
        const int pos0 = tail ? held + (u - code_units) * kUnit : u * kUnit;
        uint32_t ka[KS][4];       // K as the A operand: tokens gid, gid + 8
        uint32_t va[MT][4];       // V^T as the A operand
        float ks, vs;
        if (!tail) {
          const int64_t page = page_of(c, b, pos0 / P);
          if (page < 0) {
            if (lane == 0) atomicExch(error_word, LQ_BLOCK_BAD_PAGE);
            ks = vs = __int_as_float(0x7fffffff);
          } else {
            ks = c.k_scales[page * c.kv_heads + h];
            vs = c.v_scales[page * c.kv_heads + h];
          }
          const int64_t at = ((page < 0 ? 0 : page) * c.kv_heads + h) * P + pos0 % P;
          const int8_t* kp = c.k_pages + (at + gid) * D + q4 * 16;
          const int8_t* vp = c.v_pages + (at + q4 * 2) * D + gid * DPT;
          uint32_t kw[2][KS], vw[4][DPT / 4];
#pragma unroll
          for (int j = 0; j < D / 64; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint4 v = *reinterpret_cast<const uint4*>(kp + e * 8 * D + j * 64);
              kw[e][4 * j] = v.x; kw[e][4 * j + 1] = v.y; kw[e][4 * j + 2] = v.z; kw[e][4 * j + 3] = v.w;
            }
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // tokens 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9
            const int8_t* row = vp + ((e & 1) + (e >> 1) * 8) * D;
            if (DPT == 16) {
              const uint4 v = *reinterpret_cast<const uint4*>(row);
              vw[e][0] = v.x; vw[e][1] = v.y; vw[e][DPT / 4 - 2] = v.z; vw[e][DPT / 4 - 1] = v.w;
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(row);
              vw[e][0] = v.x; vw[e][1] = v.y;
            }
          }
#pragma unroll
          for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t w = kw[e][k] ^ 0x80808080u;
              ka[k][e] = codes_h2(w, 0x4140u);
              ka[k][e + 2] = codes_h2(w, 0x4342u);
            }
          // row gid of tile mt is dim gid * DPT + 2 mt, row gid + 8 the one after it
#pragma unroll
          for (int w = 0; w < DPT / 4; ++w)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t x = vw[2 * e][w] ^ 0x80808080u, y = vw[2 * e + 1][w] ^ 0x80808080u;
              const uint32_t lo = __byte_perm(x, y, 0x5140u), hi = __byte_perm(x, y, 0x7362u);
              va[2 * w][2 * e] = codes_h2(lo, 0x4140u);
              va[2 * w][2 * e + 1] = codes_h2(lo, 0x4342u);
              va[2 * w + 1][2 * e] = codes_h2(hi, 0x4140u);
              va[2 * w + 1][2 * e + 1] = codes_h2(hi, 0x4342u);
            }
        } else {
          // rows of the incomplete block: lifted by a power of two of their own and taken as fp16
          // (a bf16 value has 8 significant bits; the smallest are lost 2^-24 below the largest)
          float kx[2][DPT * 2], vx[4][DPT], kmax = 0.f, vmax = 0.f;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int pos = pos0 + gid + e * 8;
            const T* row = k_ring + (int64_t)(pos % (2 * P)) * D;
#pragma unroll
            for (int i = 0; i < DPT * 2; ++i) {
              kx[e][i] = pos < L ? Conv<T>::to_f32(row[(i / 16) * 64 + q4 * 16 + i % 16]) : 0.f;
              kmax = fmaxf(kmax, finite_abs(kx[e][i]));
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int pos = pos0 + q4 * 2 + (e & 1) + (e >> 1) * 8;
            const T* row = v_ring + (int64_t)(pos % (2 * P)) * D + gid * DPT;
#pragma unroll
            for (int i = 0; i < DPT; ++i) {
              vx[e][i] = pos < L ? Conv<T>::to_f32(row[i]) : 0.f;
              vmax = fmaxf(vmax, finite_abs(vx[e][i]));
            }
          }
          const float klift = lift_of(warp_max(kmax), 10, ks), vlift = lift_of(warp_max(vmax), 7, vs);
#pragma unroll
          for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float* x = &kx[e][k * 4];
              ka[k][e] = as_u32(__floats2half2_rn(x[0] * klift, x[1] * klift));
              ka[k][e + 2] = as_u32(__floats2half2_rn(x[2] * klift, x[3] * klift));
            }
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              va[i][2 * e] = as_u32(__floats2half2_rn(vx[2 * e][2 * i] * vlift, vx[2 * e + 1][2 * i] * vlift));
              va[i][2 * e + 1] = as_u32(__floats2half2_rn(vx[2 * e][2 * i + 1] * vlift, vx[2 * e + 1][2 * i + 1] * vlift));
            }
        }

        // ---- scores, weights
        const float lv = __log2f(vs), inv_vs = 1.f / vs;
        const bool masked = pos0 + kUnit - 1 > s.start + t_lo;
        float x[NT][4];
        bool rises = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < KS; ++k) mma16(acc, ka[k][0], ka[k][1], ka[k][2], ka[k][3], qb[nt][k][0], qb[nt][k][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[nt][i] = fmaf(acc[i], qu[nt][i & 1] * ks, lv);
            if (masked && pos0 + gid + (i >> 1) * 8 > seen[nt][i & 1]) x[nt][i] = -INFINITY;
            rises = rises || x[nt][i] > m[nt][i & 1] + 8.f;
          }
        }
        // M follows the maximum only when a weight would pass 2^8: any M serves, and fp16 keeps 11
        // bits of a weight up to 2^15
        if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(x[nt][e], x[nt][e + 2]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              const float to = fmaxf(m[nt][e], mx);
              const float corr = m[nt][e] == -INFINITY ? 0.f : exp2f(m[nt][e] - to);
              m[nt][e] = to;
              l[nt][e] *= corr;
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                o[nt][i][e] *= corr;
                o[nt][i][e + 2] *= corr;
              }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float base = m[nt][i & 1] == -INFINITY ? 0.f : m[nt][i & 1];
            w[i] = exp2f(x[nt][i] - base);
          }
          // the sum takes the weights as they are multiplied, rounded to fp16: their rounding then
          // cancels where few weights dominate. (Below 2^-14, where fp16 loses bits, it takes them
          // as they are: a block of small values has small w but counts in the sum by w / vs.)
          const __half2 w0 = __floats2half2_rn(w[0], w[1]), w1 = __floats2half2_rn(w[2], w[3]);
          const float2 f0 = __half22float2(w0), f1 = __half22float2(w1);
          const float least = 6.103515625e-05f;
          const float sum0 = (w[0] < least ? w[0] : f0.x) + (w[2] < least ? w[2] : f1.x);
          const float sum1 = (w[1] < least ? w[1] : f0.y) + (w[3] < least ? w[3] : f1.y);
          l[nt][0] += sum0 == 0.f ? 0.f : sum0 * inv_vs;  // (a masked token's scale may be NaN)
          l[nt][1] += sum1 == 0.f ? 0.f : sum1 * inv_vs;
          const uint32_t b0 = transpose8x8(as_u32(w0)), b1 = transpose8x8(as_u32(w1));
#pragma unroll
          for (int i = 0; i < MT; ++i) mma16(o[nt][i], va[i][0], va[i][1], va[i][2], va[i][3], b0, b1);
        }
      }

      // ---- merge the warps
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[nt][e];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int r = nt * 8 + q4 * 2 + e;
          if (gid == 0) ml_s[warp * ROWS + r] = make_float2(m[nt][e], sum);
          float* dst = o_s + (warp * ROWS + r) * SM::kO + gid * DPT;
#pragma unroll
          for (int i = 0; i < MT; ++i) *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(o[nt][i][e], o[nt][i][e + 2]);
        }
      __syncthreads();
      const bool whole = ua == 0 && ub == units;
      float* dst_part = my_part + (cta + (int64_t)b * c.kv_heads + h) * ROWS * (D + 2);
      for (int i = threadIdx.x; i < ROWS * D; i += kThreads) {
        const int r = i / D, d = i % D;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml_s[w * ROWS + r].x);
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 ml = ml_s[w * ROWS + r];
          // (a warp without units has -inf; one whose scores are NaN has NaN sums and must count)
          const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2f(ml.x - top);
          sum = fmaf(ml.y, f, sum);
          acc = fmaf(o_s[(w * ROWS + r) * SM::kO + d], f, acc);
        }
        if (whole) {
          const int row = rt * sh.tile + r, t = row / sh.G, g = row % sh.G;
          if (row < sh.rows)
            out[(((int64_t)b * sp.tokens + t) * sh.Hq + h * sh.G + g) * D + d] =
                Conv<T>::from_f32(t < s.n ? acc / sum : 0.f);
        } else {
          dst_part[r * (D + 2) + d] = acc;
          if (d == 0) {
            dst_part[r * (D + 2) + D] = top;
            dst_part[r * (D + 2) + D + 1] = sum;
          }
        }
      }
    }
    off -= (int64_t)units * c.kv_heads;  // zero where the run goes on into the next sequence
  }
}

// ---------------------------------------------------------------- join the parts
// grid (KV heads, batch, row tiles), D threads: a (sequence, head) that several CTAs shared is the
// weighted sum of their parts; one that none took (no rows that count) becomes zeros.
template <typename T>
__global__ void block_attn_join_kernel(const lq_block_kv c, const BlockSpan sp, const Shape sh, int ctas, T* __restrict__ out,
                                       const float* __restrict__ part, int* error_word) {
  __shared__ Place place_s;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int h = blockIdx.x, b = blockIdx.y, rt = blockIdx.z, D = c.head_dim, d = threadIdx.x;
  // (start and count are older than the kernel ahead, which has waited for their writer)
  SeqSpan s;
  bool bad;
  const int units = units_of(c, sp, sh, b, rt, s, bad);
  int64_t u0 = 0;
  int c0 = 0, c1 = -1;
  int64_t total = 0, n = 0;
  if (units > 0) {
    if (threadIdx.x < 32) {
      // units before sequence b: ask for the unit that b's first one is
      int64_t before = 0, all = 0;
      for (int i = threadIdx.x; i < c.batch; i += 32) {
        SeqSpan si;
        bool bi;
        const int64_t v = (int64_t)units_of(c, sp, sh, i, rt, si, bi) * c.kv_heads;
        all += v;
        if (i < b) before += v;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        all += __shfl_xor_sync(0xffffffffu, all, o);
      }
      if (threadIdx.x == 0) place_s = Place{all, before, b};
    }
    __syncthreads();
    total = place_s.total;
    n = total < ctas ? total : ctas;
    u0 = place_s.before + (int64_t)h * units;
    c0 = (int)(((u0 + 1) * n - 1) / total);
    c1 = (int)(((u0 + units) * n - 1) / total);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (units > 0 && c0 == c1) return;  // one CTA had all of it and wrote the output
  const float* mine = part + ((int64_t)rt * (ctas + (int64_t)c.batch * c.kv_heads) + (int64_t)b * c.kv_heads + h) * sh.tile * (D + 2);
  const int64_t stride = (int64_t)sh.tile * (D + 2);
  for (int r = 0; r < sh.tile; ++r) {
    const int row = rt * sh.tile + r, t = row / sh.G, g = row % sh.G;
    if (row >= sh.rows) break;
    float v = 0.f;
    if (units > 0 && t < s.n) {
      float top = -INFINITY;
      for (int k = c0; k <= c1; ++k) top = fmaxf(top, mine[k * stride + r * (D + 2) + D]);
      float sum = 0.f, acc = 0.f;
      for (int k = c0; k <= c1; ++k) {
        const float mk = mine[k * stride + r * (D + 2) + D], lk = mine[k * stride + r * (D + 2) + D + 1];
        const float f = mk == -INFINITY ? (lk == 0.f ? 0.f : 1.f) : exp2f(mk - top);
        sum = fmaf(lk, f, sum);
        acc = fmaf(mine[k * stride + r * (D + 2) + d], f, acc);
      }
      v = acc / sum;
    }
    out[(((int64_t)b * sp.tokens + t) * sh.Hq + h * sh.G + g) * D + d] = Conv<T>::from_f32(v);
  }
}

// ---------------------------------------------------------------- host
struct Plan {
  Shape sh;
  int nt, tiles, ctas;
};

Plan plan_of(const lq_block_kv& c, int Hq, int T_new) {
  Plan p;
  p.sh.Hq = Hq;
  p.sh.G = Hq / c.kv_heads;
  p.sh.rows = T_new * p.sh.G;
  p.nt = p.sh.rows <= 8 ? 1 : 2;
  p.sh.tile = 8 * p.nt;
  p.tiles = (p.sh.rows + p.sh.tile - 1) / p.sh.tile;
  p.ctas = 2 * sm_count() / p.tiles;
  if (p.ctas < 1) p.ctas = 1;
  return p;
}

int64_t scratch_bytes(const lq_block_kv& c, const Plan& p) {
  return (int64_t)p.tiles * (p.ctas + (int64_t)c.batch * c.kv_heads) * p.sh.tile * (c.head_dim + 2) * 4;
}

int check_attn(const lq_block_kv* c, int Hq, int T_new, const char* what) {
  if (const int rc = check_block_kv(c, what)) return rc;
  LQ_REQUIRE(Hq > 0 && Hq % c->kv_heads == 0 && T_new > 0, LQ_ERR_ARG,
             "%s: %d query heads do not share %d KV heads evenly, or there are no rows", what, Hq, c->kv_heads);
  LQ_REQUIRE(c->dtype != LQ_F32, LQ_ERR_UNSUPPORTED, "%s: built for float16 and bfloat16 rows", what);
  LQ_REQUIRE(c->kv_heads <= 65535 && (int64_t)T_new * (Hq / c->kv_heads) <= 65535LL * 8, LQ_ERR_ARG,
             "%s: too many rows for one call", what);
  return LQ_OK;
}

template <typename Kern, typename... Args>
int launch(Kern kern, dim3 grid, int threads, size_t smem, cudaStream_t stream, int pdl, const char* what, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
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

template <typename T, int D, int NT>
int run(const lq_block_kv& c, const BlockSpan& sp, const Plan& p, const void* q, const int64_t* qs, void* out, void* scratch,
        float scaling, int pdl, cudaStream_t stream, int* error_word, const char* what) {
  auto kern = block_attn_kernel<T, D, NT>;
  constexpr size_t smem = Smem<D, NT>::total;
  if (const int rc = ensure_smem_limit(reinterpret_cast<const void*>(kern), (int)smem, what)) return rc;
  const float qk_scale = scaling * 1.4426950408889634f;
  if (const int rc = launch(kern, dim3((unsigned)p.ctas, (unsigned)p.tiles), kThreads, smem, stream, pdl, what, c, sp, p.sh,
                            (const T*)q, qs[0], qs[1], qs[2], (T*)out, (float*)scratch, qk_scale, error_word))
    return rc;
  return launch(block_attn_join_kernel<T>, dim3((unsigned)c.kv_heads, (unsigned)c.batch, (unsigned)p.tiles), D, 0, stream, 1, what,
                c, sp, p.sh, p.ctas, (T*)out, (const float*)scratch, error_word);
}

template <typename T>
int dispatch(const lq_block_kv& c, const BlockSpan& sp, const Plan& p, const void* q, const int64_t* qs, void* out, void* scratch,
             float scaling, int pdl, cudaStream_t stream, int* error_word, const char* what) {
#define LQ_CASE(DD, NN) \
  if (c.head_dim == DD && p.nt == NN) return run<T, DD, NN>(c, sp, p, q, qs, out, scratch, scaling, pdl, stream, error_word, what);
  LQ_CASE(64, 1) LQ_CASE(64, 2)
  LQ_CASE(128, 1) LQ_CASE(128, 2)
#undef LQ_CASE
  return fail(LQ_ERR_UNSUPPORTED, "%s: no kernel for this shape", what);
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" int64_t lq_block_attn_scratch_bytes(const lq_block_kv* cache, int Hq, int T_new) {
  if (check_attn(cache, Hq, T_new, "lq_block_attn_scratch_bytes")) return -1;
  return scratch_bytes(*cache, plan_of(*cache, Hq, T_new));
}

extern "C" int lq_block_attn(const lq_block_kv* cache, const void* q, const int64_t* q_strides, void* out, void* scratch,
                             int64_t scratch_bytes_given, int Hq, int T_new, const int64_t* start_dev, int start_stride,
                             int64_t start, const int64_t* count_dev, float scaling, int pdl, void* stream) {
  const char* what = "lq_block_attn";
  if (const int rc = check_attn(cache, Hq, T_new, what)) return rc;
  LQ_REQUIRE(q && q_strides && out && scratch, LQ_ERR_ARG, "%s: null tensor pointer", what);
  LQ_REQUIRE(((uintptr_t)scratch & 15) == 0, LQ_ERR_ARG, "%s: scratch must be 16-byte aligned", what);
  const Plan p = plan_of(*cache, Hq, T_new);
  LQ_REQUIRE(scratch_bytes_given >= scratch_bytes(*cache, p), LQ_ERR_ARG, "%s: scratch of %lld bytes, %lld are needed", what,
             (long long)scratch_bytes_given, (long long)scratch_bytes(*cache, p));
  int* error_word = block_error_word();
  if (error_word == nullptr) return LQ_ERR_LAUNCH;
  const BlockSpan sp{start_dev, start, count_dev, start_stride, T_new};
  return cache->dtype == LQ_BF16
             ? dispatch<__nv_bfloat16>(*cache, sp, p, q, q_strides, out, scratch, scaling, pdl, (cudaStream_t)stream, error_word, what)
             : dispatch<__half>(*cache, sp, p, q, q_strides, out, scratch, scaling, pdl, (cudaStream_t)stream, error_word, what);
}
