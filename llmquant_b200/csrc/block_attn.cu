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
// A unit of work is 32 tokens of one KV head. The units of all sequences and heads form one line,
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

constexpr int kUnit = 32;  // tokens, as two halves of 16 (the height of an MMA tile)

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

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float inverse_of(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------- how the line of units is cut
struct Shape {
  int Hq, G, rows, tile;  // query rows per KV head: T_new * G; rows of one pass
  int warps;              // of a CTA of the main kernel
};

// The tokens row tile rt of sequence b is about.
struct Tile {
  SeqSpan s;
  int t_lo, visible, held;  // first row's token; positions some row sees; positions in complete blocks
  int code_units, units;    // per KV head: complete blocks first, then the ring's rows
  bool bad;
};
__device__ __forceinline__ Tile tile_of(const lq_block_kv& c, const BlockSpan& sp, const Shape& sh, int b, int rt) {
  Tile x;
  x.s = span_of(c, sp, b, x.bad);
  x.t_lo = rt * sh.tile / sh.G;
  const int L = x.s.start + x.s.n;
  x.visible = x.s.start + min(x.s.n, (rt * sh.tile + sh.tile - 1) / sh.G + 1);
  x.held = L & ~(c.block - 1);
  x.code_units = (min(x.visible, x.held) + kUnit - 1) / kUnit;
  x.units = x.code_units + (max(0, x.visible - x.held) + kUnit - 1) / kUnit;
  if (x.t_lo >= x.s.n) x.code_units = x.units = 0;
  return x;
}

// The line of `total` units is shared by n CTAs: n no larger than one for each round of a CTA's warps,
// but one for each (sequence, head) where those are more, so that short contexts need no join. The
// first `rem` CTAs take base + 1 units, the others base.
struct Cut {
  int total, n, base, rem;
  __device__ __forceinline__ int begin(int cta) const { return cta * base + min(cta, rem); }
  __device__ __forceinline__ int owner(int unit) const {
    const int wide = rem * (base + 1);
    return unit < wide ? unit / (base + 1) : rem + (unit - wide) / base;
  }
};
__device__ __forceinline__ Cut cut_of(int total, int ctas, int heads, int warps) {
  Cut k;
  k.total = total;
  k.n = min(min(ctas, total), max((total + warps - 1) / warps, heads));
  k.base = k.n > 0 ? total / k.n : 0;
  k.rem = total - k.n * k.base;
  return k;
}

// All units of row tile rt and, of those, the ones before sequence `b`. One warp calls it.
__device__ __forceinline__ int2 units_before(const lq_block_kv& c, const BlockSpan& sp, const Shape& sh, int rt, int b) {
  int total = 0, before = 0;
  for (int i = threadIdx.x & 31; i < c.batch; i += 32) {
    const int u = tile_of(c, sp, sh, i, rt).units;
    total += u;
    if (i < b) before += u;
  }
  total = __reduce_add_sync(0xffffffffu, total);
  before = __reduce_add_sync(0xffffffffu, before);
  return make_int2(total * c.kv_heads, before * c.kv_heads);
}

// The sequence that unit `unit` of the line lies in, and the units before that sequence.
__device__ __forceinline__ int2 sequence_of(const lq_block_kv& c, const BlockSpan& sp, const Shape& sh, int rt, int unit) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0; b0 < c.batch; b0 += 32) {
    const int mine = b0 + lane < c.batch ? tile_of(c, sp, sh, b0 + lane, rt).units * c.kv_heads : 0;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > unit);
    if (hit != 0) {
      const int at = __ffs(hit) - 1;
      return make_int2(b0 + at, before + __shfl_sync(0xffffffffu, upto - mine, at));
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return make_int2(c.batch, before);
}

// NT: groups of 8 query rows of a pass. What bounds the choice: the outputs take NT * D / 4
// registers of a thread. One group: 12 warps of 168 registers; two: 8 warps of 255.
template <int D, int NT>
struct Cfg {
  static constexpr int kWarps = NT == 1 ? 12 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRows = 8 * NT;
  static constexpr int kHalf = 16 * D;                   // bytes of 16 tokens' keys, or values
  static constexpr int kStage = 4 * kHalf + 16;          // K and V of half 0, of half 1, their scales
  static constexpr int kStages = (NT == 1 ? 2 : 3) * (128 / D);  // units in a warp's ring
  static constexpr int kQ = D + 4;                       // halves to a staged query row: rows 8 bytes apart in the banks
  static constexpr int kO = D + 4;                       // floats to a partial output row
  static constexpr int kWarpBytes = kStages * kStage;    // also a warp's partial outputs, once the ring is drained
  static constexpr size_t kQBytes = (size_t)kRows * kQ * 2;
  static constexpr size_t kMlBytes = (size_t)kWarps * kRows * 8;
  static constexpr size_t kTotal = (size_t)kWarps * kWarpBytes + kQBytes + kMlBytes + kRows * 4;
  static_assert(kWarpBytes % 16 == 0 && kQBytes % 8 == 0 && kRows * kO * 4 <= kWarpBytes && kTotal <= 227 * 1024, "");
};

// 16-byte piece `chunk` of row `row` of 16 staged tokens. Pieces are XOR-swizzled so that both readers
// are free of bank conflicts: the score product's threads (8 rows, pieces 2 q4 + j) and the value
// product's (rows 2 q4, piece gid).
template <int D>
__device__ __forceinline__ uint32_t piece_at(int row, int chunk) {
  if (D == 128) return (uint32_t)row * 128 + ((chunk ^ (row & 7)) << 4);
  return (uint32_t)(row >> 1) * 128 + (((((row & 1) << 2) + chunk) ^ ((row & 6))) << 4);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128m(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// ---------------------------------------------------------------- main kernel
// grid (CTAs that share the line, row tiles). T is the type of q, out and the ring.
template <typename T, int D, int NT>
__global__ void __launch_bounds__((Cfg<D, NT>::kThreads), 1)
block_attn_kernel(const lq_block_kv c, const BlockSpan sp, const Shape sh, const T* __restrict__ q, int64_t qsb, int64_t qst,
                  int64_t qsh, T* __restrict__ out, float* __restrict__ part, float2* __restrict__ part_ml, float qk_scale,
                  int* error_word) {
  using C = Cfg<D, NT>;
  constexpr int W = C::kWarps, ROWS = C::kRows, KS = D / 16, MT = D / 16, DPT = D / 8;  // DPT: dims of V a thread owns
  constexpr int J = D / 64;  // 16-byte pieces of a K row a thread reads
  extern __shared__ __align__(16) uint8_t smem[];
  __half* q_s = reinterpret_cast<__half*>(smem + (size_t)W * C::kWarpBytes);
  float2* ml_s = reinterpret_cast<float2*>(smem + (size_t)W * C::kWarpBytes + C::kQBytes);
  float* unit_s = reinterpret_cast<float*>(smem + (size_t)W * C::kWarpBytes + C::kQBytes + C::kMlBytes);
  __shared__ int line_s[3];

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gid = lane >> 2, q4 = lane & 3;
  const int rt = blockIdx.y, P = c.block, shift = 31 - __clz(P);
  const int cta = blockIdx.x, heads = c.batch * c.kv_heads;
  if (warp == 0) {
    const int total = units_before(c, sp, sh, rt, 0).x;
    const Cut cut = cut_of(total, gridDim.x, heads, W);
    const int2 at = sequence_of(c, sp, sh, rt, cta < cut.n ? cut.begin(cta) : total);
    if (lane == 0) {
      line_s[0] = total;
      line_s[1] = at.x;
      line_s[2] = at.y;
    }
  }
  __syncthreads();
  const Cut cut = cut_of(line_s[0], gridDim.x, heads, W);
  if (cta >= cut.n) return;
  int left = cut.begin(cta + 1) - cut.begin(cta);
  int off = cut.begin(cta) - line_s[2];
  uint8_t* ring = smem + (size_t)warp * C::kWarpBytes;
  const uint32_t ring_a = smem_u32(ring);

#pragma unroll 1
  for (int b = line_s[1]; left > 0 && b < c.batch; ++b) {
    const Tile x = tile_of(c, sp, sh, b, rt);
    if (off >= x.units * c.kv_heads) {
      off -= x.units * c.kv_heads;
      continue;
    }
    const int* table = c.table + (int64_t)b * c.max_blocks;
    const int first_seen = x.s.start + x.t_lo;  // what the tile's first row sees
#pragma unroll 1
    for (int h = off / x.units; h < c.kv_heads && left > 0; ++h) {
      const int ua = off - h * x.units;
      const int ub = min(x.units, ua + left);
      off += ub - ua;
      left -= ub - ua;

      // ---- the warp's ring: codes and scales of its units, kStages - 1 of them on their way. The page
      // ids of a unit are requested one unit earlier than its codes.
      const int last_code = min(ub, x.code_units);
      const int code_end = min(x.visible, x.held);
      int ids[2];
      auto look_up = [&](int u) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int pos = u * kUnit + 16 * e;
          ids[e] = u < last_code && pos < code_end ? table[pos >> shift] : 0;
        }
      };
      auto issue = [&](int u, int stage) {
        if (u < last_code) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int pos = u * kUnit + 16 * e;
            if (pos < code_end) {
              const uint32_t dst = ring_a + stage * C::kStage + e * 2 * C::kHalf;
              const uint32_t scale_dst = ring_a + stage * C::kStage + 4 * C::kHalf + e * 8;
              const int id = ids[e];
              if (id < 0 || id >= c.num_pages) {
                if (lane == 0) atomicExch(error_word, LQ_BLOCK_BAD_PAGE);
                if (lane < 2) asm volatile("st.shared.u32 [%0], %1;" ::"r"(scale_dst + lane * 4), "r"(0x7fffffff) : "memory");
              } else {
                const int64_t ph = (int64_t)id * c.kv_heads + h;
                const int64_t at = ((ph << shift) + (pos & (P - 1))) * D + lane * 16;
#pragma unroll
                for (int i = 0; i < C::kHalf / 512; ++i) {
                  const int idx = i * 32 + lane;
                  const uint32_t piece = piece_at<D>(idx / (D / 16), idx % (D / 16));
                  cp_async16(dst + piece, c.k_pages + at + i * 512);
                  cp_async16(dst + C::kHalf + piece, c.v_pages + at + i * 512);
                }
                if (lane < 2) cp_async4(scale_dst + lane * 4, (lane ? c.v_scales : c.k_scales) + ph);
              }
            }
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      look_up(ua + warp);
#pragma unroll
      for (int i = 0; i < C::kStages - 1; ++i) {
        issue(ua + warp + i * W, i);
        look_up(ua + warp + (i + 1) * W);
      }

      // ---- the tile's query rows as fp16, each lifted by a power of two
      for (int r = warp; r < ROWS; r += W) {
        const int row = rt * sh.tile + r, t = row / sh.G, g = row - t * sh.G;
        const bool live = row < sh.rows && t < x.s.n;
        float v[D / 32], amax = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          v[i] = live ? Conv<T>::to_f32(q[b * qsb + t * qst + (int64_t)(h * sh.G + g) * qsh + lane + 32 * i]) : 0.f;
          amax = fmaxf(amax, finite_abs(v[i]));
        }
        float unit;
        const float lift = lift_of(warp_max(amax), 10, unit);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) q_s[r * C::kQ + lane + 32 * i] = __float2half_rn(v[i] * lift);
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
          seen[nt][e] = x.s.start + (rt * sh.tile + r) / sh.G;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {  // k-step k: the four dims from q4 * 16 J + 4 k on
          const uint2 v = *reinterpret_cast<const uint2*>(q_s + (nt * 8 + gid) * C::kQ + q4 * 16 * J + k * 4);
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

      // raw products of H halves (tokens from pos0 on, positions below `end` exist) to weights as the B
      // operands of the value product
      auto weigh = [&](auto& acc, auto& wb, int pos0, int end, const auto& ks, const auto& vs) {
        constexpr int H = sizeof(ks) / sizeof(float);
        const bool masked = pos0 + 16 * H - 1 > min(first_seen, end - 1);
        bool rises = false;
        float inv[H];
#pragma unroll
        for (int e = 0; e < H; ++e) {
          const float lv = __log2f(vs[e]);
          inv[e] = inverse_of(vs[e]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[e][nt][i] = fmaf(acc[e][nt][i], qu[nt][i & 1] * ks[e], lv);
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < H; ++e)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int pos = pos0 + 16 * e + gid + (i >> 1) * 8;
                if (pos > seen[nt][i & 1] || pos >= end) acc[e][nt][i] = -INFINITY;
              }
        }
#pragma unroll
        for (int e = 0; e < H; ++e)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) rises = rises || fmaxf(acc[e][nt][i], acc[e][nt][i + 2]) > m[nt][i] + 8.f;
        // M follows the maximum only when a weight would pass 2^8: any M serves, and fp16 keeps 11
        // bits of a weight up to 2^15
        if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float mx = fmaxf(acc[0][nt][i], acc[0][nt][i + 2]);
              if (H == 2) mx = fmaxf(mx, fmaxf(acc[H - 1][nt][i], acc[H - 1][nt][i + 2]));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              const float to = fmaxf(m[nt][i], mx);
              const float corr = m[nt][i] == -INFINITY ? 0.f : exp2_of(m[nt][i] - to);
              m[nt][i] = to;
              l[nt][i] *= corr;
#pragma unroll
              for (int d = 0; d < MT; ++d) {
                o[nt][d][i] *= corr;
                o[nt][d][i + 2] *= corr;
              }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float base0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], base1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
          for (int e = 0; e < H; ++e) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = exp2_of(acc[e][nt][i] - ((i & 1) ? base1 : base0));
            // the sum takes the weights as they are multiplied, rounded to fp16: their rounding then
            // cancels where few weights dominate. (Below 2^-14, where fp16 loses bits, it takes them
            // as they are: a block of small values has small w but counts in the sum by w / vs.)
            const __half2 w0 = __floats2half2_rn(w[0], w[1]), w1 = __floats2half2_rn(w[2], w[3]);
            const float2 f0 = __half22float2(w0), f1 = __half22float2(w1);
            const float least = 6.103515625e-05f;
            const float sum0 = (w[0] < least ? w[0] : f0.x) + (w[2] < least ? w[2] : f1.x);
            const float sum1 = (w[1] < least ? w[1] : f0.y) + (w[3] < least ? w[3] : f1.y);
            l[nt][0] += sum0 == 0.f ? 0.f : sum0 * inv[e];  // (a masked token's scale may be NaN)
            l[nt][1] += sum1 == 0.f ? 0.f : sum1 * inv[e];
            wb[e][nt][0] = transpose8x8(as_u32(w0));
            wb[e][nt][1] = transpose8x8(as_u32(w1));
          }
        }
      };

      // ---- complete blocks
      int stage = 0;
#pragma unroll 1
      for (int u = ua + warp; u < last_code; u += W) {
        __syncwarp();  // every lane is done with the unit before
        issue(u + (C::kStages - 1) * W, stage == 0 ? C::kStages - 1 : stage - 1);
        look_up(u + C::kStages * W);
        asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
        __syncwarp();  // the unit is there for every lane
        const uint32_t at = ring_a + stage * C::kStage;
        stage = stage + 1 == C::kStages ? 0 : stage + 1;
        const uint4 sc = lds128m(at + 4 * C::kHalf);
        float acc[2][NT][4];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[e][nt][0] = acc[e][nt][1] = acc[e][nt][2] = acc[e][nt][3] = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          uint4 kx[2], ky[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            kx[e] = lds128m(at + e * 2 * C::kHalf + piece_at<D>(gid, q4 * J + j));
            ky[e] = lds128m(at + e * 2 * C::kHalf + piece_at<D>(gid + 8, q4 * J + j));
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t xw = (k == 0 ? kx[e].x : k == 1 ? kx[e].y : k == 2 ? kx[e].z : kx[e].w) ^ 0x80808080u;
              const uint32_t yw = (k == 0 ? ky[e].x : k == 1 ? ky[e].y : k == 2 ? ky[e].z : ky[e].w) ^ 0x80808080u;
              const uint32_t a0 = codes_h2(xw, 0x4140u), a1 = codes_h2(yw, 0x4140u);
              const uint32_t a2 = codes_h2(xw, 0x4342u), a3 = codes_h2(yw, 0x4342u);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16(acc[e][nt], a0, a1, a2, a3, qb[nt][4 * j + k][0], qb[nt][4 * j + k][1]);
            }
        }
        const float ks[2] = {__uint_as_float(sc.x), __uint_as_float(sc.z)};
        const float vs[2] = {__uint_as_float(sc.y), __uint_as_float(sc.w)};
        uint32_t wb[2][NT][2];
        weigh(acc, wb, u * kUnit, code_end, ks, vs);
        // row gid of value tile i is dim gid * DPT + 2 i, row gid + 8 the one after it
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t v_a = at + (2 * e + 1) * C::kHalf;
          uint32_t vw[4][DPT / 4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // tokens 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9
            const int row = q4 * 2 + (k & 1) + (k >> 1) * 8;
            if (D == 128) {
              const uint4 v = lds128m(v_a + piece_at<D>(row, gid));
              vw[k][0] = v.x; vw[k][1] = v.y; vw[k][DPT / 4 - 2] = v.z; vw[k][DPT / 4 - 1] = v.w;
            } else {
              const uint2 v = lds64(v_a + piece_at<D>(row, gid >> 1) + (gid & 1) * 8);
              vw[k][0] = v.x; vw[k][1] = v.y;
            }
          }
#pragma unroll
          for (int w = 0; w < DPT / 4; ++w) {
            uint32_t a[2][4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t xw = vw[2 * k][w] ^ 0x80808080u, yw = vw[2 * k + 1][w] ^ 0x80808080u;
              const uint32_t lo = __byte_perm(xw, yw, 0x5140u), hi = __byte_perm(xw, yw, 0x7362u);
              a[0][2 * k] = codes_h2(lo, 0x4140u);
              a[0][2 * k + 1] = codes_h2(lo, 0x4342u);
              a[1][2 * k] = codes_h2(hi, 0x4140u);
              a[1][2 * k + 1] = codes_h2(hi, 0x4342u);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16(o[nt][2 * w + i], a[i][0], a[i][1], a[i][2], a[i][3], wb[e][nt][0], wb[e][nt][1]);
          }
        }
      }

      // ---- rows of the incomplete block, 16 at a time: lifted by a power of two of their own and taken
      // as fp16 (a bf16 value has 8 significant bits; what is lost lies 2^-24 below the largest)
      const int first_tail = max(ua, x.code_units);
      const int ahead = (warp + W - (first_tail - ua) % W) % W;  // units go round the warps without a break
#pragma unroll 1
      for (int i16 = 2 * (first_tail + ahead); i16 < 2 * ub; i16 += (i16 & 1) ? 2 * W - 1 : 1) {
        const int pos0 = x.held + (i16 - 2 * x.code_units) * 16;
        if (pos0 >= x.visible) continue;
        const int L = x.s.start + x.s.n;
        const int64_t bh = ((int64_t)b * c.kv_heads + h) * 2 * P;
        float acc[1][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[0][nt][0] = acc[0][nt][1] = acc[0][nt][2] = acc[0][nt][3] = 0.f;
        uint4 kx[2][2 * J];
        float kmax = 0.f, vmax = 0.f;
        auto largest = [](const uint4& v, float& top) {
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 p = pair_of<T>(w[i]);
            top = fmaxf(top, fmaxf(finite_abs(p.x), finite_abs(p.y)));
          }
        };
        auto row_of = [&](const void* rows, int pos) {
          return reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(rows) + (bh + (pos & (2 * P - 1))) * D);
        };
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int pos = pos0 + gid + e * 8;
          const uint4* row = row_of(c.k_ring, pos) + q4 * 2 * J;
#pragma unroll
          for (int i = 0; i < 2 * J; ++i) {
            kx[e][i] = pos < L ? row[i] : make_uint4(0u, 0u, 0u, 0u);
            largest(kx[e][i], kmax);
          }
        }
        // (the values are read twice, the second time from L1: once for their maximum, once to multiply)
        auto value_piece = [&](int e, int i) {
          const int pos = pos0 + q4 * 2 + (e & 1) + (e >> 1) * 8;
          return pos < L ? row_of(c.v_ring, pos)[gid * (DPT / 8) + i] : make_uint4(0u, 0u, 0u, 0u);
        };
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < DPT / 8; ++i) largest(value_piece(e, i), vmax);
        float ks[1], vs[1];
        const float klift = lift_of(warp_max(kmax), 10, ks[0]), vlift = lift_of(warp_max(vmax), 7, vs[0]);
        auto lifted = [](uint32_t v, float lift) {
          const float2 p = pair_of<T>(v);
          return as_u32(__floats2half2_rn(p.x * lift, p.y * lift));
        };
#pragma unroll
        for (int i = 0; i < 2 * J; ++i) {  // 8 dims: k-steps 2 i, 2 i + 1
          const uint32_t xs[4] = {kx[0][i].x, kx[0][i].y, kx[0][i].z, kx[0][i].w};
          const uint32_t ys[4] = {kx[1][i].x, kx[1][i].y, kx[1][i].z, kx[1][i].w};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t a0 = lifted(xs[2 * k], klift), a1 = lifted(ys[2 * k], klift);
            const uint32_t a2 = lifted(xs[2 * k + 1], klift), a3 = lifted(ys[2 * k + 1], klift);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16(acc[0][nt], a0, a1, a2, a3, qb[nt][2 * i + k][0], qb[nt][2 * i + k][1]);
          }
        }
        uint32_t wb[1][NT][2];
        weigh(acc, wb, pos0, L, ks, vs);
#pragma unroll
        for (int i = 0; i < DPT / 8; ++i) {
          uint32_t y[4][4];  // [token][pair of dims], lifted
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 v = value_piece(e, i);
            y[e][0] = lifted(v.x, vlift); y[e][1] = lifted(v.y, vlift);
            y[e][2] = lifted(v.z, vlift); y[e][3] = lifted(v.w, vlift);
          }
#pragma unroll
          for (int d = 0; d < 4; ++d) {  // value tile 4 i + d: dims 2 d, 2 d + 1 of the eight
            const uint32_t a0 = __byte_perm(y[0][d], y[1][d], 0x5410u), a1 = __byte_perm(y[0][d], y[1][d], 0x7632u);
            const uint32_t a2 = __byte_perm(y[2][d], y[3][d], 0x5410u), a3 = __byte_perm(y[2][d], y[3][d], 0x7632u);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16(o[nt][4 * i + d], a0, a1, a2, a3, wb[0][nt][0], wb[0][nt][1]);
          }
        }
      }

      // ---- merge the warps, each one's outputs in its drained ring
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
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
          float* dst = reinterpret_cast<float*>(ring) + r * C::kO + gid * DPT;
#pragma unroll
          for (int i = 0; i < MT; ++i) *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(o[nt][i][e], o[nt][i][e + 2]);
        }
      __syncthreads();
      const bool whole = ua == 0 && ub == x.units;
      const int64_t slot = ((int64_t)rt * (gridDim.x + heads) + cta + b * c.kv_heads + h) * ROWS;
      const int some = min(W, ub - ua);  // warps that had units
#pragma unroll 1
      for (int i = threadIdx.x; i < ROWS * D / 4; i += C::kThreads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        const int row = rt * sh.tile + r, t = row / sh.G, g = row - t * sh.G;
        if (row >= sh.rows) break;  // (rows rise with i)
        float top = -INFINITY;
        for (int w = 0; w < some; ++w) top = fmaxf(top, ml_s[w * ROWS + r].x);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int w = 0; w < some; ++w) {
          const float2 ml = ml_s[w * ROWS + r];
          // (nothing visible: -inf and no sum; NaN scores: NaN sums, which must count)
          const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_of(ml.x - top);
          const float4 v = *reinterpret_cast<const float4*>(smem + (size_t)w * C::kWarpBytes + ((size_t)r * C::kO + d) * 4);
          sum = fmaf(ml.y, f, sum);
          acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y);
          acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
        }
        if (whole) {
          T* dst = out + (((int64_t)b * sp.tokens + t) * sh.Hq + h * sh.G + g) * D + d;
          const bool live = t < x.s.n;
          dst[0] = Conv<T>::from_f32(live ? acc.x / sum : 0.f);
          dst[1] = Conv<T>::from_f32(live ? acc.y / sum : 0.f);
          dst[2] = Conv<T>::from_f32(live ? acc.z / sum : 0.f);
          dst[3] = Conv<T>::from_f32(live ? acc.w / sum : 0.f);
        } else {
          *reinterpret_cast<float4*>(part + (slot + r) * D + d) = acc;
          if (d == 0) part_ml[slot + r] = make_float2(top, sum);
        }
      }
      __syncthreads();  // the shared memory is free for the next (sequence, head)
    }
    off -= x.units * c.kv_heads;  // zero where the run goes on into the next sequence
  }
}

// ---------------------------------------------------------------- join the parts
// grid (KV heads x rows of a tile, batch, row tiles), four warps: an output row that several CTAs
// shared is the weighted sum of their parts; one that none took (it does not count) becomes
// zeros. A warp takes every fourth part, a lane D / 32 of its values.
constexpr int kJoinWarps = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32)
block_attn_join_kernel(const lq_block_kv c, const BlockSpan sp, const Shape sh, int ctas, T* __restrict__ out,
                       const float* __restrict__ part, const float2* __restrict__ part_ml, int* error_word) {
  constexpr int V = D / 32;
  __shared__ float acc_s[kJoinWarps][D], sum_s[kJoinWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int h = blockIdx.x % c.kv_heads, r = blockIdx.x / c.kv_heads, b = blockIdx.y, rt = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = rt * sh.tile + r, t = row / sh.G, g = row - t * sh.G;
  if (row >= sh.rows) return;
  // (start and count are older than the kernel ahead, which has waited for their writer)
  const Tile x = tile_of(c, sp, sh, b, rt);
  const int heads = c.batch * c.kv_heads;
  int c0 = 0, c1 = -1;
  if (x.units > 0) {
    const int2 line = units_before(c, sp, sh, rt, b);
    const Cut cut = cut_of(line.x, ctas, heads, sh.warps);
    c0 = cut.owner(line.y + h * x.units);
    c1 = cut.owner(line.y + (h + 1) * x.units - 1);
  }
  T* dst = out + (((int64_t)b * sp.tokens + t) * sh.Hq + h * sh.G + g) * D;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (x.units > 0 && c0 == c1) return;  // one CTA had all of it and wrote the output
  if (x.bad && threadIdx.x == 0) atomicExch(error_word, LQ_BLOCK_BAD_POSITION);
  if (x.units == 0 || t >= x.s.n) {
    for (int d = threadIdx.x; d < D; d += kJoinWarps * 32) dst[d] = Conv<T>::from_f32(0.f);
    return;
  }
  const int64_t slot = ((int64_t)rt * (ctas + heads) + b * c.kv_heads + h + c0) * sh.tile + r;
  const int parts = c1 - c0 + 1;
  const float2* ml = part_ml + slot;
  const float* mine = part + slot * D + lane * V;
  float top = -INFINITY;
  for (int k = lane; k < parts; k += 32) top = fmaxf(top, ml[(int64_t)k * sh.tile].x);
  top = warp_max(top);
  float sum = 0.f, acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int k = warp; k < parts; k += kJoinWarps) {
    const float2 w = ml[(int64_t)k * sh.tile];
    const float f = w.x == -INFINITY ? (w.y == 0.f ? 0.f : 1.f) : exp2_of(w.x - top);
    const float* v = mine + (int64_t)k * sh.tile * D;
    sum = fmaf(w.y, f, sum);
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = fmaf(v[i], f, acc[i]);
  }
  if (lane == 0) sum_s[warp] = sum;
#pragma unroll
  for (int i = 0; i < V; ++i) acc_s[warp][lane * V + i] = acc[i];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kJoinWarps * 32) {
    float v = 0.f, all = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
      v += acc_s[w][d];
      all += sum_s[w];
    }
    dst[d] = Conv<T>::from_f32(v / all);
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
  p.sh.warps = p.nt == 1 ? Cfg<128, 1>::kWarps : Cfg<128, 2>::kWarps;
  p.tiles = (p.sh.rows + p.sh.tile - 1) / p.sh.tile;
  p.ctas = sm_count() / p.tiles;
  if (p.ctas < 1) p.ctas = 1;
  return p;
}

int64_t slots_of(const lq_block_kv& c, const Plan& p) {
  return (int64_t)p.tiles * (p.ctas + (int64_t)c.batch * c.kv_heads) * p.sh.tile;
}
int64_t scratch_bytes(const lq_block_kv& c, const Plan& p) { return slots_of(c, p) * (c.head_dim + 2) * 4; }

int check_attn(const lq_block_kv* c, int Hq, int T_new, const char* what) {
  if (const int rc = check_block_kv(c, what)) return rc;
  LQ_REQUIRE(Hq > 0 && Hq % c->kv_heads == 0 && T_new > 0, LQ_ERR_ARG,
             "%s: %d query heads do not share %d KV heads evenly, or there are no rows", what, Hq, c->kv_heads);
  LQ_REQUIRE(c->dtype != LQ_F32, LQ_ERR_UNSUPPORTED, "%s: built for float16 and bfloat16 rows", what);
  LQ_REQUIRE(c->kv_heads <= 65535 && (int64_t)T_new * (Hq / c->kv_heads) <= 65535LL * 8, LQ_ERR_ARG,
             "%s: too many rows for one call", what);
  LQ_REQUIRE((int64_t)c->batch * c->kv_heads * ((int64_t)c->max_blocks * c->block / kUnit + 2) < 0x7fffffffLL, LQ_ERR_ARG,
             "%s: batch, heads and positions together are too many for one call", what);
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
  constexpr size_t smem = Cfg<D, NT>::kTotal;
  if (const int rc = ensure_smem_limit(reinterpret_cast<const void*>(kern), (int)smem, what)) return rc;
  const float qk_scale = scaling * 1.4426950408889634f;
  float* part = (float*)scratch;
  float2* part_ml = (float2*)(part + slots_of(c, p) * D);
  if (const int rc = launch(kern, dim3((unsigned)p.ctas, (unsigned)p.tiles), Cfg<D, NT>::kThreads, smem, stream, pdl, what, c, sp, p.sh,
                            (const T*)q, qs[0], qs[1], qs[2], (T*)out, part, part_ml, qk_scale, error_word))
    return rc;
  const unsigned rows = (unsigned)(p.sh.rows < p.sh.tile ? p.sh.rows : p.sh.tile);
  return launch(block_attn_join_kernel<T, D>, dim3((unsigned)c.kv_heads * rows, (unsigned)c.batch, (unsigned)p.tiles),
                kJoinWarps * 32, 0, stream, 1, what, c, sp, p.sh, p.ctas, (T*)out, (const float*)part, (const float2*)part_ml,
                error_word);
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
