// Attention of the newest tokens over the block-scaled KV cache (layout: block_kv.cuh).
//
//   out[t, h] = sum_p softmax_p(scaling q[t, h] . k[p]) v[p],  p <= start + t
//
// One pass over the cache. The codes go to the tensor cores as fp16 integers (exact); the scales
// never touch an element: with key scale ks and value scale vs of a block,
//   x_p = log2(e) scaling ks (q . code_p) + log2(vs),  M = a little below the running maximum of x,
//   w_p = 2^(x_p - M)  (the weight with the value scale folded in),
//   O  += w_p code_p,  sum += (sum of the block's w_p) / vs,   out = O / sum.
//
// A unit of work is 32 tokens of one KV head. The units of all sequences and heads form one line,
// which the warps share in contiguous runs, so ragged lengths and single long contexts both fill
// the GPU without the host knowing a length. A warp is a CTA: it never waits for another one. At
// the end of a (sequence, head), or of its run, it writes the outputs where it had all of it, else a
// partial (M, sum, O) to scratch, and the second kernel joins the parts.
//
// Scores are computed as K q^T (16 tokens x 8 query rows a tile) and outputs as V^T w (16 dims x 8
// query rows), so that the few query rows of a decode step are the narrow side of the MMA: with
// queries as its 16 rows half of every product would be padding. The k index of the first product
// and the row index of the second are mapped onto the head's dims so that each thread's bytes of
// a cached row are contiguous.
#include <type_traits>

#include "block_kv.cuh"
#include "block_parts.cuh"
#include "tcgen05.cuh"

namespace lq {
namespace {

constexpr int kUnit = 32;  // tokens, as two halves of 16 (the height of an MMA tile)
constexpr float kNone = -1e30f;  // a maximum of nothing: below any score, and 2^(kNone - M) is zero
// Weights are held as fp16, which keeps 11 bits from 2^-14 to 2^15: M is set 2^kUp below the maximum and
// follows it when a weight would pass 2^kMost, so that what lies 2^-21 below the largest still has its bits.
// Long contexts have many such: with M at the maximum, 131071 weights of 1.25 * 2^-24 of the largest, 1 % of
// the sum, were off by a fifth.
constexpr float kUp = 7.f, kMost = 15.f;
constexpr int kLowestValue = -95;  // exponent below which ring values are lifted no further

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
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
__device__ __forceinline__ float lift_of(float amax, int top, float& unit, int lowest = -100) {
  int e = (int)(__float_as_uint(amax) >> 23) - 127;
  e = amax > 0.f ? max(e, lowest) : top;
  unit = __uint_as_float((unsigned)(127 + e - top) << 23);
  return __uint_as_float((unsigned)(127 - e + top) << 23);
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// Two halves, 0 in the place of one that is not finite
__device__ __forceinline__ uint32_t finite_h2(uint32_t v) {
  return v & __hle2_mask(__habs2(as_h2(v)), __floats2half2_rn(65504.f, 65504.f));
}

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_of(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float inverse_of(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values in a register pair, for the instructions that work on both
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}

// ---------------------------------------------------------------- how the line of units is cut
// Per cent of a long line that the warps which run at once take: little enough that the short runs behind
// them even out SMs of different speed. 70 / 80 / 90: one context of 131000 tokens 62.7 / 63.2 / 64.4 us, 64
// ragged sequences 67.4 / 67.6 / 71.0, 32 ragged sequences with their append 54.6 / 54.6 / 57.0: 70 and 80
// differ by less than 1 %, above that the last runs end late.
constexpr int kFirst = 80;

struct Shape {
  int Hq, G, rows, tile;  // query rows per KV head: T_new * G; rows of one pass
  uint64_t inv_G;         // ceil(2^32 / G): (row * inv_G) >> 32 = row / G for row * G < 2^32
  int unit_log2;          // tokens of a unit
  int slots, waves;       // workers of a tile's line that run at once; 2: a second wave for long lines
  uint32_t step;          // 2^32 / slots
};

__device__ __forceinline__ int token_of(const Shape& sh, int row) { return (int)((uint64_t)(unsigned)row * sh.inv_G >> 32); }

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
  x.t_lo = token_of(sh, rt * sh.tile);
  const int L = x.s.start + x.s.n;
  x.visible = x.s.start + min(x.s.n, token_of(sh, rt * sh.tile + sh.tile - 1) + 1);
  x.held = L & ~(c.block - 1);
  const int more = (1 << sh.unit_log2) - 1;
  x.code_units = (min(x.visible, x.held) + more) >> sh.unit_log2;
  x.units = x.code_units + ((max(0, x.visible - x.held) + more) >> sh.unit_log2);
  if (x.t_lo >= x.s.n) x.code_units = x.units = 0;
  return x;
}

// How the warps share the line of `total` units: up to one unit for each warp that runs at once, one
// each; up to eight, equal runs; above, with one row tile, equal runs over kFirst per cent and as many
// short ones over the rest: SMs stream at speeds up to 30 % apart, and the short runs go to those
// that are done first. (Multiplications in place of divisions: every warp begins with this.)
struct Cut {
  int total, first;  // units of the first wave
  int kind;
  __device__ __forceinline__ Cut(int total_, const Shape& sh) : total(total_), first(total_) {
    kind = total <= sh.slots ? 0 : (sh.waves == 1 || total <= 8 * sh.slots) ? 1 : 2;
    if (kind == 2) first = (int)((int64_t)total * (0x100000000LL / 100 * kFirst) >> 32);
  }
  __device__ __forceinline__ int begin(const Shape& sh, int i) const {
    if (kind == 0) return min(i, total);
    if (i < sh.slots) return (int)((uint64_t)first * ((uint64_t)sh.step * i) >> 32);
    if (kind == 1 || i >= 2 * sh.slots) return total;
    return first + (int)((uint64_t)(total - first) * ((uint64_t)sh.step * (i - sh.slots)) >> 32);
  }
};

// Where run `run` of the line lies: its length, its first sequence, and its begin behind that
// sequence's. One warp calls it.
__device__ __forceinline__ int3 run_of(const lq_block_kv& c, const BlockSpan& sp, const Shape& sh, int rt, int run) {
  const int lane = threadIdx.x & 31;
  int total = 0, mine = 0;
  for (int i = lane; i < c.batch; i += 32) total += mine = tile_of(c, sp, sh, i, rt).units * c.kv_heads;
  total = __reduce_add_sync(0xffffffffu, total);
  const Cut cut(total, sh);
  const int begin = cut.begin(sh, run), length = cut.begin(sh, run + 1) - begin;
  int before = 0;
  for (int b0 = 0; b0 < c.batch; b0 += 32) {
    if (c.batch > 32) mine = b0 + lane < c.batch ? tile_of(c, sp, sh, b0 + lane, rt).units * c.kv_heads : 0;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > begin);
    if (hit != 0) {
      const int at = __ffs(hit) - 1;
      return make_int3(length, b0 + at, begin - before - __shfl_sync(0xffffffffu, upto - mine, at));
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return make_int3(0, c.batch, 0);
}

// NT: groups of 8 query rows of a pass. The outputs take NT * D / 4 registers of a thread, so an SM holds 12
// warps with one group of 128 dims (16 of 64 dims) and 8 with two; their rings fill its shared memory.
template <int D, int NT>
struct Cfg {
  static constexpr int kWarps = NT == 1 ? (D == 64 ? 16 : 12) : 8;  // on an SM
  static constexpr int kRows = 8 * NT;
  static constexpr int kCodes = kUnit * D;               // bytes of a unit's keys, or values
  static constexpr int kStage = 2 * kCodes + 16;         // keys, values, (key, value) scales of the two halves
  static constexpr int kStages = NT == 1 ? (D == 64 ? 3 : 2) : (D == 64 ? 6 : 3);  // units in a warp's ring
  static constexpr size_t kRing = kStages * kStage;
  static_assert(kStage % 16 == 0 && kWarps * (kRing + 1024) <= 228 * 1024, "");
};

// Offset of 16-byte piece `chunk` of row `row` of a unit's staged keys or values. Pieces are
// XOR-swizzled so that both readers are free of bank conflicts: the score product's threads (8 rows
// gid, pieces 2 q4 + j) and the value product's (rows 2 q4, piece gid).
template <int D>
__device__ __forceinline__ uint32_t piece_at(int row, int chunk) {
  if (D == 128) return (uint32_t)row * 128 + ((chunk ^ (row & 7)) << 4);
  return (uint32_t)(row >> 1) * 128 + (((((row & 1) << 2) + chunk) ^ (row & 6)) << 4);
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

// 16 * J consecutive values of a 16-bit row as words
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint16_t* p, bool there, int vec) {
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = 0u;
  if (!there) return;
  if (vec) {  // on a 16-byte boundary
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
  }
}

// Largest magnitude of 16-bit pairs, INF if one is not finite
template <typename T, int N>
__device__ __forceinline__ float largest_of(const uint32_t (&w)[N]) {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  T2 top = __habs2(*reinterpret_cast<const T2*>(&w[0]));
#pragma unroll
  for (int i = 1; i < N; ++i) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const T2*>(&w[i])));
  const float lo = __low2float(top), hi = __high2float(top);
  return lo <= 3.402823466e38f && hi <= 3.402823466e38f ? fmaxf(lo, hi) : INFINITY;
}

// ---------------------------------------------------------------- main kernel
// grid (runs of the line, row tiles), one warp. T is the type of q, out and the ring. Bound by the
// latencies of a warp's units (12 warps on an SM, 1.7 instructions a cycle), by about 8 us before the
// first unit and in the join, and by SMs that stream at different speeds. One row each, 32 query heads
// on 8, bf16, with the join: one context of 131000 tokens (268 MB) 63 us, 4.3 TB/s, 0.66 of a copy's
// rate; 64 ragged contexts to 6000 with heads of 64 (299 MB) 68 us, 4.4 TB/s, 0.68. The same kernel
// that only loads the codes takes 48 us instead of 53 for the long context, before the join.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(32, (Cfg<D, NT>::kWarps))
block_attn_kernel(const lq_block_kv c, const BlockSpan sp, const Shape sh, const T* __restrict__ q, int64_t qsb, int64_t qst,
                  int64_t qsh, int q_vec, T* __restrict__ out, float* __restrict__ part, float2* __restrict__ part_ml,
                  int2* __restrict__ ends, float qk_scale, int* error_word) {
  using C = Cfg<D, NT>;
  constexpr int ROWS = C::kRows, KS = D / 16, MT = D / 16, DPT = D / 8;  // DPT: dims of V a thread owns
  constexpr int J = D / 64;  // 16-byte pieces of a K row a thread reads
  extern __shared__ __align__(16) uint8_t ring[];
  // One group of bf16 queries meets the codes as 15-bit integers in two byte planes: the codes then need
  // no conversion. fp16 queries keep their 11 bits as fp16; with more groups the conversion is shared
  // and the integer product's lower rate counts (512 rows of 32 heads on 3499 tokens, two groups: 278 us
  // by integers, 242 by fp16).
  constexpr bool kInt = NT == 1 && std::is_same<T, __nv_bfloat16>::value;
  constexpr int kTop = kInt ? 13 : 10;  // exponent that a row's largest value is lifted to

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int lane = threadIdx.x, gid = lane >> 2, q4 = lane & 3;
  const int rt = blockIdx.y, P = c.block, shift = 31 - __clz(P);
  const int heads = c.batch * c.kv_heads;
  const int3 run = run_of(c, sp, sh, rt, blockIdx.x);
  int left = run.x, off = run.z;  // units of this run; where it begins behind its first sequence
  const uint32_t ring_a = smem_u32(ring);
  // this lane's places in a stage: pieces it copies (the i-th at + 512 i, alternating at D = 128), pieces of
  // K it reads (rows gid + 8 e at + 8 D e), pieces of V (rows 2 q4 + 8 e at + 8 D e)
  const uint32_t copy_at = piece_at<D>(lane / (D / 16), lane % (D / 16));
  uint32_t k_at[J], v_at[2];
#pragma unroll
  for (int j = 0; j < J; ++j) k_at[j] = piece_at<D>(gid, q4 * J + j);
#pragma unroll
  for (int k = 0; k < 2; ++k)
    v_at[k] = C::kCodes + (D == 128 ? piece_at<D>(q4 * 2 + k, gid) : piece_at<D>(q4 * 2 + k, gid >> 1) + (gid & 1) * 8);

#pragma unroll 1
  for (int b = run.y; left > 0; ++b) {
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

      // ---- the ring: codes and scales of the next units, kStages - 1 of them on their way. The page ids
      // of a unit are requested one unit earlier than its codes.
      const int last_code = min(ub, x.code_units);
      const int code_end = min(x.visible, x.held);
      auto look_up = [&](int u) {
        const int pos = u * kUnit;
        return make_int2(u < last_code ? table[pos >> shift] : 0,
                         P == 16 && u < last_code && pos + 16 < code_end ? table[(pos >> 4) + 1] : 0);
      };
      // `halves` times 16 tokens of a page, from row `first` of it on, to half e of a stage
      auto copy = [&](int id, int first, int e, int stage, auto halves) {
        const uint32_t dst = ring_a + stage * C::kStage + e * (C::kCodes / 2);
        const uint32_t scale_dst = ring_a + stage * C::kStage + 2 * C::kCodes + e * 8;
        if (id < 0 || id >= c.num_pages) {
          if (lane == 0) atomicExch(error_word, LQ_BLOCK_BAD_PAGE);
          if (lane < 2 * halves) asm volatile("st.shared.u32 [%0], %1;" ::"r"(scale_dst + lane * 4), "r"(0x7fffffff) : "memory");
          return;
        }
        const int ph = id * c.kv_heads + h;  // (pages * heads fit 31 bits: a page takes over 2 kB)
        const int64_t at = (((int64_t)ph << shift) + first) * D + lane * 16;
        const int8_t* kp = c.k_pages + at;
        const int8_t* vp = c.v_pages + at;
#pragma unroll
        for (int i = 0; i < halves * D / 32; ++i) {
          const uint32_t to = dst + i * 512 + (D == 128 && (i & 1) ? copy_at ^ 64u : copy_at);
          cp_async16(to, kp + i * 512);
          cp_async16(to + C::kCodes, vp + i * 512);
        }
        if (lane < 2 * halves) cp_async4(scale_dst + lane * 4, ((lane & 1) ? c.v_scales : c.k_scales) + ph);
      };
      auto issue = [&](int u, int2 ids, int stage) {
        if (u < last_code) {
          const int pos = u * kUnit;
          if (P != 16) {
            copy(ids.x, pos & (P - 1), 0, stage, std::integral_constant<int, 2>());
          } else {
            copy(ids.x, 0, 0, stage, std::integral_constant<int, 1>());
            if (pos + 16 < code_end) {
              copy(ids.y, 0, 1, stage, std::integral_constant<int, 1>());
            } else if (lane < 2) {
              // A unit's second half that is not there: its weights are 0, whatever the bytes of its codes, but
              // 0 times the inverse of whatever its scales held before may be a NaN in the sum.
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring_a + stage * C::kStage + 2 * C::kCodes + 8 + lane * 4), "f"(1.f) : "memory");
            }
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      int2 page[C::kStages];
#pragma unroll
      for (int i = 0; i < C::kStages; ++i) page[i] = look_up(ua + i);
      // the query rows: row 8 nt + gid, dims from q4 * 16 J on (requested before the codes, which wait for
      // their page ids)
      uint32_t raw[NT][8 * J];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int row = rt * sh.tile + nt * 8 + gid, t = token_of(sh, row), g = row - t * sh.G;
        load_words(raw[nt], reinterpret_cast<const uint16_t*>(q) + b * qsb + t * qst + (int64_t)(h * sh.G + g) * qsh + q4 * 16 * J,
                   row < sh.rows && t < x.s.n, q_vec);
      }
      __syncwarp();  // every lane is done with the last segment's units
#pragma unroll
      for (int i = 0; i < C::kStages - 1; ++i) issue(ua + i, page[i], i);
      int2 next_page = page[C::kStages - 1];

      // ---- the query rows as B operands, each lifted by a power of two. k-step k is the four (kInt: eight)
      // dims from q4 * 16 J + 4 k (8 k) on; kInt: two k-steps hold the high and the low bytes of one.
      uint32_t qb[NT][KS][2];
      float qu[NT][2];   // what 1 of a product stands for, of the query rows 8 nt + 2 q4 (+ 1)
      int seen[NT][2];   // last position those rows see
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float amax = largest_of<T>(raw[nt]);  // INF if a value is not finite
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        float unit;
        const float lift = lift_of(is_finite(amax) ? amax : 0.f, kTop, unit);
        // (integers cannot carry a NaN: a row that is not finite gets it with its unit)
        unit = amax <= 3.402823466e38f ? unit * qk_scale : __int_as_float(0x7fffffff);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qu[nt][e] = __shfl_sync(0xffffffffu, unit, (q4 * 2 + e) * 4);
          seen[nt][e] = x.s.start + token_of(sh, rt * sh.tile + nt * 8 + q4 * 2 + e);
        }
        if constexpr (kInt) {
#pragma unroll
          for (int k = 0; k < 2 * J; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              // whole + 128 in the low bits of a sum with 1.5 * 2^23, |whole| < 2^14: its second byte is the
              // high byte (whole + 128) >> 8, its first the low byte plus 128
              const float2 v0 = pair_of<T>(raw[nt][4 * k + 2 * i]), v1 = pair_of<T>(raw[nt][4 * k + 2 * i + 1]);
              const uint32_t a0 = __float_as_uint(fmaf(v0.x, lift, 12583040.f)), a1 = __float_as_uint(fmaf(v0.y, lift, 12583040.f));
              const uint32_t a2 = __float_as_uint(fmaf(v1.x, lift, 12583040.f)), a3 = __float_as_uint(fmaf(v1.y, lift, 12583040.f));
              const uint32_t x01 = __byte_perm(a0, a1, 0x5140u), x23 = __byte_perm(a2, a3, 0x5140u);  // low, low, high, high
              qb[nt][2 * k][i] = __byte_perm(x01, x23, 0x7632u);
              qb[nt][2 * k + 1][i] = __byte_perm(x01, x23, 0x5410u) ^ 0x80808080u;
            }
        } else {
#pragma unroll
          for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 v = pair_of<T>(raw[nt][2 * k + i]);
              qb[nt][k][i] = as_u32(__floats2half2_rn(v.x * lift, v.y * lift));
            }
        }
      }
      float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = kNone;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      }

      // raw products of H halves (tokens from pos0 on, positions below `end` exist) to weights as the B
      // operands of the value product
      auto weigh = [&](auto& acc, auto& wb, int pos0, int end, const auto& ks, const auto& vs) {
        constexpr int H = sizeof(ks) / sizeof(float);
        float inv[H];
#pragma unroll
        for (int e = 0; e < H; ++e) {
          const float lv = log2_of(vs[e]);
          inv[e] = fminf(inverse_of(vs[e]), 3.0e38f);  // (of a NaN scale: a number; the weights are NaN then)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[e][nt][i] = fmaf(acc[e][nt][i], qu[nt][i & 1] * ks[e], lv);
        }
        if (pos0 + 16 * H - 1 > min(first_seen, end - 1)) {
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
        bool rises = false;
        float mx[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            mx[nt][i] = fmaxf(acc[0][nt][i], acc[0][nt][i + 2]);
            if (H == 2) mx[nt][i] = fmaxf(mx[nt][i], fmaxf(acc[H - 1][nt][i], acc[H - 1][nt][i + 2]));
            rises = rises || mx[nt][i] > m[nt][i] + kMost;
          }
        if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float to = fmaxf(mx[nt][i], __shfl_xor_sync(0xffffffffu, mx[nt][i], 4));
              to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 8));
              to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 16));
              to = fmaxf(to - kUp, m[nt][i]);
              const float corr = exp2_of(m[nt][i] - to);
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
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < H; ++e) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = exp2_of(acc[e][nt][i] - m[nt][i & 1]);
            // (the sum takes the weights in fp32: a block of small values has weights that fp16 would
            // lose, but counts in the sum by w / vs)
            l[nt][0] = fmaf(w[0] + w[2], inv[e], l[nt][0]);
            l[nt][1] = fmaf(w[1] + w[3], inv[e], l[nt][1]);
            wb[e][nt][0] = transpose8x8(as_u32(__floats2half2_rn(w[0], w[1])));
            wb[e][nt][1] = transpose8x8(as_u32(__floats2half2_rn(w[2], w[3])));
          }
      };

      // ---- complete blocks
      int stage = 0;
#pragma unroll 1
      for (int u = ua; u < last_code; ++u) {
        __syncwarp();  // every lane is done with the unit before
        issue(u + C::kStages - 1, next_page, stage == 0 ? C::kStages - 1 : stage - 1);
        next_page = look_up(u + C::kStages);
        asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
        __syncwarp();  // the unit is there for every lane
        const uint32_t at = ring_a + stage * C::kStage;
        stage = stage + 1 == C::kStages ? 0 : stage + 1;
        const uint4 sc = lds128m(at + 2 * C::kCodes);
        float acc[2][NT][4];
        if constexpr (kInt) {
          int sum[2][NT][2][4];
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[e][nt][0][i] = sum[e][nt][1][i] = 0;
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint4 kx = lds128m(at + k_at[j] + e * 16 * D), ky = lds128m(at + k_at[j] + e * 16 * D + 8 * D);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const uint32_t a0 = k ? kx.z : kx.x, a1 = k ? ky.z : ky.x, a2 = k ? kx.w : kx.y, a3 = k ? ky.w : ky.y;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int plane = 0; plane < 2; ++plane)
                    mma8(sum[e][nt][plane], a0, a1, a2, a3, qb[nt][(2 * j + k) * 2 + plane][0], qb[nt][(2 * j + k) * 2 + plane][1]);
              }
            }
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[e][nt][i] = (float)(sum[e][nt][0][i] * 256 + sum[e][nt][1][i]);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[e][nt][0] = acc[e][nt][1] = acc[e][nt][2] = acc[e][nt][3] = 0.f;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            uint4 kx[2], ky[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              kx[e] = lds128m(at + k_at[j] + e * 16 * D);
              ky[e] = lds128m(at + k_at[j] + e * 16 * D + 8 * D);
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
        }
        const float ks[2] = {__uint_as_float(sc.x), __uint_as_float(sc.z)};
        const float vs[2] = {__uint_as_float(sc.y), __uint_as_float(sc.w)};
        uint32_t wb[2][NT][2];
        weigh(acc, wb, u * kUnit, code_end, ks, vs);
        // row gid of value tile i is dim gid * DPT + 2 i, row gid + 8 the one after it
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t vw[4][DPT / 4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // tokens 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9
            const uint32_t from = at + v_at[k & 1] + e * 16 * D + (k >> 1) * 8 * D;
            if (D == 128) {
              const uint4 v = lds128m(from);
              vw[k][0] = v.x; vw[k][1] = v.y; vw[k][DPT / 4 - 2] = v.z; vw[k][DPT / 4 - 1] = v.w;
            } else {
              const uint2 v = lds64(from);
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
#pragma unroll 1
      for (int i16 = 2 * max(ua, x.code_units); i16 < 2 * ub; ++i16) {
        const int pos0 = x.held + (i16 - 2 * x.code_units) * 16;
        if (pos0 >= x.visible) break;
        const int L = x.s.start + x.s.n;
        const int64_t bh = ((int64_t)b * c.kv_heads + h) * 2 * P;
        float acc[1][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[0][nt][0] = acc[0][nt][1] = acc[0][nt][2] = acc[0][nt][3] = 0.f;
        uint4 kx[2][2 * J];
        float kmax = 0.f, vmax = 0.f;
        // A token with a value that is not finite: its key becomes NaN, and so its score for the rows that see it; the
        // value itself counts as 0, so that a row that does not see the token (weight 0) is as without it.
        uint32_t strange = 0u;
        auto row_of = [&](const void* rows, int pos) {
          return reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(rows) + (bh + (pos & (2 * P - 1))) * D);
        };
        // (the values are read twice, the second time from L1: once for their maximum, once to multiply)
        auto value_piece = [&](int e, int i) {
          const int pos = pos0 + q4 * 2 + (e & 1) + (e >> 1) * 8;
          return pos < L ? row_of(c.v_ring, pos)[gid * (DPT / 8) + i] : make_uint4(0u, 0u, 0u, 0u);
        };
        constexpr int kAtOnce = D == 64 ? 2 : 4;  // (heads of 64 have 128 registers: all four at once cost 72 us instead
        // of 68 on 64 ragged contexts to 6000)
#pragma unroll kAtOnce
        for (int e = 0; e < 4; ++e) {
          uint32_t w[DPT / 2];
#pragma unroll
          for (int i = 0; i < DPT / 8; ++i) {
            const uint4 v = value_piece(e, i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
          }
          const float top = largest_of<T>(w);
          vmax = fmaxf(vmax, is_finite(top) ? top : 0.f);
          strange |= (is_finite(top) ? 0u : 1u) << (q4 * 2 + (e & 1) + (e >> 1) * 8);
        }
        strange = __reduce_or_sync(0xffffffffu, strange);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int pos = pos0 + gid + e * 8;
          const uint4* row = row_of(c.k_ring, pos) + q4 * 2 * J;
#pragma unroll
          for (int i = 0; i < 2 * J; ++i) kx[e][i] = pos < L ? row[i] : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t w[8 * J];
#pragma unroll
          for (int i = 0; i < 2 * J; ++i) {
            w[4 * i] = kx[e][i].x; w[4 * i + 1] = kx[e][i].y; w[4 * i + 2] = kx[e][i].z; w[4 * i + 3] = kx[e][i].w;
          }
          const float top = largest_of<T>(w);
          kmax = fmaxf(kmax, is_finite(top) ? top : 0.f);
          kx[e][0].x |= !is_finite(top) || (strange >> (gid + e * 8) & 1u) ? 0x7fff7fffu : 0u;
        }
        float ks[1], vs[1];
        const float klift = lift_of(warp_max(kmax), 10, ks[0]);
        if (kInt) ks[0] *= 8.f;  // the fp16 queries are lifted 2^3 less than the integers
        // (1 / vs up to 2^102, a weight up to 2^15, fewer than 2^7 rows: the sum stays finite)
        const float vlift = lift_of(warp_max(vmax), 7, vs[0], kLowestValue);
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
            for (int nt = 0; nt < NT; ++nt) {
              uint32_t b0 = qb[nt][2 * i + k][0], b1 = qb[nt][2 * i + k][1];
              if constexpr (kInt) {  // the integers put together again: 15 bits, of which fp16 takes 11; and exactly
                // as many as a bf16 query had, down to 2^-14 of its row's largest
                const uint32_t hi = qb[nt][2 * i][k], lo = qb[nt][2 * i + 1][k];
                auto whole = [&](int n) { return (float)((int)(int8_t)(hi >> (8 * n)) * 256 + (int)(int8_t)(lo >> (8 * n))) * 0.125f; };
                b0 = as_u32(__floats2half2_rn(whole(0), whole(1)));
                b1 = as_u32(__floats2half2_rn(whole(2), whole(3)));
              }
              mma16(acc[0][nt], a0, a1, a2, a3, b0, b1);
            }
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
            y[e][0] = finite_h2(lifted(v.x, vlift)); y[e][1] = finite_h2(lifted(v.y, vlift));
            y[e][2] = finite_h2(lifted(v.z, vlift)); y[e][3] = finite_h2(lifted(v.w, vlift));
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

      // ---- what this run has of the (sequence, head): all of it, or a part
      const bool whole = ua == 0 && ub == x.units;
      const int64_t slot = part_slot(rt, gridDim.x, heads, blockIdx.x, b * c.kv_heads + h, ROWS);
      if (lane == 0) {  // for the join: the runs that begin and end it
        if (ua == 0) ends[(int64_t)rt * heads + b * c.kv_heads + h].x = blockIdx.x;
        if (ub == x.units) ends[(int64_t)rt * heads + b * c.kv_heads + h].y = blockIdx.x;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[nt][e];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int r = nt * 8 + q4 * 2 + e, row = rt * sh.tile + r, t = token_of(sh, row), g = row - t * sh.G;
          if (row >= sh.rows) continue;
          if (whole) {
            // (1 / sum is exact enough: one rounding of 2^-24 before the one of T)
            const float inv = t < x.s.n ? 1.f / sum : 0.f;
            uint32_t w[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i)
              w[i] = t < x.s.n ? pair_to<T>(o[nt][i][e] * inv, o[nt][i][e + 2] * inv) : 0u;
            uint4* dst = reinterpret_cast<uint4*>(out + (((int64_t)b * sp.tokens + t) * sh.Hq + h * sh.G + g) * D + gid * DPT);
#pragma unroll
            for (int i = 0; i < MT / 4; ++i) dst[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          } else {
            float4* dst = reinterpret_cast<float4*>(part + (slot + r) * D + gid * DPT);
#pragma unroll
            for (int i = 0; i < MT / 2; ++i)
              dst[i] = make_float4(o[nt][2 * i][e], o[nt][2 * i][e + 2], o[nt][2 * i + 1][e], o[nt][2 * i + 1][e + 2]);
            if (gid == 0) part_ml[slot + r] = make_float2(m[nt][e], sum);
          }
        }
    }
    off -= x.units * c.kv_heads;  // zero where the run goes on into the next sequence
  }
}

// ---------------------------------------------------------------- many query rows
// Prompt chunks, and drafts of many heads: 128 query rows to a CTA, one to a thread, and units of 64
// tokens, on tcgen05. The products' accumulators are in tensor memory: scores [128, 64], outputs
// [128, D]; a thread reads its row of scores, so that maximum and sum need no exchange, and writes its
// row of weights as the next product's A operand. The codes become fp16 tiles in shared memory once for
// all 128 rows, the values' tile transposed on the way (both operands of a product run along k). The
// outputs are only touched, by a warp for its 32 rows, when a row's maximum rises by 2^8 above the last one. Two CTAs on an
// SM: while one converts or exponentiates the other's products run. The weights, scales, masks and
// parts are the ones of the kernel above. Bound by the instructions around the products and their
// latencies (8 warps on an SM, 1.24 instructions a cycle, the tensor pipe busy 18 % of the time): 512 rows of
// 32 heads on 8 after 3499 tokens, 31.5 GFLOP in 115 us with 14 us of join, 274 TFLOP/s. Two threads to
// a row (16 warps on an SM) take 127 us: what is done once a unit and thread is done twice.
constexpr int kManyTile = 128, kManyThreads = 128, kManyUnit = 64, kManyCtas = 2;  // CTAs on an SM
constexpr uint32_t kManyCols = 256, kOutCol = 64;  // columns of tensor memory a CTA takes; where the outputs begin

template <int D>
struct ManyCfg {
  static constexpr int kQ = kManyTile * D * 2, kK = kManyUnit * D * 2, kV = D * kManyUnit * 2, kP = kManyTile * kManyUnit * 2;
  static constexpr int kRaw = kManyUnit * D;  // a unit's codes of keys, or values
  static constexpr size_t kTotal = 1024 + kQ + kK + kV + kP + 2 * kRaw;  // (1024: to begin on such a boundary)
  static_assert(kManyCtas * (kTotal + 1400) <= 228 * 1024, "");
};

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t a) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(a) : "memory");
}
// f32 <- f16 x f16 of kind::f16, M = 128, N columns, both operands along k
constexpr uint32_t many_idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kManyTile >> 4) << 24); }
// Address of 16-byte piece `piece` of row `row` in a tile of 128-byte rows, 128-byte swizzle
__device__ __forceinline__ uint32_t swizzled(uint32_t tile, int row, int piece) {
  return tile + row * 128 + ((piece ^ (row & 7)) << 4);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
        "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
        "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kManyThreads, kManyCtas)
block_attn_many_kernel(const lq_block_kv c, const BlockSpan sp, const Shape sh, const T* __restrict__ q, int64_t qsb,
                       int64_t qst, int64_t qsh, int q_vec, T* __restrict__ out, float* __restrict__ part,
                       float2* __restrict__ part_ml, int2* __restrict__ ends, float qk_scale, int* error_word) {
  using C = ManyCfg<D>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(8) uint64_t bar_s[2];   // scores are there, outputs are there
  __shared__ uint32_t tmem_s;
  __shared__ float4 scale_s[4];                // of 16 tokens each: ks, log2 vs, 1 / vs
  __shared__ float2 raw_scale_s[4], lift_s[4];
  __shared__ int dead_s;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t q_a = (smem_u32(smem) + 1023u) & ~1023u, k_a = q_a + C::kQ, v_a = k_a + C::kK, p_a = v_a + C::kV;
  const uint32_t raw_k = p_a + C::kP, raw_v = raw_k + C::kRaw;
  const uint32_t bar_scores = smem_u32(&bar_s[0]), bar_outputs = smem_u32(&bar_s[1]);
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_s)), "r"(kManyCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    mbar_init(bar_scores, 1);
    mbar_init(bar_outputs, 1);
    dead_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  // (only now: a dependent kernel that takes tensor memory before it waits must not come between)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = tmem_s + ((uint32_t)(warp * 32) << 16);  // this warp's rows
  const int rt = blockIdx.y, P = c.block, shift = 31 - __clz(P);
  const int heads = c.batch * c.kv_heads;
  const int3 run = run_of(c, sp, sh, rt, blockIdx.x);
  int left = run.x, off = run.z;
  uint32_t phase = 0;  // of both barriers: one completion of each per unit
  const int row = rt * kManyTile + tid, tok = token_of(sh, row), g = row - tok * sh.G;

#pragma unroll 1
  for (int b = run.y; left > 0; ++b) {
    const Tile x = tile_of(c, sp, sh, b, rt);
    if (off >= x.units * c.kv_heads) {
      off -= x.units * c.kv_heads;
      continue;
    }
    const int* table = c.table + (int64_t)b * c.max_blocks;
    const int L = x.s.start + x.s.n, code_end = min(x.visible, x.held), seen = x.s.start + tok;
    const bool live = row < sh.rows && tok < x.s.n;
#pragma unroll 1
    for (int h = off / x.units; h < c.kv_heads && left > 0; ++h) {
      const int ua = off - h * x.units;
      const int ub = min(x.units, ua + left);
      off += ub - ua;
      left -= ub - ua;
      if (dead_s) {  // a wait ran out: what this CTA would have begun has no parts
        if (tid == 0 && ua == 0) ends[(int64_t)rt * heads + b * c.kv_heads + h].x = -1;
        continue;
      }
      const int last_code = min(ub, x.code_units);

      // Codes of this warp's 16 tokens of a unit, keys and values requested apart: a unit's keys while the
      // unit before is still at its scores, its values once that one's are converted. The page id is
      // requested one unit earlier than the codes.
      auto look_up = [&](int u) {
        const int pos = u * kManyUnit + warp * 16;
        return u < last_code && pos < code_end ? table[pos >> shift] : 0;
      };
      auto issue = [&](int u, int id, auto values) {
        const int pos = u * kManyUnit + warp * 16;
        if (u < last_code && pos < code_end) {
          if (id < 0 || id >= c.num_pages) {
            if (!values && lane == 0) {
              atomicExch(error_word, LQ_BLOCK_BAD_PAGE);
              raw_scale_s[warp] = make_float2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
            }
          } else {
            const int ph = id * c.kv_heads + h;
            const int64_t at = (((int64_t)ph << shift) + (pos & (P - 1))) * D;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
              const int idx = i * 32 + lane, r = warp * 16 + idx / (D / 16), piece = idx % (D / 16);
              // (the values' pieces of a row are permuted by its pair of tokens)
              if (values) cp_async16(raw_v + r * D + ((piece ^ ((r >> 1) & (D / 16 - 1))) << 4), c.v_pages + at + idx * 16);
              else cp_async16(raw_k + r * D + piece * 16, c.k_pages + at + idx * 16);
            }
            if (!values && lane < 2) cp_async4(smem_u32(&raw_scale_s[warp]) + lane * 4, (lane ? c.v_scales : c.k_scales) + ph);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      const std::false_type keys{};
      const std::true_type values{};
      int page = look_up(ua);
      issue(ua, page, keys);
      issue(ua, page, values);
      page = look_up(ua + 1);

      // ---- this thread's query row to its row of the A tile, lifted by a power of two
      float qu;
      {
        uint32_t raw[D / 2];
        load_words(raw, reinterpret_cast<const uint16_t*>(q) + b * qsb + tok * qst + (int64_t)(h * sh.G + g) * qsh, live, q_vec);
        const float amax = largest_of<T>(raw);
        float unit;
        const float lift = lift_of(is_finite(amax) ? amax : 0.f, 10, unit);
        qu = amax <= 3.402823466e38f ? unit * qk_scale : __int_as_float(0x7fffffff);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 v = pair_of<T>(raw[4 * i + k]);
            w[k] = as_u32(__floats2half2_rn(v.x * lift, v.y * lift));
          }
          sts128(swizzled(q_a + (i >> 3) * kManyTile * 128, tid, i & 7), w[0], w[1], w[2], w[3]);
        }
      }
      float m = kNone, l = 0.f;

      int u = ua;
#pragma unroll 1
      for (; u < ub; ++u) {
        const bool tail = u >= x.code_units;
        const int pos0 = tail ? x.held + (u - x.code_units) * kManyUnit : u * kManyUnit, mine = pos0 + warp * 16;
        const int end = tail ? L : code_end;  // positions that exist
        // ---- keys: fp16 tile of the score product (its last reader, the unit before's product, has ended)
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // (the values may still be on their way)
        if (tail) {  // 16 rows of the ring to a warp: what lifts them
          const int pos = mine + (lane >> 1);
          const int64_t at = (((int64_t)b * c.kv_heads + h) * 2 * P + (pos & (2 * P - 1))) * D + (lane & 1) * (D / 2);
          float top[2] = {0.f, 0.f};
          bool strange = false;  // (as in the kernel above)
#pragma unroll
          for (int kv = 0; kv < 2; ++kv)
#pragma unroll 2
            for (int i = 0; i < D / 16; ++i) {
              const uint4 v = pos < L ? reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(kv ? c.v_ring : c.k_ring) + at)[i]
                                      : make_uint4(0u, 0u, 0u, 0u);
              const uint32_t w[4] = {v.x, v.y, v.z, v.w};
              const float m = largest_of<T>(w);
              if (is_finite(m)) top[kv] = fmaxf(top[kv], m);
              else strange = true;
            }
          float unit[2];
          const float klift = lift_of(warp_max(top[0]), 10, unit[0]), vlift = lift_of(warp_max(top[1]), 7, unit[1], kLowestValue);
          strange = __shfl_xor_sync(0xffffffffu, (int)strange, 1) != 0 || strange;  // (two lanes have a row)
          if (lane == 0) {
            lift_s[warp] = make_float2(klift, vlift);
            scale_s[warp] = make_float4(unit[0], log2_of(unit[1]), inverse_of(unit[1]), 0.f);
          }
#pragma unroll 2
          for (int i = 0; i < D / 16; ++i) {
            const uint4 v = pos < L ? reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(c.k_ring) + at)[i] : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            uint32_t z[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 p = pair_of<T>(w[k]);
              z[k] = strange ? 0x7fff7fffu : as_u32(__floats2half2_rn(p.x * klift, p.y * klift));
            }
            const int piece = (lane & 1) * (D / 16) + i;
            sts128(swizzled(k_a + (piece >> 3) * kManyUnit * 128, warp * 16 + (lane >> 1), piece & 7), z[0], z[1], z[2], z[3]);
          }
        } else {
          __syncwarp();
          const bool there = mine < code_end;
          // (a lane's two pieces in the order that keeps eight lanes on different banks)
          const int odd = D == 128 ? (lane >> 2) & 1 : 0;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const int idx = i * 32 + lane, r = warp * 16 + idx / (D / 16), piece = idx % (D / 16) * 2;
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (there) w = lds128m(raw_k + r * D + (idx % (D / 16)) * 16);
            const uint32_t a0 = (odd ? w.z : w.x) ^ 0x80808080u, a1 = (odd ? w.w : w.y) ^ 0x80808080u;
            const uint32_t a2 = (odd ? w.x : w.z) ^ 0x80808080u, a3 = (odd ? w.y : w.w) ^ 0x80808080u;
            const uint32_t tile = k_a + (piece >> 3) * kManyUnit * 128;
            sts128(swizzled(tile, r, (piece & 7) + odd), codes_h2(a0, 0x4140u), codes_h2(a0, 0x4342u), codes_h2(a1, 0x4140u), codes_h2(a1, 0x4342u));
            sts128(swizzled(tile, r, (piece & 7) + 1 - odd), codes_h2(a2, 0x4140u), codes_h2(a2, 0x4342u), codes_h2(a3, 0x4140u), codes_h2(a3, 0x4342u));
          }
          if (lane == 0) {
            const float ks = there ? raw_scale_s[warp].x : 1.f, vs = there ? raw_scale_s[warp].y : 1.f;
            scale_s[warp] = make_float4(ks, log2_of(vs), fminf(inverse_of(vs), 3.0e38f), 0.f);
          }
        }
        __syncwarp();  // (the warp has read its keys)
        issue(u + 1, page, keys);
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // this unit's values
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // generic writes -> the product's reads
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncthreads();
        if (tid == 0) {
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_f16(tmem_s, smem_desc_sw128(q_a + (k >> 2) * kManyTile * 128 + (k & 3) * 32),
                    smem_desc_sw128(k_a + (k >> 2) * kManyUnit * 128 + (k & 3) * 32), many_idesc(kManyUnit), k > 0);
          mma_commit(bar_scores);
        }

        // ---- values: fp16 tile [dim][token] of the output product. A thread takes a pair of tokens and a
        // quarter of the dims.
        if (u > ua && !mbar_wait(bar_outputs, phase ^ 1)) dead_s = 1;
        {
          constexpr int N = D / 4;  // dims
          if (tail) {
            const float vlift = lift_s[lane >> 3].y;
#pragma unroll 1
            for (int i = 0; i < N / 8; ++i) {
              uint4 v[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int pos = pos0 + 2 * lane + e;
                const int64_t at = (((int64_t)b * c.kv_heads + h) * 2 * P + (pos & (2 * P - 1))) * D + warp * N + i * 8;
                v[e] = pos < L ? *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(c.v_ring) + at) : make_uint4(0u, 0u, 0u, 0u);
              }
              const uint32_t w0[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, w1[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float2 a = pair_of<T>(w0[k]), e = pair_of<T>(w1[k]);
                const int d = warp * N + i * 8 + 2 * k;
                sts32(swizzled(v_a, d, lane >> 2) + (lane & 3) * 4, finite_h2(as_u32(__floats2half2_rn(a.x * vlift, e.x * vlift))));
                sts32(swizzled(v_a, d + 1, lane >> 2) + (lane & 3) * 4, finite_h2(as_u32(__floats2half2_rn(a.y * vlift, e.y * vlift))));
              }
            }
          } else {
            const bool there = pos0 + 2 * lane < code_end;
#pragma unroll
            for (int i = 0; i < N / 16; ++i) {
              uint4 v[2];
#pragma unroll
              for (int e = 0; e < 2; ++e)
                v[e] = there ? lds128m(raw_v + (2 * lane + e) * D + (((warp * (N / 16) + i) ^ (lane & (D / 16 - 1))) << 4)) : make_uint4(0u, 0u, 0u, 0u);
              const uint32_t w0[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, w1[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t a = w0[k] ^ 0x80808080u, e = w1[k] ^ 0x80808080u;
                const uint32_t lo = __byte_perm(a, e, 0x5140u), hi = __byte_perm(a, e, 0x7362u);
                const int d = warp * N + i * 16 + 4 * k;
                const uint32_t at = (lane & 3) * 4;
                sts32(swizzled(v_a, d, lane >> 2) + at, codes_h2(lo, 0x4140u));
                sts32(swizzled(v_a, d + 1, lane >> 2) + at, codes_h2(lo, 0x4342u));
                sts32(swizzled(v_a, d + 2, lane >> 2) + at, codes_h2(hi, 0x4140u));
                sts32(swizzled(v_a, d + 3, lane >> 2) + at, codes_h2(hi, 0x4342u));
              }
            }
          }
        }

        // ---- this thread's row of scores to weights
        if (!mbar_wait(bar_scores, phase)) dead_s = 1;
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const bool masked = pos0 + kManyUnit - 1 > min(x.s.start + x.t_lo, end - 1);
        const int last = min(seen, end - 1) - pos0;  // of this unit's tokens, the last one the row sees
        uint64_t s[kManyUnit / 2];  // pairs of scores
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t w[32];
          tmem_ld32(tmem + half * 32, w);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float4 sc = scale_s[half * 2 + (i >> 3)];
            const float by = qu * sc.x;
            s[half * 16 + i] = fma2(pack2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])), pack2(by, by), pack2(sc.y, sc.y));
          }
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < kManyUnit / 2; ++i) {
            const float2 v = unpack2(s[i]);
            s[i] = pack2(2 * i > last ? -INFINITY : v.x, 2 * i + 1 > last ? -INFINITY : v.y);
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < kManyUnit / 2; ++i) {
          const float2 v = unpack2(s[i]);
          mx = fmaxf(mx, fmaxf(v.x, v.y));
        }
        if (__any_sync(0xffffffffu, mx > m + kMost)) {
          const float to = fmaxf(m, mx - kUp), corr = exp2_of(m - to);
          m = to;
          l *= corr;
          if (u > ua) {  // (the first unit's product writes the outputs afresh)
#pragma unroll 1
            for (int i = 0; i < D / 32; ++i) {
              uint32_t w[32];
              tmem_ld32(tmem + kOutCol + i * 32, w);
#pragma unroll
              for (int k = 0; k < 32; ++k) w[k] = __float_as_uint(__uint_as_float(w[k]) * corr);
              tmem_st32(tmem + kOutCol + i * 32, w);
            }
          }
        }
        const uint64_t minus_m = pack2(-m, -m);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint64_t sums = 0;
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 v = unpack2(add2(s[e * 8 + i], minus_m));
            const float w0 = exp2_of(v.x), w1 = exp2_of(v.y);
            sums = add2(sums, pack2(w0, w1));
            w[i] = as_u32(__floats2half2_rn(w0, w1));
          }
          const float2 sum = unpack2(sums);
          l = fmaf(sum.x + sum.y, scale_s[e].z, l);
          sts128(swizzled(p_a, tid, 2 * e), w[0], w[1], w[2], w[3]);
          sts128(swizzled(p_a, tid, 2 * e + 1), w[4], w[5], w[6], w[7]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncthreads();
        if (dead_s) break;
        if (tid == 0) {
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16(tmem_s + kOutCol, smem_desc_sw128(p_a + k * 32), smem_desc_sw128(v_a + k * 32), many_idesc(D), u > ua || k > 0);
          mma_commit(bar_outputs);
        }
        issue(u + 1, page, values);  // (every thread has read this unit's)
        page = look_up(u + 2);
        phase ^= 1;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      // After a wait that ran out the products may still be at work on this memory: each is waited for once
      // more, and what there is of the row becomes NaN.
      bool gave_up = u < ub;
      if (gave_up) mbar_wait(bar_scores, phase);
      if (!mbar_wait(bar_outputs, phase ^ 1)) {
        gave_up = true;
        mbar_wait(bar_outputs, phase ^ 1);
      }
      if (gave_up) {
        dead_s = 1;
        l = __int_as_float(0x7fffffff);
      }
      __syncwarp();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");

      // ---- what this run has of the (sequence, head): all of it, or a part
      const bool whole = ua == 0 && ub == x.units;
      const int64_t slot = part_slot(rt, gridDim.x, heads, blockIdx.x, b * c.kv_heads + h, kManyTile);
      if (tid == 0) {  // for the join: the runs that begin and end it
        if (ua == 0) ends[(int64_t)rt * heads + b * c.kv_heads + h].x = blockIdx.x;
        if (ub == x.units) ends[(int64_t)rt * heads + b * c.kv_heads + h].y = blockIdx.x;
      }
      const float inv = live ? 1.f / l : 0.f;
#pragma unroll 1
      for (int i = 0; i < D / 32; ++i) {
        uint32_t w[32];
        tmem_ld32(tmem + kOutCol + i * 32, w);
        if (row >= sh.rows) {
        } else if (whole) {
          uint4* dst = reinterpret_cast<uint4*>(out + (((int64_t)b * sp.tokens + tok) * sh.Hq + h * sh.G + g) * D + i * 32);
          uint32_t y[16];
#pragma unroll
          for (int k = 0; k < 16; ++k)
            y[k] = live ? pair_to<T>(__uint_as_float(w[2 * k]) * inv, __uint_as_float(w[2 * k + 1]) * inv) : 0u;
#pragma unroll
          for (int k = 0; k < 4; ++k) dst[k] = make_uint4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
        } else {
          uint4* dst = reinterpret_cast<uint4*>(part + (slot + tid) * D + i * 32);
#pragma unroll
          for (int k = 0; k < 8; ++k) dst[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        }
        __syncwarp();
      }
      if (!whole && row < sh.rows) part_ml[slot + tid] = make_float2(m, l);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncthreads();  // shared and tensor memory are free for the next (sequence, head)
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    off -= x.units * c.kv_heads;
  }
  if (dead_s && tid == 0) atomicExch(error_word, LQ_BLOCK_WAIT);
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(kManyCols) : "memory");
}

// ---------------------------------------------------------------- join the parts
// grid (sequences x KV heads, row groups x column groups of a tile, row tiles): an output row that
// several warps shared is the weighted sum of their parts; one that none took (it does not count)
// becomes zeros. A thread has four values of a row and every `groups`-th part, eight of them requested
// at a time together with their (M, sum): three dependent trips to memory in all.
constexpr int kJoinMost = 1024;  // threads
template <typename T, int D>
__global__ void __launch_bounds__(kJoinMost)
block_attn_join_kernel(const lq_block_kv c, const BlockSpan sp, const Shape sh, int runs, int rows_each, int cols, T* __restrict__ out,
                       const float* __restrict__ part, const float2* __restrict__ part_ml, const int2* __restrict__ ends,
                       int* error_word) {
  const int V = D / 4 / cols;  // threads to a row's share of columns
  __shared__ float4 acc_s[kJoinMost];
  __shared__ float2 ml_s[kJoinMost];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int heads = c.batch * c.kv_heads;
  const int b = blockIdx.x / c.kv_heads, h = blockIdx.x - b * c.kv_heads, rt = blockIdx.z;
  // (start and count are older than the kernel ahead, which has waited for their writer)
  const Tile x = tile_of(c, sp, sh, b, rt);
  const int r0 = blockIdx.y / cols * rows_each, rows = min(rows_each, min(sh.tile, sh.rows - rt * sh.tile) - r0);
  const int items = max(rows, 1) * V, groups = max(1, (int)blockDim.x / items);
  const int group = threadIdx.x / items, item = threadIdx.x - group * items, r = item / V, d = (item - r * V + blockIdx.y % cols * V) * 4;
  const int row = rt * sh.tile + r0 + r, t = token_of(sh, row), g = row - t * sh.G;
  uint2* dst = reinterpret_cast<uint2*>(out + (((int64_t)b * sp.tokens + t) * sh.Hq + h * sh.G + g) * D + d);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (x.bad && threadIdx.x == 0) atomicExch(error_word, LQ_BLOCK_BAD_POSITION);
  if (x.units == 0) {
    if (group == 0 && rows > 0) *dst = make_uint2(0u, 0u);
    return;
  }
  const int2 end = __ldcg(ends + (int64_t)rt * heads + blockIdx.x);
  const int parts = parts_between(end.x, end.y, runs);
  if (parts == 1 || rows <= 0) return;  // one warp had all of it and wrote the output
  const bool live = t < x.s.n;
  if (parts == 0) {  // nobody took it: a wait ran out
    const float nan = live ? __int_as_float(0x7fffffff) : 0.f;
    if (group == 0) *dst = make_uint2(pair_to<T>(nan, nan), pair_to<T>(nan, nan));
    return;
  }
  const int64_t slot = part_slot(rt, runs, heads, end.x, blockIdx.x, sh.tile) + r0 + r;
  const float2* ml = part_ml + slot;
  const float* mine = part + slot * D + d;
  float m = kNone, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (group < groups) {
    for (int k = group; k < parts; k += 8 * groups) {
      float2 w[8];
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int at = k + u * groups;
        w[u] = at < parts ? __ldcg(ml + (int64_t)at * sh.tile) : make_float2(kNone, 0.f);
        v[u] = at < parts ? __ldcg(reinterpret_cast<const float4*>(mine + (int64_t)at * sh.tile * D)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < 8; ++u) top = fmaxf(top, w[u].x);
      const float corr = exp2_of(m - top);
      m = top;
      l *= corr;
      acc.x *= corr; acc.y *= corr; acc.z *= corr; acc.w *= corr;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float f = exp2_of(w[u].x - top);
        l = fmaf(w[u].y, f, l);
        acc.x = fmaf(v[u].x, f, acc.x); acc.y = fmaf(v[u].y, f, acc.y);
        acc.z = fmaf(v[u].z, f, acc.z); acc.w = fmaf(v[u].w, f, acc.w);
      }
    }
  }
  if (groups > 1) {
    acc_s[threadIdx.x] = acc;
    ml_s[threadIdx.x] = make_float2(m, l);
    __syncthreads();
    if (group == 0) {
      float top = m;
      const int used = min(groups, parts);
      for (int k = 1; k < used; ++k) top = fmaxf(top, ml_s[k * items + item].x);
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
      l = 0.f;
#pragma unroll 4
      for (int k = 0; k < used; ++k) {
        const float2 w = ml_s[k * items + item];
        const float4 v = acc_s[k * items + item];
        const float f = exp2_of(w.x - top);
        l = fmaf(w.y, f, l);
        acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
      }
    }
  }
  if (group != 0) return;
  const float inv = 1.f / l;
  *dst = live ? make_uint2(pair_to<T>(acc.x * inv, acc.y * inv), pair_to<T>(acc.z * inv, acc.w * inv)) : make_uint2(0u, 0u);
}

// ---------------------------------------------------------------- host
// Up to this many query rows (T_new * Hq / Hkv) warps work alone, 16 rows a pass, else 128 rows share a
// tcgen05 tile. Measured at 4k contexts: 32 sequences of 8 KV heads, 64 / 96 rows: 195 / 285 us alone,
// 210 / 229 shared (heads of 64, 16 sequences: 65 / 93 alone, 83 / 90 shared).
constexpr int kAloneRows = 80;

struct Plan {
  Shape sh;
  int nt, tiles, runs;
};

Plan plan_of(const lq_block_kv& c, int Hq, int T_new) {
  Plan p;
  p.sh.Hq = Hq;
  p.sh.G = Hq / c.kv_heads;
  p.sh.rows = T_new * p.sh.G;
  p.sh.inv_G = (0x100000000ULL + p.sh.G - 1) / p.sh.G;
  p.nt = p.sh.rows <= 8 ? 1 : p.sh.rows <= kAloneRows ? 2 : 0;
  p.sh.tile = p.nt ? 8 * p.nt : kManyTile;
  p.sh.unit_log2 = p.nt ? 5 : 6;
  p.tiles = (p.sh.rows + p.sh.tile - 1) / p.sh.tile;
  const int at_once = sm_count() * (p.nt == 0 ? kManyCtas : p.nt == 2 ? Cfg<128, 2>::kWarps : c.head_dim == 64 ? Cfg<64, 1>::kWarps : Cfg<128, 1>::kWarps);
  p.sh.slots = at_once / p.tiles > 1 ? at_once / p.tiles : 2;
  p.sh.step = (uint32_t)(0x100000000ULL / p.sh.slots);
  p.sh.waves = p.tiles == 1 ? 2 : 1;
  p.runs = p.sh.waves * p.sh.slots;
  return p;
}

int64_t slots_of(const lq_block_kv& c, const Plan& p) {
  return (int64_t)p.tiles * (p.runs + (int64_t)c.batch * c.kv_heads) * p.sh.tile;
}
int64_t scratch_bytes(const lq_block_kv& c, const Plan& p) {
  return slots_of(c, p) * (c.head_dim + 2) * 4 + (int64_t)p.tiles * c.batch * c.kv_heads * (int64_t)sizeof(int2);
}

int check_attn(const lq_block_kv* c, int Hq, int T_new, const char* what) {
  if (const int rc = check_block_kv(c, what)) return rc;
  LQ_REQUIRE(Hq > 0 && Hq % c->kv_heads == 0 && T_new > 0, LQ_ERR_ARG,
             "%s: %d query heads do not share %d KV heads evenly, or there are no rows", what, Hq, c->kv_heads);
  LQ_REQUIRE(c->dtype != LQ_F32, LQ_ERR_UNSUPPORTED, "%s: built for float16 and bfloat16 rows", what);
  const int64_t group = Hq / c->kv_heads, rows = T_new * group;
  // (token_of() is exact for row * group below 2^32, the rows that fill the last tile among them)
  LQ_REQUIRE(c->kv_heads <= 65535 && rows <= 65535LL * 8 && (rows + kManyTile) * group < 0x100000000LL, LQ_ERR_ARG,
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
struct Main {
  static auto kernel() { return block_attn_kernel<T, D, NT>; }
  static constexpr size_t kSmem = Cfg<D, NT>::kRing;
  static constexpr int kThreads = 32;
};
template <typename T, int D>
struct Main<T, D, 0> {
  static auto kernel() { return block_attn_many_kernel<T, D>; }
  static constexpr size_t kSmem = ManyCfg<D>::kTotal;
  static constexpr int kThreads = kManyThreads;
};

template <typename T, int D, int NT>
int run(const lq_block_kv& c, const BlockSpan& sp, const Plan& p, const void* q, const int64_t* qs, void* out, void* scratch,
        float scaling, int pdl, cudaStream_t stream, int* error_word, const char* what) {
  auto kern = Main<T, D, NT>::kernel();
  constexpr size_t smem = Main<T, D, NT>::kSmem;
  if (const int rc = ensure_smem_limit(reinterpret_cast<const void*>(kern), (int)smem, what)) return rc;
  const float qk_scale = scaling * 1.4426950408889634f;
  const int q_vec = (((uintptr_t)q | (uintptr_t)(qs[0] * 2) | (uintptr_t)(qs[1] * 2) | (uintptr_t)(qs[2] * 2)) & 15) == 0;
  float* part = (float*)scratch;
  float2* part_ml = (float2*)(part + slots_of(c, p) * D);
  int2* ends = (int2*)(part_ml + slots_of(c, p));
  if (const int rc = launch(kern, dim3((unsigned)p.runs, (unsigned)p.tiles), Main<T, D, NT>::kThreads, smem, stream, pdl, what, c, sp, p.sh,
                            (const T*)q, qs[0], qs[1], qs[2], q_vec, (T*)out, part, part_ml, ends, qk_scale,
                            error_word))
    return rc;
  // Few (sequence, head)s have many parts each (hundreds, one long context): a CTA of 512 threads for each
  // quarter of a row, so that 64 and more parts are on their way together. Many have few parts: one CTA
  // for all rows of a tile, in two groups.
  const int64_t tops = (int64_t)c.batch * c.kv_heads * p.tiles;
  const int rows = p.sh.rows < p.sh.tile ? p.sh.rows : p.sh.tile;
  const bool few = tops * rows <= 2 * sm_count();
  const int each = few ? 1 : rows < 8 ? rows : 8, cols = few ? 4 : 1, threads = few ? 512 : 2 * each * D / 4;
  return launch(block_attn_join_kernel<T, D>, dim3((unsigned)(c.batch * c.kv_heads), (unsigned)((rows + each - 1) / each * cols), (unsigned)p.tiles),
                threads, 0, stream, 1, what, c, sp, p.sh, p.runs, each, cols, (T*)out, (const float*)part, (const float2*)part_ml,
                (const int2*)ends, error_word);
}

template <typename T>
int dispatch(const lq_block_kv& c, const BlockSpan& sp, const Plan& p, const void* q, const int64_t* qs, void* out, void* scratch,
             float scaling, int pdl, cudaStream_t stream, int* error_word, const char* what) {
#define LQ_CASE(DD, NN) \
  if (c.head_dim == DD && p.nt == NN) return run<T, DD, NN>(c, sp, p, q, qs, out, scratch, scaling, pdl, stream, error_word, what);
  LQ_CASE(64, 0) LQ_CASE(64, 1) LQ_CASE(64, 2)
  LQ_CASE(128, 0) LQ_CASE(128, 1) LQ_CASE(128, 2)
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
  LQ_REQUIRE(((uintptr_t)out & 15) == 0, LQ_ERR_ARG, "%s: out must be 16-byte aligned", what);
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
