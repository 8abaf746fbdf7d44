// Paged attention over the 8-bit KV cache (kv8.hpp) for gfx950: the work lists,
// split-KV partials and merge of the 16-bit kernels, other K/V data movement.
//
// The products run on the 16-bit MFMA with the queries' type: the scaled
// converter turns four codes of one lane into two operand registers, exactly
// (a code has four significand bits and the scale is a power of two), so that
// results are those of a 16-bit cache that holds the same values.
//
//  * attn_decode_kv8_kernel: a wavefront's share of the decode stream as in
//    attn_decode_kernel, 32 tokens (two scale blocks) a step.  HBM bound: 64
//    sequences of 512 to 4096 tokens, 32/8 heads, 48.6 us, 290 MB at 6.0 TB/s
//    (47.8 with nothing computed); 16 of 32768 6.7 TB/s.
//  * attn_short_kv8_kernel: short decode batches; latency (4 of 512 tokens, 16/8
//    heads, 8.0 us).
//  * attn_tile_kv8_kernel: 64-token tiles shared by four wavefronts.  Bound by the
//    overlap of conversion, softmax and MFMA: 2048 rows over 30000 tokens 925 us,
//    1.13 PFLOP/s; 8192 prompt tokens 218 us, 0.87.
//  * attn_block_kv8_kernel: items of at most 64 columns (32 draft blocks of 16 rows
//    138 us, 4.7 TB/s and 0.59 PFLOP/s at once: issue of both, and HBM).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "attn_types.hpp"
#include "device_util.hpp"
#include "kernel_util.hpp"
#include "kv8.hpp"

namespace feattn {

int decode_wg_waves(int hkv);

// Rows of codes in LDS are 128 bytes, eight 16-byte chunks; chunk c of row t
// sits at position c ^ swz(t), which spreads every operand read below over
// all banks, whether the hardware takes 16 lanes (128 bytes) or 32 at a time.
__device__ __forceinline__ int swz_k(int t) { return ((t >> 1) & 3) | ((((t >> 3) ^ t) & 1) << 2); }
__device__ __forceinline__ int swz_v(int t) {
  return ((t >> 1) & 1) | (((t >> 4) & 1) << 1) | ((((t >> 2) ^ t) & 1) << 2);
}

// Reference maximum of a column that has seen no token.  (Finite: differences
// with it need no special case.)
constexpr float kEmpty = -3.4028234663852886e38f;

// Softmax of a step's scores against the running reference maximum m of each
// column, in log2 units, which is lazy: the probabilities p = 2^(s scale - m) are
// taken with the m there is, and only where a lane's sum of them passes 2^9 (so
// that a single one might, or is infinite: a column's first step) is m raised to
// the column's maximum, l and o with it rescaled, and the step taken again.  No
// maximum and no exchange between the lanes of a column otherwise.  (With the
// columns' maxima exchanged every step 32 draft blocks took 147 us and 2048 rows
// over 30000 1105 us, with each lane's maximum compared 143 and 1070.)
// P: the step's 16-token blocks; put(cb, p) takes a column block's values.
template <int P, int NCB, typename PUT>
__device__ __forceinline__ void softmax_step(f32x4 (&sc)[P][NCB], float scale, float (&m)[NCB], float (&lsum)[NCB],
                                             f32x4 (&o)[8][NCB], PUT put) {
  constexpr float kMost = 512.f;
  float ps[NCB];
  auto exponentials = [&](int cb) {
    float x[P][4];
    float t = 0.f;
#pragma unroll
    for (int tb = 0; tb < P; ++tb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[tb][r] = fast_exp2(__builtin_fmaf(sc[tb][cb][r], scale, -m[cb]));
        t += x[tb][r];
      }
    ps[cb] = t;
    put(cb, x);
  };
  bool above = false;
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    exponentials(cb);
    above = above || ps[cb] > kMost;
  }
  if (__builtin_amdgcn_ballot_w64(above) != 0) {
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      float mx = kNegInf;
#pragma unroll
      for (int tb = 0; tb < P; ++tb)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[tb][cb][r]);
      const float mt = max_x32(max_x16(mx)) * scale;
      const bool up = mt > m[cb];
      const float alpha = up ? fast_exp2(m[cb] - mt) : 1.f;
      if (up) m[cb] = mt;
      lsum[cb] *= alpha;
#pragma unroll
      for (int db = 0; db < 8; ++db) o[db][cb] *= alpha;
      exponentials(cb);
    }
  }
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) lsum[cb] += ps[cb];
}

// Probabilities as two 16-bit operands whose sum they are within 2^-17 (bf16) or
// 2^-23 (fp16): hi rounded, lo the rest.  The decode kernels wait for memory,
// not for the MFMA, so the second product costs them nothing (two column blocks:
// 1.1 us of 46.4), and their results carry the output's rounding alone (with hi
// only the error was 1.4 times that).
template <bool BF16>
__device__ __forceinline__ void pack2_split(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2<BF16>(a, b);
  lo = pack2<BF16>(a - lo_f32<BF16>(hi), b - hi_f32<BF16>(hi));
}

template <bool BF16>
__device__ __forceinline__ void pack8_split(const float (&x)[4], const float (&y)[4], u32x4& hi, u32x4& lo) {
  uint32_t h[4], l[4];
  pack2_split<BF16>(x[0], x[1], h[0], l[0]);
  pack2_split<BF16>(x[2], x[3], h[1], l[1]);
  pack2_split<BF16>(y[0], y[1], h[2], l[2]);
  pack2_split<BF16>(y[2], y[3], h[3], l[3]);
  hi = u32x4{h[0], h[1], h[2], h[3]};
  lo = u32x4{l[0], l[1], l[2], l[3]};
}

// V^T operand of a 32-token step: lane 16 J + L of the read for dim block db
// points at 8 bytes (dims 16 db + 8 m ..) of row k's token, L = 2 k + m: tokens
// 4 J + k of the first 16 (k < 4) and 4 J + k - 4 of the second, the tokens
// that the lane's own S^T values belong to.
__device__ __forceinline__ void v_operand_addr(int J, int L, uint32_t (&v_lds)[8]) {
  const int k = L >> 1, m = L & 1;
  const int t = k < 4 ? 4 * J + k : 16 + 4 * J + k - 4;
#pragma unroll
  for (int db = 0; db < 8; ++db) v_lds[db] = (uint32_t)(128 * t + 16 * (db ^ swz_v(t)) + 8 * m);
}

// Four values of a partial row, already under its scale, to element `at`; the
// codes of what their rounding leaves are returned for part_lo, where a row has
// dims 16 db + 4 J .. + 3 at byte 32 J + 4 db: a column's lane stores 32 bytes.
template <bool BF16>
__device__ __forceinline__ uint32_t put_part(const AttnArgs& a, size_t at, f32x4 v) {
  const u32x2 hi = {pack2<false>(v[0], v[1]), pack2<false>(v[2], v[3])};
  *reinterpret_cast<u32x2*>(a.part_o + at) = hi;
  if constexpr (BF16) return 0u;
  v = (v - f32x4{lo_f32<false>(hi[0]), hi_f32<false>(hi[0]), lo_f32<false>(hi[1]), hi_f32<false>(hi[1])}) * kPartLo;
  return kv8_encode4(v[0], v[1], v[2], v[3]);
}

// A column's results (lane 16 J + L: dims 16 db + 4 J + r): to `out` and `lse`,
// or to partial row `slot` when the row is split.
template <bool BF16>
__device__ __forceinline__ void put_column(const AttnArgs& a, const f32x4 (&o)[8], float ls, float m, int part,
                                           int row, int slot, int head, int J) {
  const float inv = ls > 0.f ? 1.f / ls : 0.f;
  const float l2 = ls > 0.f ? m + __log2f(ls) : kNegInf;
  if (part < 0) {
    const size_t oi = (size_t)row * a.hq + head;
    uint16_t* op = a.out + oi * kHeadDim + 4 * J;
#pragma unroll
    for (int db = 0; db < 8; ++db)
      *reinterpret_cast<u32x2*>(op + 16 * db) =
          u32x2{pack2<BF16>(o[db][0] * inv, o[db][1] * inv), pack2<BF16>(o[db][2] * inv, o[db][3] * inv)};
    if (a.lse != nullptr && J == 0) a.lse[oi] = l2 * kLn2;
    return;
  }
  float mx = 0.f;
#pragma unroll
  for (int db = 0; db < 8; ++db)
#pragma unroll
    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, fabsf(o[db][r]));
  mx = max_x32(max_x16(mx)) * inv;
  float is;
  const float sc = part_scale_of(mx, is);
  const size_t oi = (size_t)slot * a.hq + head;
  u32x4 low[2];
#pragma unroll
  for (int db = 0; db < 8; ++db)
    low[db >> 2][db & 3] = put_part<BF16>(a, oi * kHeadDim + 4 * J + 16 * db, o[db] * inv * is);
  if (!BF16 && a.part_lo != nullptr) {
    u32x4* to = reinterpret_cast<u32x4*>(a.part_lo + oi * kHeadDim + 32 * J);
    to[0] = low[0];
    to[1] = low[1];
  }
  if (J == 0) {
    a.part_lse[oi] = l2;
    a.part_scale[oi] = sc;
  }
}

// The same for a combined column that 32 lanes hold (lane c: dims 4 c .. + 3).
template <bool BF16>
__device__ __forceinline__ void put_combined(const AttnArgs& a, f32x4 acc, float ls, float top, int part, int row,
                                             int slot, int head, int c) {
  const float inv = ls > 0.f ? 1.f / ls : 0.f;
  const float l2 = ls > 0.f ? top + __log2f(ls) : kNegInf;
  acc *= inv;
  if (part < 0) {
    const size_t oi = (size_t)row * a.hq + head;
    *reinterpret_cast<u32x2*>(a.out + oi * kHeadDim + 4 * c) =
        u32x2{pack2<BF16>(acc[0], acc[1]), pack2<BF16>(acc[2], acc[3])};
    if (a.lse != nullptr && c == 0) a.lse[oi] = l2 * kLn2;
    return;
  }
  float mx = fmaxf(fmaxf(fabsf(acc[0]), fabsf(acc[1])), fmaxf(fabsf(acc[2]), fabsf(acc[3])));
#pragma unroll
  for (int d = 1; d <= 16; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
  float is;
  const float sc = part_scale_of(mx, is);
  const size_t oi = (size_t)slot * a.hq + head;
  const uint32_t low = put_part<BF16>(a, oi * kHeadDim + 4 * c, acc * is);
  if (!BF16 && a.part_lo != nullptr)
    *reinterpret_cast<uint32_t*>(a.part_lo + oi * kHeadDim + 32 * (c & 3) + 4 * (c >> 2)) = low;
  if (c == 0) {
    a.part_lse[oi] = l2;
    a.part_scale[oi] = sc;
  }
}

// ===========================================================================
// Decode
// ===========================================================================
// A wavefront owns a ring of U units in LDS, one stream of units per share: K
// and V of every 32 tokens of its items (4 KB of codes each).  A unit is five
// copies, four of 1 KB and one for its scales (the two blocks' K or V scale).
//
// Lane = 16*J + L.  Per 32 tokens:
//   S^T = K Q^T: A = K rows (lane: token L, dims 16 (J + 4 s) .. +15 with one
//                ds_read_b128 of codes, two k-steps), B = Q^T (the same dims);
//                C: lane holds tokens 4J+r of column L.
//   O^T += V^T P^T: A = V^T (v_operand_addr), B = the lane's own S^T values.
constexpr int kKv8Unit = 4096;
constexpr int kKv8Slot = kKv8Unit + 256;  // with the scales

constexpr int kKv8Units = 2;  // 16 sequences of 32768 tokens 161 us, 163 with three; 64 of 512 to 4096 52.3, 52.9, 53.8 with four

// ---- short-context items (see attn_short.hpp for the 16-bit form)
constexpr int kShort8Wave = 16384;  // a wavefront's LDS: 64 tokens of V codes, then its 32 x 128 fp32 results
template <int WAVES>
constexpr size_t short8_lds() {
  return (size_t)WAVES * kShort8Wave + (size_t)WAVES * kDecodeCols * 2 * sizeof(float);
}

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef int32_t i32x2 __attribute__((ext_vector_type(2)));

// K and V scale of a scale block, by a scalar load.
__device__ __forceinline__ f32x2 ldc_scales(const float* scales, size_t at) {
  typedef const __attribute__((address_space(4))) f32x2* cp;
  return *(cp)(scales + 2 * at);
}

template <bool BF16, int WAVES, int NCB, bool GRID2>
__device__ __forceinline__ void short_items_kv8(const AttnArgs& a, int causal, int n_items, uint8_t* dsm) {
  const int lane = threadIdx.x & 63;
  const int J = lane >> 4;
  const int L = lane & 15;
  const int wave = uniform(threadIdx.x >> 6);
  const int G = a.group;
  const int row_bytes = a.hkv * kHeadDim;
  const uint32_t lbase = (uint32_t)(uintptr_t)dsm;
  const uint32_t vst = lbase + (uint32_t)(wave * kShort8Wave);
  const uint32_t mlbase = lbase + (uint32_t)(WAVES * kShort8Wave);
  typedef __attribute__((address_space(3))) float lds_f32;
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

  const uint32_t k_goff = (uint32_t)(L * row_bytes + 16 * J);
  uint32_t v_goff[4];  // 8 rows each: blocks 2 i (0, 1) and 2 i + 1 (2, 3) of a 32-token step
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int t = 8 * r + (lane >> 3);
    v_goff[r] = (uint32_t)((t & 15) * row_bytes + 16 * ((lane & 7) ^ swz_v(t)));
  }
  uint32_t v_lds[8];
  v_operand_addr(J, L, v_lds);

  for (int it = GRID2 ? 0 : blockIdx.x; it < n_items; it += gridDim.x) {
    const int ri = GRID2 ? (int)blockIdx.y : uniform(it / a.hkv);
    const int kvh = GRID2 ? (int)blockIdx.x : uniform(it) - ri * a.hkv;
    const ShortItem* rec = a.shorts + ri;
    typedef const __attribute__((address_space(4))) i32x8* c_i32x8;
    typedef const __attribute__((address_space(4))) i32x4* c_i32x4;
    const i32x8 h = *(c_i32x8)rec;
    const i32x4 first = *(c_i32x4)(rec->block + 4 * wave);
    const int q0 = h[0], nq = h[1], vis = h[2], t0 = h[3], t1 = h[4], part = h[5], page_off = h[6];
    const int ncols = nq * G;
    const int nblk = (t1 - t0 + 15) >> 4;
    const int nbw = (nblk + WAVES - 1) / WAVES;     // blocks per wavefront
    const int nact = (nblk + nbw - 1) / nbw;        // wavefronts with blocks
    const int b0 = wave * nbw;
    const int nb = min(nblk, b0 + nbw) - b0;        // this wavefront's blocks (<= 0: none)
    const int wt0 = t0 + 16 * b0;
    const int wt1 = min(t1, wt0 + 16 * nb);

    float m[NCB], lsum[NCB];
    f32x4 o[8][NCB];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      m[cb] = kEmpty;
      lsum[cb] = 0.f;
#pragma unroll
      for (int db = 0; db < 8; ++db) o[db][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    if (nb > 0) {
      const char* khead = reinterpret_cast<const char*>(a.kc) + (size_t)kvh * kHeadDim;
      const char* vhead = reinterpret_cast<const char*>(a.vc) + (size_t)kvh * kHeadDim;
      size_t blk[4];   // scale blocks of the cache
      f32x2 sc8[4];   // their scales
      u32x4 kf[4][2];
      // Blocks past the wavefront's last are read as its last one: every
      // address is one of the item's, and what they hold is masked.
      auto locate = [&](int tok, int i) {
        const int t = min(tok + 16 * i, wt0 + 16 * (nb - 1));
        const int pg = ldc(a.pages, page_off + (t >> a.page_shift));
        return ((size_t)pg << (a.page_shift - 4)) + (size_t)((t & ((1 << a.page_shift) - 1)) >> 4);
      };
      auto load_k = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int s = 0; s < 2; ++s)
            kf[i][s] = *reinterpret_cast<const u32x4*>(khead + blk[i] * (size_t)(16 * row_bytes) + k_goff + 64 * s);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc8[i] = ldc_scales(a.scales, blk[i] * (size_t)a.hkv + (size_t)kvh);
      };
      auto copy_v = [&](int live) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < live) {
#pragma unroll
            for (int r = 0; r < 2; ++r)
              lds_dma16(vhead + blk[i] * (size_t)(16 * row_bytes), v_goff[2 * (i & 1) + r],
                        vst + (uint32_t)(2048 * i + 1024 * r));
          }
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) blk[i] = (size_t)(uint32_t)first[i];
      u32x4 qf[NCB][4];
      int lim[NCB];
      int lq = lane;
      asm volatile("" : "+v"(lq));  // (what is derived from the lane alone is not to be held through the item loop)
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        const int n = 16 * cb + (lq & 15);
        const bool ok = n < ncols;
        const int nn = ok ? n : 0;
        const int r = nn / G;
        lim[cb] = ok ? min(causal ? vis + r : t1 - 1, wt1 - 1) : -1;
        const uint16_t* qp = a.q + ((size_t)(q0 + r) * a.hq + kvh * G + (nn - r * G)) * kHeadDim + 16 * (lq >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) qf[cb][k] = ld16(qp + 64 * (k >> 1) + 8 * (k & 1));
      }
      load_k();
      copy_v(nb);

      for (int tok = wt0; tok < wt1; tok += 64) {
        const int live = min(4, (wt1 - tok + 15) >> 4);
        wait_vmem<0>();
        f32x2 sv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[i] = sc8[i];
        f32x4 sc[4][NCB];
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) {
#pragma unroll
          for (int cb = 0; cb < NCB; ++cb) sc[tb][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (tb < live) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const u32x4 w = kf[tb][k >> 1];
              const u32x4 ka = kv8_decode8<BF16>(w[2 * (k & 1)], w[2 * (k & 1) + 1], sv[tb][0], sv[tb][0]);
#pragma unroll
              for (int cb = 0; cb < NCB; ++cb) sc[tb][cb] = mfma16<BF16>(ka, qf[cb][k], sc[tb][cb]);
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        const bool more = tok + 64 < wt1;
        if (more) {
#pragma unroll
          for (int i = 0; i < 4; ++i) blk[i] = locate(tok + 64, i);
          load_k();  // under the softmax
        }

#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
          for (int tb = 0; tb < 4; ++tb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (tok + 16 * tb + 4 * J + r > lim[cb]) sc[tb][cb][r] = kNegInf;
        u32x4 pf[2][NCB], pl[2][NCB];
        softmax_step<4, NCB>(sc, a.scale_log2, m, lsum, o, [&](int cb, const float (&x)[4][4]) {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) pack8_split<BF16>(x[2 * ks], x[2 * ks + 1], pf[ks][cb], pl[ks][cb]);
        });

        __builtin_amdgcn_sched_barrier(0);
        // V rows past the last token, up to the 32-token step they end in,
        // hold stale cache or LDS contents: zero (0 * stale must stay 0).
        const int valid = wt1 - tok;
        const int rows = live > 2 ? 64 : 32;
        if (valid < rows) {
          for (int q = 8 * valid + lane; q < 8 * rows; q += 64) lds_zero16(vst + 16 * q);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
          if (ks == 0 || live > 2) {
#pragma unroll
            for (int db = 0; db < 8; ++db) {
              const u32x2 w = lds_read_tr8(vst + v_lds[db] + ks * 4096);
              const u32x4 vf = kv8_decode8<BF16>(w[0], w[1], sv[2 * ks][1], sv[2 * ks + 1][1]);
#pragma unroll
              for (int cb = 0; cb < NCB; ++cb) o[db][cb] = mfma16<BF16>(vf, pf[ks][cb], o[db][cb]);
#pragma unroll
              for (int cb = 0; cb < NCB; ++cb) o[db][cb] = mfma16<BF16>(vf, pl[ks][cb], o[db][cb]);
            }
          }
        if (more) {
          wait_lds();  // the reads of this step's V are complete
          copy_v((wt1 - tok - 64 + 15) >> 4);
        }
      }
      // fp32 results and statistics to LDS: row = column, 16-byte chunk c
      // (dims 4 c ..) at chunk position c ^ L.
      wait_lds();
      int ln = lane;
      asm volatile("" : "+v"(ln));
      const int Lo = ln & 15, Jo = ln >> 4;
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        const float ls = sum_x32(sum_x16(lsum[cb]));
#pragma unroll
        for (int db = 0; db < 8; ++db)
          *(lds_f32x4*)(uintptr_t)(vst + (uint32_t)(512 * (16 * cb + Lo) + 16 * ((4 * db + Jo) ^ Lo))) = o[db][cb];
        if (Jo == 0) {
          const uint32_t ml = mlbase + (uint32_t)(8 * (wave * kDecodeCols + 16 * cb + Lo));
          *(lds_f32*)(uintptr_t)ml = m[cb];
          *(lds_f32*)(uintptr_t)(ml + 4) = ls;
        }
      }
    }
    __syncthreads();

    // Combine: a 32-lane half per column, 4 dims per lane.
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int c = ln & 31;
    for (int n = 2 * wave + (ln >> 5); n < 16 * NCB; n += 2 * WAVES) {
      if (n >= ncols) break;
      float mw[WAVES], lw[WAVES];
      float top = kNegInf;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        mw[w] = kNegInf;
        lw[w] = 0.f;
        if (w < nact) {
          const uint32_t ml = mlbase + (uint32_t)(8 * (w * kDecodeCols + n));
          mw[w] = *(lds_f32*)(uintptr_t)ml;
          lw[w] = *(lds_f32*)(uintptr_t)(ml + 4);
        }
        top = fmaxf(top, mw[w]);
      }
      const float base = top == kNegInf ? 0.f : top;
      float ls = 0.f;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
        if (w < nact) {
          const float wt = fast_exp2(mw[w] - base);
          ls += lw[w] * wt;
          acc += *(lds_f32x4*)(uintptr_t)(lbase + (uint32_t)(w * kShort8Wave + 512 * n + 16 * (c ^ (n & 15)))) * wt;
        }
      const int r = n / G, head = kvh * G + (n - r * G);
      put_combined<BF16>(a, acc, ls, top, part, q0 + r, part + r, head, c);
    }
    if constexpr (GRID2) break;
    if (it + (int)gridDim.x < n_items) __syncthreads();  // the regions are the next item's V
  }
}

template <bool BF16, int WAVES, int NCB>
__global__ __launch_bounds__(64 * WAVES, 2) void attn_short_kv8_kernel(AttnArgs a, int causal) {
  extern __shared__ __attribute__((aligned(16))) uint8_t dsm[];
  short_items_kv8<BF16, WAVES, NCB, true>(a, causal, 1, dsm);
}

// NCB: 16-column blocks per item.  ANY: a graph plan's launch, whose later
// prepares may plan the batch as short-context items.
template <bool BF16, int WAVES, int NCB, bool ANY>
__global__ __launch_bounds__(64 * WAVES, ANY ? 2 : 1) void attn_decode_kv8_kernel(AttnArgs a, int causal) {
  constexpr int U = kKv8Units;
  static_assert(U * WAVES * kKv8Slot <= kLdsBytes, "decode ring exceeds LDS");
  extern __shared__ __attribute__((aligned(16))) uint8_t dsm[];
  const int lane = threadIdx.x & 63;
  const int J = lane >> 4;
  const int L = lane & 15;
  const int wave = uniform(threadIdx.x >> 6);
  const int G = a.group;
  const int pshift = a.page_shift;
  const int pmask = (1 << pshift) - 1;
  const uint32_t ring = (uint32_t)(uintptr_t)dsm + (uint32_t)(wave * U * kKv8Slot);

  const int slot = blockIdx.x * WAVES + wave;
  const int kvh = slot % a.hkv;
  const int share = slot / a.hkv;
  if (!ANY && share >= a.n_share_cap) return;
  const ShareStart rec = ldc_share(a.shares, ANY ? min(share, a.n_share_cap - 1) : share);
  if constexpr (ANY) {
    if constexpr (WAVES >= kShortMinWaves) {
      if (rec.n_short > 0) {
        short_items_kv8<BF16, WAVES, NCB, false>(a, causal, rec.n_short, dsm);
        return;
      }
    }
    if (share >= a.n_share_cap) return;
  }
  const int it_begin = rec.it_begin;
  const int it_end = rec.it_end;
  if (it_begin >= it_end) return;

  // Copy instruction r of a unit of codes, lane i: row 8 r + i / 8 of its 32,
  // chunk position i % 8.
  const int row_bytes = a.hkv * kHeadDim;
  uint32_t k_goff[2], v_goff[4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int t = 8 * r + (lane >> 3);
    k_goff[r] = (uint32_t)(t * row_bytes + 16 * ((lane & 7) ^ swz_k(t)));
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int t = 8 * r + (lane >> 3);
    v_goff[r] = (uint32_t)((t & 15) * row_bytes + 16 * ((lane & 7) ^ swz_v(t)));
  }
  // K operand: token L, chunk J + 4 s; Q operand for k-step 2 s + h: column L,
  // the 16-byte chunk of dims 16 (J + 4 s) + 8 h.
  uint32_t k_lds[2], v_lds[8];
#pragma unroll
  for (int s = 0; s < 2; ++s) k_lds[s] = (uint32_t)(128 * L + 16 * ((J + 4 * s) ^ swz_k(L)));
  v_operand_addr(J, L, v_lds);

  const size_t head_off = (size_t)kvh * kHeadDim;
  auto page_id = [&](const DecodeItem& d, int tok) { return ldc(a.pages, d.page_off + (tok >> pshift)); };
  auto block_of = [&](int tok, int pg) {
    return ((size_t)pg << (pshift - 4)) + (size_t)((tok & pmask) >> 4);
  };
  auto block_addr = [&](const void* cache, size_t blk) {
    return reinterpret_cast<const char*>(cache) + head_off + blk * (size_t)(16 * row_bytes);
  };

  // ---- copy side: the next unit of the share's stream --------------------
  // K (c_key) or V of the 32 tokens at c_tok of item c_it.  The following item
  // (nw) and the next K unit's page ids are requested one item / one unit
  // before they are needed.  A unit whose tokens end in its first block copies
  // that one twice (what it brings is masked).
  int c_it = it_begin;
  DecodeItem cw = rec.first;
  DecodeItem nw = cw;
  if (c_it + 1 < it_end) nw = ldc_ditem(a.ditems, c_it + 1);
  bool c_key = true;
  int c_tok = cw.t0;
  int pg0 = rec.pg0;
  int pg1 = cw.t0 + 16 < cw.t1 ? rec.pg1 : rec.pg0;
  size_t blk0 = 0, blk1 = 0;
  bool c_live = true;
  int issued = 0;
  int c_slot = 0;

  auto issue_codes = [&](const void* cache, const uint32_t (&goff)[4], int side, uint32_t dst) {
    const char* b0 = block_addr(cache, blk0);
    const char* b1 = block_addr(cache, blk1);
    lds_dma16<true>(b0, goff[0], dst);
    lds_dma16<true>(b0, goff[1], dst + 1024);
    lds_dma16<true>(b1, goff[2], dst + 2048);
    lds_dma16<true>(b1, goff[3], dst + 3 * 1024);
    const size_t at = (lane & 1) ? blk1 : blk0;
    lds_dma4(a.scales + 2 * (at * (size_t)a.hkv + (size_t)kvh) + side, dst + kKv8Unit);
  };
  auto issue_one = [&]() {
    const uint32_t dst = ring + (uint32_t)(c_slot * kKv8Slot);
    if (c_key) {
      blk0 = block_of(c_tok, pg0);
      blk1 = c_tok + 16 < cw.t1 ? block_of(c_tok + 16, pg1) : blk0;
      const uint32_t kg[4] = {k_goff[0], k_goff[1], k_goff[0], k_goff[1]};
      issue_codes(a.kc, kg, 0, dst);
      // pages of the next K unit: later in this item, or the next item's first
      if (c_tok + 32 < cw.t1) {
        pg0 = page_id(cw, c_tok + 32);
        pg1 = page_id(cw, min(c_tok + 48, cw.t1 - 1));
      } else if (c_it + 1 < it_end) {
        pg0 = page_id(nw, nw.t0);
        pg1 = page_id(nw, min(nw.t0 + 16, nw.t1 - 1));
      }
    } else {
      issue_codes(a.vc, v_goff, 1, dst);
      c_tok += 32;
      if (c_tok >= cw.t1) {
        ++c_it;
        if (c_it < it_end) {
          cw = nw;
          c_tok = cw.t0;
          if (c_it + 1 < it_end) nw = ldc_ditem(a.ditems, c_it + 1);
        } else {
          c_live = false;
        }
      }
    }
    c_key = !c_key;
    ++issued;
    c_slot = c_slot + 1 == U ? 0 : c_slot + 1;
  };

  // ---- compute side --------------------------------------------------------
  int consumed = 0;
  int r_slot = 0;
  auto refill = [&]() {
    wait_lds();
    while (c_live && issued - consumed < U) issue_one();
  };
  auto refill_after_reads = [&]() {  // the unit read last is done with
    consumed += 1;
    refill();
  };
  typedef __attribute__((address_space(3))) f32x2 lds_f32x2;

  for (int it = it_begin; it < it_end; ++it) {
    const DecodeItem w = it == it_begin ? rec.first : ldc_ditem(a.ditems, it);
    const int t0 = w.t0;
    const int t1 = w.t1;
    const int ncols = w.nq * G;
    bool col_ok[NCB];
    int crow[NCB], chead[NCB], lim[NCB];  // lim: last visible token of the lane's column
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      const int n = 16 * cb + L;
      col_ok[cb] = n < ncols;
      crow[cb] = w.q0 + (col_ok[cb] ? n / G : 0);
      chead[cb] = kvh * G + (col_ok[cb] ? n % G : 0);
      lim[cb] = -1;
      if (col_ok[cb]) lim[cb] = min(causal ? w.len - w.nq + (crow[cb] - w.q0) : w.len - 1, t1 - 1);
    }

    // Q goes to registers: as units of the ring, in front of the item's K and V,
    // it kept those from being asked for until it had come (two column blocks:
    // 24 sequences of 5 rows 48.4 us, 47.6 so).
    u32x4 qf[NCB][4];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      const uint16_t* qp = a.q + ((size_t)crow[cb] * a.hq + chead[cb]) * kHeadDim + 16 * J;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        qf[cb][k] = ld16(qp + 64 * (k >> 1) + 8 * (k & 1));
        if (!col_ok[cb]) qf[cb][k] = u32x4{0u, 0u, 0u, 0u};
      }
    }
    refill();

    float m[NCB], lsum[NCB];
    f32x4 o[8][NCB];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      m[cb] = kEmpty;
      lsum[cb] = 0.f;
#pragma unroll
      for (int db = 0; db < 8; ++db) o[db][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    for (int tok = t0; tok < t1; tok += 32) {
      // The workgroup's wavefronts are brought back in step every 64 tokens,
      // so that each page is requested by all of them at about the same time.
      if (((tok - t0) & 32) == 0) __builtin_amdgcn_s_barrier();
      refill();
      // ---- S^T; the K unit's slot is refilled as soon as it is read
      wait_units<U, 5>(issued - consumed - 1);
      const uint32_t kst = ring + (uint32_t)(r_slot * kKv8Slot);
      r_slot = r_slot + 1 == U ? 0 : r_slot + 1;
      const f32x2 ks = *(lds_f32x2*)(uintptr_t)(kst + kKv8Unit);
      u32x4 kw[2][2];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) kw[tb][s] = lds_read16(kst + 2048 * tb + k_lds[s]);
      refill_after_reads();
      f32x4 sc[2][NCB];
#pragma unroll
      for (int tb = 0; tb < 2; ++tb) {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) sc[tb][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const u32x4 kf = kv8_decode8<BF16>(kw[tb][k >> 1][2 * (k & 1)], kw[tb][k >> 1][2 * (k & 1) + 1], ks[tb], ks[tb]);
#pragma unroll
          for (int cb = 0; cb < NCB; ++cb) sc[tb][cb] = mfma16<BF16>(kf, qf[cb][k], sc[tb][cb]);
        }
      }

#pragma unroll
      for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (tok + 16 * tb + 4 * J + r > lim[cb]) sc[tb][cb][r] = kNegInf;

      // ---- the reads of V, and the exponentials under them
      wait_units<U, 5>(issued - consumed - 1);
      const uint32_t vst = ring + (uint32_t)(r_slot * kKv8Slot);
      r_slot = r_slot + 1 == U ? 0 : r_slot + 1;
      if (t1 - tok < 32) {
        // Rows past the item end hold stale contents: zero them, so that
        // 0 * (stale) can never become NaN.  (16-byte chunk q lies in row q / 8.)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int q = lane + 64 * u;
          if ((q >> 3) >= t1 - tok) lds_zero16(vst + 16 * q);
        }
      }
      const f32x2 vs = *(lds_f32x2*)(uintptr_t)(vst + kKv8Unit);
      u32x2 vw[8];
#pragma unroll
      for (int db = 0; db < 8; ++db) vw[db] = lds_read_tr8(vst + v_lds[db]);
      // With two column blocks V's slot is refilled at once (24 sequences of 5
      // rows 46.2 us, 47.2 a step later); with one the wait costs more.
      if constexpr (NCB > 1) refill_after_reads();
      __builtin_amdgcn_sched_barrier(0);
      u32x4 pf[NCB], pl[NCB];
      softmax_step<2, NCB>(sc, a.scale_log2, m, lsum, o, [&](int cb, const float (&x)[2][4]) {
        pack8_split<BF16>(x[0], x[1], pf[cb], pl[cb]);
      });

      // ---- O^T
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        const u32x4 vf = kv8_decode8<BF16>(vw[db][0], vw[db][1], vs[0], vs[1]);
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) o[db][cb] = mfma16<BF16>(vf, pf[cb], o[db][cb]);
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) o[db][cb] = mfma16<BF16>(vf, pl[cb], o[db][cb]);
      }
      if constexpr (NCB == 1) consumed += 1;
    }

#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      const float ls = sum_x32(sum_x16(lsum[cb]));
      if (col_ok[cb]) {
        f32x4 oc[8];
#pragma unroll
        for (int db = 0; db < 8; ++db) oc[db] = o[db][cb];
        put_column<BF16>(a, oc, ls, m[cb], w.part, crow[cb], w.part + (16 * cb + L) / G, chead[cb], J);
      }
    }
  }
}

// ===========================================================================
// Tiles
// ===========================================================================
// Four wavefronts share 64-token tiles.  Wavefront w copies the codes of block
// w of the next tile to a region of its own (4 KB) while the current one is
// computed; once they have landed it converts them, once for all four, into
// the 16-bit tile (32 KB: K blocks, then V blocks, 16 tokens x 256 bytes, the
// chunks of a row permuted), of which there are two.
constexpr int kTile8Block = 4096;
constexpr int kTile8Stage = 8 * kTile8Block;
constexpr int kTile8Raw = 2 * kTile8Stage;           // offset of the wavefronts' code regions
constexpr int kTile8Lds = kTile8Raw + 4 * 4096;      // 80 KB: two workgroups a compute unit

// The lane's index, from the hardware: neither it nor what follows from it is
// held in registers through items of the other kind.
__device__ __forceinline__ int fresh_lane() {
  uint32_t zero;
  asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
  return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
}

struct Tile8Lanes {
  uint32_t goff[2];
  uint32_t k_lds[4], v_lds[8];
};

// Row of a block and 16 codes of it that a lane copies and converts in
// instruction u, and the chunk positions (c ^ these) of row t in the 16-bit tile.
// A write of 16 bytes goes eight lanes at a time over 32 banks: four lanes with
// the even (or odd) chunks of a half of row t and four with row t + 8's, whose
// positions differ in the lowest bit, meet no bank twice (eight lanes of one row
// did: 8 cycles more a write, 944 us against 932 for 2048 rows over 30000).  The operand reads, of 16 rows (K) and
// of eight consecutive ones (V), do not either.
__device__ __forceinline__ int tile8_row(int lane, int u) { return 8 * ((lane >> 2) & 1) + (lane >> 4) + 4 * u; }
__device__ __forceinline__ int tile8_part(int lane) { return (lane & 3) | ((lane >> 1) & 4); }
__device__ __forceinline__ int tile8_swz_k(int t) { return t ^ (t >> 3); }
__device__ __forceinline__ int tile8_swz_v(int t) { return ((2 * t) & 15) | (t >> 3); }

__device__ __forceinline__ Tile8Lanes tile8_lanes(const AttnArgs& a, int lane) {
  const int J = lane >> 4, L = lane & 15;
  const int row_bytes = a.hkv * kHeadDim;
  Tile8Lanes tl;
#pragma unroll
  for (int r = 0; r < 2; ++r) tl.goff[r] = (uint32_t)(tile8_row(lane, r) * row_bytes + 16 * tile8_part(lane));
#pragma unroll
  for (int s = 0; s < 4; ++s) tl.k_lds[s] = (uint32_t)(16 * (16 * L + ((4 * s + J) ^ tile8_swz_k(L))));
  const int k = L >> 2, m = L & 3, t = 4 * J + k;
#pragma unroll
  for (int db = 0; db < 8; ++db) {
    const int c = 2 * db + (m >> 1);
    tl.v_lds[db] = (uint32_t)(16 * (16 * t + (c ^ tile8_swz_v(t))) + 8 * (m & 1));
  }
  return tl;
}

// Requests the codes of this wavefront's block (tokens T + 16 wave ..) of item
// w's tile at T, and returns its scales; blocks at or past the item end are
// skipped.
template <bool STREAM>
__device__ __forceinline__ f32x2 tile8_copy(const AttnArgs& a, const WorkItem& w, const SeqInfo& s,
                                             const uint32_t (&goff)[2], uint32_t lbase, int wave, int T) {
  const int tok = T + 16 * wave;
  if (tok >= w.t1) return f32x2{1.f, 1.f};
  const int pshift = a.page_shift;
  const int row_bytes = a.hkv * kHeadDim;
  const int pg = ldc(a.pages, s.page_off + (tok >> pshift));
  const size_t blk = ((size_t)pg << (pshift - 4)) + (size_t)((tok & ((1 << pshift) - 1)) >> 4);
  const size_t off = blk * (size_t)(16 * row_bytes) + (size_t)w.kvh * kHeadDim;
  const char* kb = reinterpret_cast<const char*>(a.kc) + off;
  const char* vb = reinterpret_cast<const char*>(a.vc) + off;
  const uint32_t raw = lbase + (uint32_t)(kTile8Raw + wave * 4096);
#pragma unroll
  for (int r = 0; r < 2; ++r) lds_dma16<STREAM>(kb, goff[r], raw + 1024 * r);
#pragma unroll
  for (int r = 0; r < 2; ++r) lds_dma16<STREAM>(vb, goff[r], raw + 2048 + 1024 * r);
  return ldc_scales(a.scales, blk * (size_t)a.hkv + (size_t)w.kvh);
}

template <bool BF16, bool CAUSAL, int NCB, bool STREAM>
__device__ __forceinline__ int tile8_item(const AttnArgs& a, const WorkItem& w, const SeqInfo& s, bool has_next,
                                          const WorkItem& wn, const SeqInfo& sn, const Tile8Lanes& tl, uint32_t lbase,
                                          int wave, int lane, int stage0, f32x2& scales) {
  const int J = lane >> 4;
  const int L = lane & 15;
  const int G = a.group;
  const int kvh = w.kvh;
  const int t0 = w.t0;
  const int t1 = w.t1;
  const int ncols = w.nq * G;
  constexpr int kWcols = 16 * NCB;  // columns per wavefront
  const bool wave_on = wave * kWcols < ncols;

  int lim[NCB], crow[NCB], chead[NCB];
  u32x4 qf[NCB][4];
  int lim_min = 1 << 30;
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    const int n = wave * kWcols + 16 * cb + L;
    const bool ok = n < ncols;
    crow[cb] = w.q0 + (ok ? n / G : 0);
    chead[cb] = kvh * G + (ok ? n % G : 0);
    lim[cb] = -1;
    if (ok) lim[cb] = min(CAUSAL ? s.len - s.qlen + (crow[cb] - s.qo) : s.len - 1, t1 - 1);
    if (ok) lim_min = min(lim_min, lim[cb]);
    const uint16_t* qp = a.q + ((size_t)crow[cb] * a.hq + chead[cb]) * kHeadDim + 8 * J;
#pragma unroll
    for (int k = 0; k < 4; ++k) qf[cb][k] = ld16(qp + 32 * k);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!ok) qf[cb][k] = u32x4{0u, 0u, 0u, 0u};
      // (Q has landed past this point: no wait for it inside the tile loop)
      asm volatile("" : "+v"(qf[cb][k]));
    }
  }
#pragma unroll
  for (int o_ = 32; o_ >= 1; o_ >>= 1) lim_min = min(lim_min, __shfl_xor(lim_min, o_, 64));

  float m[NCB], lsum[NCB];
  f32x4 o[8][NCB];
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    m[cb] = kEmpty;
    lsum[cb] = 0.f;
#pragma unroll
    for (int db = 0; db < 8; ++db) o[db][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto compute = [&](uint32_t st, int T, auto masked) {
    constexpr bool MASK = decltype(masked)::value;
    f32x4 sc[4][NCB];
#pragma unroll
    for (int tb = 0; tb < 4; ++tb)
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) sc[tb][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t kb = st + tl.k_lds[k];
#pragma unroll
      for (int tb = 0; tb < 4; ++tb) {
        const u32x4 kf = lds_read16(kb + tb * kTile8Block);
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) sc[tb][cb] = mfma16<BF16>(kf, qf[cb][k], sc[tb][cb]);
      }
    }

    if constexpr (MASK) {
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int tb = 0; tb < 4; ++tb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (T + 16 * tb + 4 * J + r > lim[cb]) sc[tb][cb][r] = kNegInf;
    }
    u32x4 pf[2][NCB];
    softmax_step<4, NCB>(sc, a.scale_log2, m, lsum, o, [&](int cb, const float (&x)[4][4]) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        pf[ks][cb] = u32x4{pack2<BF16>(x[2 * ks][0], x[2 * ks][1]), pack2<BF16>(x[2 * ks][2], x[2 * ks][3]),
                           pack2<BF16>(x[2 * ks + 1][0], x[2 * ks + 1][1]),
                           pack2<BF16>(x[2 * ks + 1][2], x[2 * ks + 1][3])};
    });

#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        const uint32_t vb = st + tl.v_lds[db];
        const u32x2 lo = lds_read_tr16(vb + (4 + 2 * ks) * kTile8Block);
        const u32x2 hi = lds_read_tr16(vb + (5 + 2 * ks) * kTile8Block);
        const u32x4 vf = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) o[db][cb] = mfma16<BF16>(vf, pf[ks][cb], o[db][cb]);
      }
    // V^T operand reads three blocks ahead of their MFMAs (LDS latency)
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
    for (int i = 0; i < 13; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, NCB, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 3 * NCB, 0);
  };

  int stage = stage0;
  for (int T = t0; T < t1; T += kTileTokens) {
    wait_vmem<0>();  // this wavefront's codes have landed
    // From here until the next tile's copies are on their way a wavefront comes
    // first on its SIMD: the other three wait for what it converts, and memory
    // for what it asks (2048 rows over 30000: 1059 us without, 938 so; the 16-bit
    // arithmetic first instead, 1014; 8192 prompt tokens 232 and 234).
    __builtin_amdgcn_s_setprio(2);
    const uint32_t st = lbase + (uint32_t)(stage * kTile8Stage);
    {
      // Rows at or past the item end become zero in V (0 * stale must stay 0).
      const uint32_t raw = lbase + (uint32_t)(kTile8Raw + wave * 4096);
      const int valid = t1 - (T + 16 * wave);
      const int c = tile8_part(lane);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = tile8_row(lane, u);
        const u32x4 kw = lds_read16(raw + 16 * lane + 1024 * u);
        u32x4 vw = lds_read16(raw + 2048 + 16 * lane + 1024 * u);
        if (t >= valid) vw = u32x4{0u, 0u, 0u, 0u};
        const uint32_t kd = st + (uint32_t)(wave * kTile8Block + 256 * t);
        const uint32_t vd = kd + 4 * kTile8Block;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          lds_write16(kd + 16 * ((2 * c + h) ^ tile8_swz_k(t)),
                      kv8_decode8<BF16>(kw[2 * h], kw[2 * h + 1], scales[0], scales[0]));
          lds_write16(vd + 16 * ((2 * c + h) ^ tile8_swz_v(t)),
                      kv8_decode8<BF16>(vw[2 * h], vw[2 * h + 1], scales[1], scales[1]));
        }
      }
    }
    __syncthreads();  // the tile is in LDS, its codes are read, the other tile is free
    if (T + kTileTokens < t1) scales = tile8_copy<STREAM>(a, w, s, tl.goff, lbase, wave, T + kTileTokens);
    else if (has_next) scales = tile8_copy<STREAM>(a, wn, sn, tl.goff, lbase, wave, wn.t0);
    __builtin_amdgcn_s_setprio(0);
    if (wave_on) {
      if (T + kTileTokens - 1 <= lim_min) compute(st, T, std::false_type{});
      else compute(st, T, std::true_type{});
    }
    stage ^= 1;
  }

  if (wave_on) {
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      const float ln = sum_x32(sum_x16(lsum[cb]));
      const int n = wave * kWcols + 16 * cb + L;
      if (n < ncols) {
        f32x4 oc[8];
#pragma unroll
        for (int db = 0; db < 8; ++db) oc[db] = o[db][cb];
        put_column<BF16>(a, oc, ln, m[cb], w.part, crow[cb], w.part + n / G, chead[cb], J);
      }
    }
  }
  return stage;
}

// ---------------------------------------------------------------------------
// Items of at most 64 columns (draft blocks, verify rows): HBM bound
// ---------------------------------------------------------------------------
// Here each wavefront owns tokens instead of columns: an item's steps of 32
// tokens go to four wavefronts in turn, each computes all 64 columns on its own,
// from codes that it alone copies, converts and reads once, with no barrier
// inside an item.  The ring of units runs on into the next item while the four
// results of one are combined.  Q (64 columns, 16 KB) lies in LDS, in the region
// that combining uses in its turn.
//
// Two such groups of four wavefronts, neighbouring kv heads of the same tokens,
// make a workgroup where the list is an equal cut of the tokens (pairs):
// their reads meet in 256 bytes of a cache row.  One kv head's 128 bytes a row
// are what such a stream reads alone, 5.8 TB/s with nothing computed against
// 6.5 for two heads and 6.9 for four and more.
constexpr int kBlk8Units = 2;  // (32 blocks of 16 rows over 2048 to 16384: 138.0 us, 140.4 with three)
constexpr int kBlk8Wave = kBlk8Units * kKv8Slot;
constexpr int kBlk8Head = kTile8Lds - 4 * kBlk8Wave;  // Q, or: exchange, then statistics
constexpr int kBlk8Stats = 4 * 3 * 2048;  // what the wavefronts hand each other of 16 columns
static_assert(kBlk8Head >= 64 * 256 && kBlk8Head >= kBlk8Stats + 4 * 64 * 12 && kBlk8Head % 256 == 0, "");

// Items [it0, it1) of the list, by the four wavefronts (wv) that share `qbase`;
// every wavefront of the workgroup makes the same number of calls and items.
template <bool BF16, bool CAUSAL, bool STREAM>
__device__ __forceinline__ void block8_items(const AttnArgs& a, int it0, int it1, uint32_t qbase, uint32_t ring,
                                             int wv, int lane) {
  constexpr int NCB = 4;
  const int J = lane >> 4;
  const int L = lane & 15;
  const int G = a.group;
  const int pshift = a.page_shift;
  const int pmask = (1 << pshift) - 1;
  const int row_bytes = a.hkv * kHeadDim;
  typedef __attribute__((address_space(3))) float lds_f32;
  typedef __attribute__((address_space(3))) f32x2 lds_f32x2;
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

  uint32_t k_goff[2], v_goff[4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int t = 8 * r + (lane >> 3);
    k_goff[r] = (uint32_t)(t * row_bytes + 16 * ((lane & 7) ^ swz_k(t)));
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int t = 8 * r + (lane >> 3);
    v_goff[r] = (uint32_t)((t & 15) * row_bytes + 16 * ((lane & 7) ^ swz_v(t)));
  }
  // Operand reads: chunk J of row L (K; J + 4: ^ 64), chunk 2 J of row L (Q; the
  // k-step 2 i + h: ^ 16 (8 i + h)), v_operand_addr's of dim block 0 (db: ^ 16 db).
  uint32_t k_at = (uint32_t)(128 * L + 16 * (J ^ swz_k(L)));
  uint32_t q_at = (uint32_t)(256 * L + 16 * ((2 * J) ^ L));
  uint32_t v_at;
  {
    const int k = L >> 1, t = k < 4 ? 4 * J + k : 16 + 4 * J + k - 4;
    v_at = (uint32_t)(128 * t + 16 * swz_v(t) + 8 * (L & 1));
  }

  // ---- copy side: K, then V of this wavefront's steps (tokens c_tok .. + 31)
  // of item c_it, through the items.
  int c_it = it0 - 1, c_tok = 0, c_t1 = 0, c_pages = 0, c_kvh = 0;
  int pg0 = 0, pg1 = 0;
  bool c_live = true, c_key = true;
  size_t blk0 = 0, blk1 = 0;
  int issued = 0, consumed = 0, c_slot = 0, r_slot = 0;
  auto next_item = [&]() {  // the next item with a step of this wavefront
    while (c_tok >= c_t1) {
      if (++c_it >= it1) {
        c_live = false;
        return;
      }
      const WorkItem n = ldc_item(a.items, c_it);
      c_tok = n.t0 + 32 * wv;
      c_t1 = n.t1;
      c_kvh = n.kvh;
      c_pages = ldc_seq(a.seqs, n.seq).page_off;
    }
    pg0 = ldc(a.pages, c_pages + (c_tok >> pshift));
    pg1 = ldc(a.pages, c_pages + (min(c_tok + 16, c_t1 - 1) >> pshift));
  };
  auto block_of = [&](int tok, int pg) { return ((size_t)pg << (pshift - 4)) + (size_t)((tok & pmask) >> 4); };
  auto issue_codes = [&](const void* cache, const uint32_t (&goff)[4], int side, uint32_t dst) {
    const char* base = reinterpret_cast<const char*>(cache) + (size_t)c_kvh * kHeadDim;
    const char* b0 = base + blk0 * (size_t)(16 * row_bytes);
    const char* b1 = base + blk1 * (size_t)(16 * row_bytes);
    lds_dma16<STREAM>(b0, goff[0], dst);
    lds_dma16<STREAM>(b0, goff[1], dst + 1024);
    lds_dma16<STREAM>(b1, goff[2], dst + 2048);
    lds_dma16<STREAM>(b1, goff[3], dst + 3 * 1024);
    const size_t at = (lane & 1) ? blk1 : blk0;
    lds_dma4(a.scales + 2 * (at * (size_t)a.hkv + (size_t)c_kvh) + side, dst + kKv8Unit);
  };
  auto refill = [&]() {  // (the caller has waited for its reads of the slot freed last)
    while (c_live && issued - consumed < kBlk8Units) {
      const uint32_t dst = ring + (uint32_t)(c_slot * kKv8Slot);
      if (c_key) {
        blk0 = block_of(c_tok, pg0);
        blk1 = c_tok + 16 < c_t1 ? block_of(c_tok + 16, pg1) : blk0;
        const uint32_t kg[4] = {k_goff[0], k_goff[1], k_goff[0], k_goff[1]};
        issue_codes(a.kc, kg, 0, dst);
        if (c_tok + 128 < c_t1) {
          pg0 = ldc(a.pages, c_pages + ((c_tok + 128) >> pshift));
          pg1 = ldc(a.pages, c_pages + (min(c_tok + 144, c_t1 - 1) >> pshift));
        }
      } else {
        issue_codes(a.vc, v_goff, 1, dst);
        c_tok += 128;
        if (c_tok >= c_t1) next_item();
      }
      c_key = !c_key;
      ++issued;
      c_slot = c_slot + 1 == kBlk8Units ? 0 : c_slot + 1;
    }
  };
  auto barrier = [&]() {  // of LDS reads and writes; copies stay in flight
    wait_lds();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  next_item();

  for (int it = it0; it < it1; ++it) {
    const WorkItem w = ldc_item(a.items, it);
    const SeqInfo s = ldc_seq(a.seqs, w.seq);
    const int t0 = w.t0, t1 = w.t1, kvh = w.kvh;
    const int ncols = w.nq * G;

    // Q: wavefront wv copies column block wv; columns past the item repeat its first.
    {
      const int before = issued;
      const int ln = fresh_lane();
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = 4 * r + (ln >> 4);
        const int col = 16 * wv + n;
        const int nn = col < ncols ? col : 0;
        lds_dma16(a.q + ((size_t)(w.q0 + nn / G) * a.hq + kvh * G + nn % G) * kHeadDim + 8 * ((ln & 15) ^ n),
                  qbase + (uint32_t)(4096 * wv + 1024 * r));
      }
      refill();
      wait_units<kBlk8Units, 5>(issued - before);
    }

    int lim[NCB];
    int lim_min = 1 << 30;
    const int lq = fresh_lane() & 15;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      const int n = 16 * cb + lq;
      lim[cb] = -1;
      if (n < ncols) {
        lim[cb] = min(CAUSAL ? s.len - s.qlen + (w.q0 + n / G - s.qo) : s.len - 1, t1 - 1);
        lim_min = min(lim_min, lim[cb]);
      }
    }
#pragma unroll
    for (int o_ = 8; o_ >= 1; o_ >>= 1) lim_min = min(lim_min, __shfl_xor(lim_min, o_, 64));
    lim_min = uniform(lim_min);

    float m[NCB], lsum[NCB];
    f32x4 o[8][NCB];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      m[cb] = kEmpty;
      lsum[cb] = 0.f;
#pragma unroll
      for (int db = 0; db < 8; ++db) o[db][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    barrier();  // Q is in LDS

    for (int tok = t0 + 32 * wv; tok < t1; tok += 128) {
      asm volatile("" : "+v"(k_at), "+v"(q_at), "+v"(v_at));  // (the derived addresses are not to be held)
      // ---- S^T
      wait_units<kBlk8Units, 5>(issued - consumed - 1);
      const uint32_t kst = ring + (uint32_t)(r_slot * kKv8Slot);
      r_slot = r_slot + 1 == kBlk8Units ? 0 : r_slot + 1;
      const f32x2 ks = *(lds_f32x2*)(uintptr_t)(kst + kKv8Unit);
      u32x4 kw[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) kw[i][tb] = lds_read16(kst + 2048 * tb + (k_at ^ (64 * i)));
      u32x4 qf[2][NCB];  // this k-step's and the next one's
      auto read_q = [&](int k) {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
          qf[k & 1][cb] = lds_read16(qbase + (q_at ^ (16 * (8 * (k >> 1) + (k & 1)))) + 4096 * cb);
      };
      read_q(0);
      f32x4 sc[2][NCB];
#pragma unroll
      for (int tb = 0; tb < 2; ++tb)
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) sc[tb][cb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k < 3) read_q(k + 1);
        __builtin_amdgcn_sched_barrier(0);  // (else the reads sink to their use, behind a full LDS latency each)
        u32x4 kf[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
          kf[tb] = kv8_decode8<BF16>(kw[k >> 1][tb][2 * (k & 1)], kw[k >> 1][tb][2 * (k & 1) + 1], ks[tb], ks[tb]);
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
          for (int tb = 0; tb < 2; ++tb) sc[tb][cb] = mfma16<BF16>(kf[tb], qf[k & 1][cb], sc[tb][cb]);
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_lds();
      consumed += 1;
      refill();

      // ---- softmax
      if (tok + 31 > lim_min) {
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
          for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (tok + 16 * tb + 4 * J + r > lim[cb]) sc[tb][cb][r] = kNegInf;
      }
      // (V^T operands are read ahead of the exponentials)
      wait_units<kBlk8Units, 5>(issued - consumed - 1);
      const uint32_t vst = ring + (uint32_t)(r_slot * kKv8Slot);
      r_slot = r_slot + 1 == kBlk8Units ? 0 : r_slot + 1;
      if (t1 - tok < 32) {
        // rows past the item end: zero (0 * stale must stay 0)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int q = lane + 64 * u;
          if ((q >> 3) >= t1 - tok) lds_zero16(vst + 16 * q);
        }
      }
      const f32x2 vs = *(lds_f32x2*)(uintptr_t)(vst + kKv8Unit);
      u32x2 vw[8];
#pragma unroll
      for (int db = 0; db < 8; ++db) vw[db] = lds_read_tr8(vst + (v_at ^ (16 * db)));
      __builtin_amdgcn_sched_barrier(0);
      u32x4 pf[NCB];
      softmax_step<2, NCB>(sc, a.scale_log2, m, lsum, o, [&](int cb, const float (&x)[2][4]) {
        pf[cb] = u32x4{pack2<BF16>(x[0][0], x[0][1]), pack2<BF16>(x[0][2], x[0][3]), pack2<BF16>(x[1][0], x[1][1]),
                       pack2<BF16>(x[1][2], x[1][3])};
      });

      // ---- O^T
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        const u32x4 vf = kv8_decode8<BF16>(vw[db][0], vw[db][1], vs[0], vs[1]);
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) o[db][cb] = mfma16<BF16>(vf, pf[cb], o[db][cb]);
      }
      wait_lds();
      consumed += 1;
      refill();
    }

    // ---- combine, 16 columns a round: wavefront v finishes dims 32 v .. + 31,
    // which the other three hand it.
    const int ln = fresh_lane(), Jc = ln >> 4, Lc = ln & 15;
    const uint32_t stats = qbase + kBlk8Stats;
    barrier();  // every step's reads of Q are done
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      lsum[cb] = sum_x32(sum_x16(lsum[cb]));
      float mx = 0.f;
#pragma unroll
      for (int db = 0; db < 8; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, fabsf(o[db][cb][r]));
      mx = max_x32(max_x16(mx));
      if (Jc == 0) {
        const uint32_t at = stats + (uint32_t)(12 * (64 * wv + 16 * cb + Lc));
        *(lds_f32*)(uintptr_t)at = m[cb];
        *(lds_f32*)(uintptr_t)(at + 4) = lsum[cb];
        *(lds_f32*)(uintptr_t)(at + 8) = mx;
      }
    }
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      if (16 * cb < ncols) {
        if (cb > 0) barrier();  // the round before is read
        f32x4 acc[2];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          if (v == wv) {
            acc[0] = o[2 * v][cb];
            acc[1] = o[2 * v + 1][cb];
          } else {
            const uint32_t to = qbase + (uint32_t)(2048 * (3 * v + (wv < v ? wv : wv - 1)) + 16 * ln);
            *(lds_f32x4*)(uintptr_t)to = o[2 * v][cb];
            *(lds_f32x4*)(uintptr_t)(to + 1024) = o[2 * v + 1][cb];
          }
        }
        barrier();
        float mv[4], lv[4], xv[4];
        float top = kNegInf;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const uint32_t at = stats + (uint32_t)(12 * (64 * v + 16 * cb + Lc));
          mv[v] = *(lds_f32*)(uintptr_t)at;
          lv[v] = *(lds_f32*)(uintptr_t)(at + 4);
          xv[v] = *(lds_f32*)(uintptr_t)(at + 8);
          top = fmaxf(top, mv[v]);
        }
        const float base = top;
        float ls = 0.f, bound = 0.f, own = 0.f;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          mv[v] = fast_exp2(mv[v] - base);
          ls += lv[v] * mv[v];
          bound += xv[v] * mv[v];
          if (v == wv) own = mv[v];
        }
        acc[0] *= own;
        acc[1] *= own;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          if (v == wv) continue;
          const uint32_t from = qbase + (uint32_t)(2048 * (3 * wv + (v < wv ? v : v - 1)) + 16 * ln);
          acc[0] += *(lds_f32x4*)(uintptr_t)from * mv[v];
          acc[1] += *(lds_f32x4*)(uintptr_t)(from + 1024) * mv[v];
        }
        const int col = 16 * cb + Lc;
        if (col < ncols) {
          const float inv = ls > 0.f ? 1.f / ls : 0.f;
          const float l2 = ls > 0.f ? top + __log2f(ls) : kNegInf;
          const int r = col / G, head = kvh * G + (col - r * G);
          acc[0] *= inv;
          acc[1] *= inv;
          if (w.part < 0) {
            const size_t oi = (size_t)(w.q0 + r) * a.hq + head;
#pragma unroll
            for (int i = 0; i < 2; ++i)
              *reinterpret_cast<u32x2*>(a.out + oi * kHeadDim + 32 * wv + 16 * i + 4 * Jc) =
                  u32x2{pack2<BF16>(acc[i][0], acc[i][1]), pack2<BF16>(acc[i][2], acc[i][3])};
            if (a.lse != nullptr && wv == 0 && Jc == 0) a.lse[oi] = l2 * kLn2;
          } else {
            // (the parts' largest magnitudes bound the row's: within a few times)
            float is;
            const float sc = part_scale_of(bound * inv, is);
            const size_t oi = (size_t)(w.part + r) * a.hq + head;
            u32x2 low;
#pragma unroll
            for (int i = 0; i < 2; ++i)
              low[i] = put_part<BF16>(a, oi * kHeadDim + 32 * wv + 16 * i + 4 * Jc, acc[i] * is);
            if (!BF16 && a.part_lo != nullptr)
              *reinterpret_cast<u32x2*>(a.part_lo + oi * kHeadDim + 32 * Jc + 8 * wv) = low;
            if (wv == 0 && Jc == 0) {
              a.part_lse[oi] = l2;
              a.part_scale[oi] = sc;
            }
          }
        }
      }
    }
    if (it + 1 < it1) barrier();  // the region is the next item's Q
  }
}

template <bool BF16, bool CAUSAL, bool STREAM, int HEADS>
__global__ __launch_bounds__(256 * HEADS, 2) void attn_block_kv8_kernel(AttnArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t dsm[];
  const int wave = uniform(threadIdx.x >> 6);
  const uint32_t lbase = (uint32_t)(uintptr_t)dsm;
  // Workgroups of one XCD (every eighth) take neighbouring shares, the kv heads
  // of one token range, so that its L2 channels see all of a page's lines.
  const int n_wg = (int)gridDim.x;
  const int b = n_wg % 8 == 0 ? (int)(blockIdx.x % 8) * (n_wg / 8) + (int)blockIdx.x / 8 : (int)blockIdx.x;
  const int share = HEADS * b + (wave >> 2);
  const int it = ldc(a.tile_off, share);
  const int end = min(ldc(a.tile_off, share + 1), uniform(*a.n_items));
  if (it >= end) return;
  block8_items<BF16, CAUSAL, STREAM>(a, it, end, lbase + (uint32_t)((wave >> 2) * kBlk8Head),
                                     lbase + (uint32_t)(HEADS * kBlk8Head + wave * kBlk8Wave), wave & 3,
                                     threadIdx.x & 63);
}

// Wide: any items, as tiles.  Even: the same, with the two shares of a compute
// unit evened out.  Any: the launch of a graph plan, whose later
// prepares may bring either kind: items of at most 64 columns as blocks.  (That
// one for eager launches too took 262 us for 8192 prompt tokens, 234 without
// the narrow items' path beside it.)
enum class Tile8 { Wide, Even, Any };

// The planner's longest-first lists give the first-dispatched workgroup of a
// compute unit's two (share b < pair) 3/2 of the other's work, what the 16-bit
// kernel's unequal pairs get through in the same time.  Here a wavefront's
// priority at the copies keeps the two alike: the last items of share b, from
// the one whose middle lies past half of both shares, go to share b + pair
// (8192 prompt tokens 219 us, 234 as listed, 221 at 5/9).  Both workgroups read
// the costs and come to the same border; who takes an item changes no result.
__device__ __forceinline__ void tile8_even_out(const AttnArgs& a, int n_items, int lane, int& last, int& more,
                                               int& more_end) {
  const int b = (int)blockIdx.x;
  const int first = b < a.pair ? b : b - a.pair;
  const int second = first + a.pair;
  if (second >= (int)gridDim.x) return;
  const int a0 = ldc(a.tile_off, first), a1 = min(ldc(a.tile_off, first + 1), n_items);
  const int b0 = ldc(a.tile_off, second), b1 = min(ldc(a.tile_off, second + 1), n_items);
  if (a0 >= a1 || b0 >= b1) return;          // an empty share's workgroup has ended
  if (a1 - a0 > 64 || b1 - b0 > 64) return;  // more than a lane each: left as listed
  const int ca = lane < a1 - a0 ? a.items[a0 + lane].cost : 0;
  int both = ca + (lane < b1 - b0 ? a.items[b0 + lane].cost : 0);
  int upto = ca;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(upto, d, 64);
    if (lane >= d) upto += v;
    both += __shfl_xor(both, d, 64);
  }
  const bool keeps = lane < a1 - a0 && 2 * upto - ca <= both;
  const int border = a0 + (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(keeps));
  if (b == first) {
    last = max(border, a0 + 1);
  } else {
    more = max(border, a0 + 1);
    more_end = a1;
  }
}

template <bool BF16, bool CAUSAL, bool STREAM, Tile8 KIND>
__global__ __launch_bounds__(256, 2) void attn_tile_kv8_kernel(AttnArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t dsm[];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int n_items = uniform(*a.n_items);
  const uint32_t lbase = (uint32_t)(uintptr_t)dsm;

  Tile8Lanes tl;
  if constexpr (KIND != Tile8::Any) tl = tile8_lanes(a, lane);

  int it = ldc(a.tile_off, blockIdx.x);
  const int end = min(ldc(a.tile_off, blockIdx.x + 1), n_items);
  if (it >= end) return;
  WorkItem w = ldc_item(a.items, it);
  SeqInfo s = ldc_seq(a.seqs, w.seq);
  f32x2 scales = {1.f, 1.f};
  int stage = 0;
  bool primed = false;  // w's first tile was requested during the item before
  int last = end, more = 0, more_end = 0;  // this workgroup's items: [it, last), then [more, more_end)
  if constexpr (KIND != Tile8::Any) {
    scales = tile8_copy<STREAM>(a, w, s, tl.goff, lbase, wave, w.t0);
    primed = true;
  }
  if constexpr (KIND == Tile8::Even) tile8_even_out(a, n_items, lane, last, more, more_end);
  for (;;) {
    int nit = it + 1;
    bool has_next = nit < end;
    if constexpr (KIND == Tile8::Even) {
      if (nit == last) nit = more;
      has_next = nit != more_end && (nit < last || more < more_end);
    }
    WorkItem wn = w;
    SeqInfo sn = s;
    if (has_next) {
      wn = ldc_item(a.items, nit);
      sn = ldc_seq(a.seqs, wn.seq);
    }
    if constexpr (KIND != Tile8::Any) {
      if (w.nq * a.group <= 64)
        stage = tile8_item<BF16, CAUSAL, 1, STREAM>(a, w, s, has_next, wn, sn, tl, lbase, wave, lane, stage, scales);
      else
        stage = tile8_item<BF16, CAUSAL, 2, STREAM>(a, w, s, has_next, wn, sn, tl, lbase, wave, lane, stage, scales);
    } else if (w.nq * a.group <= 64) {
      block8_items<BF16, CAUSAL, STREAM>(a, it, it + 1, lbase, lbase + (uint32_t)(kBlk8Head + wave * kBlk8Wave), wave,
                                         fresh_lane());
    } else {
      const int ln = fresh_lane();
      const Tile8Lanes tw = tile8_lanes(a, ln);
      if (!primed) scales = tile8_copy<STREAM>(a, w, s, tw.goff, lbase, wave, w.t0);
      primed = has_next && wn.nq * a.group > 64;
      stage = tile8_item<BF16, CAUSAL, 2, STREAM>(a, w, s, primed, wn, sn, tw, lbase, wave, ln, stage, scales);
    }
    if (!has_next) break;
    if (!primed) __syncthreads();  // the next item lays out LDS anew
    it = nit;
    w = wn;
    s = sn;
  }
}

// ===========================================================================
// Launchers
// ===========================================================================
enum class Decode8 { Shares, Short, Any };

template <bool BF16, int WAVES, int NCB, Decode8 KIND>
static hipError_t decode8_launch(const AttnArgs& a, int causal, int grid, hipStream_t st) {
  void (*fn)(AttnArgs, int);
  size_t lds = 0;
  if constexpr (KIND != Decode8::Short) lds = (size_t)WAVES * kKv8Units * kKv8Slot;
  if constexpr (KIND != Decode8::Shares) lds = std::max(lds, short8_lds<WAVES>());
  if constexpr (KIND == Decode8::Short) fn = attn_short_kv8_kernel<BF16, WAVES, NCB>;
  else fn = attn_decode_kv8_kernel<BF16, WAVES, NCB, KIND == Decode8::Any>;
  static std::atomic<uint64_t> lds_ok{0};
  const hipError_t e = allow_lds((const void*)fn, lds, lds_ok);
  if (e != hipSuccess) return e;
  const dim3 g = KIND == Decode8::Short ? dim3(a.hkv, grid / a.hkv) : dim3(grid);
  hipLaunchKernelGGL(fn, g, dim3(64 * WAVES), lds, st, a, causal);
  return hipGetLastError();
}

template <bool BF16, int WAVES, Decode8 KIND>
static hipError_t decode8_ncb(const AttnArgs& a, int ncb, int causal, int grid, hipStream_t st) {
  switch (ncb) {
    case 1: return decode8_launch<BF16, WAVES, 1, KIND>(a, causal, grid, st);
    case 2: return decode8_launch<BF16, WAVES, 2, KIND>(a, causal, grid, st);
    default: return hipErrorInvalidValue;
  }
}

template <bool BF16, int WAVES>
static hipError_t decode8_kind(const AttnArgs& a, int ncb, int causal, bool any, int grid, hipStream_t st) {
  if constexpr (WAVES >= kShortMinWaves) {
    if (any) return decode8_ncb<BF16, WAVES, Decode8::Any>(a, ncb, causal, grid, st);
    if (a.n_short > 0) return decode8_ncb<BF16, WAVES, Decode8::Short>(a, ncb, causal, grid, st);
  } else if (a.n_short > 0) {
    return hipErrorInvalidValue;
  }
  return decode8_ncb<BF16, WAVES, Decode8::Shares>(a, ncb, causal, grid, st);
}

template <bool BF16>
static hipError_t decode8_waves(const AttnArgs& a, int waves, int ncb, int causal, bool any, int grid,
                                hipStream_t st) {
  switch (waves) {
    case 8: return decode8_kind<BF16, 8>(a, ncb, causal, any, grid, st);
    case 4: return decode8_kind<BF16, 4>(a, ncb, causal, any, grid, st);
    case 2: return decode8_kind<BF16, 2>(a, ncb, causal, any, grid, st);
    case 1: return decode8_kind<BF16, 1>(a, ncb, causal, any, grid, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_decode_kv8(const AttnArgs& a, bool bf16, int waves, int ncb, int causal, bool any, int grid,
                             hipStream_t st) {
  return bf16 ? decode8_waves<true>(a, waves, ncb, causal, any, grid, st)
              : decode8_waves<false>(a, waves, ncb, causal, any, grid, st);
}

template <bool BF16, bool CAUSAL, bool STREAM, Tile8 KIND>
static hipError_t tile8_launch(const AttnArgs& a, int grid, hipStream_t st) {
  static std::atomic<uint64_t> lds_ok{0};
  const hipError_t e = allow_lds((const void*)attn_tile_kv8_kernel<BF16, CAUSAL, STREAM, KIND>, kTile8Lds, lds_ok);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((attn_tile_kv8_kernel<BF16, CAUSAL, STREAM, KIND>), dim3(grid), dim3(256), kTile8Lds, st, a);
  return hipGetLastError();
}

// (HEADS = 2: `grid` shares are an equal cut's, all kv heads of a token range
// together, so that neighbours have the same items.)
template <bool BF16, bool CAUSAL, bool STREAM, int HEADS>
static hipError_t block8_launch(const AttnArgs& a, int grid, hipStream_t st) {
  constexpr size_t lds = (size_t)HEADS * kTile8Lds;
  static std::atomic<uint64_t> lds_ok{0};
  const hipError_t e = allow_lds((const void*)attn_block_kv8_kernel<BF16, CAUSAL, STREAM, HEADS>, lds, lds_ok);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((attn_block_kv8_kernel<BF16, CAUSAL, STREAM, HEADS>), dim3(grid / HEADS), dim3(256 * HEADS), lds,
                     st, a);
  return hipGetLastError();
}

template <bool BF16, bool CAUSAL>
static hipError_t tile8_kind(const AttnArgs& a, bool stream, bool any, bool narrow, bool pairs, int grid,
                             hipStream_t st) {
  auto go = [&](auto streamed) {
    constexpr bool S = decltype(streamed)::value;
    if (any) return tile8_launch<BF16, CAUSAL, S, Tile8::Any>(a, grid, st);
    if (!narrow)
      return a.pair > 0 ? tile8_launch<BF16, CAUSAL, S, Tile8::Even>(a, grid, st)
                        : tile8_launch<BF16, CAUSAL, S, Tile8::Wide>(a, grid, st);
    return pairs ? block8_launch<BF16, CAUSAL, S, 2>(a, grid, st) : block8_launch<BF16, CAUSAL, S, 1>(a, grid, st);
  };
  return stream ? go(std::true_type{}) : go(std::false_type{});
}

// any: a graph plan's launch; else narrow: every item has at most 64 columns;
// pairs: and the list is an equal cut over an even number of kv heads.
hipError_t launch_tile_kv8(const AttnArgs& a, bool bf16, bool causal, bool stream, bool any, bool narrow, bool pairs,
                           int grid, hipStream_t st) {
  if (bf16)
    return causal ? tile8_kind<true, true>(a, stream, any, narrow, pairs, grid, st)
                  : tile8_kind<true, false>(a, stream, any, narrow, pairs, grid, st);
  return causal ? tile8_kind<false, true>(a, stream, any, narrow, pairs, grid, st)
                : tile8_kind<false, false>(a, stream, any, narrow, pairs, grid, st);
}

}  // namespace feattn
