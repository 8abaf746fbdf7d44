// Append to the 8-bit paged KV cache (kv8.hpp), with q/k RMSNorm and RoPE on
// the way, and reading its tokens back as 16-bit rows, for gfx950.
//
// Append: for every scale block and kv head that the call writes,
//   need  = the smallest power of two s with max |x| <= 448 s over the finite
//           values x that the call puts there
//   scale = need where the call writes the block's first slot (which starts
//           the block), else max(old scale, need); where that grows, the codes
//           already in the block are rescaled
//   code  = e4m3(x / scale), round to nearest even, rounded once from the fp32
//           value (normalised, rotated); infinities and NaNs become NaN codes.
// This file is compiled with -ffp-contract=off (the rope form's queries are
// bit-identical to fe_rope's).
#include "kv8.hpp"
#include "rope_math.hpp"

namespace feattn {

enum class Kv8Form { Store, Rope, NormRope };

struct Kv8Args {
  const uint16_t* q;  // Rope: rotated in place through q_out (the same tensor)
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_stride, kv_stride;  // elements from row to row
  const uint16_t* qw;
  const uint16_t* kw;
  float eps;
  uint16_t* q_out;  // [rows][hq][128]
  uint8_t* kc;
  uint8_t* vc;
  uint32_t* scales;
  const int64_t* pos;
  const int64_t* slots;
  const float* table;
  int rows, hq, hkv, max_pos, cache_slots;
};

// Sum and maximum over an aligned group of eight lanes, in registers.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_bits(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141;

__device__ __forceinline__ float sum8(float v) {
  v += __uint_as_float(dpp_bits<kXor1>(__float_as_uint(v)));
  v += __uint_as_float(dpp_bits<kXor2>(__float_as_uint(v)));
  return v + __uint_as_float(dpp_bits<kHalfMirror>(__float_as_uint(v)));
}
__device__ __forceinline__ uint32_t max8(uint32_t v) {
  v = max(v, dpp_bits<kXor1>(v));
  v = max(v, dpp_bits<kXor2>(v));
  return max(v, dpp_bits<kHalfMirror>(v));
}

// A head's 128 elements lie on eight lanes: lane c holds elements 8c..8c+7 and
// 64+8c..64+8c+7 (the RoPE pairs), x[0..7] and x[8..15].
template <bool BF16>
__device__ __forceinline__ void unpack16(u32x4 lo, u32x4 hi, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = lo_f32<BF16>(lo[i]);
    x[2 * i + 1] = hi_f32<BF16>(lo[i]);
    x[8 + 2 * i] = lo_f32<BF16>(hi[i]);
    x[9 + 2 * i] = hi_f32<BF16>(hi[i]);
  }
}

// Normalization and rotation stay in fp32 up to the one rounding at the end;
// sums in pairs and fused products keep them within a few 2^-24.
__device__ __forceinline__ float rms16(const float (&x)[16], float eps) {
  float s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[i] = x[4 * i] * x[4 * i];
#pragma unroll
    for (int e = 1; e < 4; ++e) s[i] = __builtin_fmaf(x[4 * i + e], x[4 * i + e], s[i]);
  }
  return rsqrtf(sum8((s[0] + s[1]) + (s[2] + s[3])) * (1.f / 128.f) + eps);
}

__device__ __forceinline__ void scale16(float (&x)[16], float r, const float (&w)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = x[e] * r * w[e];
}

// cs: the lane's cos entries, then its sin entries.
__device__ __forceinline__ void rotate16(float (&x)[16], const float (&cs)[16]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = x[e], b = x[8 + e];
    x[e] = __builtin_fmaf(a, cs[e], -(b * cs[8 + e]));
    x[8 + e] = __builtin_fmaf(b, cs[e], a * cs[8 + e]);
  }
}

__device__ __forceinline__ void load_angles(const float* at, float (&cs)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(at + (i < 2 ? 4 * i : 64 + 4 * (i - 2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) cs[4 * i + e] = v[e];
  }
}

// Query heads: eight lanes take kQHeads heads of one row, which share the
// row's angles (512 bytes, as much as two heads).
constexpr int kQHeads = 4;

template <bool BF16, Kv8Form FORM>
__device__ __forceinline__ void kv8_query(const Kv8Args& a, int64_t unit, int c) {
  const int groups = (a.hq + kQHeads - 1) / kQHeads;
  const int64_t units = (int64_t)a.rows * groups;
  if (unit >= units) return;  // whole groups of eight lanes
  const int64_t row = units <= UINT32_MAX ? (int64_t)((uint32_t)unit / (uint32_t)groups) : unit / groups;
  const int head = (int)(unit - row * groups) * kQHeads;
  const uint16_t* src = a.q + row * a.q_stride + (int64_t)head * 128 + 8 * c;
  uint16_t* dst = a.q_out + (row * a.hq + head) * 128 + 8 * c;
  const int64_t p = a.pos[row];
  const bool rot = p >= 0 && p < a.max_pos;
  const float* at = a.table + (rot ? p : 0) * 128 + 8 * c;
  u32x4 lo[kQHeads], hi[kQHeads];
#pragma unroll
  for (int i = 0; i < kQHeads; ++i) {
    const int h = head + i < a.hq ? 128 * i : 0;
    lo[i] = ldv(src + h);
    hi[i] = ldv(src + h + 64);
  }
  if constexpr (FORM == Kv8Form::Rope) {
    if (!rot) return;  // in place
#pragma unroll
    for (int i = 0; i < kQHeads; ++i) rotate8<BF16>(lo[i], hi[i], at, at + 64);
  } else {
    float cs[16], w[16];
    load_angles(at, cs);
    unpack16<BF16>(ldv(a.qw + 8 * c), ldv(a.qw + 64 + 8 * c), w);
#pragma unroll
    for (int i = 0; i < kQHeads; ++i) {
      float x[16];
      unpack16<BF16>(lo[i], hi[i], x);
      scale16(x, rms16(x, a.eps), w);
      if (rot) rotate16(x, cs);
      float l[8], h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        l[e] = x[e];
        h[e] = x[8 + e];
      }
      lo[i] = pack8_rne<BF16>(l);
      hi[i] = pack8_rne<BF16>(h);
    }
  }
#pragma unroll
  for (int i = 0; i < kQHeads; ++i)
    if (head + i < a.hq) {
      stv(dst + 128 * i, lo[i]);
      stv(dst + 128 * i + 64, hi[i]);
    }
}

// Keys take the codes of their 64-bit values.  A code has so few bits that an
// error of 2^-24 before its rounding shows as a whole step of an element now and
// then.  So a lane computes its 16 elements in fp32, within t = 1.25 * 2^-22
// (|a| + |b|) (r, r w and x r w round to 2^-24 each, b s and the result once
// more), and where an interval of that size around one holds a number of at
// most five significant bits, as all borders between codes are whatever the
// block's scale will be, it computes them again in 64 bits and rounds them to
// odd: towards zero, and the rest as a last bit, so that the code's rounding is
// that of the 64-bit value.  (One pass over eight rows in seven does; in 64 bits
// throughout the keys and values of 8192 rows of 8 heads took 22 us, 13 with no
// arithmetic on the keys.)
__device__ __forceinline__ float round_odd(double d) {
  const float f = (float)d;
  uint32_t u = __float_as_uint(f);
  const double back = (double)f;
  if (fabs(back) > fabs(d)) --u;
  if (back != d) u |= 1u;
  return f == f && fabsf(f) < __builtin_huge_valf() ? __uint_as_float(u) : f;
}

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)dpp_bits<CTRL>((uint32_t)b) | (uint64_t)dpp_bits<CTRL>((uint32_t)(b >> 32)) << 32);
}

template <bool BF16, bool NORM>
__device__ __forceinline__ void key_row(u32x4 lo, u32x4 hi, const uint16_t* kw, float eps, int c, bool rot,
                                        const float* angles, float (&out)[16]) {
  float in[16], w[16] = {}, cs[16];
  load_angles(angles, cs);
  if constexpr (NORM) unpack16<BF16>(ldv(kw + 8 * c), ldv(kw + 64 + 8 * c), w);
  unpack16<BF16>(lo, hi, in);
  double r = 1.0;
  if constexpr (NORM) {
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < 16; ++e) s = __builtin_fma((double)in[e], (double)in[e], s);
    s += dpp64<kXor1>(s);
    s += dpp64<kXor2>(s);
    s += dpp64<kHalfMirror>(s);
    s = s * (1.0 / 128.0) + (double)eps;
    r = __builtin_amdgcn_rsq(s);  // good to some 2^-23: one step of Newton's iteration
    if (s < __builtin_huge_val()) r *= 1.5 - 0.5 * s * r * r;
  }
  const float rf = (float)r;
  // (rows of a size whose fp32 factors would leave the normal range: in 64 bits)
  uint32_t crossed = NORM && !(rf > 0x1p-100f && rf < 0x1p100f) ? 1u << 31 : 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float a = in[e], b = in[8 + e];
    if constexpr (NORM) {
      a *= rf * w[e];
      b *= rf * w[8 + e];
    }
    out[e] = rot ? __builtin_fmaf(a, cs[e], -(b * cs[8 + e])) : a;
    out[8 + e] = rot ? __builtin_fmaf(b, cs[e], a * cs[8 + e]) : b;
    const float t = (fabsf(a) + fabsf(b)) * 0x1.4p-22f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float y = fabsf(out[8 * h + e]);
      crossed |= __float_as_uint(y - t) ^ __float_as_uint(y + t);
    }
  }
  if ((crossed >> 19) != 0) {
    // (read again: nothing of the first computation is to be held for this one)
    asm volatile("" : "+v"(angles), "+v"(kw));
    load_angles(angles, cs);
    if constexpr (NORM) unpack16<BF16>(ldv(kw + 8 * c), ldv(kw + 64 + 8 * c), w);
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(lo[i]), "+v"(hi[i]));
    unpack16<BF16>(lo, hi, in);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      double a = (double)in[e], b = (double)in[8 + e];
      if constexpr (NORM) {
        a *= r * (double)w[e];
        b *= r * (double)w[8 + e];
      }
      const double co = (double)cs[e], si = (double)cs[8 + e];
      out[e] = round_odd(rot ? __builtin_fma(a, co, -(b * si)) : a);
      out[8 + e] = round_odd(rot ? __builtin_fma(b, co, a * si) : b);
      __builtin_amdgcn_sched_barrier(0);  // (one pair's 64-bit values at a time)
    }
  }
}

// One wavefront takes a window of 16 rows and one (kv head, K or V).  The rows
// of a call that go to one scale block follow one another; such a run belongs
// to the window its first row lies in, whose wavefront is the only one to
// write that block and head: no atomics, and the same bits every time.  The
// window's runs (they end within 32 rows of its first) are taken in batches of
// whole runs, at most 16 rows, whose values are all in registers at once, eight
// lanes to a row, while the runs' scales are found: a prompt's window is one
// batch or two, a decode batch's 16 runs of one row are one.  (All 32 rows in
// registers at once took 31 us for 8192 rows of 8 heads, keys and values
// alone, of which 17 were without the arithmetic on the keys.)
// Lane i (1 <= i <= 32) keeps the books of row r0 - 1 + i.
template <bool BF16, Kv8Form FORM>
__device__ __forceinline__ void kv8_window(const Kv8Args& a, int64_t unit) {
  const int lane = threadIdx.x & 63;
  const int c = lane & 7;
  const int g = lane >> 3;
  const int heads = 2 * a.hkv;
  const int64_t win = unit <= INT32_MAX ? (int64_t)((uint32_t)unit / (uint32_t)heads) : unit / heads;
  const int hs = uniform((int)(unit - win * heads));
  const int side = hs >= a.hkv ? 1 : 0;
  const int head = side ? hs - a.hkv : hs;
  const int64_t r0 = win * 16;
  const bool keys = FORM != Kv8Form::Store && side == 0;

  // ---- runs
  const int64_t row = r0 - 1 + lane;
  int slot = -1, p = -1;
  if (lane <= 32 && row >= 0 && row < a.rows) {
    const int64_t s = a.slots[row];
    if (s >= 0 && s < a.cache_slots) slot = (int)s;
    if (keys) {
      const int64_t q = a.pos[row];
      if (q >= 0 && q < a.max_pos) p = (int)q;
    }
  }
  const int block = slot >> 4;  // -1: the row is not stored
  const int before = __shfl_up(block, 1, 64);
  // (lane 0: the row before the window, whose run another window owns)
  const uint64_t run_heads = __builtin_amdgcn_ballot_w64(lane == 0 || block != before);
  const int start = 63 - __builtin_clzll(run_heads & ((uint64_t(2) << lane) - 1));
  const bool member = block >= 0 && start >= 1 && start <= 16 && lane <= 32;
  uint64_t left = __builtin_amdgcn_ballot_w64(member);
  if (left == 0) return;

  uint32_t* const scale_at = a.scales + ((int64_t)(member ? block : 0) * a.hkv + head) * 2 + side;
  uint32_t old = 0;
  if (member) old = *scale_at;
  old &= kInfBits;
  if (old == kInfBits) old = 0;

  const uint16_t* src = (side ? a.v : a.k) + (int64_t)head * 128 + 8 * c;
  uint8_t* cache = (side ? a.vc : a.kc) + (int64_t)head * 128;
  const int64_t row_bytes = (int64_t)a.hkv * 128;
  do {
    // The batch: lanes [i0, i1), from a run's first row up to the last border of
    // two runs that is at most 16 rows away.
    const int i0 = __builtin_ctzll(left);
    const uint64_t borders = run_heads & (uint64_t(0x1fffe) << i0);
    const int i1 = borders != 0 ? 63 - __builtin_clzll(borders) : i0 + 16;
    const uint64_t rows_of = left & ((uint64_t(1) << i1) - 1);
    left &= ~(((uint64_t(1) << i1) - 1));

    float x[2][16];
    uint32_t top[2];
    u32x4 lo[2], hi[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      top[s] = 0;
      if (s > 0 && (rows_of >> (i0 + 8)) == 0) continue;
      const int64_t r = min(r0 - 1 + i0 + 8 * s + g, (int64_t)a.rows - 1);
      const uint16_t* at = src + r * a.kv_stride;
      lo[s] = ldv(at);
      hi[s] = ldv(at + 64);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s > 0 && (rows_of >> (i0 + 8)) == 0) continue;
      if (keys) {
        const int at = __shfl(p, i0 + 8 * s + g, 64);
        key_row<BF16, FORM == Kv8Form::NormRope>(lo[s], hi[s], a.kw, a.eps, c, at >= 0,
                                                 a.table + (int64_t)max(at, 0) * 128 + 8 * c, x[s]);
      } else {
        unpack16<BF16>(lo[s], hi[s], x[s]);
      }
      float mx = 0.f;  // (a NaN leaves it as it is)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, fabsf(x[s][e]));
      const float cap = kv8_cap<BF16>();
      if (__builtin_amdgcn_ballot_w64(!(mx <= cap)) != 0) {
        // infinities, which like NaNs have no code but NaN's and count for no
        // scale, and magnitudes past the cap
        mx = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float y = x[s][e];
          if (fabsf(y) < __builtin_huge_valf()) {
            if (fabsf(y) > cap) x[s][e] = __builtin_copysignf(cap, y);
            mx = fmaxf(mx, fabsf(x[s][e]));
          }
        }
      }
      top[s] = __float_as_uint(mx);
      top[s] = max8(top[s]);
    }

    // ---- the runs' scales, from the rows' maxima
    const bool mine = (rows_of >> lane) & 1;
    const int j = lane - i0;
    const uint32_t t0 = (uint32_t)__shfl((int)top[0], (8 * j) & 63, 64);
    const uint32_t t1 = (uint32_t)__shfl((int)top[1], (8 * j) & 63, 64);
    uint32_t amax = mine ? (j < 8 ? t0 : t1) : 0u;
    uint32_t written = mine ? 1u << (slot & 15) : 0u;
#pragma unroll
    for (int d = 1; d <= 8; d <<= 1) {  // over the lanes behind, within the run
      const uint32_t am = (uint32_t)__shfl_down((int)amax, d, 64);
      const uint32_t wr = (uint32_t)__shfl_down((int)written, d, 64);
      const int st = __shfl_down(start, d, 64);
      if (lane + d < 64 && st == start) {
        amax = max(amax, am);
        written |= wr;
      }
    }
    amax = (uint32_t)__shfl((int)amax, start, 64);
    written = (uint32_t)__shfl((int)written, start, 64);
    const uint32_t held = (written & 1u) ? 0u : old;
    const uint32_t scale = max(kv8_need(amax), held);
    const bool leader = mine && start == lane;
    if (leader) *scale_at = scale;

    // ---- the codes
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s > 0 && (rows_of >> (i0 + 8)) == 0) continue;
      const int from = i0 + 8 * s + g;
      const float inv = kv8_inverse((uint32_t)__shfl((int)scale, from, 64));
      const int to = __shfl(mine ? slot : -1, from, 64);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[s][e] *= inv;
      if (to >= 0) {
        uint8_t* dst = cache + (int64_t)to * row_bytes + 8 * c;
        const u32x2 lo = {kv8_encode4(x[s][0], x[s][1], x[s][2], x[s][3]),
                          kv8_encode4(x[s][4], x[s][5], x[s][6], x[s][7])};
        const u32x2 hi = {kv8_encode4(x[s][8], x[s][9], x[s][10], x[s][11]),
                          kv8_encode4(x[s][12], x[s][13], x[s][14], x[s][15])};
        *reinterpret_cast<u32x2*>(dst) = lo;
        *reinterpret_cast<u32x2*>(dst + 64) = hi;
      }
    }

    // ---- earlier tokens of blocks whose scale grew: four lanes a token
    uint64_t grown = __builtin_amdgcn_ballot_w64(leader && scale > held && !(written & 1u));
    while (grown != 0) {
      const int l = __builtin_ctzll(grown);
      grown &= grown - 1;
      const int b = __builtin_amdgcn_readlane(block, l);
      const uint32_t wr = (uint32_t)__builtin_amdgcn_readlane((int)written, l);
      const int de = (__builtin_amdgcn_readlane((int)held, l) - __builtin_amdgcn_readlane((int)scale, l)) >> 23;
      const float ratio = __builtin_ldexpf(1.f, de);
      const int t = lane >> 2;
      if (((wr >> t) & 1u) == 0) {
        u32x4* codes = reinterpret_cast<u32x4*>(cache + ((int64_t)b * 16 + t) * row_bytes + 32 * (lane & 3));
        u32x4 q[2] = {codes[0], codes[1]};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const auto f0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i][k], false);
            const auto f1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i][k], true);
            q[i][k] = kv8_encode4(f0[0] * ratio, f0[1] * ratio, f1[0] * ratio, f1[1] * ratio);
          }
        codes[0] = q[0];
        codes[1] = q[1];
      }
    }
  } while (left != 0);
}

// Windows first: they take longest.  (Windows and queries in turns, so that
// what waits and what streams would overlap: 45.7 us for 8192 rows of 32/8
// heads, 43.5 so, against 20.7 and 23.1 alone; queries first 44.4.  The queries
// stream 5.8 TB/s; keys and values are bound by their dependent loads and the
// arithmetic on the keys.)  Four wavefronts per SIMD: 128 registers.
template <bool BF16, Kv8Form FORM>
__global__ __launch_bounds__(256, 4) void kv8_append_kernel(Kv8Args a) {
  const int64_t wave = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  const int64_t windows = ((int64_t)a.rows + 15) / 16 * (2 * a.hkv);
  if (wave < windows) {
    kv8_window<BF16, FORM>(a, wave);
  } else if constexpr (FORM != Kv8Form::Store) {
    const int lane = threadIdx.x & 63;
    kv8_query<BF16, FORM>(a, (wave - windows) * 8 + (lane >> 3), lane & 7);
  }
}

template <Kv8Form FORM>
static hipError_t kv8_launch(const Kv8Args& a, bool bf16, hipStream_t st) {
  const int64_t windows = ((int64_t)a.rows + 15) / 16 * (2 * a.hkv);
  const int64_t queries = FORM == Kv8Form::Store ? 0 : (int64_t)a.rows * ((a.hq + kQHeads - 1) / kQHeads);
  const int64_t grid = (windows + (queries + 7) / 8 + 3) / 4;
  if (grid == 0) return hipSuccess;
  if (grid > INT32_MAX) return hipErrorInvalidValue;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(256), 0, st, a); };
  if (bf16) go(kv8_append_kernel<true, FORM>);
  else go(kv8_append_kernel<false, FORM>);
  return hipGetLastError();
}

hipError_t launch_store_kv8(const void* k, const void* v, void* kc, void* vc, float* scales, const int64_t* slots,
                            int rows, int hkv, bool bf16, int cache_slots, hipStream_t st) {
  Kv8Args a{};
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.kv_stride = (int64_t)hkv * 128;
  a.kc = (uint8_t*)kc;
  a.vc = (uint8_t*)vc;
  a.scales = (uint32_t*)scales;
  a.slots = slots;
  a.rows = rows;
  a.hkv = hkv;
  a.cache_slots = cache_slots;
  return kv8_launch<Kv8Form::Store>(a, bf16, st);
}

hipError_t launch_rope_append_kv8(void* q, const void* k, const void* v, void* kc, void* vc, float* scales,
                                  const int64_t* pos, const int64_t* slots, const float* table, int rows, int hq,
                                  int hkv, bool bf16, int max_pos, int cache_slots, hipStream_t st) {
  Kv8Args a{};
  a.q = (const uint16_t*)q;
  a.q_out = (uint16_t*)q;
  a.q_stride = (int64_t)hq * 128;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.kv_stride = (int64_t)hkv * 128;
  a.kc = (uint8_t*)kc;
  a.vc = (uint8_t*)vc;
  a.scales = (uint32_t*)scales;
  a.pos = pos;
  a.slots = slots;
  a.table = table;
  a.rows = rows;
  a.hq = hq;
  a.hkv = hkv;
  a.max_pos = max_pos;
  a.cache_slots = cache_slots;
  return kv8_launch<Kv8Form::Rope>(a, bf16, st);
}

hipError_t launch_norm_rope_append_kv8(const void* qkv, int64_t row_stride, const void* qw, const void* kw, float eps,
                                       void* q_out, void* kc, void* vc, float* scales, const int64_t* pos,
                                       const int64_t* slots, const float* table, int rows, int hq, int hkv, bool bf16,
                                       int max_pos, int cache_slots, hipStream_t st) {
  Kv8Args a{};
  a.q = (const uint16_t*)qkv;
  a.k = a.q + (int64_t)hq * 128;
  a.v = a.k + (int64_t)hkv * 128;
  a.q_stride = a.kv_stride = row_stride;
  a.qw = (const uint16_t*)qw;
  a.kw = (const uint16_t*)kw;
  a.eps = eps;
  a.q_out = (uint16_t*)q_out;
  a.kc = (uint8_t*)kc;
  a.vc = (uint8_t*)vc;
  a.scales = (uint32_t*)scales;
  a.pos = pos;
  a.slots = slots;
  a.table = table;
  a.rows = rows;
  a.hq = hq;
  a.hkv = hkv;
  a.max_pos = max_pos;
  a.cache_slots = cache_slots;
  return kv8_launch<Kv8Form::NormRope>(a, bf16, st);
}

// Tokens of the cache as 16-bit rows: a thread takes 8 codes of K and of V, so
// that both the loads (8 bytes) and the stores (16 bytes) of a wavefront are
// contiguous (HBM bound: 30000 rows of 4 heads 14.6 us, 6.3 TB/s).  Rows whose slot is outside the cache are left as they are.
template <bool BF16>
__global__ __launch_bounds__(256) void kv8_load_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                       const float* __restrict__ scales,
                                                       const int64_t* __restrict__ slots, uint16_t* __restrict__ k_out,
                                                       uint16_t* __restrict__ v_out, int64_t total, int hkv,
                                                       int cache_slots) {
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= total) return;
  const int64_t unit = idx >> 4;  // (row, head)
  const int c = (int)(idx & 15);
  const int64_t row = total <= UINT32_MAX ? (int64_t)((uint32_t)unit / (uint32_t)hkv) : unit / hkv;
  const int head = (int)(unit - row * hkv);
  const int64_t slot = slots[row];
  if (slot < 0 || slot >= cache_slots) return;
  const int64_t from = (slot * hkv + head) * 128 + 8 * c;
  const u32x2 kw = *reinterpret_cast<const u32x2*>(kc + from);
  const u32x2 vw = *reinterpret_cast<const u32x2*>(vc + from);
  const f32x2 s = *reinterpret_cast<const f32x2*>(scales + ((slot >> 4) * hkv + head) * 2);
  stv(k_out + 8 * idx, kv8_decode8<BF16>(kw[0], kw[1], s[0], s[0]));
  stv(v_out + 8 * idx, kv8_decode8<BF16>(vw[0], vw[1], s[1], s[1]));
}

hipError_t launch_load_kv8(const void* kc, const void* vc, const float* scales, const int64_t* slots, void* k_out,
                           void* v_out, int rows, int hkv, bool bf16, int cache_slots, hipStream_t st) {
  const int64_t total = (int64_t)rows * hkv * 16;
  if (total == 0) return hipSuccess;
  const int64_t grid = (total + 255) / 256;
  if (grid > INT32_MAX) return hipErrorInvalidValue;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(256), 0, st, (const uint8_t*)kc, (const uint8_t*)vc, scales,
                       slots, (uint16_t*)k_out, (uint16_t*)v_out, total, hkv, cache_slots);
  };
  if (bf16) go(kv8_load_kernel<true>);
  else go(kv8_load_kernel<false>);
  return hipGetLastError();
}

}  // namespace feattn
