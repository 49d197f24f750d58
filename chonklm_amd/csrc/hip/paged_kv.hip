// The quantised, paged K/V cache for gfx950: new rows normalised, rotated and
// quantised into their pages (k_kv_append), values read back (k_kv_read), and
// attention of one new token a row over the pages, split over the length and
// joined (k_kv_attend, k_kv_join). The C entry points are at the end.
//
// A page holds 64 positions; per kv head K codes | K scales | V codes | V scales.
// Codes come in units of 32 positions x 32 dims, in the order in which lane
// n = 16 g + i of a wave feeds the 16x16x32 matrix product:
//   scores   S[position][head] = K Q^T: A row i = position 16 t + i, k = dims 8 g + e
//   output   O[dim][head]      = V^T P^T: A row i = dim 16 h + i, k = positions
//            4 g + (e & 3) + 16 (e >> 2)
// The scores' result leaves lane (g, head) with positions 4 g + r of both tiles
// t = 0, 1: exactly the eight positions that the second product's B operand
// wants there, so the probabilities never leave their lane.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "chonk.h"
#include "errors.h"
#include "kernel_common.h"
#include "part_sum.h"
#include "paged_kv.h"

namespace chonk {
namespace {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

constexpr int kMostWgs = 2048;  // segments of a split attention, at most
constexpr int kWholeHalves = 32;  // half pages of a row that is never cut
// ... of at least so many half pages (5 x 8 rows of 4094 positions of 64 dims in 4 bits: 10.8 us in
// segments of 8, 12.3 of 16; 48 rows of 512 of 256 dims in fp16: 12.8 of 8, 13.0 of 4)
constexpr int kMinHalves = 8;

__device__ __forceinline__ f4_t mfma(h8_t a, h8_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ void fault(const KvCache& c, int bit) {
  if (c.fault) atomicOr(c.fault, bit);
}

// The page of (seq, pos), or -1 (and the fault noted) where there is none.
__device__ __forceinline__ int page_of(const KvCache& c, int seq, int pos, bool note) {
  const int bad = seq >= c.n_seqs ? KVF_SEQ : pos < 0 || pos / kKvPage >= c.max_pages ? KVF_POS : 0;
  if (bad) {
    if (note) fault(c, bad);
    return -1;
  }
  const int page = c.table[(size_t)seq * c.max_pages + pos / kKvPage];
  if (page < 0 || page >= c.n_pages) {
    if (note) fault(c, KVF_PAGE);
    return -1;
  }
  return page;
}

// Place of position p (0..31 of its half) in the order of the scales and of
// the V operand: lane group 4 bits up, its eight positions below.
__device__ __forceinline__ int place_of(int p) { return ((p & 15) >> 2) * 8 + (p & 3) + 4 * (p >> 4); }

// ---- writing ----------------------------------------------------------------------

typedef float f4u_t __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 h4u_t __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 h8u_t __attribute__((ext_vector_type(8), aligned(2)));

// Sums and maxima over the L lanes of a (row, head), without the LDS crossbar.
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int L>
__device__ __forceinline__ double lanes_sum(double v) {
  v += dpp64<0xb1>(v);
  v += dpp64<0x4e>(v);
  v += dpp64<0x141>(v);
  if constexpr (L >= 16) v += dpp64<0x140>(v);
  if constexpr (L >= 32) v += __shfl_xor(v, 16);
  if constexpr (L >= 64) v += __shfl_xor(v, 32);
  return v;
}

// a / b from r = 1 / b rounded once: the quotient's error, exact in one fused step, times r
// puts it right, as a division would round it (Markstein; b and the quotient are
// far from the ends of fp32's range, or the quotient does not matter).
__device__ __forceinline__ float quotient(float a, float b, float r) {
  const float q = a * r;
  return fmaf(fmaf(-q, b, a), r, q);
}

// Codes and scale of eight lanes' 32 values, four consecutive dims a lane. A
// scale is the fp16 nearest to the exact one, and the codes count in units of
// that fp16 number, so a code is off by at most half a unit of what is stored.
template <int KV>
__device__ __forceinline__ uint32_t quantise(const float (&y)[4], int (&c)[4]) {
  constexpr float kTop = KV == CHONK_KV_Q8 ? 127.f : 7.f, kLow = KV == CHONK_KV_Q8 ? -127.f : -8.f;
  // the largest magnitude; a NaN or an infinity makes it infinite
  float m = y[0];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (fabsf(y[i]) > fabsf(m)) m = y[i];
    bad |= !(fabsf(y[i]) <= 3.402823466e38f);
  }
  if (bad) m = INFINITY;
  // (of equal magnitudes the lower dim's: every lane must find the same one)
  auto step = [&](float o, int x) {
    if (fabsf(o) > fabsf(m) || (fabsf(o) == fabsf(m) && (threadIdx.x & x))) m = o;
  };
  step(dpp<0xb1>(m), 1);
  step(dpp<0x4e>(m), 2);
  step(dpp<0x141>(m), 4);  // (the other four's: a mirrored row of eight)
  bad = fabsf(m) == INFINITY;
  float d = KV == CHONK_KV_Q8 ? quotient(fabsf(m), 127.f, 1.f / 127.f) : m * -0.125f;
  d = fminf(fmaxf(d, -65504.f), 65504.f);
  const _Float16 h = (_Float16)d;
  const float dh = (float)h, rh = __fdiv_rn(1.f, dh);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c[i] = bad || dh == 0.f ? 0 : (int)fminf(fmaxf(rintf(quotient(y[i], dh, rh)), kLow), kTop);
  return bad ? 0x7e00u : (uint32_t)__builtin_bit_cast(unsigned short, h);
}

// Where position p (of a half page) and dim i (of a block) lie in a unit's K codes
// (run of eight dims) and V codes (place of the dim), as a count of pieces.
__device__ __forceinline__ int k_piece(int p, int i) { return (i >> 3) * 16 + (p & 15); }
__device__ __forceinline__ int v_piece(int p, int i) { return (place_of(p) >> 3) * 16 + (i & 15); }

// Four consecutive dims' stored values of one position: codes with their bias, or halves.
template <int KV>
__device__ __forceinline__ void stored4(const float (&y)[4], uint32_t (&c)[4], uint32_t& d) {
  if constexpr (KV == CHONK_KV_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __builtin_bit_cast(unsigned short, (_Float16)y[i]);
  } else {
    int q[4];
    d = quantise<KV>(y, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = (uint32_t)(q[i] + (KV == CHONK_KV_Q8 ? 128 : 8));
  }
}
// K of position j, dims d0 .. d0 + 3. (4 bits: the lane with the byte's low nibbles stores.)
template <int KV>
__device__ __forceinline__ void put_k(uint8_t* base, int hd, int j, int d0, const uint32_t (&c)[4], bool ok) {
  const int unit = (j / 32) * (hd / 32) + d0 / 32, p = j & 31, i0 = d0 & 31, n = k_piece(p, i0);
  if constexpr (KV == CHONK_KV_Q4) {
    uint32_t w = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
    w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xb1, 0xf, 0xf, false) << 4;  // dims + 4: the next lane's
    if (ok && !(threadIdx.x & 1)) *(uint32_t*)(base + (size_t)unit * 512 + n * 8 + (p >> 4) * 4) = w;
  } else if (ok) {
    if constexpr (KV == CHONK_KV_Q8)
      *(uint32_t*)(base + (size_t)unit * 1024 + n * 16 + (p >> 4) * 8 + (i0 & 7)) = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
    else
      *(uint2*)(base + (size_t)unit * 2048 + (p >> 4) * 1024 + n * 16 + (i0 & 7) * 2) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
  }
}
// V of position j, dims d0 .. d0 + 3: places of their own, 16 bytes (4 bits: 8) apart. (Four
// positions gathered first, a prompt's bytes went out four in a store, a quarter of the stores:
// 18.6 us instead of 17.8 for 2047 rows of 24 heads x 128 in 8 bits, for the gathering.)
template <int KV>
__device__ __forceinline__ void put_v(uint8_t* base, int hd, int j, int d0, const uint32_t (&c)[4], bool ok) {
  const int unit = (j / 32) * (hd / 32) + d0 / 32, p = j & 31, i0 = d0 & 31, n = v_piece(p, i0), e = place_of(p) & 7;
  if constexpr (KV == CHONK_KV_F16) {
    uint16_t* o = (uint16_t*)(base + (size_t)unit * 2048 + (i0 >> 4) * 1024) + n * 8 + e;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (ok) o[8 * i] = (uint16_t)c[i];
  } else {
    uint32_t w = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
    uint8_t* o;
    if constexpr (KV == CHONK_KV_Q8) {
      o = base + (size_t)unit * 1024 + n * 16 + (i0 >> 4) * 8 + e;
    } else {
      w |= __shfl_xor(w, 4) << 4;  // dims + 16: the lane four on
      ok = ok && !(threadIdx.x & 4);
      o = base + (size_t)unit * 512 + n * 8 + e;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (ok) o[(KV == CHONK_KV_Q8 ? 16 : 8) * i] = (uint8_t)(w >> (8 * i));
  }
}

// Four consecutive elements of a row.
template <bool F16>
__device__ __forceinline__ void row4(const PartSum& P, const _Float16* p16, int64_t ld, int r, int col, float (&v)[4]) {
  if constexpr (F16) {
    const h4u_t x = *(const h4u_t*)(p16 + r * ld + col);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)x[i];
  } else {
    const float* p = P.p + r * ld + col;
    const f4u_t x = *(const f4u_t*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x[i];
    for (int z = 1; z < P.ks; ++z) {
      const f4u_t w = *(const f4u_t*)(p + z * P.zs);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += w[i];
    }
  }
}

// A workgroup takes 32 / NB consecutive rows, 8 NB lanes a row with four dims a lane,
// and walks a range of their slots (q heads, then K's heads, then V's): a row's place, its page
// and its angles are fetched once, not once a head, and the next slot's values are on
// their way while one is worked on. (A slot a workgroup, a 2047-row prompt of 16 + 8 heads x
// 128 took 22 us, most of it three dependent trips to memory for each of 32000 waves.)
// Every product and sum after the norm's is rounded by itself (no fused multiply-add)
// and the norm's sum of squares is taken in 64 bits: the codes do not depend on which
// path (prompt rows or single tokens) wrote them.
// Measured: 17.7 us for 2047 rows of 16 + 8 + 8 heads x 128 fp32 to 8 bits (34 MB read, 21 MB
// written, 3.1 of the 4.7 TB/s that a large copy makes: V's codes leave a byte at a time), 4 to
// 4.5 us for up to 64 rows, of which a launch and its dependent trips to memory are all.
template <int KV, bool F16, int NB>
__global__ __launch_bounds__(kWg) void k_kv_append(KvAppendArgs a) {
#pragma clang fp contract(off)
  constexpr int L = 8 * NB, R = kWg / L, HD = 32 * NB, PART = kv_part_bytes(KV, HD);
  __shared__ __align__(16) float xs[kWg * 4];
  const int tid = threadIdx.x, d0 = (tid & (L - 1)) * 4, row = tid / L;
  const int qh = (F16 ? a.q16 != nullptr : a.q.p != nullptr) ? a.heads : 0, kvh = a.c.kv_heads, slots = qh + 2 * kvh;
  const int per = (slots + gridDim.y - 1) / gridDim.y, from = blockIdx.y * per, to = min(from + per, slots);
  const int r = min((int)blockIdx.x * R + row, a.rows - 1);
  const bool in = (int)blockIdx.x * R + row < a.rows;
  auto fetch = [&](int slot, float (&y)[4]) {
    const bool is_q = slot < qh, is_v = slot >= qh + kvh;
    const int h = is_q ? slot : is_v ? slot - qh - kvh : slot - qh;
    row4<F16>(is_q ? a.q : is_v ? a.v : a.k, is_q ? a.q16 : is_v ? a.v16 : a.k16, is_q ? a.q_ld : is_v ? a.v_ld : a.k_ld, r,
              h * HD + d0, y);
  };
  const int seq = a.at.seq ? a.at.seq[r] : a.at.seq0, pos = a.at.pos ? a.at.pos[r] : a.at.p0 + r;
  float y[4], ahead[4];
  if (from < to) fetch(from, ahead);
  f4u_t wq = f4u_t{1.f, 1.f, 1.f, 1.f}, wk = wq;
  if (a.qn_w) wq = *(const f4u_t*)(a.qn_w + d0);
  if (a.kn_w) wk = *(const f4u_t*)(a.kn_w + d0);
  // where the row goes; one that names no place goes nowhere
  int page = 0;
  bool ok = in && seq >= 0;
  if (ok) {
    page = page_of(a.c, seq, pos, d0 == 0);
    ok = page >= 0;
    if (ok && a.rope && pos >= a.rope_n) {
      if (d0 == 0) fault(a.c, KVF_POS);
      ok = false;
    }
  }
  // the lane's dims' angles, and where the other of each pair is
  float2 cs[4];
  int other[4];
  const int half = a.rope_dim / 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = d0 + i;
    const bool turned = a.rope && d < a.rope_dim;
    const int pair = !turned ? 0 : a.interleaved ? d >> 1 : d < half ? d : d - half;
    other[i] = !turned ? -1 : a.interleaved ? d ^ 1 : d < half ? d + half : d - half;
    cs[i] = turned && ok ? a.rope[(size_t)pos * half + pair] : make_float2(1.f, 0.f);
  }
  const int j = pos & (kKvPage - 1);

  for (int slot = from; slot < to; ++slot) {
    const bool is_q = slot < qh, is_v = slot >= qh + kvh;
    const int h = is_q ? slot : is_v ? slot - qh - kvh : slot - qh;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = ahead[i];
    if (slot + 1 < to) fetch(slot + 1, ahead);
    if (is_q ? a.qn_w != nullptr : !is_v && a.kn_w != nullptr) {
      const f4u_t w = is_q ? wq : wk;
      double sq = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sq += (double)y[i] * (double)y[i];
      sq = lanes_sum<L>(sq);
      const float inv = (float)rsqrt(sq * (1.0 / HD) + a.eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = y[i] * inv * w[i];
    }
    if (a.rope && !is_v) {
      float x[4];
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = y[i ^ 1];
      } else {  // other lanes' dims
        *(float4*)(xs + 4 * tid) = make_float4(y[0], y[1], y[2], y[3]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = xs[4 * tid - d0 + max(other[i], 0)];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (other[i] >= 0)
          y[i] = other[i] < d0 + i ? x[i] * cs[i].y + y[i] * cs[i].x : y[i] * cs[i].x - x[i] * cs[i].y;
    }
    if (is_q) {
      const int64_t o = r * a.qo_ld + h * HD + d0;
      if (!ok) continue;
      if constexpr (F16)
        *(h4u_t*)((_Float16*)a.q_out + o) = h4u_t{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
      else
        *(f4u_t*)((float*)a.q_out + o) = f4u_t{y[0], y[1], y[2], y[3]};
      continue;
    }
    uint8_t* base = a.c.pages + (((size_t)page * kvh + h) * 2 + (is_v ? 1 : 0)) * PART;
    uint32_t c[4], d = 0;
    stored4<KV>(y, c, d);
    if (KV != CHONK_KV_F16 && ok && (d0 & 31) == 0)
      ((uint16_t*)(base + kv_code_bytes(KV, HD)))[((j / 32) * NB + d0 / 32) * 32 + place_of(j & 31)] = (uint16_t)d;
    if (is_v)
      put_v<KV>(base, HD, j, d0, c, ok);
    else
      put_k<KV>(base, HD, j, d0, c, ok);
  }
}

// ---- reading back -----------------------------------------------------------------

// Eight dims of a row's place in `page`.
template <int KV, bool F16>
__device__ __forceinline__ void read8(const KvReadArgs& a, int r, int kv, int d0, int page, int pos) {
  const int hd = a.c.hd;
  const int part = kv_part_bytes(KV, hd), j = pos & (kKvPage - 1), p = j & 31, pl = place_of(p);
  const int unit = (j / 32) * (hd / 32) + d0 / 32, i0 = d0 & 31;
  const uint8_t* base = a.c.pages + ((size_t)page * a.c.kv_heads + kv) * 2 * part;
  const int64_t o = r * a.row_ld + kv * a.head_ld + d0;
#pragma unroll
  for (int is_v = 0; is_v < 2; ++is_v) {
    void* out = is_v ? a.v : a.k;
    if (!out) continue;
    const uint8_t* src = base + is_v * part;
    float x[8];
    const int nk = k_piece(p, i0), nv = v_piece(p, i0);
    if constexpr (KV == CHONK_KV_F16) {
      const _Float16* h = (const _Float16*)src + (size_t)unit * 1024;
      const h8_t k = __builtin_bit_cast(h8_t, ldg4(h + (p >> 4) * 512 + nk * 8));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)(is_v ? h[(i0 >> 4) * 512 + (nv + i) * 8 + (pl & 7)] : k[i]);
    } else {
      const float d = h2f(((const uint16_t*)(src + kv_code_bytes(KV, hd)))[unit * 32 + pl]);
      uint32_t c[8];
      if constexpr (KV == CHONK_KV_Q8) {
        const uint8_t* q = src + (size_t)unit * 1024;
        const uint2 k = ldg2(q + nk * 16 + (p >> 4) * 8);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          c[i] = is_v ? q[(nv + i) * 16 + (i0 >> 4) * 8 + (pl & 7)] : (i < 4 ? k.x : k.y) >> (8 * (i & 3)) & 255;
      } else {
        const uint8_t* q = src + (size_t)unit * 512;
        const uint32_t k = ldg1(q + nk * 8 + (p >> 4) * 4);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          c[i] = is_v ? q[(nv + i) * 8 + (pl & 7)] >> (i0 >> 4 ? 4 : 0) & 15 : k >> (8 * (i & 3) + 4 * (i >> 2)) & 15;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)((int)c[i] - (KV == CHONK_KV_Q8 ? 128 : 8)) * d;
    }
    if constexpr (F16) {
#pragma unroll
      for (int i = 0; i < 8; i += 4)
        *(h4u_t*)((_Float16*)out + o + i) = h4u_t{(_Float16)x[i], (_Float16)x[i + 1], (_Float16)x[i + 2], (_Float16)x[i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += 4) *(f4u_t*)((float*)out + o + i) = f4u_t{x[i], x[i + 1], x[i + 2], x[i + 3]};
    }
  }
}

// Byte (or nibble pair) k of a piece's words.
__device__ __forceinline__ int byte_of(uint32_t w, int k) { return (int)(w >> (8 * k) & 0xff); }

// A wave per (32 rows, kv head, block of 32 dims). Rows that are a half page's
// positions (what a prompt's and a history's are, but at its ends) are read in the pages' own
// order, a unit of 1 KiB (8 bits) at a time, and leave in whole 64-byte pieces; others
// one by one. The rows' groups start where row 0's half page does.
// Bound by the bytes: 25 to 27 us for 11003 positions of 8 heads x 128 from 8 bits to fp32, 114
// MB, 4.2 to 4.5 TB/s (a large copy makes 4.7; 20 us where the last cache still holds the memory
// that the results go to); 3 us for one row.
template <int KV, bool F16>
__global__ __launch_bounds__(kWg) void k_kv_read(KvReadArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hd = a.c.hd, nb = hd / 32;
  const int shift = (a.at.pos ? a.at.pos[0] : a.at.p0) & 31;
  const int groups = (a.rows + shift + 31) / 32;
  // (kv heads and blocks before rows: a row's pieces are written close in time)
  const uint32_t task = blockIdx.x * 4 + wave, per = (uint32_t)(a.c.kv_heads * nb);
  const int grp = (int)(task / per), it = (int)(task % per), kv = it / nb, b = it % nb;
  if (grp >= groups) return;
  const int r0 = grp * 32 - shift, r = r0 + (lane & 31);
  const bool in = r >= 0 && r < a.rows;
  const int rc = min(max(r, 0), a.rows - 1);
  const int seq = a.at.seq ? a.at.seq[rc] : a.at.seq0, pos = a.at.pos ? a.at.pos[rc] : a.at.p0 + rc;
  // the half page that the first of the group's rows would make it
  const int first = __builtin_ctzll(__ballot(in));
  const int s0 = __builtin_amdgcn_readlane(seq, first), p0 = __builtin_amdgcn_readlane(pos, first) - first;
  const bool odd = in && (seq != s0 || pos != p0 + (lane & 31));
  if (__ballot(odd) || (p0 & 31) || p0 < 0 || s0 < 0) {
    // two lanes a row, 16 of the block's dims each
    if (!in || seq < 0) return;
    const int page = page_of(a.c, seq, pos, it == 0 && lane < 32);
    if (page < 0) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) read8<KV, F16>(a, r, kv, 32 * b + 16 * (lane >> 5) + 8 * i, page, pos);
    return;
  }
  const int page = page_of(a.c, s0, p0, lane == 0);
  if (page < 0) return;
  const int part = kv_part_bytes(KV, hd), u = p0 / 32 & 1, unit = u * nb + b, g = lane >> 4, i = lane & 15;
  const uint8_t* base = a.c.pages + ((size_t)page * a.c.kv_heads + kv) * 2 * part;
  const int64_t o = r0 * a.row_ld + kv * a.head_ld + 32 * b;  // (of the group's row 0, which may lie before the first)
  constexpr int W = KV == CHONK_KV_F16 ? 8 : KV == CHONK_KV_Q8 ? 4 : 2;
  uint32_t w[2][W];
  uint4 dk[2];
  uint32_t ds[2];
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const uint8_t* src = base + v * part + (size_t)unit * (256 * W);
    if constexpr (KV == CHONK_KV_Q4) {
      const uint2 x = ldg2(src + lane * 8);
      w[v][0] = x.x, w[v][1] = x.y;
    } else {
#pragma unroll
      for (int t = 0; t < W / 4; ++t) {
        const uint4 x = ldg4(src + t * 1024 + lane * 16);
        w[v][4 * t] = x.x, w[v][4 * t + 1] = x.y, w[v][4 * t + 2] = x.z, w[v][4 * t + 3] = x.w;
      }
    }
    if constexpr (KV != CHONK_KV_F16) {
      const uint8_t* s = base + v * part + kv_code_bytes(KV, hd) + unit * 64;
      if (v) {
        dk[1] = ldg4(s + g * 16);  // V: of the lane's eight positions
      } else {                     // K: of positions i and 16 + i
        ds[0] = ((const uint16_t*)s)[place_of(i)];
        ds[1] = ((const uint16_t*)s)[place_of(16 + i)];
      }
    }
  }
  if (a.k) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (KV == CHONK_KV_F16)
          x[e] = h2f(w[0][4 * t + e / 2] >> (16 * (e & 1)));
        else if constexpr (KV == CHONK_KV_Q8)
          x[e] = (float)(byte_of(w[0][2 * t + e / 4], e & 3) - 128) * h2f(ds[t]);
        else
          x[e] = (float)((int)(w[0][t] >> (8 * (e & 3) + 4 * (e >> 2)) & 15) - 8) * h2f(ds[t]);
      }
      const int rr = r0 + 16 * t + i;
      if (rr < 0 || rr >= a.rows) continue;
      const int64_t at = o + (16 * t + i) * a.row_ld + 8 * g;
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        if constexpr (F16)
          *(h4u_t*)((_Float16*)a.k + at + e) =
              h4u_t{(_Float16)x[e], (_Float16)x[e + 1], (_Float16)x[e + 2], (_Float16)x[e + 3]};
        else
          *(f4u_t*)((float*)a.k + at + e) = f4u_t{x[e], x[e + 1], x[e + 2], x[e + 3]};
      }
    }
  }
  if (a.v) {
    const uint32_t dw[4] = {dk[1].x, dk[1].y, dk[1].z, dk[1].w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = 4 * g + (e & 3) + 16 * (e >> 2), rr = r0 + j;
      const float d = KV == CHONK_KV_F16 ? 1.f : h2f(dw[e / 2] >> (16 * (e & 1)));
      float x[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (KV == CHONK_KV_F16)
          x[h] = h2f(w[1][4 * h + e / 2] >> (16 * (e & 1)));
        else if constexpr (KV == CHONK_KV_Q8)
          x[h] = (float)(byte_of(w[1][2 * h + e / 4], e & 3) - 128) * d;
        else
          x[h] = (float)((int)(w[1][e / 4] >> (8 * (e & 3) + 4 * h) & 15) - 8) * d;
      }
      const int64_t at = o + j * a.row_ld + i;
      if constexpr (F16) {
        // neighbours trade halves, so that each stores two dims together: the even lane
        // those of the block's first 16, the odd lane those of its last
        const uint32_t mine = (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)x[0]) |
                              (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)x[1]) << 16;
        const uint32_t its = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mine, 0xb1, 0xf, 0xf, false);
        const uint32_t two = __builtin_amdgcn_perm(its, mine, i & 1 ? 0x03020706u : 0x05040100u);
        if (rr < 0 || rr >= a.rows) continue;
        typedef uint32_t u1_t __attribute__((aligned(2)));
        *(u1_t*)((_Float16*)a.v + at + (i & 1 ? 15 : 0)) = two;
      } else {
        if (rr < 0 || rr >= a.rows) continue;
        ((float*)a.v)[at] = x[0];
        ((float*)a.v)[at + 16] = x[1];
      }
    }
  }
}

// ---- attention --------------------------------------------------------------------

// Codes become exact fp16 operands two at a time: put under the exponent of 1024,
// where the last bit counts 1 (bytes by v_perm beside 0x64, nibbles by an and with an
// or; 16 times the code for high nibbles), and 1024 and the bias subtracted, exactly.
// Bytes 0 and 2 of a word share a register, and 1 and 3, so the order of eight is
// (0, 2, 1, 3, 4, 6, 5, 7): both products take their k in that order.
// (As denormals, one operation for two codes, the matrix unit takes them too; but it
// aligns such a product by the exponent 2^-14 that denormals share, and a code of b bits
// loses 10 - b of the product's 24: results were off by 1e-5 with 4 bits and by
// 2.5e-6 instead of 9e-7 with 8, and no call was faster.)
__device__ __forceinline__ uint32_t less2(uint32_t v, uint32_t k) {
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, v) - __builtin_bit_cast(h2_t, k));
}
__device__ __forceinline__ uint32_t even_bytes(uint32_t w) {
  return less2(__builtin_amdgcn_perm(0x64646464u, w, 0x04020400u), 0x64806480u);
}
__device__ __forceinline__ uint32_t odd_bytes(uint32_t w) {
  return less2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030401u), 0x64806480u);
}
__device__ __forceinline__ uint32_t low_nibbles(uint32_t w) {
  uint32_t e = 0x64006400u;
  asm("" : "+v"(e));  // (a register: with two literals the and and the or would be two instructions)
  return less2((w & 0x000f000fu) | e, 0x64086408u);
}
__device__ __forceinline__ uint32_t high_nibbles(uint32_t w) {
  uint32_t e = 0x64006400u;
  asm("" : "+v"(e));
  return less2((w & 0x00f000f0u) | e, 0x64806480u);
}
__device__ __forceinline__ h8_t halves(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(h8_t, u32x4_t{a, b, c, d});
}

template <int KV>
constexpr int kOrder(int e) {  // element e of an operand's k: which of the eight
  if (KV == CHONK_KV_F16) return e;
  constexpr int o[8] = {0, 2, 1, 3, 4, 6, 5, 7};
  return o[e];
}

// One half page (32 positions) of a head's K or V in a lane's registers.
template <int KV, int NB>
struct Codes {
  static constexpr int kWords = KV == CHONK_KV_F16 ? 8 : KV == CHONK_KV_Q8 ? 4 : 2;  // a block
  uint32_t w[NB * kWords];
  uint32_t d[NB == 8 ? 2 : 1];  // the half's scales, two (four) of its 32 NB a lane

  __device__ __forceinline__ void load(const uint8_t* part, int u, int lane) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint8_t* unit = part + (u * NB + b) * (kv_code_bytes(KV, 32) / 2);
      if constexpr (KV == CHONK_KV_Q4) {
        const uint2 x = ldg2(unit + lane * 8);
        w[2 * b] = x.x, w[2 * b + 1] = x.y;
      } else {
#pragma unroll
        for (int t = 0; t < kWords / 4; ++t) {
          const uint4 x = ldg4(unit + t * 1024 + lane * 16);
          w[kWords * b + 4 * t] = x.x, w[kWords * b + 4 * t + 1] = x.y;
          w[kWords * b + 4 * t + 2] = x.z, w[kWords * b + 4 * t + 3] = x.w;
        }
      }
    }
  }
  // (apart, and asked for first: the half page's work begins with them)
  __device__ __forceinline__ void load_scales(const uint8_t* part, int u, int lane) {
    if constexpr (KV != CHONK_KV_F16) {
      const uint8_t* s = part + kv_code_bytes(KV, 32 * NB) + u * NB * 64;
      if constexpr (NB == 8) {
        const uint2 x = ldg2(s + lane * 8);
        d[0] = x.x, d[1] = x.y;
      } else {
        d[0] = ldg1(s + (lane & (NB * 16 - 1)) * 4);
      }
    }
  }
  // The A operands of block b: K's two tiles of 16 positions, V's two of 16 dims.
  // High nibbles are 16 times their code.
  __device__ __forceinline__ void k_tiles(int b, h8_t& a0, h8_t& a1) const {
    const uint32_t* x = w + kWords * b;
    if constexpr (KV == CHONK_KV_F16) {
      a0 = halves(x[0], x[1], x[2], x[3]);
      a1 = halves(x[4], x[5], x[6], x[7]);
    } else if constexpr (KV == CHONK_KV_Q8) {
      a0 = halves(even_bytes(x[0]), odd_bytes(x[0]), even_bytes(x[1]), odd_bytes(x[1]));
      a1 = halves(even_bytes(x[2]), odd_bytes(x[2]), even_bytes(x[3]), odd_bytes(x[3]));
    } else {
      const uint32_t y0 = x[0] >> 8, y1 = x[1] >> 8;
      a0 = halves(low_nibbles(x[0]), low_nibbles(y0), high_nibbles(x[0]), high_nibbles(y0));
      a1 = halves(low_nibbles(x[1]), low_nibbles(y1), high_nibbles(x[1]), high_nibbles(y1));
    }
  }
  __device__ __forceinline__ void v_tiles(int b, h8_t& a0, h8_t& a1) const {
    if constexpr (KV == CHONK_KV_Q4) {
      const uint32_t* x = w + kWords * b;
      const uint32_t y0 = x[0] >> 8, y1 = x[1] >> 8;
      a0 = halves(low_nibbles(x[0]), low_nibbles(y0), low_nibbles(x[1]), low_nibbles(y1));
      a1 = halves(high_nibbles(x[0]), high_nibbles(y0), high_nibbles(x[1]), high_nibbles(y1));
    } else {
      k_tiles(b, a0, a1);
    }
  }
};

// A row's visible positions, as half pages.
struct Span {
  int seq, len, first, h0, h1;
  bool bad;
  __device__ __forceinline__ Span(const KvAttendArgs& a, int seq_, int len_, bool note) : seq(seq_), len(len_ + a.len_add) {
    bad = seq >= 0 && len > 0 && (seq >= a.c.n_seqs || len > a.c.max_pages * kKvPage);
    if (bad && note) fault(a.c, seq >= a.c.n_seqs ? KVF_SEQ : KVF_POS);
    if (bad || seq < 0) len = 0;
    len = max(len, 0);
    first = a.window > 0 ? max(0, len - a.window) : 0;
    h0 = first / 32;
    h1 = (len + 31) / 32;
  }
};

// The rows' cut into segments, the same in every wave: at most `want` segments (at least
// kMinHalves long) of about as many halves each, found from all the rows' lengths, so that
// ragged rows keep the device as evenly busy as equal ones and the host needs to know no
// length. Rows none of which is long, and many of like length (the longest within 1.5 times the
// mean), stay whole. A lane looks at rows 4 lane .. 4 lane + 3 (at most 256 rows). The row
// that `mine` holds for comes back in all lanes (row -1: none).
struct Cut {
  int row, seq, len, before, segs;  // segments of the rows before it (an item each), segments of its items
};
template <class F>
__device__ __forceinline__ Cut cut_rows(const KvAttendArgs& a, int items, F mine) {
  constexpr int R = 4;
  const int lane = threadIdx.x & 63, r0 = R * lane;
  int seq[R], len[R], n[R], sum = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = min(r0 + i, a.rows - 1);
    seq[i] = a.seq[r];
    len[i] = a.len[r];
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const Span s(a, seq[i], len[i], false);
    n[i] = r0 + i < a.rows ? s.h1 - s.h0 : 0;
  }
  // The shortest length of a segment that leaves at most `want` of them: between an
  // even share and what must do (every item's last segment may be short), by halving. As
  // floats: whatever the length, the segments it gives are the same in every wave.
  float total = 0.f, longest = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    total += (float)n[i];
    longest = fmaxf(longest, (float)n[i]);
  }
  total = wave_sum(total) * (float)items;
  longest = wave_max(longest);
  const float want = (float)a.want;
  float lo = total / want, hi = total / (want - (float)(a.rows * items)) * 1.0001f + 1.f;
  auto pieces = [&](int i, float most) { return r0 + i < a.rows ? max(1, (int)ceilf((float)n[i] / most)) : 0; };
  const bool whole = longest <= (float)a.whole || (a.many && longest * (float)(a.rows * items) <= 1.5f * total);
  if (whole) {
    hi = fmaxf(longest, 1.f);
  } else if (hi > (float)kMinHalves) {
    for (int k = 0; k < 4; ++k) {
      const float mid = 0.5f * (lo + hi);
      int t = 0;
#pragma unroll
      for (int i = 0; i < R; ++i) t += pieces(i, mid);
      if (wave_sum((float)t) * (float)items <= want)
        hi = mid;
      else
        lo = mid;
    }
  }
  const float most = fmaxf(hi, (float)kMinHalves);
  int segs[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    segs[i] = pieces(i, most);
    sum += segs[i];
  }
  int before = sum;
#pragma unroll
  for (int x = 1; x < 64; x *= 2) {
    const int o = __shfl_up(before, x);
    if (lane >= x) before += o;
  }
  before -= sum;
  Cut c{-1, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (r0 + i < a.rows && mine(r0 + i, before, segs[i])) c = Cut{r0 + i, seq[i], len[i], before, segs[i]};
    before += segs[i];
  }
  const uint64_t found = __ballot(c.row >= 0);
  if (!found) return Cut{-1, 0, 0, 0, 0};
  const int at = __builtin_ctzll(found);
  return Cut{__builtin_amdgcn_readlane(c.row, at), __builtin_amdgcn_readlane(c.seq, at),
             __builtin_amdgcn_readlane(c.len, at), __builtin_amdgcn_readlane(c.before, at),
             __builtin_amdgcn_readlane(c.segs, at)};
}

// The maximum over the 16 lanes of a row, a step an instruction. (Through the compiler a
// step is a move, two quietings of NaNs and the maximum. A lane's value may not be
// read across lanes for two cycles after it is written: hence the waits.)
__device__ __forceinline__ float row_max(float v) {
  asm("s_nop 1\n\tv_max_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_mirror row_mask:0xf bank_mask:0xf"
      : "+v"(v));
  return v;
}
// The larger of the two, and of the magnitudes of packed halves (their bits grow with them).
__device__ __forceinline__ uint32_t top2(uint32_t a, uint32_t b) {
  typedef unsigned short s2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s2_t, a), __builtin_bit_cast(s2_t, b)));
}
// fp16's exponent field of the largest of a lane's V scales (NaN and infinities as the largest
// finite one): the scale is below 2^(field - 14)
__device__ __forceinline__ float scale_field(uint32_t w) {
  const uint32_t x = max(w & 0x7fffu, w >> 16 & 0x7fffu);
  return (float)min(x >> 10, 30u);
}

// w * half H of d: the sum with 0 makes it one mixed instruction. (Not in asm: w
// comes from an exponential, whose result the next instruction cannot take
// without a wait that the compiler sees to.)
template <int H>
__device__ __forceinline__ float mul_half(float w, uint32_t d) {
  return fmaf((float)__builtin_bit_cast(h2_t, d)[H], w, 0.f);
}
// w less half H of h, in one instruction. h is a conversion's result, w that or what the
// conversion took, so neither is an exponential's fresh one.
template <int H>
__device__ __forceinline__ float less_half(float w, uint32_t h) {
  float o;
  if constexpr (H == 0)
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(o) : "v"(h), "v"(w));
  else
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(o) : "v"(h), "v"(w));
  return o;
}
// Two weights as fp16 pairs hi + lo (22 bits; both cut, the second from what the first leaves).
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
  lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(less_half<0>(x, hi), less_half<1>(y, hi)));
}

// Where a split call keeps each row's segments and its first one's workgroup: behind
// the segments' rows and their (maximum, sum).
__device__ __forceinline__ int* cuts(const KvAttendArgs& a, int nhm) {
  return (int*)(a.part + (int64_t)a.want * nhm * (a.c.hd + 2));
}

// One workgroup per segment of a (row, kv head, up to 16 of its q heads); its
// NW waves take the segment's half pages in turn, each with its own running
// maximum, sum and output, and meet in LDS at the end.
//
// q and the weights are split into two fp16 halves each, hi + lo. With more than four heads
// that is two products. PACK (at most four heads): the products have 16 columns for
// them, so columns 0 .. 3 take the heads' hi and 4 .. 7 their lo in one product (8 .. 15 a copy);
// and as what is done to the scores between the products (exponentials, weights times
// V's scales, their split) would be done on all 16, the scores of a half page, 4 heads
// x 32 positions, go through LDS to two a lane, and the split weights back. Half the
// products and a third fewer vector instructions.
//
// Bound by the pages' bytes where rows are long: 32 rows of up to 16k positions of 8 heads x 128 in
// 4 bits take 67 us for 302 MB, 4.5 of the 4.7 TB/s that a large copy makes; one row of 41k in 8
// bits 20 us for 89 MB, 4.4 TB/s. Short rows are bound by the chain of dependent trips to memory
// (length, page id, K and V, for split rows the cut before it): 5.2 us for one of 301 x 3 heads x 64.
template <int KV, int NB, bool PACK, int NW>
__global__ __launch_bounds__(64 * NW, NB == 8 || (NB == 4 && (NW == 8 || (KV == CHONK_KV_F16 && !PACK))) ? 2 : NB == 4 ? 3 : 4) void k_kv_attend(KvAttendArgs a) {
  constexpr int HD = 32 * NB, PART = kv_part_bytes(KV, HD), WG = 64 * NW;
  constexpr bool F = KV == CHONK_KV_F16;
  constexpr int WB = F ? 1 : NB;            // blocks with weights of their own
  // What registers cannot hold beside K and V of a half page and the output: q's halves
  // go to LDS, and fp16's 256-wide rows are fetched one of K and V at a time.
  constexpr bool QL = NB == 8 || (NB == 4 && KV != CHONK_KV_Q4 && !PACK);
  constexpr int QP = PACK ? 1 : 2;          // halves of q that a lane holds
  constexpr bool ONE = F && NB == 8;
  extern __shared__ __align__(16) float sm[];  // [wave][head][HD] | [wave][head][m, l]
  __shared__ __align__(16) uint32_t sck[NW][F ? 4 : NB * 16];          // K's scales, as stored
  __shared__ __align__(16) uint32_t scv[NW][F ? 4 : NB * 16];          // V's (PACK: [pair][block])
  __shared__ __align__(16) float ss[NW][PACK ? 8 * 32 : 4];            // scores [column][place]
  __shared__ __align__(16) uint32_t sw[NW][PACK ? WB * 2 * 64 : 4];    // weights [block][hi, lo][head][16 pairs]
  __shared__ __align__(16) uint32_t sq[QL ? NB * QP * 64 * 4 : 4];
  const int G = a.heads / a.c.kv_heads, hgs = (G + 15) / 16, items = a.c.kv_heads * hgs;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15;
  int r, it, seq, len, seg = 0, segs = 1;
  if (a.split) {
    const int id = blockIdx.x;
    const Cut c = cut_rows(a, items, [&](int, int before, int n) { return id >= before * items && id < (before + n) * items; });
    if (c.row < 0) return;
    r = c.row, seq = c.seq, len = c.len, segs = c.segs;
    it = (id - c.before * items) / segs;
    seg = (id - c.before * items) % segs;
    if (it == 0 && seg == 0 && tid == 0) {  // for the join
      int* cut = cuts(a, min(G, 16)) + 2 * r;
      cut[0] = seq < 0 ? 1 : segs;
      cut[1] = id;
    }
  } else {
    r = blockIdx.x / items;
    it = blockIdx.x % items;
    seq = ld_scalar(a.seq + r);
    len = ld_scalar(a.len + r);
  }
  const int kv = it / hgs, hg = it % hgs;
  const int h0 = kv * G + hg * 16, nh = min(16, G - hg * 16);
  // q on its way first (eight dims of each block, in their own order): it hangs on nothing.
  // (`out` may be q: a row's heads are written after the waves that read them have met, or by the join)
  f4u_t qx[NB][2];
  {
    const int64_t o = r * a.q_ld + (int64_t)(h0 + min(PACK ? col & 3 : col, nh - 1)) * HD + 8 * g;
    if (a.f16) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const h8u_t x = *(const h8u_t*)((const _Float16*)a.q + o + 32 * b);
#pragma unroll
        for (int e = 0; e < 8; ++e) qx[b][e / 4][e & 3] = (float)x[e];
      }
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        qx[b][0] = *(const f4u_t*)((const float*)a.q + o + 32 * b);
        qx[b][1] = *(const f4u_t*)((const float*)a.q + o + 32 * b + 4);
      }
    }
  }
  const Span sp(a, seq, len, tid == 0);
  if (sp.seq < 0) return;  // (the join leaves the row alone too)
  const int per = (sp.h1 - sp.h0 + segs - 1) / segs;
  const int to = min(sp.h0 + (seg + 1) * per, sp.h1);
  int hx = sp.h0 + seg * per + wave;

  // The first half page's K and V are on their way before anything else. The pages of
  // the wave's next 64 half pages are one load, an id a lane.
  const int32_t* tab = a.c.table + (size_t)sp.seq * a.c.max_pages;
  const uint8_t* pool = a.c.pages + (size_t)kv * 2 * PART;
  const size_t page_bytes = (size_t)a.c.kv_heads * 2 * PART;
  bool poison = sp.bad;
  int ids = 0, asked = 0;  // half pages asked for so far
  const int hx0 = hx;
  auto next_part = [&]() {
    if ((asked & 63) == 0) {
      const int h = hx0 + (asked + lane) * NW;
      ids = h < to ? tab[h / 2] : 0;
      const bool out = ids < 0 || ids >= a.c.n_pages;
      if (__ballot(out)) {
        if (out) fault(a.c, KVF_PAGE);
        ids = out ? 0 : ids;
        poison = true;
      }
    }
    return pool + (size_t)__builtin_amdgcn_readlane(ids, asked++ & 63) * page_bytes;
  };
  Codes<KV, NB> kc, vc;
  const uint8_t* vnext = nullptr;  // ONE: where the V of K's half page is
  if (hx < to) {
    const uint8_t* p = next_part();
    kc.load_scales(p, hx & 1, lane);
    vc.load_scales(p + PART, hx & 1, lane);
    kc.load(p, hx & 1, lane);
    if constexpr (ONE)
      vnext = p + PART;
    else
      vc.load(p + PART, hx & 1, lane);
  }

  // q: this lane's head at dims 32 b + 8 g + e, scaled by a power of two so that the
  // head's largest lies in [2^13, 2^14) and split into two halves of 11 bits each
  h8_t qr[QL ? 1 : NB][QP];
  float mul;             // score of S in powers of two
  {
    float top = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(qx[b][e / 4][e & 3]));
    float t0, t1;
    swap16(top, t0, t1);
    top = fmaxf(t0, t1);
    swap32(top, t0, t1);
    top = fmaxf(t0, t1);
    // (a power of two of the head's largest, and the sign of the scale, into q: mul is positive)
    const int sh = top > 0.f ? min(13 - ((int)(__float_as_uint(top) >> 23) - 127), 100) : 0;
    mul = a.scale == 0.f ? 1.f : ldexpf(fabsf(a.scale) * 1.44269504f, -sh);
    const float f = a.scale == 0.f ? 0.f : copysignf(ldexpf(1.f, sh), a.scale);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      h8_t hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float part = KV == CHONK_KV_Q4 && e >= 4 ? 0.0625f : 1.f;  // (high nibbles are 16 times their code)
        const int k = kOrder<KV>(e);
        const float y = qx[b][k / 4][k & 3] * f * part;
        hi[e] = (_Float16)y;
        lo[e] = (_Float16)(y - (float)hi[e]);
      }
      if constexpr (PACK) hi = col & 4 ? lo : hi;
      if constexpr (QL) {
        if (wave == 0) {
          *(h8_t*)(sq + (QP * b * 64 + lane) * 4) = hi;
          if constexpr (!PACK) *(h8_t*)(sq + ((QP * b + 1) * 64 + lane) * 4) = lo;
        }
      } else {
        qr[b][0] = hi;
        if constexpr (!PACK) qr[b][1] = lo;
      }
    }
  }
  if constexpr (QL) __syncthreads();

  // With PACK a lane's two scores are head `hc`'s at places pa and pb, the pair
  // pc of the 16 that make up the second product's operand.
  const int hc = lane >> 4, pc = lane & 15;
  const int pa = F ? 2 * pc : 8 * (pc >> 2) + (pc & 1) + 4 * ((pc >> 1) & 1), pb = pa + (F ? 1 : 2);
  if constexpr (PACK) mul = __shfl(mul, hc);

  // m is the reference of the exponents: the running maximum of score (in powers of
  // two) and V scale together, less what keeps weight * scale below 2^14 and its
  // bits above fp16's denormals. (A field is 0 at least, so no weight is above 2^29.)
  float m = -1e30f, l = 0.f;
  f4_t acc[2 * NB];
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) acc[i] = f4_t{0.f, 0.f, 0.f, 0.f};

  for (; hx < to; hx += NW) {
    const int j0 = 32 * hx;
    const bool edge = j0 < sp.first || j0 + 32 > sp.len;
    const bool more = hx + NW < to;
    const uint8_t* next = nullptr;
    if constexpr (!F) {
      constexpr int D = NB == 8 ? 2 : 1;
      if (edge) {  // scales of unseen places may be anything
#pragma unroll
        for (int i = 0; i < D; ++i) {
          const int n = ((D * lane + i) & 15) * 2;  // place of the word's first
          const int j = j0 + 4 * (n >> 3) + (n & 3) + 16 * ((n >> 2) & 1);
          if (j < sp.first || j >= sp.len) vc.d[i] &= 0xffff0000u;
          if (j + 1 < sp.first || j + 1 >= sp.len) vc.d[i] &= 0xffffu;
        }
      }
      // (PACK: the words re-paired as the weights are, (0, 2), (1, 3) of each four)
      if constexpr (NB == 8) {
        *(uint2*)(sck[wave] + 2 * lane) = make_uint2(kc.d[0], kc.d[1]);
        if constexpr (PACK) {
          uint32_t* o = scv[wave] + (2 * lane & 15) * NB + (lane >> 3);
          o[0] = __builtin_amdgcn_perm(vc.d[1], vc.d[0], 0x05040100u);
          o[NB] = __builtin_amdgcn_perm(vc.d[1], vc.d[0], 0x07060302u);
        } else {
          *(uint2*)(scv[wave] + 2 * lane) = make_uint2(vc.d[0], vc.d[1]);
        }
      } else {
        uint32_t v = vc.d[0];
        if constexpr (PACK) {
          const uint32_t w = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false);
          v = __builtin_amdgcn_perm(w, v, lane & 1 ? 0x03020706u : 0x05040100u);
        }
        if (lane < NB * 16) {
          sck[wave][lane] = kc.d[0];
          scv[wave][PACK ? (lane & 15) * NB + (lane >> 4) : lane] = v;
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      h8_t k0, k1;
      kc.k_tiles(b, k0, k1);
      f4_t s0 = f4_t{0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
      for (int i = 0; i < QP; ++i) {
        h8_t q;
        if constexpr (QL)
          q = *(const h8_t*)(sq + ((QP * b + i) * 64 + lane) * 4);
        else
          q = qr[b][i];
        s0 = mfma(k0, q, s0);
        s1 = mfma(k1, q, s1);
      }
      if constexpr (F) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[e] += s0[e];
          s[4 + e] += s1[e];
        }
      } else {
        const h8_t d = *(const h8_t*)(sck[wave] + b * 16 + g * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[e] = fmaf((float)d[e], s0[e], s[e]);
          s[4 + e] = fmaf((float)d[4 + e], s1[e], s[4 + e]);
        }
      }
    }
    // (an even number of halves on: the same half of its page)
    if constexpr (ONE) {
      vc.load(vnext, hx & 1, lane);
    } else if (more) {
      next = next_part();
      kc.load_scales(next, hx & 1, lane);
      vc.load_scales(next + PART, hx & 1, lane);
      kc.load(next, hx & 1, lane);
    }
    if (edge) {
      uint32_t out = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = j0 + 4 * g + (e & 3) + 16 * (e >> 2);
        const bool o = j < sp.first || j >= sp.len;
        out |= (uint32_t)o << e;
        s[e] = o ? -INFINITY : s[e];
      }
      if constexpr (F) {
        uint32_t seen[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) seen[i] = (out >> (2 * i) & 1 ? 0 : 0xffffu) | (out >> (2 * i + 1) & 1 ? 0 : 0xffff0000u);
#pragma unroll
        for (int i = 0; i < NB * 8; ++i) vc.w[i] &= seen[i & 3];
      }
    }
    float s0 = 0.f, s1 = 0.f, top;
    uint32_t dv[NB];
    if constexpr (PACK) {
      if (col < 8) {
        *(float4*)(ss[wave] + col * 32 + 8 * g) = make_float4(s[0], s[1], s[2], s[3]);
        *(float4*)(ss[wave] + col * 32 + 8 * g + 4) = make_float4(s[4], s[5], s[6], s[7]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      s0 = ss[wave][hc * 32 + pa] + ss[wave][(hc + 4) * 32 + pa];
      s1 = ss[wave][hc * 32 + pb] + ss[wave][(hc + 4) * 32 + pb];
      top = fmaxf(s0, s1) * mul;
      if constexpr (!F) {
#pragma unroll
        for (int b = 0; b < NB; ++b) dv[b] = scv[wave][pc * NB + b];
        uint32_t x = dv[0] & 0x7fff7fffu;
#pragma unroll
        for (int b = 1; b < NB; ++b) x = top2(x, dv[b] & 0x7fff7fffu);
        top += scale_field(x);
      }
      top = row_max(top);
    } else {
      top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7]))) * mul;
      if constexpr (!F) {
        uint32_t x = 0;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint4 d = *(const uint4*)(scv[wave] + b * 16 + g * 4);
          x = top2(x, top2(top2(d.x & 0x7fff7fffu, d.y & 0x7fff7fffu), top2(d.z & 0x7fff7fffu, d.w & 0x7fff7fffu)));
        }
        top += scale_field(x);
      }
      float t0, t1;
      swap16(top, t0, t1);
      top = fmaxf(t0, t1);
      swap32(top, t0, t1);
      top = fmaxf(t0, t1);
    }
    // weight < 2^14, or weight * scale < 2^(28 - field + field - 14)
    const float ref = fmaxf(m, top - (F ? 14.f : 28.f));
    if (__ballot(ref != m)) {
      const float f = __builtin_amdgcn_exp2f(m - ref);
      l *= f;
      m = ref;
      const float fa = PACK ? __shfl(f, (col & 3) * 16) : f;
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) acc[i] *= fa;
    }
    float p[PACK ? 2 : 8];
    if constexpr (PACK) {
      p[0] = __builtin_amdgcn_exp2f(fmaf(s0, mul, -m));
      p[1] = __builtin_amdgcn_exp2f(fmaf(s1, mul, -m));
      l += p[0] + p[1];
#pragma unroll
      for (int b = 0; b < WB; ++b) {
        uint32_t hi, lo;
        if constexpr (F)
          split2(p[0], p[1], hi, lo);
        else
          split2(mul_half<0>(p[0], dv[b]), mul_half<1>(p[1], dv[b]), hi, lo);
        sw[wave][2 * b * 64 + lane] = hi;
        sw[wave][(2 * b + 1) * 64 + lane] = lo;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(fmaf(s[e], mul, -m));
        l += p[e];
      }
    }
    [[maybe_unused]] uint32_t ph[4], pl[4];
    if constexpr (F && !PACK) {
#pragma unroll
      for (int i = 0; i < 4; ++i) split2(p[2 * i], p[2 * i + 1], ph[i], pl[i]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      h8_t wh, v0, v1;
      vc.v_tiles(b, v0, v1);
      if constexpr (PACK) {
        wh = *(const h8_t*)(sw[wave] + (2 * (F ? 0 : b) + (col >> 2 & 1)) * 64 + (col & 3) * 16 + 4 * g);
      } else {
        if constexpr (!F) {
          const uint4 d = *(const uint4*)(scv[wave] + b * 16 + g * 4);
          split2(mul_half<0>(p[0], d.x), mul_half<0>(p[2], d.y), ph[0], pl[0]);
          split2(mul_half<1>(p[1], d.x), mul_half<1>(p[3], d.y), ph[1], pl[1]);
          split2(mul_half<0>(p[4], d.z), mul_half<0>(p[6], d.w), ph[2], pl[2]);
          split2(mul_half<1>(p[5], d.z), mul_half<1>(p[7], d.w), ph[3], pl[3]);
        }
        wh = halves(ph[0], ph[1], ph[2], ph[3]);
        const h8_t wl = halves(pl[0], pl[1], pl[2], pl[3]);
        acc[2 * b] = mfma(v0, wl, acc[2 * b]);
        acc[2 * b + 1] = mfma(v1, wl, acc[2 * b + 1]);
      }
      acc[2 * b] = mfma(v0, wh, acc[2 * b]);
      acc[2 * b + 1] = mfma(v1, wh, acc[2 * b + 1]);
    }
    if constexpr (ONE) {
      if (more) {
        next = next_part();
        kc.load(next, hx & 1, lane);
        vnext = next + PART;
      }
    } else if (more) {
      vc.load(next + PART, hx & 1, lane);
    }
  }
  if constexpr (PACK) {
    l = group_sum<16>(l);
    // column c + 4 into column c: the lo weights' share
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] += dpp<0x104>(acc[i][e]);
  } else {
    float t0, t1;
    swap16(l, t0, t1);
    l = t0 + t1;
    swap32(l, t0, t1);
    l = t0 + t1;
  }
  if (poison) l = __builtin_nanf("");
  // the waves' rows meet in LDS
  float* ml = sm + NW * nh * HD;
  if (col < nh) {
    float* o = sm + (wave * nh + col) * HD;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
      // (codes of high nibbles were 16 times themselves)
      const float f = KV == CHONK_KV_Q4 && (i & 1) ? 0.0625f : 1.f;
      *(float4*)(o + 16 * i + 4 * g) = make_float4(acc[i][0] * f, acc[i][1] * f, acc[i][2] * f, acc[i][3] * f);
    }
  }
  if (PACK ? pc == 0 && hc < nh : g == 0 && col < nh) {
    float* o = ml + (wave * nh + (PACK ? hc : col)) * 2;
    o[0] = m;
    o[1] = l;
  }
  __syncthreads();
  const int nhm = min(G, 16);
  float* prow = a.part + (int64_t)blockIdx.x * nhm * HD;
  float* pml = a.part + (int64_t)a.want * nhm * HD + (int64_t)blockIdx.x * nhm * 2;
  for (int x = tid; x < nh * HD; x += WG) {
    const int h = x / HD, d = x % HD;
    float M = -1e30f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, ml[(w * nh + h) * 2]);
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(ml[(w * nh + h) * 2] - M);
      L += f * ml[(w * nh + h) * 2 + 1];
      O += f * sm[(w * nh + h) * HD + d];
    }
    if (segs > 1) {
      prow[x] = O;
      if (d == 0) {
        pml[2 * h] = M;
        pml[2 * h + 1] = L;
      }
    } else {
      const float y = L == 0.f ? 0.f : O / L;
      const int64_t o = r * a.o_ld + (int64_t)(h0 + h) * HD + d;
      if (a.f16)
        ((_Float16*)a.out)[o] = (_Float16)y;
      else
        ((float*)a.out)[o] = y;
    }
  }
}

// Joins a (row, head)'s segments: HD / 4 columns of float4, the segments over
// groups of threads, every group's in order and the groups in order: the result does not
// hang on which workgroup ended first. Bound by its launch and two trips to memory: 3.9 us for 5
// rows of 16 heads x 64, 4.5 for 16 heads x 128 of one row in 96 segments each.
__global__ __launch_bounds__(kWg) void k_kv_join(KvAttendArgs a) {
  __shared__ float wt[kMostWgs];
  __shared__ float red[8];
  __shared__ __align__(16) float so[kWg * 4];
  const int G = a.heads / a.c.kv_heads, hgs = (G + 15) / 16, nhm = min(G, 16);
  const int h = blockIdx.x, r = blockIdx.y, hd = a.c.hd, tid = threadIdx.x;
  const int* cut = cuts(a, nhm) + 2 * r;
  const int segs = ld_scalar(cut), slot = ld_scalar(cut + 1);
  if (segs == 1) return;
  const int it = h / G * hgs + h % G / 16, hh = h % G % 16;
  const int slot0 = slot + it * segs;
  const float* rows = a.part + ((int64_t)slot0 * nhm + hh) * hd;
  const float* ml = a.part + (int64_t)a.want * nhm * hd + ((int64_t)slot0 * nhm + hh) * 2;
  float M = -1e30f;
  for (int s = tid; s < segs; s += kWg) M = fmaxf(M, ml[(int64_t)s * nhm * 2]);
  M = wave_max(M);
  if ((tid & 63) == 0) red[tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float L = 0.f;
  for (int s = tid; s < segs; s += kWg) {
    const float f = __builtin_amdgcn_exp2f(ml[(int64_t)s * nhm * 2] - M);
    wt[s] = f;
    L += f * ml[(int64_t)s * nhm * 2 + 1];
  }
  L = wave_sum(L);
  if ((tid & 63) == 0) red[4 + (tid >> 6)] = L;
  __syncthreads();
  L = (red[4] + red[5]) + (red[6] + red[7]);
  const int cols = hd / 4, c = tid % cols, grp = tid / cols, groups = kWg / cols;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = grp; s < segs; s += groups) {
    const float4 v = ldg4f(rows + (int64_t)s * nhm * hd + 4 * c);
    const float f = wt[s];
    o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
  }
  *(float4*)(so + 4 * tid) = o;
  __syncthreads();
  for (int d = tid; d < hd; d += kWg) {
    float y = 0.f;
    for (int g = 0; g < groups; ++g) y += so[4 * (g * cols) + d];
    y = L == 0.f ? 0.f : y / L;
    const int64_t at = r * a.o_ld + (int64_t)h * hd + d;
    if (a.f16)
      ((_Float16*)a.out)[at] = (_Float16)y;
    else
      ((float*)a.out)[at] = y;
  }
}

int64_t attend_items(const KvCache& c, int rows, int heads) {
  return (int64_t)rows * c.kv_heads * ((heads / c.kv_heads + 15) / 16);
}
// Workgroups of four waves that the registers let the 256 CUs hold at once: segments wanted of
// few (row, head)s (more would wait for a place: 41k positions of 128 dims took 28 us in
// 1024, 22 in 768).
int attend_once(const KvCache& c) { return c.hd >= 256 ? 512 : c.hd == 128 ? 768 : 1024; }
bool attend_many(const KvCache& c, int64_t items) { return items > attend_once(c) / 2; }
// Many of them, which fill half of the device or more as they are: twice that, two segments
// for each at least.
int attend_want(const KvCache& c, int64_t items) { return attend_once(c) * (attend_many(c, items) ? 2 : 1); }
// Half pages up to which rows stay whole: one workgroup walks them in the time of the
// shorter walk and its join. (24 x 12 rows of up to 1024 positions of 64 dims in 8 bits: 11.7 us
// whole, 13.4 + 4.2 cut; 48 rows of 512 positions of 256 dims in fp16: 14.5 whole, 12.8 + 3.9
// cut; 32 x 8 of 640 of 128 dims in 8 bits: 14.1 whole, 18.3 cut.) Many rows longer than that
// share the device well unless their lengths differ (64 x 8 of 128 dims in 4 bits, of up to
// 2048: 29.9 us whole, 34.4 cut; of 1 to 16384: 205 whole, 133 cut).
int attend_whole(const KvCache& c, int64_t items) { return attend_many(c, items) ? 4 * kWholeHalves : kWholeHalves; }
// Whether rows may be cut: the lengths are the device's to know (cut_rows), the table's
// width is known here. (Rows that could have been cut and were not, 64 x 8 of 640: 16.5 us
// instead of 13.7.)
bool attend_splits(const KvCache& c, int rows, int heads, int window) {
  const int64_t most = std::min<int64_t>(2 * (int64_t)c.max_pages, window > 0 ? (int64_t)window / 32 + 2 : INT32_MAX);
  const int64_t items = attend_items(c, rows, heads);
  return rows <= 256 && items <= attend_once(c) && most > attend_whole(c, items);
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t s) {
  const int slots = ((a.f16 ? a.q16 != nullptr : a.q.p != nullptr) ? a.heads : 0) + 2 * a.c.kv_heads;
  // as many ranges of slots as fill the device (2047 rows of 32 heads x 128: 18.6 us in 1024
  // workgroups, 19.1 in 2048, whose rows are fetched again for every range)
  const int groups = (a.rows + kWg / (a.c.hd / 4) - 1) / (kWg / (a.c.hd / 4));
  const dim3 grid(groups, std::max(1, std::min(slots, 1024 / groups)));
#define CHONK_KV_CASE(T, B)                                                                 \
  if (a.c.type == T && a.c.hd == 32 * B) {                                                  \
    if (a.f16)                                                                              \
      hipLaunchKernelGGL((k_kv_append<T, true, B>), grid, dim3(kWg), 0, s, a);              \
    else                                                                                    \
      hipLaunchKernelGGL((k_kv_append<T, false, B>), grid, dim3(kWg), 0, s, a);             \
  } else
#define CHONK_KV_CASES(T) CHONK_KV_CASE(T, 1) CHONK_KV_CASE(T, 2) CHONK_KV_CASE(T, 4) CHONK_KV_CASE(T, 8)
  CHONK_KV_CASES(CHONK_KV_F16)
  CHONK_KV_CASES(CHONK_KV_Q8)
  CHONK_KV_CASES(CHONK_KV_Q4)
  return hipErrorInvalidValue;
#undef CHONK_KV_CASES
#undef CHONK_KV_CASE
  return hipGetLastError();
}

hipError_t launch_kv_read(const KvReadArgs& a, hipStream_t s) {
  // (one group more than the rows fill: where the first half page starts is the device's to know)
  const int64_t waves = ((int64_t)a.rows + 31 + 31) / 32 * a.c.kv_heads * (a.c.hd / 32);
  const dim3 grid((uint32_t)((waves + 3) / 4));
#define CHONK_KV_CASE(T)                                                                \
  case T:                                                                               \
    if (a.f16)                                                                          \
      hipLaunchKernelGGL((k_kv_read<T, true>), grid, dim3(kWg), 0, s, a);               \
    else                                                                                \
      hipLaunchKernelGGL((k_kv_read<T, false>), grid, dim3(kWg), 0, s, a);              \
    return hipGetLastError();
  switch (a.c.type) {
    CHONK_KV_CASE(CHONK_KV_F16)
    CHONK_KV_CASE(CHONK_KV_Q8)
    CHONK_KV_CASE(CHONK_KV_Q4)
    default: return hipErrorInvalidValue;
  }
#undef CHONK_KV_CASE
}

int64_t kv_attend_floats(const KvCache& c, int rows, int heads) {
  return attend_splits(c, rows, heads, 0) ? (int64_t)attend_want(c, attend_items(c, rows, heads)) * std::min(heads / c.kv_heads, 16) * (c.hd + 2) + 2 * rows : 0;
}

hipError_t launch_kv_attend(const KvAttendArgs& a0, hipStream_t s) {
  KvAttendArgs a = a0;
  const int G = a.heads / a.c.kv_heads, nh = std::min(G, 16);
  const int64_t items = attend_items(a.c, a.rows, a.heads);
  a.split = attend_splits(a.c, a.rows, a.heads, a.window) ? 1 : 0;
  a.want = attend_want(a.c, items);
  a.many = attend_many(a.c, items);
  a.whole = attend_whole(a.c, items);
  if (a.split && !a.part) return hipErrorInvalidValue;
  const dim3 grid(a.split ? a.want : (uint32_t)items);
  // whole rows of few workgroups: eight waves each, as long as all of them fit the CUs (a row
  // of 301 positions of 3 heads x 64: 5.2 us, 6.5 with four waves; 64 rows of up to 640 of 8 x
  // 128 need two rounds of the CUs with eight, and are walked in one, 13 us, with four)
  const bool wide = !a.split && items <= (a.c.hd >= 128 ? 256 : 512);
  const size_t sh = (size_t)(wide ? 8 : 4) * nh * (a.c.hd + 2) * 4;
#define CHONK_KV_LAUNCH(T, B, P, W)                                                                      \
  {                                                                                                      \
    if (sh > 32768) {                                                                                    \
      const hipError_t e = hipFuncSetAttribute((const void*)k_kv_attend<T, B, P, W>,                     \
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)sh);     \
      if (e != hipSuccess) return e;                                                                     \
    }                                                                                                    \
    hipLaunchKernelGGL((k_kv_attend<T, B, P, W>), grid, dim3(64 * W), sh, s, a);                         \
  }
#define CHONK_KV_CASE(T, B, P)                                                                           \
  if (a.c.type == T && a.c.hd == 32 * B && P == (nh <= 4)) {                                             \
    if (wide)                                                                                            \
      CHONK_KV_LAUNCH(T, B, P, 8)                                                                        \
    else                                                                                                 \
      CHONK_KV_LAUNCH(T, B, P, 4)                                                                        \
  } else
#define CHONK_KV_CASES(T, P) CHONK_KV_CASE(T, 1, P) CHONK_KV_CASE(T, 2, P) CHONK_KV_CASE(T, 4, P) CHONK_KV_CASE(T, 8, P)
  CHONK_KV_CASES(CHONK_KV_F16, false)
  CHONK_KV_CASES(CHONK_KV_F16, true)
  CHONK_KV_CASES(CHONK_KV_Q8, false)
  CHONK_KV_CASES(CHONK_KV_Q8, true)
  CHONK_KV_CASES(CHONK_KV_Q4, false)
  CHONK_KV_CASES(CHONK_KV_Q4, true)
  return hipErrorInvalidValue;
#undef CHONK_KV_CASES
#undef CHONK_KV_CASE
#undef CHONK_KV_LAUNCH
  if (a.split) hipLaunchKernelGGL(k_kv_join, dim3(a.heads, a.rows), dim3(kWg), 0, s, a);
  return hipGetLastError();
}

}  // namespace chonk

// ---- C entry points -----------------------------------------------------------------

namespace chonk {
namespace {

std::string no(const char* what, long long v) { return std::string(what) + " " + std::to_string(v); }

void check_format(int32_t kv_type, int32_t kv_heads, int32_t head_dim) {
  if (!kv_type_ok(kv_type)) throw Error(CHONK_EINVAL, no("paged K/V cache: unsupported kv type", kv_type));
  if (kv_heads <= 0 || kv_heads > 4096) throw Error(CHONK_EINVAL, no("paged K/V cache: bad kv head count", kv_heads));
  if (!kv_hd_ok(head_dim))
    throw Error(CHONK_EINVAL, no("paged K/V cache: head_dim must be 32, 64, 128 or 256, not", head_dim));
}

KvCache checked(const chonk_kv_cache* c) {
  if (!c) throw Error(CHONK_EINVAL, "null argument");
  check_format(c->kv_type, c->kv_heads, c->head_dim);
  if (c->n_pages <= 0 || c->n_seqs <= 0 || c->max_pages <= 0 || c->max_pages > (1 << 24) || !c->pages || !c->table)
    throw Error(CHONK_EINVAL, "paged K/V cache: empty pool or table");
  if ((uintptr_t)c->pages % 16) throw Error(CHONK_EINVAL, "paged K/V cache: pages must be 16-byte aligned");
  KvCache k{};
  k.pages = (uint8_t*)c->pages;
  k.table = c->table;
  k.fault = c->fault;
  k.type = c->kv_type;
  k.kv_heads = c->kv_heads;
  k.hd = c->head_dim;
  k.n_pages = c->n_pages;
  k.n_seqs = c->n_seqs;
  k.max_pages = c->max_pages;
  return k;
}

void check_heads(int32_t heads, int32_t kv_heads) {
  if (heads <= 0 || heads > 65536 || heads % kv_heads)
    throw Error(CHONK_EINVAL, no("paged K/V cache: query heads must be a multiple of the kv heads, not", heads));
}
// A launch holds fewer than 2^32 threads.
void check_grid(int64_t wgs) {
  if (wgs >= (1 << 24)) throw Error(CHONK_EINVAL, "paged K/V cache: too many rows and heads for one call");
}
void check_rows(int32_t rows) {
  if (rows < 0 || rows > (1 << 22)) throw Error(CHONK_EINVAL, no("paged K/V cache: bad row count", rows));
}
void check_act(int32_t type) {
  if (type != CHONK_F32 && type != CHONK_F16) throw Error(CHONK_EINVAL, no("paged K/V cache: bad element type", type));
}
// Rows must not overlap (a row of a result) or run backwards.
void check_stride(const char* what, int64_t ld, int64_t least) {
  if (ld < least) throw Error(CHONK_EINVAL, std::string("paged K/V cache: ") + what + " rows are closer than their width");
}

// The cache's device for the length of a call.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    HIP_OK(hipGetDevice(&was_));
    if (device != was_) HIP_OK(hipSetDevice(device));
    now_ = device;
  }
  ~OnDevice() {
    if (now_ != was_) (void)hipSetDevice(was_);
  }

 private:
  int was_ = 0, now_ = 0;
};

}  // namespace
}  // namespace chonk

using namespace chonk;

extern "C" {

int64_t chonk_kv_page_bytes(int32_t kv_type, int32_t kv_heads, int32_t head_dim) {
  int64_t n = 0;
  const int rc = api_free([&] {
    check_format(kv_type, kv_heads, head_dim);
    n = (int64_t)kv_heads * 2 * kv_part_bytes(kv_type, head_dim);
  });
  return rc == CHONK_OK ? n : rc;
}

int chonk_kv_append(const chonk_kv_cache* cache, const chonk_kv_rows* rows, const chonk_kv_append_args* x,
                    void* stream) {
  return api_free([&] {
    KvAppendArgs a{};
    a.c = checked(cache);
    if (!rows || !x) throw Error(CHONK_EINVAL, "null argument");
    check_rows(rows->n);
    check_act(x->type);
    if (rows->n == 0) return;
    if (!rows->seq || !rows->pos || !x->k || !x->v) throw Error(CHONK_EINVAL, "null argument");
    const int64_t kvw = (int64_t)a.c.kv_heads * a.c.hd;
    check_stride("k", x->k_stride, kvw);
    check_stride("v", x->v_stride, kvw);
    if (x->q) {
      check_heads(x->heads, a.c.kv_heads);
      if (!x->q_out) throw Error(CHONK_EINVAL, "null argument");
      check_stride("q", x->q_stride, (int64_t)x->heads * a.c.hd);
      check_stride("q_out", x->q_out_stride, (int64_t)x->heads * a.c.hd);
    }
    if (x->rope && (x->rope_dim <= 0 || x->rope_dim > a.c.hd || x->rope_dim % 2 || x->rope_positions <= 0))
      throw Error(CHONK_EINVAL, no("paged K/V cache: rope_dim must be even and at most head_dim, not", x->rope_dim));
    if (x->k_norm || x->q_norm) {
      if (!(x->eps >= 0.0)) throw Error(CHONK_EINVAL, "paged K/V cache: eps must not be negative");
    }
    check_grid((int64_t)rows->n * (a.c.hd / 4) / kWg + 2048);
    a.at.seq = rows->seq;
    a.at.pos = rows->pos;
    a.rows = rows->n;
    a.heads = x->heads;
    a.f16 = x->type == CHONK_F16;
    a.q_ld = x->q_stride;
    a.k_ld = x->k_stride;
    a.v_ld = x->v_stride;
    a.qo_ld = x->q_out_stride;
    a.q_out = x->q_out;
    if (a.f16) {
      a.q16 = (const _Float16*)x->q;
      a.k16 = (const _Float16*)x->k;
      a.v16 = (const _Float16*)x->v;
    } else {
      const void* src[3] = {x->q, x->k, x->v};
      PartSum* dst[3] = {&a.q, &a.k, &a.v};
      for (int i = 0; i < 3; ++i) {
        dst[i]->p = (const float*)src[i];
        dst[i]->ks = 1;
      }
    }
    a.qn_w = x->q_norm;
    a.kn_w = x->k_norm;
    a.eps = x->eps;
    a.rope = (const float2*)x->rope;
    a.rope_dim = x->rope_dim;
    a.rope_n = x->rope_positions;
    a.interleaved = x->interleaved != 0;
    OnDevice on(cache->device);
    HIP_OK(launch_kv_append(a, (hipStream_t)stream));
  });
}

int chonk_kv_read(const chonk_kv_cache* cache, const chonk_kv_rows* rows, int32_t type, void* k, void* v,
                  int64_t row_stride, int64_t head_stride, void* stream) {
  return api_free([&] {
    KvReadArgs a{};
    a.c = checked(cache);
    if (!rows || (!k && !v)) throw Error(CHONK_EINVAL, "null argument");
    check_rows(rows->n);
    check_act(type);
    if (rows->n == 0) return;
    if (!rows->seq || !rows->pos) throw Error(CHONK_EINVAL, "null argument");
    // either order of rows and heads, none inside another
    const int64_t hd = a.c.hd;
    const bool rows_out = head_stride >= hd && row_stride >= (a.c.kv_heads - 1) * head_stride + hd;
    const bool heads_out = row_stride >= hd && head_stride >= (int64_t)(rows->n - 1) * row_stride + hd;
    if (!rows_out && !heads_out) throw Error(CHONK_EINVAL, "paged K/V cache: result rows overlap");
    check_grid(((int64_t)rows->n / 32 + 2) * a.c.kv_heads * (a.c.hd / 32) / 4);
    a.at.seq = rows->seq;
    a.at.pos = rows->pos;
    a.rows = rows->n;
    a.k = k;
    a.v = v;
    a.row_ld = row_stride;
    a.head_ld = head_stride;
    a.f16 = type == CHONK_F16;
    OnDevice on(cache->device);
    HIP_OK(launch_kv_read(a, (hipStream_t)stream));
  });
}

int64_t chonk_kv_attend_workspace(const chonk_kv_cache* cache, int32_t n_rows, int32_t heads) {
  int64_t n = 0;
  const int rc = api_free([&] {
    const KvCache c = checked(cache);
    check_rows(n_rows);
    check_heads(heads, c.kv_heads);
    n = n_rows ? kv_attend_floats(c, n_rows, heads) * 4 : 0;
  });
  return rc == CHONK_OK ? n : rc;
}

int chonk_kv_attend(const chonk_kv_cache* cache, const chonk_kv_attend_args* x, void* stream) {
  return api_free([&] {
    KvAttendArgs a{};
    a.c = checked(cache);
    if (!x) throw Error(CHONK_EINVAL, "null argument");
    check_rows(x->n);
    check_act(x->type);
    check_heads(x->heads, a.c.kv_heads);
    if (x->window < 0) throw Error(CHONK_EINVAL, no("paged K/V cache: bad window", x->window));
    if (x->n == 0) return;
    if (!x->seq || !x->lengths || !x->q || !x->out) throw Error(CHONK_EINVAL, "null argument");
    check_stride("q", x->q_stride, (int64_t)x->heads * a.c.hd);
    check_stride("out", x->out_stride, (int64_t)x->heads * a.c.hd);
    const int G = x->heads / a.c.kv_heads;
    check_grid((int64_t)x->n * a.c.kv_heads * ((G + 15) / 16));
    const int64_t need = kv_attend_floats(a.c, x->n, x->heads) * 4;
    if (need > 0 && (!x->workspace || x->workspace_bytes < need || (uintptr_t)x->workspace % 16))
      throw Error(CHONK_EINVAL, "paged K/V cache: attention needs " + std::to_string(need) +
                                    " bytes of 16-byte aligned workspace, got " + std::to_string(x->workspace_bytes));
    a.seq = x->seq;
    a.len = x->lengths;
    a.q = x->q;
    a.out = x->out;
    a.q_ld = x->q_stride;
    a.o_ld = x->out_stride;
    a.rows = x->n;
    a.heads = x->heads;
    a.f16 = x->type == CHONK_F16;
    a.window = x->window;
    a.scale = x->scale;
    a.part = (float*)x->workspace;
    OnDevice on(cache->device);
    HIP_OK(launch_kv_attend(a, (hipStream_t)stream));
  });
}

}  // extern "C"
