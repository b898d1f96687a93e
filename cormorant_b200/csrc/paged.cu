// The paged KV cache's operators (see the header's section on it): the row
// preparation that norms, rotates and writes, the read-back, and the attention
// of few rows a sequence.
#include "paged.cuh"

#include <atomic>
#include <type_traits>

#include "gemm_i8x4.h"
#include "paged_tile.h"

namespace paged {

int check_cache(const corm_paged_cache* c, const char* what) {
  if (c->B == 0 || c->rows == 0) return CORM_OK;
  if (!c->kc || !c->vc || !c->table || !c->cu || !c->pos) return corm::fail(CORM_EINVAL, "%s: null cache buffer", what);
  if (c->bits != 16 && c->bits != 8) return corm::fail(CORM_EINVAL, "%s: %u bits (16 or 8)", what, c->bits);
  if (c->bits == 8 && (!c->ks || !c->vs)) return corm::fail(CORM_EINVAL, "%s: 8-bit pages without shifts", what);
  if (c->HD != 16 && c->HD != 32 && c->HD != 64 && c->HD != 128 && c->HD != 256)
    return corm::fail(CORM_EINVAL, "%s: HD %u (16, 32, 64, 128 or 256)", what, c->HD);
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128 && c->page != 256)
    return corm::fail(CORM_EINVAL, "%s: page %u (16, 32, 64, 128 or 256)", what, c->page);
  if (c->KV == 0 || c->KV > 65535u || c->B > 65535u)
    return corm::fail(CORM_ELIMIT, "%s: KV %u, B %u (up to 65535)", what, c->KV, c->B);
  if (c->pages > 0x7FFFFFFFu || c->rows > 0x7FFFFFFFu || (uint64_t)c->table_width * c->page > 0x7FFFFFFFull)
    return corm::fail(CORM_ELIMIT, "%s: pages, rows or positions beyond 2^31", what);
  uintptr_t m = (uintptr_t)c->kc | (uintptr_t)c->vc;
  if (c->bits == 8) m |= (uintptr_t)c->ks | (uintptr_t)c->vs;
  if (m & 15u) return corm::fail(CORM_EINVAL, "%s: unaligned pages", what);
  if (((uintptr_t)c->table | (uintptr_t)c->cu | (uintptr_t)c->pos) & 3u)
    return corm::fail(CORM_EINVAL, "%s: unaligned table, cu or pos", what);
  return CORM_OK;
}

}  // namespace paged

namespace {

using namespace paged;

// ---------------------------------------------------------------- preparation
// A warp per row, or per part of a row's heads where there are few rows: HD / 8 lanes
// a head, a lane holding the 8 elements of four pairs, the heads in turns of 256 / HD
// (the rotated ones, then v's).  A row's sequence, page, cosines and sines are looked
// up once for all its heads, and a lane's entries once for all its rows.  Norm: the
// squares' sum by shuffles over the head, the divisor by the unit's table and Newton
// step, 64-bit throughout (D < 2^63, |x Rm| < 2^48, |P1 G| < 2^56).
//
// Bound by its instructions: a rotated element is two wide products and a rounding of
// a 64-bit sum, a third of some 290 instructions a turn (20 k rows x 25 heads of 64: 67
// us, 60% of the issue slots, 2.4 TB/s; a thread per 8 elements of one head, a row looked
// up by each: 113 us).  Three blocks an SM, so 80 registers; the next turn's elements are
// loaded before this one's are worked on, as 24 warps hold too few loads otherwise.
constexpr uint32_t kTurns = 8;  // turns of a part: their entries' forms are a byte each of one word
struct PrepArgs {
  corm_llm_paged_prep_desc d;
  const uint32_t* rsq;
  uint32_t turned, turns, per, parts;  // turns of the rotated heads, of all; a part's; parts of a row
};

// the row-ops unit's 1 / sqrt(D) ~ Rm 2^-sh for 1 <= D < 2^63: Dm = D 2^-d (d even) below
// 2^32 with one of its two top bits, a table's y0 and a Newton step, all in 32 bits but the last
__device__ __forceinline__ void rsqrt64(uint64_t D, uint32_t& Rm, int& sh, const uint32_t* __restrict__ rsq) {
  int d = 32 - __clzll((long long)D);
  if (d & 1) d += 1;
  const uint32_t Dm = (uint32_t)((D << (32 - d)) >> 32);  // (32 - d <= the leading zeros)
  const uint32_t y0 = __ldg(rsq + (Dm >> 19));
  const uint32_t u = __umulhi(__umulhi(Dm, y0), y0);
  // |y0 (2^30 - u)| < 2^62: the table's y0 is within 2^-13 of 1 / sqrt
  const int64_t y1 = (int64_t)y0 + (((int64_t)y0 * (int32_t)((1u << 30) - u)) >> 31);
  Rm = (uint32_t)min(max(y1, (int64_t)1 << 31), ((int64_t)1 << 32) - 1);
  sh = 47 + d / 2;
}

// one rotated element with any entry s = sh_a | sh_b << 8 | sh_c << 16; 64-bit
// while the up-shifts are at most 22 (|c| < 2^24: both terms below 2^61)
__device__ __noinline__ int32_t rot_any(int32_t x, int32_t cs, int32_t y, int32_t sn, uint32_t s) {
  const int a = (int)(s & 63u), b = (int)((s >> 8) & 63u), c = (int)(s >> 16);
  const int64_t u = (int64_t)x * cs, v = (int64_t)y * sn;
  if (max(a, b) <= 22) return (int32_t)corm_sat16(corm_rne_shr64f((u << a) + (v << b), c));
  return (int32_t)corm_sat16_128(corm_rne_shr128(((__int128)u << a) + ((__int128)v << b), c));
}
// no up-shift, a down-shift k <= 31 whose quotient is below 2^31 (sums stay below
// 2^40: k >= 9, or an element that is not rotated).  To nearest, ties to even: with
// half1 = 2^(k - 1) - 1 added first, the bit at 2^k is still the quotient's parity in a
// tie, and where it is not, adding it carries nothing.  par = 1; both 0 for k = 0
__device__ __forceinline__ int32_t rot_plain(int32_t x, int32_t cs, int32_t y, int32_t sn, uint32_t k, int64_t half1,
                                             uint32_t par) {
  const int64_t v = (int64_t)x * cs + ((int64_t)y * sn + half1);
  const int64_t u = v + (int64_t)(__funnelshift_r((uint32_t)v, (uint32_t)(v >> 32), k) & par);
  return (int32_t)__funnelshift_r((uint32_t)u, (uint32_t)(u >> 32), k);
}

// A row of the batch: its sequence (rows ascend: b goes forward), position and page
struct RowAt {
  bool in;        // a row of a sequence
  bool held;      // its position has a page
  uint32_t p;     // its position (< 2^32: positions and rows are below 2^31)
  uint64_t line;  // the page's first cached row of head 0, plus the row's place in a page
};
__device__ __forceinline__ uint32_t first_sequence(const corm_paged_cache& c, uint32_t row) {
  uint32_t b = 0, hi = c.B;  // the last b with cu[b] <= row lies in [b, hi)
  while (hi - b > 1u) {
    const uint32_t mid = (b + hi) / 2u;
    if (c.cu[mid] <= (int32_t)row) b = mid;
    else hi = mid;
  }
  return b;
}
__device__ __forceinline__ RowAt row_at(const corm_paged_cache& c, uint32_t row, uint32_t& b) {
  while (b + 1u < c.B && c.cu[b + 1] <= (int32_t)row) b++;
  const SeqRows s = seq_rows(c, b, c.rows);
  RowAt o;
  o.in = row >= s.lo && row < s.lo + s.n;
  o.p = s.pos + (row - s.lo);
  o.held = false;
  o.line = 0;
  if (o.in && o.p < s.cap) {
    const uint32_t sh = 31u - __clz(c.page);
    const int32_t pg = c.table[(uint64_t)b * c.table_width + (o.p >> sh)];
    o.held = (uint32_t)pg < c.pages;
    if (o.held) o.line = (uint64_t)((uint32_t)pg * (uint64_t)(c.KV << sh)) + (o.p & (c.page - 1u));
  }
  return o;
}

template <int HD, bool VEC, bool NORM>
__global__ void __launch_bounds__(256, 3) paged_prep_kernel(const __grid_constant__ PrepArgs A) {
  constexpr uint32_t LPH = HD / 8, HPT = 32 / LPH;  // lanes a head, heads a turn
  // the norms' entries, q's and k's, a lane's eight LPH apart (no bank is asked twice):
  // factor, down-shift n, 2^(n - 1) - 1 (0 for n = 0)
  __shared__ int4 s_norm[NORM ? 2 : 1][NORM ? HD : 1];
  corm_pdl_wait();
  corm_pdl_trigger();
  const corm_llm_paged_prep_desc& d = A.d;
  const corm_paged_cache& c = d.c;
  const uint32_t KV = c.KV, lane = threadIdx.x % LPH, sub = (threadIdx.x & 31u) / LPH, hr = d.rot / 2u;
  const uint32_t gw = blockIdx.x * 8u + (threadIdx.x >> 5), row_step = gridDim.x * 8u / A.parts, part = gw % A.parts;
  uint32_t row = gw / A.parts;
  const uint32_t rows = min(c.rows, (uint32_t)max(c.cu[c.B], 0));
  // the dimensions of a lane's pairs: a rotated pair p at (p, p + rot / 2) or
  // (2 p, 2 p + 1); the rest of the head, and v's, in neighbouring pairs
  auto first_of = [&](uint32_t p, bool v) { return p < hr && !d.interleaved && !v ? p : 2u * p; };
  auto second_of = [&](uint32_t p, bool v) { return p < hr && !d.interleaved && !v ? p + hr : 2u * p + 1u; };
  auto dim_a = [&](uint32_t k, bool v) { return first_of(4u * lane + k, v); };
  auto dim_b = [&](uint32_t k, bool v) { return second_of(4u * lane + k, v); };
  bool high = true;  // every down-shift is 32 .. 62: the usual entries
  if (NORM) {
    for (uint32_t i = threadIdx.x; i < 2u * HD; i += 256u) {
      const uint8_t* ne = (const uint8_t*)(i < HD ? d.nq : d.nk);
      if (!ne) continue;
      const uint32_t l = i % LPH, e = i % HD / LPH, p = 4u * l + (e & 3u);
      ne += 16u * (e < 4u ? first_of(p, false) : second_of(p, false));
      const uint32_t n = ne[10] & 63u;
      const uint64_t h = n ? (1ull << (n - 1u)) - 1ull : 0ull;
      s_norm[i / HD][i % HD] = make_int4(*(const int32_t*)ne, (int)n, (int)(uint32_t)h, (int)(uint32_t)(h >> 32));
      high = high && n >= 32u && n <= 62u;
    }
    high = __syncthreads_and(high);
  }
  if (row >= rows || row >= row_step) return;
  const uint32_t it0 = part * A.per, it1 = min(it0 + A.per, A.turns);
  // a turn's head: whether there is one for this lane, of what, which
  struct Slot {
    bool any, is_q, is_v;
    uint32_t head;
  };
  auto slot_of = [&](uint32_t it) {
    Slot s;
    const bool v = it >= A.turned;
    const uint32_t i = (v ? it - A.turned : it) * HPT + sub;
    s.is_v = v;
    s.any = i < (v ? KV : d.H + KV);
    s.is_q = !v && i < d.H;
    s.head = v || s.is_q ? i : i - d.H;
    return s;
  };
  auto shifts = [&](const Slot& s, uint32_t dim) -> uint32_t {  // sh_a | sh_b << 8 | sh_c << 16
    const uint8_t* ent = (const uint8_t*)(s.is_q ? d.pq : (s.is_v ? d.pv : d.pk));
    const bool bc = d.flags & (s.is_q ? 1u : (s.is_v ? 4u : 2u));
    return s.is_v && (d.flags & 8u) ? 0u : *(const uint32_t*)(ent + 16ull * (bc ? 0u : s.head * HD + dim) + 8) & 0x3F3F3Fu;
  };
  // the usual entries: no up-shift and one down-shift for the lane's elements, whose
  // quotients fit 32 bits: the down-shift, a byte a turn; any others (255) are read
  // again where they are used
  uint64_t forms = 0;
#pragma unroll 1
  for (uint32_t it = it0; it < it1; it++) {
    const Slot s = slot_of(it);
    uint32_t kd = 255;
    if (s.any) {
      const uint32_t k0 = shifts(s, dim_a(0, s.is_v));
      kd = k0 >> 16;
      bool plain = (k0 & 0xFFFFu) == 0u && kd <= 31u && (kd >= 9u || s.is_v || 4u * lane >= hr);
      if (!(s.is_v && (d.flags & 8u)) && !(d.flags & (s.is_q ? 1u : (s.is_v ? 4u : 2u)))) {  // an entry a dimension
        const uint8_t* const e = (const uint8_t*)(s.is_q ? d.pq : (s.is_v ? d.pv : d.pk)) + 16ull * (s.head * HD) + 8u;
#pragma unroll
        for (uint32_t k = 0; k < 4; k++)
          plain = plain && ((*(const uint32_t*)(e + 16u * dim_a(k, s.is_v)) ^ k0) & 0x3F3F3Fu) == 0u &&
                  ((*(const uint32_t*)(e + 16u * dim_b(k, s.is_v)) ^ k0) & 0x3F3F3Fu) == 0u;
      }
      if (!plain) kd = 255;
    }
    forms |= (uint64_t)kd << (8u * (it - it0));
  }
  const bool spl = 4u * lane < hr && !d.interleaved;  // VEC: alike for the lane's four pairs
  const bool all_spl = VEC && d.rot == HD && !d.interleaved;
  // the next row's heads, q's and k's counted as one (k's head i - H), this lane's place
  // in them; the second four of its elements are `far` on (VEC)
  const uint32_t place = VEC ? (spl ? 4u : 8u) * lane : 0u, far = spl ? hr : 4u, place_v = VEC ? 8u * lane : 0u;
  const int16_t* nq = d.q0 + (uint64_t)row * d.ldq0 + place;
  const int16_t* nk = d.k0 + (uint64_t)row * d.ldk + place - (uint64_t)d.H * HD;
  const int16_t* nv = d.v0 + (uint64_t)row * d.ldv + place_v;
  int16_t* yq = d.q + (uint64_t)row * d.ldq + place;
  // the 8 elements of a turn: two words of 4, the pairs' firsts and seconds where `spl`
  // (or not VEC), else as they lie
  auto load = [&](uint32_t it) {
    uint4 w = make_uint4(0, 0, 0, 0);
    const bool v = it >= A.turned;
    const uint32_t i = (v ? it - A.turned : it) * HPT + sub;
    if (i >= (v ? KV : d.H + KV)) return w;
    const int16_t* x = (v ? nv : (i < d.H ? nq : nk)) + (uint64_t)i * HD;
    if (VEC) {
      const uint2 a = *(const uint2*)x, b = *(const uint2*)(x + (v ? 4u : far));
      w = make_uint4(a.x, a.y, b.x, b.y);
    } else {
      w = make_uint4(pack16(x[dim_a(0, v)], x[dim_a(1, v)]), pack16(x[dim_a(2, v)], x[dim_a(3, v)]),
                     pack16(x[dim_b(0, v)], x[dim_b(1, v)]), pack16(x[dim_b(2, v)], x[dim_b(3, v)]));
    }
    return w;
  };
  uint32_t b = first_sequence(c, row);
  uint4 w = load(it0);
#pragma unroll 1
  for (; row < rows; row += row_step, yq += row_step * d.ldq) {
    const RowAt at = row_at(c, row, b);
    const uint32_t rb = c.bits == 8u ? HD : 2 * HD;
    int8_t* const kr = c.kc + at.line * rb;
    int8_t* const vr = c.vc + at.line * rb;
    int32_t cs[4], sn[4];
    {
      const int32_t* tr = d.rope + (uint64_t)min(at.in ? at.p : 0u, d.rope_rows - 1u) * d.rot;
      if (VEC && 4u * lane < hr) {
        const int4 c4 = __ldg((const int4*)(tr + 4u * lane)), s4 = __ldg((const int4*)(tr + hr + 4u * lane));
        cs[0] = c4.x, cs[1] = c4.y, cs[2] = c4.z, cs[3] = c4.w;
        sn[0] = s4.x, sn[1] = s4.y, sn[2] = s4.z, sn[3] = s4.w;
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t pr = 4u * lane + k;
          cs[k] = pr < hr ? __ldg(tr + pr) : 1;  // past the rotated part: x << sh_a alone
          sn[k] = pr < hr ? __ldg(tr + hr + pr) : 0;
        }
      }
    }
#pragma unroll 1
    for (uint32_t it = it0; it < it1; it++) {
      const uint4 x = w;
      // the next turn's elements, while this one's are worked on
      if (it + 1u < it1) {
        w = load(it + 1u);
      } else if (row + row_step < rows) {
        nq += row_step * d.ldq0;
        nk += row_step * d.ldk;
        nv += row_step * d.ldv;
        w = load(it0);
      }
      if (!at.in) continue;  // a row of no sequence
      const Slot s = slot_of(it);
      const bool sp = VEC ? spl && !s.is_v : true;
      uint4 ab = x;  // the pairs' firsts, then their seconds
      if (VEC && !(all_spl && !s.is_v)) {
        if (!sp)
          ab = make_uint4(__byte_perm(x.x, x.y, 0x5410), __byte_perm(x.z, x.w, 0x5410), __byte_perm(x.x, x.y, 0x7632),
                          __byte_perm(x.z, x.w, 0x7632));
      }
      int32_t va[4] = {(int16_t)ab.x, (int32_t)ab.x >> 16, (int16_t)ab.y, (int32_t)ab.y >> 16};
      int32_t vb[4] = {(int16_t)ab.z, (int32_t)ab.z >> 16, (int16_t)ab.w, (int32_t)ab.w >> 16};
      if (NORM && !s.is_v) {  // (alike over the warp; a head's lanes all have it or not)
        uint64_t s2 = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) s2 = (uint64_t)((int64_t)vb[k] * vb[k] + (int64_t)((uint64_t)((int64_t)va[k] * va[k]) + s2));
#pragma unroll
        for (uint32_t o = LPH / 2; o > 0; o >>= 1) s2 += __shfl_xor_sync(0xffffffffu, s2, o);
        if (s.is_q ? d.nq : d.nk) {
          uint32_t Rm;
          int sh;
          rsqrt64(max(s2 + (s.is_q ? d.eps_q : d.eps_k), (uint64_t)1), Rm, sh, A.rsq);
          sh -= 24;
          // |x| <= sqrt(D): P1 = floor(x Rm 2^-sh) is 2^24 at most, and the table's error;
          // Rm has its top bit: x Rm is x times it as a signed word, and 2^32 x.  P1 G to
          // nearest, ties to even, as rot_plain rounds: the quotient is in the high word
          const bool fast = high && __all_sync(__activemask(), sh < 32);
          auto normed = [&](int32_t x, uint32_t i) {
            const int4 e = s_norm[s.is_q ? 0 : 1][NORM ? i * LPH + lane : 0];
            const int64_t xr = (int64_t)x * (int32_t)Rm + ((int64_t)x << 32);
            if (fast) {
              const int32_t p1 = (int32_t)__funnelshift_r((uint32_t)xr, (uint32_t)(xr >> 32), (uint32_t)sh);
              const int64_t v = (int64_t)p1 * e.x + (int64_t)((uint64_t)(uint32_t)e.w << 32 | (uint32_t)e.z);
              const uint32_t n = (uint32_t)e.y - 32u;
              const int64_t u = v + (((int32_t)(v >> 32) >> n) & 1);
              return min(max((int32_t)(u >> 32) >> n, -32768), 32767);
            }
            return (int32_t)corm_sat16(corm_rne_shr64f((xr >> sh) * e.x, e.y));
          };
#pragma unroll
          for (uint32_t k = 0; k < 4; k++) {
            va[k] = normed(va[k], k);
            vb[k] = normed(vb[k], 4u + k);
          }
        }
      }
      const uint32_t kd = (uint32_t)(forms >> (8u * (it - it0))) & 255u;
      if (kd != 255u) {
        const uint32_t half1 = kd ? (1u << kd) / 2u - 1u : 0u, par = kd ? 1u : 0u;
        if (s.is_v) {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            va[k] = (va[k] + (int32_t)(half1 + ((uint32_t)(va[k] >> kd) & par))) >> kd;
            vb[k] = (vb[k] + (int32_t)(half1 + ((uint32_t)(vb[k] >> kd) & par))) >> kd;
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const int32_t a = va[k], bb = vb[k];
            va[k] = rot_plain(a, cs[k], -bb, sn[k], kd, half1, par);
            vb[k] = rot_plain(bb, cs[k], a, sn[k], kd, half1, par);
          }
        }
      } else if (s.any) {
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
          const int32_t a = va[k], bb = vb[k];
          va[k] = rot_any(a, s.is_v ? 1 : cs[k], -bb, s.is_v ? 0 : sn[k], shifts(s, dim_a(k, s.is_v)));
          vb[k] = rot_any(bb, s.is_v ? 1 : cs[k], a, s.is_v ? 0 : sn[k], shifts(s, dim_b(k, s.is_v)));
        }
      }
      // (saturates)
      uint32_t w0 = pack_s16(va[0], va[1]), w1 = pack_s16(va[2], va[3]), w2 = pack_s16(vb[0], vb[1]), w3 = pack_s16(vb[2], vb[3]);
      if (s.is_q) {
        int16_t* y = yq + (uint64_t)s.head * HD;
        if (VEC) {
          *(uint2*)y = sp ? make_uint2(w0, w1) : make_uint2(__byte_perm(w0, w2, 0x5410), __byte_perm(w0, w2, 0x7632));
          *(uint2*)(y + far) = sp ? make_uint2(w2, w3) : make_uint2(__byte_perm(w1, w3, 0x5410), __byte_perm(w1, w3, 0x7632));
        } else {
          const uint32_t ww[4] = {w0, w1, w2, w3};
#pragma unroll
          for (uint32_t k = 0; k < 4; k++) {
            y[dim_a(k, false)] = (int16_t)(ww[k >> 1] >> (16u * (k & 1u)));
            y[dim_b(k, false)] = (int16_t)(ww[2 + (k >> 1)] >> (16u * (k & 1u)));
          }
        }
      }
      uint32_t shift = 0;
      if (c.bits == 8u) {  // (every lane: the head's largest element)
        // x or its complement, two of 16 bits a word (a permutation repeats the signs)
        auto mag = [](uint32_t w) {
          uint32_t sign;
          asm("prmt.b32 %0, %1, 0, 0xBB99;" : "=r"(sign) : "r"(w));
          return w ^ sign;
        };
        uint32_t t = __vmaxu2(__vmaxu2(mag(w0), mag(w1)), __vmaxu2(mag(w2), mag(w3)));
#pragma unroll
        for (uint32_t o = LPH / 2; o > 0; o >>= 1) t = __vmaxu2(t, __shfl_xor_sync(0xffffffffu, t, o));
        t = max(t & 0xFFFFu, t >> 16);
        const int bits = 32 - __clz((int)t);
        shift = bits > 7 ? (uint32_t)(bits - 7) : 0u;
      }
      if (s.is_q || !s.any || !at.held) continue;
      int8_t* y = (s.is_v ? vr : kr) + (uint64_t)s.head * (c.page * rb);
      if (c.bits == 8u) {
        // RNE by shift <= 8; only the upper end can round past the codes
        const int32_t h = (1 << shift) >> 1, r = h ? h - 1 : 0;
        va[0] = (int16_t)w0, va[1] = (int32_t)w0 >> 16, va[2] = (int16_t)w1, va[3] = (int32_t)w1 >> 16;
        vb[0] = (int16_t)w2, vb[1] = (int32_t)w2 >> 16, vb[2] = (int16_t)w3, vb[3] = (int32_t)w3 >> 16;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          va[k] = min((va[k] + r + (h ? (va[k] >> shift) & 1 : 0)) >> shift, 127);
          vb[k] = min((vb[k] + r + (h ? (vb[k] >> shift) & 1 : 0)) >> shift, 127);
        }
        if (lane == 0) (s.is_v ? c.vs : c.ks)[at.line + (uint64_t)s.head * c.page] = (uint8_t)shift;
        w0 = pack_s16(va[0], va[1]), w1 = pack_s16(va[2], va[3]), w2 = pack_s16(vb[0], vb[1]), w3 = pack_s16(vb[2], vb[3]);
      }
      if (VEC) {
        // bytes of va, of vb: low (or code), then high
        const uint32_t wb[4] = {__byte_perm(w0, w1, 0x6420), __byte_perm(w2, w3, 0x6420), __byte_perm(w0, w1, 0x7531),
                                __byte_perm(w2, w3, 0x7531)};
#pragma unroll
        for (int pl = 0; pl < 2; pl++) {  // low bytes (codes), high bytes
          if (pl && c.bits == 8u) break;
          int8_t* yp = y + (c.bits == 8u || pl ? 0 : HD);
          if (sp) {
            *(uint32_t*)(yp + 4u * lane) = wb[2 * pl];
            *(uint32_t*)(yp + 4u * lane + hr) = wb[2 * pl + 1];
          } else {
            *(uint2*)(yp + 8u * lane) = make_uint2(__byte_perm(wb[2 * pl], wb[2 * pl + 1], 0x5140),
                                                   __byte_perm(wb[2 * pl], wb[2 * pl + 1], 0x7362));
          }
        }
      } else {
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
          const uint32_t da = dim_a(k, s.is_v), db = dim_b(k, s.is_v), m = 16u * (k & 1u);
          const uint32_t a = (k < 2 ? w0 : w1) >> m, bb = (k < 2 ? w2 : w3) >> m;
          if (c.bits == 8u) {
            y[da] = (int8_t)a;
            y[db] = (int8_t)bb;
          } else {
            y[da] = (int8_t)(a >> 8);
            y[db] = (int8_t)(bb >> 8);
            y[HD + da] = (int8_t)a;
            y[HD + db] = (int8_t)bb;
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------- read-back
// A warp per row, or per part of its heads (K's, then V's) where there are few rows;
// HD / 8 lanes a head, 8 elements a lane: 8-byte loads of each plane, four heads' under
// way at once, one 16-byte store (words where the output is not on 16 bytes).  Bound by
// the loads' latency and the copies' instructions: 3 sequences of 20 k cached rows at 8
// bits 13.6 us (3.8 TB/s), 16 of up to 640 5.3 us.
struct ReadArgs {
  corm_llm_paged_read_desc d;
  uint32_t vec, heads, turns, per, parts;  // heads: K's and V's, or one of them
};
template <int HD>
__global__ void __launch_bounds__(256) paged_read_kernel(const __grid_constant__ ReadArgs A) {
  corm_pdl_wait();
  corm_pdl_trigger();
  constexpr uint32_t LPH = HD / 8, HPT = 32 / LPH, U = 4;
  const corm_llm_paged_read_desc& d = A.d;
  const corm_paged_cache& c = d.c;
  const uint32_t lane = threadIdx.x % LPH, sub = (threadIdx.x & 31u) / LPH, nk = d.k ? c.KV : 0u;
  const uint32_t gw = blockIdx.x * 8u + (threadIdx.x >> 5), row_step = gridDim.x * 8u / A.parts;
  const uint32_t part = gw % A.parts, it0 = part * A.per, it1 = min(it0 + A.per, A.turns);
  uint32_t row = gw / A.parts;
  const uint32_t rows = min(c.rows, (uint32_t)max(c.cu[c.B], 0));
  if (row >= rows || row >= row_step) return;
  const bool b8 = c.bits == 8u;
  const uint32_t rb = b8 ? HD : 2 * HD, hb = c.page * rb;  // bytes from head to head
  uint32_t b = first_sequence(c, row);
#pragma unroll 1
  for (; row < rows; row += row_step) {
    const RowAt at = row_at(c, row, b);
    if (!at.in) continue;
    const int8_t* const kr = c.kc + at.line * rb + 8u * lane;
    const int8_t* const vr = c.vc + at.line * rb + 8u * lane;
    int16_t* const ko = d.k + (uint64_t)row * d.ldk + 8u * lane;
    int16_t* const vo = d.v + (uint64_t)row * d.ldv + 8u * lane;
#pragma unroll 1
    for (uint32_t t = it0; t < it1; t += U) {
      uint2 h[U], l[U];
#pragma unroll
      for (uint32_t u = 0; u < U; u++) {
        const uint32_t i = (t + u) * HPT + sub;
        const bool is_v = i >= nk;
        const uint32_t g = is_v ? i - nk : i;
        h[u] = l[u] = make_uint2(0, 0);
        if (at.held && t + u < it1 && i < A.heads) {
          const int8_t* const y = (is_v ? vr : kr) + (uint64_t)g * hb;
          h[u] = *(const uint2*)y;
          if (b8) l[u].x = (is_v ? c.vs : c.ks)[at.line + (uint64_t)g * c.page];
          else l[u] = *(const uint2*)(y + HD);
        }
      }
#pragma unroll
      for (uint32_t u = 0; u < U; u++) {
        const uint32_t i = (t + u) * HPT + sub;
        const bool is_v = i >= nk;
        const uint32_t g = is_v ? i - nk : i;
        if (t + u >= it1 || i >= A.heads) continue;
        uint32_t w[4];
        if (b8) {
          const uint32_t sh = l[u].x;  // (a shift from 16 up leaves nothing)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const uint32_t q = k < 2 ? h[u].x : h[u].y;
            const uint32_t v0 = (uint32_t)(int32_t)(int8_t)(q >> (16 * (k & 1))), v1 = (uint32_t)(int32_t)(int8_t)(q >> (16 * (k & 1) + 8));
            w[k] = sh < 16u ? __byte_perm(v0 << sh, v1 << sh, 0x5410) : 0u;
          }
        } else {
          w[0] = __byte_perm(l[u].x, h[u].x, 0x5140);
          w[1] = __byte_perm(l[u].x, h[u].x, 0x7362);
          w[2] = __byte_perm(l[u].y, h[u].y, 0x5140);
          w[3] = __byte_perm(l[u].y, h[u].y, 0x7362);
        }
        int16_t* const o = (is_v ? vo : ko) + (uint64_t)g * HD;
        if (A.vec) {
          *(uint4*)o = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            o[2 * k] = (int16_t)w[k];
            o[2 * k + 1] = (int16_t)(w[k] >> 16);
          }
        }
      }
    }
  }
}

// The launch of a kernel with a warp per row and part: `turns` of work a row in parts of
// at most `most` turns, smaller ones while the warps that are resident at once (`blocks_sm`
// blocks of 8 an SM) have fewer than `each` / 2 parts each: the preparation, whose turns
// are long, evens out its last round (4.5k rows of 12 turns: 76 us against 92); the
// read-back, short beside a row's lookups, only fills the SMs (14 us against 22)
struct RowGrid {
  uint32_t per, parts, grid;
};
RowGrid row_grid(uint64_t rows, uint32_t turns, uint32_t most, uint32_t blocks_sm, uint32_t each) {
  const uint64_t room = 148ull * 8u * blocks_sm;
  RowGrid g;
  g.parts = (turns + most - 1u) / most;
  while (g.parts < turns && rows * g.parts * 2u < each * room) g.parts++;
  g.per = (turns + g.parts - 1u) / g.parts;
  g.parts = (turns + g.per - 1u) / g.per;
  const uint64_t want = (rows * g.parts + 7u) / 8u, least = (g.parts + 7u) / 8u;  // (a row's parts at least)
  const uint64_t grid = want < room / 8u ? want : room / 8u;
  g.grid = (uint32_t)(grid < least ? least : grid);
  return g;
}

// ---------------------------------------------------------------- attention, few rows
// A cluster of X CTAs per (sequence, KV head, 8 rows), a row being (token,
// head of the group), token-major; the CTAs share the keys.  The unit's e(d) is
// a table of d = m - score, so sums cannot be rescaled as a running maximum
// moves; instead the scores stay on the chip: those of a CTA's keys are formed
// once (int16 in shared memory), the maxima meet over the cluster, then e in
// place and the sums meet, then P in place and P.V over the V rows, whose
// partial sums (modulo 2^32, so in any order) meet last.  K and V are read once.
// Keys beyond the shared memory: windows, the scores formed again in each of
// the three passes.
//
// The eight warps work apart: a warp has every eighth block of keys (32 or 64),
// copies them itself into stages of its own (16 bytes a lane, the next under way
// while it computes; the V rows arrive under the softmax), and
// nothing but the maxima, the sums and the output meets.  Warp-level MMAs with the
// keys, then the output's dimensions, as the 16 rows of an MMA and the query rows as
// its 8 columns: a decoded token's group of heads is far below the 128 rows of a
// tcgen05 tile, and the copies are to bound the kernel.  The contraction over the
// keys takes them in the order in which the scores' words hold them (word i of 16
// keys: keys i and i + 8); V's rows are transposed on the way to the registers.
//
// Measured (64 dimensions, 3 query heads a KV head, in a graph): 64 sequences of 128 to
// 639 keys 12.4 us, bound by its chain of waits (page, K, maximum, sum, V; 6.4 us with one
// sequence of 33 keys, 4 of them the kernel's); 8 sequences of 21k to 32k keys at 8 bits
// 39 us, 3.3 TB/s: the K and V phases run at three quarters of the memory's rate, the
// softmax between them (about 250 of 1000 instructions a block) keeps only the stages'
// copies under way; 128 dimensions, 4 query heads, 16 bits, 16 x 4k keys: 41 us, 4.9 TB/s.
// A ring of 64-key stages that all warps share, a copy warp and 16-row MMAs: 29 and 146
// us for the first two.
constexpr uint32_t kRows = 8;     // rows of a tile
constexpr uint32_t kWarps = 8;
constexpr uint32_t kMaxCluster = 8;

struct SplitArgs {
  corm_llm_paged_attn_desc d;
  const int32_t* tab;
  int* err;
  Waits waits;
  uint32_t G, Ginv, X, stages, win, rcap;  // Ginv: ceil(2^16 / G); stages of a warp; win: blocks of a warp's window; rcap: rows held
};

template <int HD, int BITS>
struct SplitShape {
  static constexpr uint32_t RB = HD * (BITS / 8);             // bytes of a cached row
  static constexpr uint32_t KS = RB <= 64 ? 64 : 32;          // keys of a block (a stage)
  static constexpr uint32_t STB = KS * RB + (BITS == 8 ? 128u : 0u);  // a stage (its shifts last)
  static constexpr uint32_t NKS = HD < 32 ? 1 : HD / 32;      // MMA steps of a score
  static constexpr uint32_t MT = HD / 16;                     // 16-dimension tiles of the output
  static constexpr uint32_t PW = KS / 2;                      // words of a row's scores in a block
  static constexpr uint32_t OCC = HD <= 64 ? 3 : (HD == 128 ? 2 : 1);  // CTAs an SM that the registers allow
};

// A stage's rows, 16-byte pieces in another order by the row (byte offsets ^ this), so
// that eight keys' pieces of one place, keys 0 .. 7 or 0 .. 3 and 8 .. 11, meet no bank
// twice; linear in the row's bits
template <uint32_t RB>
__host__ __device__ constexpr uint32_t stage_swizzle(uint32_t row) {
  return RB == 16 ? 0u
                  : (RB == 32 ? 16u * (((row >> 2) ^ (row >> 3)) & 1u)
                              : (RB == 64 ? 16u * (((row >> 1) & 3u) ^ (2u * ((row >> 3) & 1u)))
                                          : 16u * ((row & 7u) ^ (4u * ((row >> 3) & 1u)))));
}
// word i of row r's scores in a block: groups of 8 words trade places by the row, so that
// four rows' reads meet no bank twice
template <uint32_t PW>
__device__ __forceinline__ uint32_t score_word(uint32_t r, uint32_t i) {
  return r * PW + (i ^ (PW == 32 ? 8u * (r & 3u) : 8u * ((r >> 1) & 1u)));
}

// OCC: CTAs an SM.  64 dimensions have a form of three, for batches that fill them, and
// one of two whose registers hold the output's sums apart (8 sequences of 21k to 32k keys
// at 8 bits 39 us against 43; 64 of 128 to 639 15.4 against 12.9)
template <int HD, int BITS, int OCC>
__global__ void __launch_bounds__(256, OCC) paged_attn_split_kernel(const __grid_constant__ SplitArgs A) {
  using Sh = SplitShape<HD, BITS>;
  constexpr uint32_t RB = Sh::RB, KS = Sh::KS, STB = Sh::STB, NKS = Sh::NKS, PW = Sh::PW;
  extern __shared__ __align__(128) uint8_t pa_sm[];
  __shared__ uint64_t cbar;
  __shared__ int32_t s_wmax[kWarps][kRows], s_m[kRows];
  __shared__ unsigned long long s_ws[kWarps][kRows], s_s[kRows];
  __shared__ uint32_t s_lo[kRows], s_hi[kRows], s_cm[kRows], s_cs[kRows], s_fp[kRows];
  const corm_paged_cache& c = A.d.c;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t X = A.X, g = blockIdx.y, b = blockIdx.z, G = A.G;
  const uint32_t tile = X == 1u ? blockIdx.x : blockIdx.x / X, rank = X == 1u ? 0u : blockIdx.x % X;
  const uint32_t NST = A.stages, rcap = A.rcap, WIN = A.win;
  uint8_t* const ring = pa_sm + warp * NST * STB;                                          // this warp's stages
  uint32_t* const S = (uint32_t*)(pa_sm + kWarps * NST * STB) + warp * WIN * rcap * PW;  // and scores: [block][row][PW]
  uint16_t* const tab = (uint16_t*)(pa_sm + kWarps * (NST * STB + WIN * rcap * PW * 4u));
  uint32_t* const s_O = (uint32_t*)(tab + 4096);
  // before the wait for the kernel in front: the table, which no kernel writes
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    const int4 v = ((const int4*)A.tab)[tid + 256u * i];
    ((uint2*)tab)[tid + 256u * i] = make_uint2(pack16(v.x - 1, v.y - 1), pack16(v.z - 1, v.w - 1));
  }
  if (tid < kWarps * kRows) ((unsigned long long*)s_ws)[tid] = 0;
  if (tid == 0) {
    sm100::mbar_init(&cbar, X);
    sm100::fence_mbar_init();
  }
  corm_pdl_wait();
  corm_pdl_trigger();
  const SeqRows sq = seq_rows(c, b, c.rows);
  const uint32_t n = min(sq.n, A.d.max_q), r0 = tile * kRows;
  if ((uint64_t)r0 >= (uint64_t)n * G) return;  // the cluster's CTAs alike
  const uint32_t nr = min(kRows, n * G - r0);
  // row r0 + d (d < 8) is token i0 + t, head o of the group: t = (o0 + d) / G, exact by Ginv
  const uint32_t i0 = tile ? r0 / G : 0u, o0 = r0 - i0 * G;
  auto token = [&](uint32_t d) { return ((o0 + d) * A.Ginv) >> 16; };
  const uint32_t i1 = i0 + token(nr - 1u);
  // the keys some row of the tile sees: [lo, hi), in blocks from lo rounded down
  const uint32_t hi = min(sq.pos + i1 + 1u, sq.cap);
  const uint32_t w = A.d.window;
  const uint32_t lo = (w && sq.pos + i0 + 1u > w) ? sq.pos + i0 + 1u - w : 0u;
  const uint32_t tile0 = lo / KS, ntile = hi > lo ? (hi + KS - 1u) / KS - tile0 : 0u;
  const uint32_t per = (ntile + X - 1u) / X;
  const uint32_t first = tile0 + min(rank * per, ntile) + warp, end = tile0 + min(rank * per + per, ntile);
  const uint32_t own = first < end ? (end - first + kWarps - 1u) / kWarps : 0u;  // blocks first, first + 8, ...
  const bool again = own > WIN;  // more than a window (a warp's own affair)

  const uint32_t qn = lane >> 2, qt = lane & 3u;
  uint2 qw[NKS][2];  // q of row qn: four dimensions of each operand word
  {
    const uint32_t d = min(qn, nr - 1u), t = token(d);
    const int16_t* const q = A.d.q + (uint64_t)(sq.lo + i0 + t) * A.d.ldq + (uint64_t)(g * G + o0 + d - t * G) * HD + 4u * qt;
    const bool q8 = (((uintptr_t)A.d.q | (A.d.ldq * 2u)) & 7u) == 0;
#pragma unroll
    for (uint32_t ks = 0; ks < NKS; ks++)
#pragma unroll
      for (uint32_t half = 0; half < 2; half++) {
        qw[ks][half] = make_uint2(0, 0);
        if (qn < nr && (HD > 16 || half == 0)) {
          const int16_t* const p = q + 32u * ks + 16u * half;
          qw[ks][half] = q8 ? *(const uint2*)p : make_uint2(pack16(p[0], p[1]), pack16(p[2], p[3]));
        }
      }
  }
  // ---------------- the copies: K's blocks, then V's; in windows K's blocks for each of
  // the first two passes, then each window's K and V
  const uint32_t sub = min(c.page, KS), psh = 31u - __clz(c.page), ssh = 31u - __clz(sub);
  const uint32_t pieces = KS >> ssh, pcs = 31u - __clz(pieces);  // pieces of a block
  const int32_t* const tb = c.table + (uint64_t)b * c.table_width;
  const uint32_t total = again ? 4u * own : 2u * own;
  uint32_t eq = 0, ej = 0, ea = 0, ep = 0, es = 0;  // the next copy's number, block, window and pass and stage
  bool ev = false;                                  // of V
  const uint32_t held = 32u >> pcs;                 // blocks whose pages the lanes hold, a piece each: from block ib on
  uint32_t ib = 0;
  auto pages_from = [&](uint32_t j) -> int32_t {  // below 0: no page
    const uint32_t bj = j + (lane >> pcs), key = (first + bj * kWarps) * KS + ((lane & (pieces - 1u)) << ssh);
    int32_t id = -1;
    if (bj < own && key < hi) id = tb[key >> psh];
    return (uint32_t)id < c.pages ? id : -1;
  };
  int32_t ids = pages_from(0);
  // one group of asynchronous copies, 16 bytes a lane (empty after the last block);
  // pieces without a page are zeros
  auto emit = [&]() {
    if (eq < total) {
      if (ej - ib >= held) {
        ib = ej & ~(held - 1u);
        ids = pages_from(ib);
      }
      const uint32_t at = (ej - ib) * pieces;
      uint8_t* const st = ring + es * STB;
      const uint8_t* const rows = ev ? (const uint8_t*)c.vc : (const uint8_t*)c.kc;
      const uint32_t in0 = ((first + ej * kWarps) * KS) & (c.page - 1u);  // a block in a page: its first row
      if (pieces == 1u) {
        const int32_t pg = __shfl_sync(0xffffffffu, ids, at);
        const uint32_t n = pg < 0 ? 0u : 16u;
        const uint64_t line = ((uint64_t)(uint32_t)max(pg, 0) * c.KV + g) * c.page + in0;
        const uint8_t* const src = rows + line * RB + lane * 16u;
        const uint32_t to = (lane * 16u) ^ stage_swizzle<RB>(lane * 16u / RB);
#pragma unroll
        for (uint32_t i = 0; i < KS * RB / 512u; i++)
          cp_async16(st + (to ^ stage_swizzle<RB>(i * 512u / RB)) + i * 512u, src + i * 512u, n);
        if (BITS == 8 && lane < KS / 16u) cp_async16(st + KS * RB + lane * 16u, (ev ? c.vs : c.ks) + line + lane * 16u, n);
      } else {
#pragma unroll 1
        for (uint32_t i = lane * 16u; i < KS * RB; i += 512u) {
          const uint32_t row = i / RB;
          const int32_t pg = __shfl_sync(0xffffffffu, ids, at + (row >> ssh));
          const uint64_t line = ((uint64_t)(uint32_t)max(pg, 0) * c.KV + g) * c.page + (row & (sub - 1u));
          cp_async16(st + (i ^ stage_swizzle<RB>(row)), rows + line * RB + i % RB, pg < 0 ? 0u : 16u);
        }
        if (BITS == 8) {
          const int32_t pg = __shfl_sync(0xffffffffu, ids, (at + (lane * 16u >> ssh)) & 31u);
          const uint64_t line = ((uint64_t)(uint32_t)max(pg, 0) * c.KV + g) * c.page + (lane * 16u & (sub - 1u));
          if (lane < KS / 16u) cp_async16(st + KS * RB + lane * 16u, (ev ? c.vs : c.ks) + line, pg < 0 ? 0u : 16u);
        }
      }
      if (++es == NST) es = 0;
      eq++;
      ej++;
      if (!again) {
        if (ej == own) ej = 0, ev = true;
      } else if (ep < 2u) {
        if (ej == own) ej = 0, ep++;
      } else if (ej == min(ea + WIN, own)) {
        if (ev) ea += WIN;
        ev = !ev;
        ej = ea;
      }
    }
    cp_async_commit();
  };
  for (uint32_t i = 0; i < NST; i++) emit();

  // ---------------- the rows
  if (tid < kRows) {
    const uint32_t d = min(tid, nr - 1u), t = token(d), h = g * G + o0 + d - t * G;
    const uint32_t p = sq.pos + i0 + t;
    s_hi[tid] = min(p + 1u, sq.cap);
    s_lo[tid] = (w && p + 1u > w) ? p + 1u - w : 0u;
    s_cm[tid] = A.d.smx[2u * h];
    const uint32_t cfg = A.d.smx[2u * h + 1u];
    s_cs[tid] = cfg & 63u;
    s_fp[tid] = (cfg >> 8) & 31u;
  }
  uint32_t bh[NKS][2], bl[NKS][2];  // q's planes
#pragma unroll
  for (uint32_t ks = 0; ks < NKS; ks++)
#pragma unroll
    for (uint32_t half = 0; half < 2; half++) {
      bh[ks][half] = __byte_perm(qw[ks][half].x, qw[ks][half].y, 0x7531);
      bl[ks][half] = __byte_perm(qw[ks][half].x, qw[ks][half].y, 0x6420);
    }
  if (X > 1) cluster_sync();
  else __syncthreads();

  const uint32_t lo_last = s_lo[nr - 1u], hi_first = s_hi[0];  // every row sees [lo_last, hi_first)
  const uint32_t ra = 2u * qt, rb = ra + 1u;                   // the rows of this lane's columns
  uint32_t cst = 0;                                            // the next stage
  bool ok = true;
  auto stage_in = [&]() {  // all but the last NST - 1 groups are here
    if (NST == 1u) cp_async_wait<0>();
    else if (NST == 2u) cp_async_wait<1>();
    else cp_async_wait<3>();
    __syncwarp();
    return ring + cst * STB;
  };
  auto stage_out = [&]() {
    __syncwarp();
    if (++cst == NST) cst = 0;
    emit();
  };
  // a lane's row of an MMA's 16 x 32 operand: key (lane mod 16), the piece of 16 bytes lane / 16
  const uint32_t krow = lane & 15u, kx = (HD >= 32 ? 16u * (lane >> 4) : 0u) ^ stage_swizzle<RB>(lane & 15u);
  // of a transposed one's (32 keys as the scores' words hold them): key vrow
  const uint32_t vr16 = 2u * ((lane >> 2) & 3u) + ((lane >> 1) & 1u) + 8u * (lane & 1u);
  const uint32_t vrow = 16u * (lane >> 4) + vr16, vx = stage_swizzle<RB>(vr16);
  // the scores of block t into the window's slot; the running maxima of the keys the rows ra and rb see
  uint32_t mxa = 0x80008000u, mxb = 0x80008000u;
  auto scores = [&](uint32_t t, uint32_t slot) {
    const uint8_t* const st = stage_in();
    const uint32_t st_a = sm100::smem_u32(st) + krow * RB;
    uint32_t* const d = S + slot * rcap * PW;
    const bool whole = t * KS >= lo_last && (t + 1u) * KS <= hi_first;
#pragma unroll
    for (uint32_t k16 = 0; k16 < KS / 16; k16++) {
      const uint32_t row = st_a + 16u * k16 * RB;
      uint32_t hh[4], mid[4], ll[4], h[4] = {0, 0, 0, 0}, l[4] = {0, 0, 0, 0};
#pragma unroll
      for (uint32_t ks = 0; ks < NKS; ks++) {
        if constexpr (HD >= 32) {
          ldmatrix_x4(h, row + ((32u * ks) ^ kx));
          if (BITS == 16) ldmatrix_x4(l, row + ((HD + 32u * ks) ^ kx));
        } else {
          ldmatrix_x2(h, row + kx);
          if (BITS == 16) ldmatrix_x2(l, row + (HD ^ kx));
        }
        if (ks == 0) {
          mma_ss_first(hh, h, bh[ks][0], bh[ks][1]);
          mma_su_first(mid, h, bl[ks][0], bl[ks][1]);
          if (BITS == 16) mma_uu_first(ll, l, bl[ks][0], bl[ks][1]);
        } else {
          mma_ss(hh, h, bh[ks][0], bh[ks][1]);
          mma_su(mid, h, bl[ks][0], bl[ks][1]);
          if (BITS == 16) mma_uu(ll, l, bl[ks][0], bl[ks][1]);
        }
        if (BITS == 16) mma_us(mid, l, bh[ks][0], bh[ks][1]);
      }
      // columns ra and rb of keys qn (sums 0, 1) and qn + 8 (2, 3)
      uint32_t y[4];
      if (BITS == 16) {
#pragma unroll
        for (int x = 0; x < 4; x++) y[x] = (uint32_t)((int32_t)((hh[x] << 16) + (mid[x] << 8) + ll[x]) >> 8);
      } else {
        const uint8_t* const sp = st + KS * RB + 16u * k16 + qn;
        const uint32_t s0 = sp[0] & 31u, s1 = sp[8] & 31u;
#pragma unroll
        for (int x = 0; x < 4; x++) y[x] = (uint32_t)((int32_t)(((hh[x] << 8) + mid[x]) << (x < 2 ? s0 : s1)) >> 8);
      }
      uint32_t wa = pack_s16(y[0], y[2]), wb = pack_s16(y[1], y[3]);
      if (ra < nr) d[score_word<PW>(ra, 8u * k16 + qn)] = wa;
      if (rb < nr) d[score_word<PW>(rb, 8u * k16 + qn)] = wb;
      if (!whole) {
        const uint32_t k0 = t * KS + 16u * k16 + qn, k1 = k0 + 8u;
        const uint32_t la = s_lo[ra], ha = s_hi[ra], lb = s_lo[rb], hb = s_hi[rb];
        wa = __byte_perm(k0 >= la && k0 < ha ? wa : 0x8000u, k1 >= la && k1 < ha ? wa : 0x80000000u, 0x7610);
        wb = __byte_perm(k0 >= lb && k0 < hb ? wb : 0x8000u, k1 >= lb && k1 < hb ? wb : 0x80000000u, 0x7610);
      }
      mxa = __vmaxs2(mxa, wa);
      mxb = __vmaxs2(mxb, wb);
    }
    stage_out();
  };
  uint32_t cphase = 0;
  // every CTA of the cluster is here, and what it wrote before is visible
  auto cluster_meet = [&]() {
    __syncthreads();
    if (X > 1) {
      if (tid < X) mbar_arrive_remote(&cbar, tid);
      if (ok) ok = mbar_wait_cluster(&cbar, cphase, A.err, 303, A.waits);
      cphase ^= 1u;
    }
  };

  // pass 1: the maxima
#pragma unroll 1
  for (uint32_t j = 0; j < own; j++) scores(first + j * kWarps, again ? 0u : j);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    mxa = __vmaxs2(mxa, __shfl_xor_sync(0xffffffffu, mxa, o));
    mxb = __vmaxs2(mxb, __shfl_xor_sync(0xffffffffu, mxb, o));
  }
  if (qn == 0) {
    s_wmax[warp][ra] = max((int32_t)(int16_t)(mxa & 0xFFFFu), (int32_t)mxa >> 16);
    s_wmax[warp][rb] = max((int32_t)(int16_t)(mxb & 0xFFFFu), (int32_t)mxb >> 16);
  }
  __syncthreads();
  if (X > 1) {
    if (tid < kRows) {
      int32_t m = s_wmax[0][tid];
#pragma unroll
      for (uint32_t i = 1; i < kWarps; i++) m = max(m, s_wmax[i][tid]);
      s_m[tid] = m;
    }
    cluster_meet();
  }
  // the row's maximum over the CTA's warps, or the cluster's CTAs
  auto row_max = [&](uint32_t r) {
    int32_t m = INT32_MIN;
    if (X == 1) {
#pragma unroll
      for (uint32_t i = 0; i < kWarps; i++) m = max(m, s_wmax[i][r]);
    } else {
      for (uint32_t i = 0; i < X; i++) m = max(m, (int32_t)cluster_ld32(cluster_addr(&s_m[r], i)));
    }
    return m;
  };
  const int32_t mx = row_max(lane & 7u);
  // a word (two keys) a lane, PW lanes a row, the rows in turn
  const uint32_t rl = lane % PW, rh = lane / PW;
  constexpr uint32_t RSTEP = 32 / PW;
  const uint32_t word_key = 16u * (rl >> 3) + (rl & 7u);  // the word's first key in its block; the second is 8 on
  // e of a word's two scores, 0 where the row does not see the key.  With 9 <= Cs the
  // product of d 2^16 and Cm 2^8, shifted down, is floor(d Cm / 2^(Cs - 1)) = 2 y and a
  // bit: the table's byte offset is it mod 2^13 without the bit, the octave it / 2^13
  struct Row {
    uint32_t cm, cs, klo, khi, m0, cm8, sh;
  };
  auto row_of = [&](uint32_t r, uint32_t m0) {  // m0: the maximum at 2^16
    Row o;
    o.cm = s_cm[r], o.cs = s_cs[r], o.klo = s_lo[r], o.khi = s_hi[r];
    o.m0 = m0;
    o.cm8 = o.cs >= 40u ? 0u : (o.cm & 0xFFFFFFu) << 8;
    o.sh = min(o.cs, 40u) - 9u;
    return o;
  };
  auto e_of = [&](auto narrow, const Row& o, uint32_t x, uint32_t t, uint32_t& e0, uint32_t& e1) {
    const uint32_t d0 = o.m0 - (x << 16), d1 = o.m0 - (x & 0xFFFF0000u);
    if constexpr (decltype(narrow)::value) {
      const uint32_t t0 = __umulhi(d0, o.cm8) >> o.sh, t1 = __umulhi(d1, o.cm8) >> o.sh;
      e0 = shr_clamp((uint32_t)*(const uint16_t*)((const uint8_t*)tab + (t0 & 0x1FFEu)) + 1u, t0 >> 13);
      e1 = shr_clamp((uint32_t)*(const uint16_t*)((const uint8_t*)tab + (t1 & 0x1FFEu)) + 1u, t1 >> 13);
    } else {
      e0 = smx_e_wide(d0 >> 16, o.cm, o.cs, tab);
      e1 = smx_e_wide(d1 >> 16, o.cm, o.cs, tab);
    }
    if (t * KS < lo_last || (t + 1u) * KS > hi_first) {  // (alike over the warp)
      const uint32_t k0 = t * KS + word_key, k1 = k0 + 8u;
      e0 = k0 >= o.klo && k0 < o.khi ? e0 : 0u;
      e1 = k1 >= o.klo && k1 < o.khi ? e1 : 0u;
    }
  };
  // pass 2: e of blocks [a, z) in place (or only the sums)
  auto e_pass = [&](uint32_t a, uint32_t z, bool keep) {
#pragma unroll 1
    for (uint32_t q = 0; q < nr; q += RSTEP) {
      const uint32_t r = min(q + rh, nr - 1u);
      const bool mine = q + rh < nr;
      const Row o = row_of(r, (uint32_t)__shfl_sync(0xffffffffu, mx, r) << 16);
      uint32_t sum = 0;  // (of a window: below 2^32 over the row)
      auto go = [&](auto narrow) {
        uint32_t* p = S + score_word<PW>(r, rl);
#pragma unroll 4
        for (uint32_t j = a; j < z; j++, p += rcap * PW) {
          uint32_t e0, e1;
          e_of(narrow, o, *p, first + j * kWarps, e0, e1);
          sum += e0 + e1;
          if (keep && mine) *p = pack_u16(e0, e1);
        }
      };
      if (__all_sync(0xffffffffu, o.cs >= 9u)) go(std::true_type());
      else go(std::false_type());
#pragma unroll
      for (int o = PW / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (rl == 0 && mine) s_ws[warp][r] += sum;
    }
  };
  if (!again) {
    e_pass(0, own, true);
  } else {
#pragma unroll 1
    for (uint32_t a = 0; a < own; a += WIN) {
      const uint32_t z = min(a + WIN, own);
#pragma unroll 1
      for (uint32_t j = a; j < z; j++) scores(first + j * kWarps, j - a);
      e_pass(a, z, false);
      __syncwarp();
    }
  }
  __syncthreads();
  if (X > 1) {
    if (tid < kRows) {
      unsigned long long sum = 0;
#pragma unroll
      for (uint32_t i = 0; i < kWarps; i++) sum += s_ws[i][tid];
      s_s[tid] = sum;
    }
    cluster_meet();
  }
  auto row_r = [&](uint32_t r) {
    unsigned long long sum = 0;
    if (X == 1) {
#pragma unroll
      for (uint32_t i = 0; i < kWarps; i++) sum += s_ws[i][r];
    } else {
      for (uint32_t i = 0; i < X; i++) sum += cluster_ld64(cluster_addr(&s_s[r], i));
    }
    return smx_r(sum);
  };
  const uint32_t Rs = row_r(lane & 7u);

  // pass 3: P of blocks [a, z) in place (in windows from the scores), then P.V
  auto p_pass = [&](uint32_t a, uint32_t z) {
#pragma unroll 1
    for (uint32_t q = 0; q < nr; q += RSTEP) {
      const uint32_t r = min(q + rh, kRows - 1u), R = __shfl_sync(0xffffffffu, Rs, r), m0 = (uint32_t)__shfl_sync(0xffffffffu, mx, r) << 16;
      if (r >= nr) continue;
      uint32_t* p = S + score_word<PW>(r, rl);
      const uint32_t fp = s_fp[r];
      if (again) {
        const Row o = row_of(r, m0);
        uint32_t* v = p;
#pragma unroll 1
        for (uint32_t j = a; j < z; j++, v += rcap * PW) {
          uint32_t e0, e1;
          if (o.cs >= 9u) e_of(std::true_type(), o, *v, first + j * kWarps, e0, e1);
          else e_of(std::false_type(), o, *v, first + j * kWarps, e0, e1);
          *v = pack_u16(e0, e1);
        }
      }
      if (fp >= 8u && fp <= 15u) {  // the high word of e R 2^(f_p - 8) + 2^31
        const uint32_t Rp = R << (fp - 8u);
#pragma unroll 4
        for (uint32_t j = a; j < z; j++, p += rcap * PW) {
          const uint32_t x = *p, u0 = x & 0xFFFFu, u1 = x >> 16;
          const uint32_t e0 = u0 + ((u0 + 1u) >> 16), e1 = u1 + ((u1 + 1u) >> 16);
          *p = pack_s16((uint32_t)(((uint64_t)e0 * Rp + (1ull << 31)) >> 32), (uint32_t)(((uint64_t)e1 * Rp + (1ull << 31)) >> 32));
        }
      } else {
#pragma unroll 1
        for (uint32_t j = a; j < z; j++, p += rcap * PW) {
          const uint32_t x = *p;
          *p = smx_p(e_unpack(x & 0xFFFFu), R, fp) | smx_p(e_unpack(x >> 16), R, fp) << 16;
        }
      }
    }
    __syncwarp();
  };
  // the output's sums of weight 1, 2^8 and 2^16 apart, or (many dimensions) in one
  constexpr bool APART = HD <= 32 || (HD == 64 && OCC == 2);
  uint32_t acc[Sh::MT][4], acc1[APART ? Sh::MT : 1][4], acc2[APART ? Sh::MT : 1][4];
#pragma unroll
  for (uint32_t j = 0; j < Sh::MT; j++)
#pragma unroll
    for (int x = 0; x < 4; x++) {
      acc[j][x] = 0;
      if (APART) acc1[j][x] = acc2[j][x] = 0;
    }
  auto values = [&](uint32_t slot) {
    const uint8_t* const st = stage_in();
    const uint32_t* const pr = S + slot * rcap * PW;
    const uint32_t st_a = sm100::smem_u32(st) + vrow * RB;
#pragma unroll(HD <= 64 ? KS / 32 : 1)
    for (uint32_t k32 = 0; k32 < KS / 32; k32++) {
      uint32_t p0[2], p1[2], p2[2] = {0, 0};
#pragma unroll
      for (uint32_t h = 0; h < 2; h++) {
        uint2 v = make_uint2(0, 0);
        if (qn < nr) v = *(const uint2*)(pr + score_word<PW>(qn, 16u * k32 + 8u * h + 2u * qt));
        if (BITS == 16) {
          p0[h] = __byte_perm(v.x, v.y, 0x6420);
          p1[h] = __byte_perm(v.x, v.y, 0x7531);
        } else {  // P << shift: 23 bits, three planes against the codes
          const uint8_t* const sp = st + KS * RB + 32u * k32 + 16u * h + 2u * qt;
          const uint32_t sa = *(const uint16_t*)sp, sb = *(const uint16_t*)(sp + 8);
          const uint32_t y0 = (v.x & 0xFFFFu) << (sa & 31u), y1 = (v.x >> 16) << (sb & 31u);
          const uint32_t y2 = (v.y & 0xFFFFu) << ((sa >> 8) & 31u), y3 = (v.y >> 16) << ((sb >> 8) & 31u);
          const uint32_t f = __byte_perm(y0, y1, 0x5140), z = __byte_perm(y2, y3, 0x5140);
          p0[h] = __byte_perm(f, z, 0x5410);
          p1[h] = __byte_perm(f, z, 0x7632);
          p2[h] = __byte_perm(__byte_perm(y0, y1, 0x0062), __byte_perm(y2, y3, 0x0062), 0x5410);
        }
      }
#pragma unroll
      for (uint32_t j = 0; j < Sh::MT; j++) {
        uint32_t ah[4], al[4];
        ldmatrix_t8(ah, st_a + 32u * k32 * RB + ((16u * j) ^ vx));
        if (BITS == 16) ldmatrix_t8(al, st_a + 32u * k32 * RB + ((HD + 16u * j) ^ vx));
        if constexpr (APART) {
          if (BITS == 16) {
            mma_uu(acc[j], al, p0[0], p0[1]);
            mma_su(acc1[j], ah, p0[0], p0[1]);
            mma_uu(acc1[j], al, p1[0], p1[1]);
            mma_su(acc2[j], ah, p1[0], p1[1]);
          } else {
            mma_su(acc[j], ah, p0[0], p0[1]);
            mma_su(acc1[j], ah, p1[0], p1[1]);
            mma_su(acc2[j], ah, p2[0], p2[1]);
          }
        } else {
          uint32_t a1[4], a2[4];
          if (BITS == 16) {
            mma_uu(acc[j], al, p0[0], p0[1]);
            mma_su_first(a1, ah, p0[0], p0[1]);
            mma_uu(a1, al, p1[0], p1[1]);
            mma_su_first(a2, ah, p1[0], p1[1]);
          } else {
            mma_su(acc[j], ah, p0[0], p0[1]);
            mma_su_first(a1, ah, p1[0], p1[1]);
            mma_su_first(a2, ah, p2[0], p2[1]);
          }
#pragma unroll
          for (int x = 0; x < 4; x++) acc[j][x] += (a1[x] << 8) + (a2[x] << 16);
        }
      }
    }
    stage_out();
  };
#pragma unroll 1
  for (uint32_t a = 0; a < own; a += WIN) {
    const uint32_t z = min(a + WIN, own);
    if (again)
#pragma unroll 1
      for (uint32_t j = a; j < z; j++) scores(first + j * kWarps, j - a);
    p_pass(a, z);
#pragma unroll 1
    for (uint32_t j = a; j < z; j++) values(j - a);
  }
  // the warps' sums (modulo 2^32: any order) through their stages, which are read and
  // hold kRows HD words at least; then the cluster's
  uint32_t* const part = (uint32_t*)ring;  // [row][HD]
#pragma unroll
  for (uint32_t j = 0; j < Sh::MT; j++) {
    // sums 0, 1: dimension 16 j + qn of rows ra, rb; 2, 3: 8 dimensions on
    if (APART)
#pragma unroll
      for (int x = 0; x < 4; x++) acc[j][x] += (acc1[j][x] << 8) + (acc2[j][x] << 16);
    if (ra < nr) part[ra * HD + 16u * j + qn] = acc[j][0], part[ra * HD + 16u * j + qn + 8u] = acc[j][2];
    if (rb < nr) part[rb * HD + 16u * j + qn] = acc[j][1], part[rb * HD + 16u * j + qn + 8u] = acc[j][3];
  }
  __syncthreads();
  auto put = [&](uint32_t i, uint32_t v) {
    const uint32_t d = i / HD, t = token(d);
    A.d.o[(uint64_t)(sq.lo + i0 + t) * A.d.ldo + (uint64_t)(g * G + o0 + d - t * G) * HD + i % HD] = (int16_t)out16(v);
  };
  for (uint32_t i = tid; i < nr * HD; i += 256u) {
    uint32_t v = 0;
#pragma unroll
    for (uint32_t k = 0; k < kWarps; k++) v += *(const uint32_t*)(pa_sm + k * NST * STB + 4u * i);
    if (X > 1) s_O[i] = v;
    else put(i, v);
  }
  if (X > 1) {
    cluster_meet();
    for (uint32_t i = rank * 256u + tid; i < nr * HD; i += X * 256u) {
      uint32_t v = 0;
      for (uint32_t k = 0; k < X; k++) v += cluster_ld32(cluster_addr(&s_O[i], k));
      put(i, v);
    }
    cluster_sync();  // no CTA leaves while another reads its sums
  }
}

// dynamic shared memory of a CTA, occ of them an SM
constexpr uint32_t split_smem(uint32_t occ) { return (occ == 3u ? 73u : (occ == 2u ? 111u : 222u)) * 1024u; }

// how many clusters of X CTAs, d an SM, the current device holds at once (asked for once)
template <int HD, int BITS>
uint32_t resident_clusters(uint32_t X, uint32_t d) {
  static std::atomic<int> known[16][kMaxCluster + 1][4];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 16)
    if (const int n = known[dev][X][d].load(std::memory_order_relaxed)) return (uint32_t)n - 1u;
  auto kern = paged_attn_split_kernel<HD, BITS, SplitShape<HD, BITS>::OCC>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(X * 1024u);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = split_smem(d);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = X;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)split_smem(1)) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  if (dev < 16) known[dev][X][d].store(n + 1, std::memory_order_relaxed);
  return (uint32_t)n;
}

template <int HD, int BITS>
int launch_split(SplitArgs A, uint32_t tiles, cudaStream_t st) {
  using Sh = SplitShape<HD, BITS>;
  const corm_paged_cache& c = A.d.c;
  const uint64_t blocks = paged::live_tiles(A.d, kRows, tiles);
  const uint32_t cap = c.table_width * c.page, keys = A.d.max_keys < cap ? A.d.max_keys : cap;
  const uint32_t span = A.d.window && A.d.window < keys ? A.d.window + A.d.max_q : keys;
  const uint32_t kblocks = (span < keys ? span : keys) / Sh::KS + 2u;
  // the CTAs an SM that the registers allow, or fewer: so many that the scores fit beside
  // a stage a warp, but no more than are used.  A cluster lies within a GPC, so X CTAs of
  // it are at once resident for all `blocks` when the device holds so many clusters at
  // some d CTAs an SM.  d CTAs share an SM's issue slots but hide one another's waits: the
  // least (d + 1) / X is taken that leaves a warp two blocks (in the form of three CTAs, 8
  // sequences x 5 heads of 21k to 32k keys: X = 3 77 us, 4 64, 5 56, 6 43, and 59 for 8,
  // which is not resident at once; 4 x 5 heads at 16 bits: 104, 80, 68, 46, 8 43)
  uint32_t X, occ = Sh::OCC, room, need, fixed;
  const uint32_t block = kWarps * A.rcap * Sh::PW * 4u;
  for (;; occ--) {
    uint64_t bd = (blocks + 147u) / 148u;
    X = 1;
    for (uint32_t x = 2; x <= kMaxCluster && kblocks >= 2u * kWarps * x; x++) {
      uint32_t d = 1;
      while (d <= occ && resident_clusters<HD, BITS>(x, d) < blocks) d++;
      if (d <= occ && (d + 1u) * X < (bd + 1u) * x) X = x, bd = d;
    }
    fixed = 8192u + (X > 1 ? A.rcap * HD * 4u : 0u);
    need = ((kblocks + X - 1u) / X + kWarps - 1u) / kWarps;  // of a warp
    room = split_smem(occ) - fixed;
    if (occ == 1u || ((uint64_t)need * block + kWarps * Sh::STB <= room && (occ == 2u || bd > 2u))) break;
  }
  A.X = X;
  A.Ginv = (65536u + A.G - 1u) / A.G;
  uint32_t stages = 1;
  const uint32_t most = (room - kWarps * Sh::STB) / block;
  A.win = min(min(need, most), 512u);  // (a row's sum of e over a window fits 32 bits)
  while (stages < 4u && A.win * block + 2u * stages * kWarps * Sh::STB <= room) stages *= 2u;  // 1, 2 or 4
  A.stages = stages;
  const size_t smem = kWarps * stages * Sh::STB + (size_t)A.win * block + fixed;
  auto kern = paged_attn_split_kernel<HD, BITS, Sh::OCC>;
  if constexpr (HD == 64)
    if (occ < 3u) kern = paged_attn_split_kernel<HD, BITS, 2>;
  // (one limit for every launch: another thread's may be between its limit and its launch)
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)split_smem(1)) != cudaSuccess)
    return corm::cuda_status("llm_paged_attn");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * X, c.KV, c.B);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = corm_pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = X;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  {
    corm::ProfScope prof_("paged_attn_split_kernel", st);
    cudaLaunchKernelEx(&cfg, kern, A);
  }
  return corm::cuda_status("llm_paged_attn");
}

}  // namespace

extern "C" int corm_llm_paged_prep(const corm_llm_paged_prep_desc* d, corm_stream_t stream) {
  if (!d) return corm::fail(CORM_EINVAL, "corm_llm_paged_prep: null descriptor");
  const corm_paged_cache& c = d->c;
  if (int rc = paged::check_cache(&c, "corm_llm_paged_prep")) return rc;
  if (c.B == 0 || c.rows == 0) return CORM_OK;
  if (!d->q0 || !d->k0 || !d->v0 || !d->q || !d->rope || !d->pq || !d->pk || (!d->pv && !(d->flags & 8u)))
    return corm::fail(CORM_EINVAL, "corm_llm_paged_prep: null buffer");
  if (d->H == 0 || d->H > 65535u || (d->rot & 1u) || d->rot == 0 || d->rot > c.HD || d->rope_rows == 0)
    return corm::fail(CORM_EINVAL, "corm_llm_paged_prep: H %u, rot %u (even, 2 .. HD %u), rope_rows %u", d->H, d->rot,
                      c.HD, d->rope_rows);
  if (d->ldq0 < (uint64_t)d->H * c.HD || d->ldq < (uint64_t)d->H * c.HD || d->ldk < (uint64_t)c.KV * c.HD ||
      d->ldv < (uint64_t)c.KV * c.HD)
    return corm::fail(CORM_EINVAL, "corm_llm_paged_prep: row strides below the row lengths");
  if ((d->nq && d->eps_q >> 62) || (d->nk && d->eps_k >> 62))
    return corm::fail(CORM_ELIMIT, "corm_llm_paged_prep: eps beyond 2^62");
  if ((((uintptr_t)d->nq | (uintptr_t)d->nk | (uintptr_t)d->rope | (uintptr_t)d->pq | (uintptr_t)d->pk |
        (uintptr_t)d->pv) & 3u) ||
      (((uintptr_t)d->q0 | (uintptr_t)d->k0 | (uintptr_t)d->v0 | (uintptr_t)d->q) & 1u))
    return corm::fail(CORM_EINVAL, "corm_llm_paged_prep: unaligned buffers");
  if (int rc = corm::check_device()) return rc;
  const corm::DeviceTables* tb = corm::tables();
  if (!tb) return CORM_ECUDA;
  PrepArgs A;
  A.d = *d;
  A.rsq = tb->ro_rsq;
  // 8-byte rows, 16-byte table rows, whole lanes of one kind of pair
  const bool vec = !(((uintptr_t)d->q0 | (uintptr_t)d->k0 | (uintptr_t)d->v0 | (uintptr_t)d->q) & 7u) &&
                   !((d->ldq0 | d->ldk | d->ldv | d->ldq) & 3u) && !((uintptr_t)d->rope & 15u) && d->rot % 8u == 0;
  cudaStream_t st = (cudaStream_t)stream;
  const uint32_t hpt = 256u / c.HD;
  A.turned = (d->H + c.KV + hpt - 1u) / hpt;
  A.turns = A.turned + (c.KV + hpt - 1u) / hpt;
  const RowGrid rg = row_grid(c.rows, A.turns, kTurns, 3, 8);
  A.per = rg.per;
  A.parts = rg.parts;
  auto launch = [&](auto kern) { corm_launch_pdl(kern, dim3(rg.grid), dim3(256), 0, st, A); };
  {
    corm::ProfScope prof_("paged_prep_kernel", st);
    auto pick = [&](auto hd) {
      constexpr int W = decltype(hd)::value;
      if (d->nq || d->nk) {
        if (vec) launch(paged_prep_kernel<W, true, true>);
        else launch(paged_prep_kernel<W, false, true>);
      } else {
        if (vec) launch(paged_prep_kernel<W, true, false>);
        else launch(paged_prep_kernel<W, false, false>);
      }
    };
    switch (c.HD) {
      case 16: pick(std::integral_constant<int, 16>()); break;
      case 32: pick(std::integral_constant<int, 32>()); break;
      case 64: pick(std::integral_constant<int, 64>()); break;
      case 128: pick(std::integral_constant<int, 128>()); break;
      default: pick(std::integral_constant<int, 256>()); break;
    }
  }
  return corm::cuda_status("llm_paged_prep");
}

extern "C" int corm_llm_paged_read(const corm_llm_paged_read_desc* d, corm_stream_t stream) {
  if (!d) return corm::fail(CORM_EINVAL, "corm_llm_paged_read: null descriptor");
  const corm_paged_cache& c = d->c;
  if (int rc = paged::check_cache(&c, "corm_llm_paged_read")) return rc;
  if (c.B == 0 || c.rows == 0 || (!d->k && !d->v)) return CORM_OK;
  if ((d->k && d->ldk < (uint64_t)c.KV * c.HD) || (d->v && d->ldv < (uint64_t)c.KV * c.HD))
    return corm::fail(CORM_EINVAL, "corm_llm_paged_read: row strides below the row lengths");
  if (((uintptr_t)d->k | (uintptr_t)d->v) & 1u) return corm::fail(CORM_EINVAL, "corm_llm_paged_read: unaligned rows");
  if (int rc = corm::check_device()) return rc;
  ReadArgs A;
  A.d = *d;
  A.vec = !(((uintptr_t)d->k | (uintptr_t)d->v) & 15u) && !((d->k ? d->ldk : 0) & 7u) && !((d->v ? d->ldv : 0) & 7u);
  A.heads = (d->k ? c.KV : 0u) + (d->v ? c.KV : 0u);
  cudaStream_t st = (cudaStream_t)stream;
  const uint32_t hpt = 256u / c.HD;
  A.turns = (A.heads + hpt - 1u) / hpt;
  const RowGrid rg = row_grid(c.rows, A.turns, A.turns, 6, 1);
  A.per = rg.per;
  A.parts = rg.parts;
  auto launch = [&](auto kern) { corm_launch_pdl(kern, dim3(rg.grid), dim3(256), 0, st, A); };
  {
    corm::ProfScope prof_("paged_read_kernel", st);
    switch (c.HD) {
      case 16: launch(paged_read_kernel<16>); break;
      case 32: launch(paged_read_kernel<32>); break;
      case 64: launch(paged_read_kernel<64>); break;
      case 128: launch(paged_read_kernel<128>); break;
      default: launch(paged_read_kernel<256>); break;
    }
  }
  return corm::cuda_status("llm_paged_read");
}

extern "C" int corm_llm_paged_attn(const corm_llm_paged_attn_desc* d, corm_stream_t stream) {
  if (!d) return corm::fail(CORM_EINVAL, "corm_llm_paged_attn: null descriptor");
  const corm_paged_cache& c = d->c;
  if (int rc = paged::check_cache(&c, "corm_llm_paged_attn")) return rc;
  if (c.B == 0 || c.rows == 0 || d->max_q == 0) return CORM_OK;
  if (!d->q || !d->o || !d->smx) return corm::fail(CORM_EINVAL, "corm_llm_paged_attn: null buffer");
  if (d->H == 0 || d->H % c.KV || d->H / c.KV > 16u)
    return corm::fail(CORM_EINVAL, "corm_llm_paged_attn: H %u over KV %u (1 .. 16 query heads a KV head)", d->H, c.KV);
  if (d->ldq < (uint64_t)d->H * c.HD || d->ldo < (uint64_t)d->H * c.HD)
    return corm::fail(CORM_EINVAL, "corm_llm_paged_attn: row strides below the row length");
  if (((uintptr_t)d->smx & 3u) || (((uintptr_t)d->q | (uintptr_t)d->o) & 1u))
    return corm::fail(CORM_EINVAL, "corm_llm_paged_attn: unaligned buffers");
  if (int rc = corm::check_device()) return rc;
  const corm::DeviceTables* tb = corm::tables();
  if (!tb) return CORM_ECUDA;
  SplitArgs A{};
  A.d = *d;
  A.d.max_q = d->max_q < c.rows ? d->max_q : c.rows;
  A.tab = tb->smx_tab;
  A.err = corm::device_error_word();
  if (!A.err) return CORM_ECUDA;
  A.waits = paged::waits();
  A.G = d->H / c.KV;
  const uint64_t rows = (uint64_t)A.d.max_q * A.G;
  A.rcap = rows < kRows ? (uint32_t)rows : kRows;
  const uint64_t tiles = (rows + kRows - 1u) / kRows;
  if (tiles > (1ull << 27)) return corm::fail(CORM_ELIMIT, "corm_llm_paged_attn: max_q %u", d->max_q);
  cudaStream_t st = (cudaStream_t)stream;
  // this form or 128-row tiles: up to 32 rows a sequence and KV head this one (8 rows cost
  // it the time that 128 cost the other).  Beyond, where its CTAs leave SMs idle (8 groups
  // of 600 keys: 128 rows 14 us against 37), and up to 64 rows where they are at once
  // resident (32 groups of 600: 64 rows 16 us against 31) or the other's scores do not fit
  // (128 groups of 4000: 64 rows 223 us against 229, 40 rows 151 against 243; of 600, 64
  // rows: 52 against 45)
  const uint32_t cap = c.table_width * c.page, span = A.d.window ? A.d.window + A.d.max_q : cap;
  const uint32_t keys = min(A.d.max_keys, min(cap, span < A.d.window ? cap : span));
  const uint64_t ctas = paged::live_tiles(A.d, kRows, tiles);
  const bool few = rows <= 32u || (rows <= 64u && (keys > 640u || ctas <= 444u)) || (rows <= 128u && ctas <= 148u);
  if (!few && paged::tile_takes(A.d)) return paged::launch_tiles(A.d, A.tab, A.err, st);
  switch (c.HD * 2u + (c.bits == 8u)) {
    case 32: return launch_split<16, 16>(A, (uint32_t)tiles, st);
    case 33: return launch_split<16, 8>(A, (uint32_t)tiles, st);
    case 64: return launch_split<32, 16>(A, (uint32_t)tiles, st);
    case 65: return launch_split<32, 8>(A, (uint32_t)tiles, st);
    case 128: return launch_split<64, 16>(A, (uint32_t)tiles, st);
    case 129: return launch_split<64, 8>(A, (uint32_t)tiles, st);
    case 256: return launch_split<128, 16>(A, (uint32_t)tiles, st);
    case 257: return launch_split<128, 8>(A, (uint32_t)tiles, st);
    case 512: return launch_split<256, 16>(A, (uint32_t)tiles, st);
    default: return launch_split<256, 8>(A, (uint32_t)tiles, st);
  }
}
