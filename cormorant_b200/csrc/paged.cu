// The paged KV cache's operators (see the header's section on it): the row
// preparation that norms, rotates and writes, the read-back, and the attention
// of few rows a sequence.
#include "paged.cuh"

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
// A group of HD / 8 lanes per (row, head slot), a lane holding the 8 elements of
// four pairs; a thread keeps its slot over all its rows (the grid's step is a
// multiple of the slots), so its entries are decoded once.  Norm: the squares'
// sum by shuffles over the group, the divisor by the unit's table and Newton
// step, 64-bit throughout (D < 2^63, |x Rm| < 2^48, |P1 G| < 2^56).
struct PrepArgs {
  corm_llm_paged_prep_desc d;
  const uint32_t* rsq;
  uint32_t vec;  // 8-byte loads and stores are aligned and whole
};

// the row-ops unit's 1 / sqrt(D) ~ Rm 2^-sh for 1 <= D < 2^63
__device__ __forceinline__ void rsqrt64(uint64_t D, uint64_t& Rm, int& sh, const uint32_t* __restrict__ rsq) {
  int d = 32 - __clzll((long long)D);
  if (d & 1) d += 1;
  const uint64_t Dm = d >= 0 ? D >> d : D << -d;  // < 2^32
  const uint64_t y0 = __ldg(rsq + (Dm >> 19));
  const uint64_t u = (((Dm * y0) >> 32) * y0) >> 32;
  // |y0 (2^30 - u)| < 2^62: the table's y0 is within 2^-13 of 1 / sqrt
  int64_t y1 = (int64_t)y0 + (((int64_t)y0 * ((1ll << 30) - (int64_t)u)) >> 31);
  y1 = max(y1, (int64_t)1 << 31);
  Rm = (uint64_t)min(y1, ((int64_t)1 << 32) - 1);
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
// 2^40: k >= 9, or an element that is not rotated): both roundings (floor for the
// parity, then the result) are one funnel shift each.  half1 = 2^(k - 1) - 1 and
// par = 1, both 0 for k = 0
__device__ __forceinline__ int32_t rot_plain(int32_t x, int32_t cs, int32_t y, int32_t sn, uint32_t k, uint32_t half1,
                                             uint32_t par) {
  const int64_t v = (int64_t)x * cs + (int64_t)y * sn;
  const uint32_t odd = __funnelshift_r((uint32_t)v, (uint32_t)(v >> 32), k) & par;
  const int64_t u = v + (int64_t)(half1 + odd);
  return (int32_t)__funnelshift_r((uint32_t)u, (uint32_t)(u >> 32), k);
}

template <int HD, bool VEC, bool NORM>
__global__ void __launch_bounds__(256, 3) paged_prep_kernel(const __grid_constant__ PrepArgs A) {
  corm_pdl_wait();
  corm_pdl_trigger();
  constexpr uint32_t LPH = HD / 8;     // lanes per head
  constexpr uint32_t SPB = 256 / LPH;  // heads per block and pass
  const corm_llm_paged_prep_desc& d = A.d;
  const corm_paged_cache& c = d.c;
  const uint32_t KV = c.KV, slots = d.H + 2u * KV;
  const uint32_t lane = threadIdx.x % LPH;
  const uint64_t item0 = (uint64_t)blockIdx.x * SPB + threadIdx.x / LPH, step = (uint64_t)gridDim.x * SPB;  // step % slots == 0
  const uint32_t slot = (uint32_t)(item0 % slots);
  const uint32_t row_step = (uint32_t)(step / slots);
  const bool is_q = slot < d.H, is_v = slot >= d.H + KV;
  const uint32_t head = is_q ? slot : (is_v ? slot - d.H - KV : slot - d.H);
  const uint32_t rot = is_v ? 0u : d.rot, hr = rot / 2u;
  // the dimensions of this lane's pairs: a rotated pair p at (p, p + rot / 2) or
  // (2 p, 2 p + 1); the rest of the head in neighbouring pairs
  uint32_t da[4], db[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const uint32_t p = 4u * lane + k;
    const bool split = p < hr && !d.interleaved;
    da[k] = split ? p : 2u * p;
    db[k] = split ? p + hr : 2u * p + 1u;
  }
  const bool spl = 4u * lane < hr && !d.interleaved;  // VEC: alike for the lane's four pairs
  // the usual entries: no up-shift and one down-shift for the lane's elements, whose
  // quotients fit 32 bits; any others are read again where they are used
  const uint8_t* ent = (const uint8_t*)(is_q ? d.pq : (is_v ? d.pv : d.pk));
  const bool bc = d.flags & (is_q ? 1u : (is_v ? 4u : 2u)), direct = is_v && (d.flags & 8u);
  auto shifts = [&](uint32_t dim) -> uint32_t {  // sh_a | sh_b << 8 | sh_c << 16
    return direct ? 0u : *(const uint32_t*)(ent + 16ull * (bc ? 0u : head * HD + dim) + 8) & 0x3F3F3Fu;
  };
  const uint32_t k0 = shifts(da[0]), kd = k0 >> 16;
  bool plain = (k0 & 0xFFFFu) == 0u && kd <= 31u && (kd >= 9u || 4u * lane >= hr);
#pragma unroll
  for (int k = 0; k < 4; k++) plain = plain && shifts(da[k]) == k0 && shifts(db[k]) == k0;
  const uint32_t half1 = kd ? (1u << (kd & 31u)) / 2u - 1u : 0u, par = kd ? 1u : 0u;
  const uint8_t* ne = (const uint8_t*)(is_q ? d.nq : (is_v ? nullptr : d.nk));
  int32_t ga[4], gb[4];
  uint32_t na = 0, nb = 0;  // the norm's down-shifts, a byte each
  if (NORM && ne) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint8_t* ea = ne + 16u * da[k];
      const uint8_t* eb = ne + 16u * db[k];
      ga[k] = *(const int32_t*)ea;
      gb[k] = *(const int32_t*)eb;
      na |= (ea[10] & 63u) << (8 * k);
      nb |= (eb[10] & 63u) << (8 * k);
    }
  }
  const uint64_t eps = is_q ? d.eps_q : d.eps_k;
  const int16_t* src = is_q ? d.q0 : (is_v ? d.v0 : d.k0);
  const uint64_t ld = is_q ? d.ldq0 : (is_v ? d.ldv : d.ldk);
  const unsigned mask = LPH == 32 ? 0xffffffffu : ((1u << LPH) - 1u) << ((threadIdx.x & 31u) / LPH * LPH);
  const int32_t total = c.cu[c.B];
  const uint64_t rows = min((uint64_t)c.rows, (uint64_t)max(total, 0));
  // the sequence of the first row: the last b with cu[b] <= row (cu ascends), then
  // forward as the rows do
  uint32_t b = 0;
  {
    uint32_t hi = c.B;  // the answer lies in [b, hi)
    const int64_t r = (int64_t)(item0 / slots);
    while (hi - b > 1u) {
      const uint32_t mid = (b + hi) / 2u;
      if ((int64_t)c.cu[mid] <= r) b = mid;
      else hi = mid;
    }
  }
  for (uint64_t row = item0 / slots; row < rows; row += row_step) {
    while (b + 1u < c.B && (int64_t)c.cu[b + 1] <= (int64_t)row) b++;
    const SeqRows s = seq_rows(c, b, c.rows);
    if (row < s.lo || row >= s.lo + s.n) continue;  // a row of no sequence (alike over the group)
    const uint64_t p = (uint64_t)s.pos + (row - s.lo);
    const int16_t* x = src + row * ld + (uint64_t)head * HD;
    int32_t va[4], vb[4];
    if (VEC) {
      uint2 w0, w1;
      if (spl) {
        w0 = *(const uint2*)(x + 4u * lane);
        w1 = *(const uint2*)(x + 4u * lane + hr);
      } else {
        w0 = *(const uint2*)(x + 8u * lane);
        w1 = *(const uint2*)(x + 8u * lane + 4u);
      }
      const int32_t v8[8] = {(int16_t)w0.x, (int32_t)w0.x >> 16, (int16_t)w0.y, (int32_t)w0.y >> 16,
                             (int16_t)w1.x, (int32_t)w1.x >> 16, (int16_t)w1.y, (int32_t)w1.y >> 16};
#pragma unroll
      for (int k = 0; k < 4; k++) {
        va[k] = spl ? v8[k] : v8[2 * k];
        vb[k] = spl ? v8[4 + k] : v8[2 * k + 1];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        va[k] = x[da[k]];
        vb[k] = x[db[k]];
      }
    }
    if (NORM && ne) {
      uint64_t s2 = 0;
#pragma unroll
      for (int k = 0; k < 4; k++) s2 += (uint64_t)(uint32_t)(va[k] * va[k]) + (uint32_t)(vb[k] * vb[k]);
#pragma unroll
      for (uint32_t o = LPH / 2; o > 0; o >>= 1) s2 += __shfl_xor_sync(mask, s2, o);
      uint64_t Rm;
      int sh;
      rsqrt64(max(s2 + eps, (uint64_t)1), Rm, sh, A.rsq);
      sh -= 24;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        va[k] = (int32_t)corm_sat16(corm_rne_shr64f((((int64_t)va[k] * (int64_t)Rm) >> sh) * ga[k], (int)(na >> (8 * k)) & 63));
        vb[k] = (int32_t)corm_sat16(corm_rne_shr64f((((int64_t)vb[k] * (int64_t)Rm) >> sh) * gb[k], (int)(nb >> (8 * k)) & 63));
      }
    }
    const int32_t* tr = d.rope + (uint64_t)min(p, (uint64_t)(d.rope_rows - 1u)) * d.rot;
    int32_t cs[4], sn[4];
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
    if (plain) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int32_t a = va[k], bb = vb[k];
        va[k] = min(max(rot_plain(a, cs[k], -bb, sn[k], kd, half1, par), -32768), 32767);
        vb[k] = min(max(rot_plain(bb, cs[k], a, sn[k], kd, half1, par), -32768), 32767);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int32_t a = va[k], bb = vb[k];
        va[k] = rot_any(a, cs[k], -bb, sn[k], shifts(da[k]));
        vb[k] = rot_any(bb, cs[k], a, sn[k], shifts(db[k]));
      }
    }
    if (is_q) {
      int16_t* y = d.q + row * d.ldq + (uint64_t)head * HD;
      if (VEC) {
        if (spl) {
          *(uint2*)(y + 4u * lane) = make_uint2(pack16(va[0], va[1]), pack16(va[2], va[3]));
          *(uint2*)(y + 4u * lane + hr) = make_uint2(pack16(vb[0], vb[1]), pack16(vb[2], vb[3]));
        } else {
          *(uint2*)(y + 8u * lane) = make_uint2(pack16(va[0], vb[0]), pack16(va[1], vb[1]));
          *(uint2*)(y + 8u * lane + 4u) = make_uint2(pack16(va[2], vb[2]), pack16(va[3], vb[3]));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
          y[da[k]] = (int16_t)va[k];
          y[db[k]] = (int16_t)vb[k];
        }
      }
      continue;
    }
    uint32_t shift = 0;
    if (c.bits == 8u) {  // (every lane of the group, also where nothing is written)
      uint32_t t = 0;
#pragma unroll
      for (int k = 0; k < 4; k++) t = max(t, max((uint32_t)(va[k] ^ (va[k] >> 31)), (uint32_t)(vb[k] ^ (vb[k] >> 31))));
#pragma unroll
      for (uint32_t o = LPH / 2; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(mask, t, o));
      const int bits = 32 - __clz((int)t);
      shift = bits > 7 ? (uint32_t)(bits - 7) : 0u;
      // RNE by shift <= 8; only the upper end can round past the codes
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int32_t h = (1 << shift) >> 1, r = h ? h - 1 : 0;
        va[k] = min((va[k] + r + (h ? (va[k] >> shift) & 1 : 0)) >> shift, 127);
        vb[k] = min((vb[k] + r + (h ? (vb[k] >> shift) & 1 : 0)) >> shift, 127);
      }
    }
    if (p >= s.cap) continue;
    const int32_t pg = c.table[(uint64_t)b * c.table_width + p / c.page];
    if ((uint32_t)pg >= c.pages) continue;
    const uint64_t line = ((uint64_t)pg * KV + head) * c.page + p % c.page;
    int8_t* y = (is_v ? c.vc : c.kc) + line * (c.bits == 8u ? HD : 2 * HD);
    if (VEC) {
      uint32_t w[4];  // bytes of va, of vb: low (or code), then high
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const int32_t* v = q ? vb : va;
        const uint32_t l0 = pack16(v[0], v[1]), l1 = pack16(v[2], v[3]);
        w[q] = __byte_perm(l0, l1, 0x6420);
        w[2 + q] = __byte_perm(l0, l1, 0x7531);
      }
#pragma unroll
      for (int pl = 0; pl < 2; pl++) {  // low bytes (codes), high bytes
        if (pl && c.bits == 8u) break;
        int8_t* yp = y + (c.bits == 8u || pl ? 0 : HD);
        if (spl) {
          *(uint32_t*)(yp + 4u * lane) = w[2 * pl];
          *(uint32_t*)(yp + 4u * lane + hr) = w[2 * pl + 1];
        } else {
          *(uint2*)(yp + 8u * lane) =
              make_uint2(__byte_perm(w[2 * pl], w[2 * pl + 1], 0x5140), __byte_perm(w[2 * pl], w[2 * pl + 1], 0x7362));
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if (c.bits == 8u) {
          y[da[k]] = (int8_t)va[k];
          y[db[k]] = (int8_t)vb[k];
        } else {
          y[da[k]] = (int8_t)(va[k] >> 8);
          y[db[k]] = (int8_t)(vb[k] >> 8);
          y[HD + da[k]] = (int8_t)va[k];
          y[HD + db[k]] = (int8_t)vb[k];
        }
      }
    }
    if (c.bits == 8u && lane == 0) (is_v ? c.vs : c.ks)[line] = (uint8_t)shift;
  }
}

// ---------------------------------------------------------------- read-back
// A lane per 8 elements of (row, KV head, K or V): 8-byte loads of each plane,
// one 16-byte store (8-byte stores where the output is not on 16 bytes).
template <int HD>
__global__ void __launch_bounds__(256) paged_read_kernel(const __grid_constant__ corm_llm_paged_read_desc d, uint32_t vec) {
  corm_pdl_wait();
  corm_pdl_trigger();
  constexpr uint32_t LPH = HD / 8;
  const corm_paged_cache& c = d.c;
  const uint32_t slots = 2u * c.KV;
  const int32_t last = c.cu[c.B];
  const uint64_t rows = min((uint64_t)c.rows, (uint64_t)max(last, 0));
  const uint64_t total = rows * slots * LPH;
  uint32_t b = 0;
  bool first = true;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256u) {
    const uint32_t lane = (uint32_t)(i % LPH);
    const uint64_t it = i / LPH;
    const uint64_t row = it / slots;
    const uint32_t slot = (uint32_t)(it - row * slots);
    if (first) {
      uint32_t hi = c.B;
      while (hi - b > 1u) {
        const uint32_t mid = (b + hi) / 2u;
        if ((int64_t)c.cu[mid] <= (int64_t)row) b = mid;
        else hi = mid;
      }
      first = false;
    }
    while (b + 1u < c.B && (int64_t)c.cu[b + 1] <= (int64_t)row) b++;
    const bool is_v = slot >= c.KV;
    int16_t* out = is_v ? d.v : d.k;
    if (!out) continue;
    const SeqRows s = seq_rows(c, b, c.rows);
    if (row < s.lo || row >= s.lo + s.n) continue;
    const uint32_t g = is_v ? slot - c.KV : slot;
    const uint64_t p = (uint64_t)s.pos + (row - s.lo);
    const int32_t pg = p < s.cap ? c.table[(uint64_t)b * c.table_width + p / c.page] : -1;
    uint32_t w[4] = {0, 0, 0, 0};
    if ((uint32_t)pg < c.pages) {
      const uint64_t line = ((uint64_t)pg * c.KV + g) * c.page + p % c.page;
      const int8_t* y = (is_v ? c.vc : c.kc) + line * (c.bits == 8u ? HD : 2 * HD) + 8u * lane;
      const uint2 h = *(const uint2*)y;
      if (c.bits == 8u) {
        const uint32_t sh = (is_v ? c.vs : c.ks)[line];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t q = k < 2 ? h.x : h.y;
          const int32_t v0 = (int8_t)(q >> (16 * (k & 1))), v1 = (int8_t)(q >> (16 * (k & 1) + 8));
          w[k] = pack16(sh < 16u ? v0 << sh : 0, sh < 16u ? v1 << sh : 0);
        }
      } else {
        const uint2 l = *(const uint2*)(y + HD);
        w[0] = __byte_perm(l.x, h.x, 0x5140);
        w[1] = __byte_perm(l.x, h.x, 0x7362);
        w[2] = __byte_perm(l.y, h.y, 0x5140);
        w[3] = __byte_perm(l.y, h.y, 0x7362);
      }
    }
    int16_t* o = out + row * (is_v ? d.ldv : d.ldk) + (uint64_t)g * HD + 8u * lane;
    if (vec) {
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

// ---------------------------------------------------------------- attention, few rows
// A cluster of X CTAs per (sequence, KV head, 16 rows), a row being (token,
// head of the group), token-major; the CTAs share the keys.  The unit's e(d) is
// a table of d = m - score, so sums cannot be rescaled as a running maximum
// moves; instead the scores stay on the chip: every CTA forms those of its keys
// once (int16 in shared memory), the maxima meet over the cluster, then e in
// place and the sums meet, then P in place and P.V over the V rows, whose
// partial sums (modulo 2^32, so in any order) meet last.  K and V are read once.
// Keys beyond the shared memory: windows, the scores formed again in each of
// the three passes.
//
// A ninth warp copies the pages (64 keys a stage, one bulk copy per page piece)
// into a ring, running ahead across the phases, so the V rows arrive under the
// softmax.  Warp-level MMAs: the 16-row tile is far below the 128 rows of a
// tcgen05 tile, and the copies bound the kernel.  The contraction over HD takes
// the dimensions in the order in which a lane's 16-byte pieces hold them (the q
// fragments alike); V's bytes are transposed 4 x 4 in registers.
constexpr uint32_t kT = 64;       // keys of a stage
constexpr uint32_t kRows = 16;    // rows of a tile
constexpr uint32_t kWarps = 8;    // computing warps
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kSplitRows = 32;  // rows of a sequence and KV head up to which this form runs

struct SplitArgs {
  corm_llm_paged_attn_desc d;
  const int32_t* tab;
  int* err;
  uint32_t G, X, stages, win, rcap;  // win: tiles of a window; rcap: rows held
};

template <int HD, int BITS>
struct SplitShape {
  static constexpr uint32_t RB = HD * (BITS / 8);                     // bytes of a cached row
  static constexpr uint32_t STB = kT * RB + (BITS == 8 ? 128u : 0u);  // a stage (its shifts last)
  static constexpr uint32_t NKS = HD < 32 ? 1 : HD / 32;              // MMA steps of a score
  static constexpr uint32_t DW = HD < 32 ? HD : 32;                   // output dimensions of a warp
  static constexpr uint32_t DG = HD / DW, KG = kWarps / DG;           // dimension and key groups of warps
  static constexpr uint32_t NT = DW / 8;
};
__host__ __device__ constexpr uint32_t split_pitch(uint32_t win) { return win * kT + 16u; }  // int16 of a score row

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int HD, int BITS>
__global__ void __launch_bounds__(288, HD <= 128 ? 2 : 1) paged_attn_split_kernel(const __grid_constant__ SplitArgs A) {
  using Sh = SplitShape<HD, BITS>;
  constexpr uint32_t RB = Sh::RB, STB = Sh::STB, NKS = Sh::NKS, DW = Sh::DW, DG = Sh::DG, KG = Sh::KG, NT = Sh::NT;
  extern __shared__ __align__(128) uint8_t pa_sm[];
  __shared__ uint64_t full[8], empty[8], cbar;
  __shared__ int32_t s_wmax[kWarps][kRows], s_m[kRows], s_gm[kRows];
  __shared__ unsigned long long s_s[kRows];
  __shared__ uint32_t s_R[kRows], s_lo[kRows], s_hi[kRows], s_cm[kRows], s_cs[kRows], s_fp[kRows];
  const corm_paged_cache& c = A.d.c;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t X = A.X, tile = blockIdx.x / X, rank = blockIdx.x % X, g = blockIdx.y, b = blockIdx.z, G = A.G;
  const uint32_t NST = A.stages;
  uint8_t* ring = pa_sm;
  int16_t* S = (int16_t*)(ring + NST * STB);
  const uint32_t pitch = split_pitch(A.win);
  uint32_t* s_O = (uint32_t*)(S + A.rcap * pitch);
  uint16_t* tab = (uint16_t*)(s_O + A.rcap * HD);
  if (tid == 0) {
    for (uint32_t i = 0; i < NST; i++) {
      sm100::mbar_init(&full[i], 1);
      sm100::mbar_init(&empty[i], kWarps);
    }
    sm100::mbar_init(&cbar, X);
    sm100::fence_mbar_init();
  }
  corm_pdl_wait();
  corm_pdl_trigger();
  const SeqRows sq = seq_rows(c, b, c.rows);
  const uint32_t n = min(sq.n, A.d.max_q), r0 = tile * kRows;
  if ((uint64_t)r0 >= (uint64_t)n * G) return;  // the cluster's CTAs alike
  const uint32_t nr = min(kRows, n * G - r0);
  const uint32_t i0 = r0 / G, i1 = (r0 + nr - 1u) / G;
  // the keys some row of the tile sees: [lo, hi), in tiles from lo rounded down
  const uint32_t hi = min(sq.pos + i1 + 1u, sq.cap);
  const uint32_t w = A.d.window;
  const uint32_t lo = (w && sq.pos + i0 + 1u > w) ? sq.pos + i0 + 1u - w : 0u;
  const uint32_t tile0 = lo / kT, ntile = hi > lo ? (hi + kT - 1u) / kT - tile0 : 0u;
  const uint32_t per = (ntile + X - 1u) / X;
  const uint32_t t0 = tile0 + min(rank * per, ntile), t1 = tile0 + min(rank * per + per, ntile);
  const uint32_t nwin = (t1 - t0 + A.win - 1u) / A.win;
  if (X > 1) cluster_sync();
  else __syncthreads();

  if (warp == kWarps) {
    // ---------------- the copies
    const uint32_t sub = min(c.page, kT), pieces = kT / sub;
    const int32_t* tb = c.table + (uint64_t)b * c.table_width;
    const uint32_t psh = 31u - __clz(c.page);
    uint32_t gi = 0, base = 0xFFFFFF00u;
    int32_t ids = -1;
    bool ok = true;
    auto emit = [&](bool is_v, uint32_t t) {
      const uint32_t s = gi % NST;
      if (gi >= NST && ok) ok = wait_for(&empty[s], ((gi / NST) - 1u) & 1u, A.err, 301);
      ok = __all_sync(0xffffffffu, ok);
      gi++;
      if (!ok) return;
      const uint32_t b0 = (t * kT) >> psh, b1 = (t * kT + kT - 1u) >> psh;
      if (b0 < base || b1 >= base + 32u) {  // 32 table entries at a time
        base = b0;
        ids = base + lane < c.table_width ? tb[base + lane] : -1;
      }
      const uint32_t key = t * kT + lane * sub;
      const bool in = lane < pieces && key < hi;
      const int32_t id = __shfl_sync(0xffffffffu, ids, in ? (key >> psh) - base : 0u);
      const bool good = in && (uint32_t)id < c.pages;
      uint8_t* dst = ring + s * STB + lane * sub * RB;
      if (in && !good) {  // a page of zeros
        for (uint32_t i = 0; i < sub * RB; i += 16u) *(int4*)(dst + i) = make_int4(0, 0, 0, 0);
        if (BITS == 8)
          for (uint32_t i = 0; i < sub; i += 16u) *(int4*)(ring + s * STB + kT * RB + lane * sub + i) = make_int4(0, 0, 0, 0);
        sm100::fence_proxy_async_smem();
      }
      const uint32_t cnt = __popc(__ballot_sync(0xffffffffu, good));
      if (lane == 0) sm100::mbar_expect_tx(&full[s], cnt * sub * (RB + (BITS == 8 ? 1u : 0u)));
      __syncwarp();
      if (good) {
        const uint64_t line = ((uint64_t)(uint32_t)id * c.KV + g) * c.page + (key & (c.page - 1u));
        bulk_g2s(dst, (is_v ? c.vc : c.kc) + line * RB, sub * RB, &full[s]);
        if (BITS == 8) bulk_g2s(ring + s * STB + kT * RB + lane * sub, (is_v ? c.vs : c.ks) + line, sub, &full[s]);
      }
    };
    // K (v = 0) for the first pass and, in windows, again for the other two; V (v = 1)
    // behind each window's K of the last
#pragma unroll 1
    for (uint32_t pass = 0; pass < 3; pass++)
#pragma unroll 1
      for (uint32_t a = t0; a < t1; a += A.win)
#pragma unroll 1
        for (uint32_t v = (pass == 0 || nwin > 1) ? 0u : 1u; v < (pass == 2 ? 2u : 1u); v++)
#pragma unroll 1
          for (uint32_t t = a; t < min(a + A.win, t1); t++) emit(v == 1u, t);
    // every copy lands before the CTA's shared memory goes away
    for (uint32_t q = gi > NST ? gi - NST : 0u; ok && q < gi; q++)
      wait_for(&full[q % NST], (q / NST) & 1u, nullptr, 0);
    __syncwarp();
    if (X > 1) cluster_sync();
    return;
  }

  // ---------------- the rows
  if (tid < kRows) {
    const uint32_t rr = r0 + min(tid, nr - 1u), i = rr / G, h = g * G + rr % G;
    const uint32_t p = sq.pos + i;
    s_hi[tid] = min(p + 1u, sq.cap);
    s_lo[tid] = (w && p + 1u > w) ? p + 1u - w : 0u;
    s_cm[tid] = A.d.smx[2u * h];
    const uint32_t cfg = A.d.smx[2u * h + 1u];
    s_cs[tid] = cfg & 63u;
    s_fp[tid] = (cfg >> 8) & 31u;
    s_s[tid] = 0;
  }
  for (uint32_t i = tid; i < 4096u; i += 256u) tab[i] = (uint16_t)(A.tab[i] - 1);
  for (uint32_t i = tid; i < nr * HD; i += 256u) s_O[i] = 0;
  const uint32_t qn = lane >> 2, qt = lane & 3u;  // a fragment's row (and row + 8; a key; a column) and quarter
  uint32_t ah[NKS][4], al[NKS][4];
#pragma unroll
  for (uint32_t ks = 0; ks < NKS; ks++)
#pragma unroll
    for (uint32_t x = 0; x < 4; x++) {
      const uint32_t row = qn + 8u * (x & 1u), half = x >> 1;  // a0: row, a1: row + 8, a2 / a3: the second half
      // word v of the lane's pieces: dimensions 64 (v / 4) + 16 t + 4 (v % 4) (rows of 64 up)
      const uint32_t v = 2u * ks + half;
      const uint32_t dim = HD >= 64 ? 64u * (v >> 2) + 16u * qt + 4u * (v & 3u) : (HD == 32 ? 8u * qt + 4u * half : 4u * qt);
      ah[ks][x] = al[ks][x] = 0;
      if (row < nr && (HD > 16 || half == 0)) {
        const uint32_t rr = r0 + row;
        const int16_t* q = A.d.q + (uint64_t)(sq.lo + rr / G) * A.d.ldq + (uint64_t)(g * G + rr % G) * HD + dim;
        const uint32_t x0 = pack16(q[0], q[1]), x1 = pack16(q[2], q[3]);
        ah[ks][x] = __byte_perm(x0, x1, 0x7531);
        al[ks][x] = __byte_perm(x0, x1, 0x6420);
      }
    }
  consumer_sync();
  const uint32_t lo0 = s_lo[qn], hi0 = qn < nr ? s_hi[qn] : 0u, lo1 = s_lo[qn + 8u], hi1 = qn + 8u < nr ? s_hi[qn + 8u] : 0u;
  uint32_t gi = 0;
  bool ok = true;
  // the scores of tile t into the window's rows; the running maxima of the keys each row sees
  int32_t mx0 = INT32_MIN, mx1 = INT32_MIN;
  auto scores = [&](uint32_t t, uint32_t a) {
    const uint32_t s = gi % NST;
    if (ok) ok = wait_for(&full[s], (gi / NST) & 1u, A.err, 302);
    __syncwarp();
    gi++;
    const uint8_t* row = ring + s * STB + (8u * warp + qn) * RB;
    uint32_t hh[4] = {0, 0, 0, 0}, mid[4] = {0, 0, 0, 0}, ll[4] = {0, 0, 0, 0};
    if (HD >= 64) {
#pragma unroll
      for (uint32_t k = 0; k < (HD >= 64 ? HD / 64 : 1); k++) {
        const uint8_t* p = row + 64u * k + 16u * qt;
        uint4 h, l = make_uint4(0, 0, 0, 0);
        if (BITS == 16) {  // odd keys take the planes in the other order: no bank is asked twice
          const uint4 u = *(const uint4*)(p + ((qn & 1u) ? HD : 0)), v = *(const uint4*)(p + ((qn & 1u) ? 0 : HD));
          h = (qn & 1u) ? v : u;
          l = (qn & 1u) ? u : v;
        } else {
          h = *(const uint4*)p;
        }
        const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
        for (uint32_t j = 0; j < 2; j++) {
          const uint32_t ks = NKS > 1 ? 2u * k + j : 0u;
          mma_ss(hh, ah[ks], hw[2 * j], hw[2 * j + 1]);
          mma_us(mid, al[ks], hw[2 * j], hw[2 * j + 1]);
          if (BITS == 16) {
            mma_su(mid, ah[ks], lw[2 * j], lw[2 * j + 1]);
            mma_uu(ll, al[ks], lw[2 * j], lw[2 * j + 1]);
          }
        }
      }
    } else {
      uint32_t h0, h1 = 0, l0 = 0, l1 = 0;
      if (HD == 32) {
        const uint2 u = *(const uint2*)(row + 8u * qt);
        h0 = u.x, h1 = u.y;
        if (BITS == 16) {
          const uint2 v = *(const uint2*)(row + HD + 8u * qt);
          l0 = v.x, l1 = v.y;
        }
      } else {
        h0 = *(const uint32_t*)(row + 4u * qt);
        if (BITS == 16) l0 = *(const uint32_t*)(row + HD + 4u * qt);
      }
      mma_ss(hh, ah[0], h0, h1);
      mma_us(mid, al[0], h0, h1);
      if (BITS == 16) {
        mma_su(mid, ah[0], l0, l1);
        mma_uu(ll, al[0], l0, l1);
      }
    }
    uint32_t s0 = 0, s1 = 0;
    if (BITS == 8) {
      const uint32_t sh = *(const uint16_t*)(ring + s * STB + kT * RB + 8u * warp + 2u * qt);
      s0 = sh & 31u;
      s1 = (sh >> 8) & 31u;
    }
    __syncwarp();
    if (lane == 0) sm100::mbar_arrive(&empty[s]);
    int32_t v[4];
#pragma unroll
    for (int x = 0; x < 4; x++) {
      uint32_t acc = BITS == 16 ? (hh[x] << 16) + (mid[x] << 8) + ll[x] : ((hh[x] << 8) + mid[x]) << ((x & 1) ? s1 : s0);
      v[x] = out16(acc);
    }
    const uint32_t key = t * kT + 8u * warp + 2u * qt;
    if (key >= lo0 && key < hi0) mx0 = max(mx0, v[0]);
    if (key + 1u >= lo0 && key + 1u < hi0) mx0 = max(mx0, v[1]);
    if (key >= lo1 && key < hi1) mx1 = max(mx1, v[2]);
    if (key + 1u >= lo1 && key + 1u < hi1) mx1 = max(mx1, v[3]);
    int16_t* d = S + (t - a) * kT + 8u * warp + 2u * qt;
    if (qn < nr) *(uint32_t*)(d + qn * pitch) = pack16(v[0], v[1]);
    if (qn + 8u < nr) *(uint32_t*)(d + (qn + 8u) * pitch) = pack16(v[2], v[3]);
  };
  uint32_t cphase = 0;
  // every CTA of the cluster is here, and what it wrote before is visible
  auto cluster_meet = [&]() {
    consumer_sync();
    if (X > 1) {
      if (tid < X) mbar_arrive_remote(&cbar, tid);
      if (ok) ok = mbar_wait_cluster(&cbar, cphase, A.err, 303);
      cphase ^= 1u;
    }
  };

  // pass 1: the maxima
  for (uint32_t a = t0; a < t1; a += A.win)
    for (uint32_t t = a; t < min(a + A.win, t1); t++) scores(t, a);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    mx0 = max(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
    mx1 = max(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
  }
  if (qt == 0) {
    s_wmax[warp][qn] = mx0;
    s_wmax[warp][qn + 8u] = mx1;
  }
  consumer_sync();
  if (tid < kRows) {
    int32_t m = s_wmax[0][tid];
    for (uint32_t i = 1; i < kWarps; i++) m = max(m, s_wmax[i][tid]);
    s_m[tid] = m;
  }
  cluster_meet();
  if (tid < kRows) {
    int32_t m = s_m[tid];
    if (X > 1)
      for (uint32_t i = 0; i < X; i++) m = max(m, (int32_t)cluster_ld32(cluster_addr(&s_m[tid], i)));
    s_gm[tid] = m;
  }
  consumer_sync();

  // rows over the warps: one each from eight rows on, else wpr warps a row
  const uint32_t wpr = nr > 4u ? 1u : (nr > 2u ? 2u : (nr > 1u ? 4u : 8u)), wgr = kWarps / wpr;
  const uint32_t rw = warp / wpr, rl = (warp % wpr) * 32u + lane, rstep = 32u * wpr;
  // pass 2: e of the window [a, e) in place (or only its sum), the sum of the row r
  auto e_pass = [&](uint32_t a, uint32_t e, bool keep) {
    for (uint32_t r = rw; r < nr; r += wgr) {
      uint32_t* row = (uint32_t*)(S + r * pitch);
      const uint32_t cm = s_cm[r], cs = s_cs[r], klo = s_lo[r], khi = s_hi[r];
      const int32_t m = s_gm[r];
      const SmxScale sc = smx_scale(cm, max(cs, 8u));
      unsigned long long sum = 0;
      for (uint32_t i = rl; i < (e - a) * (kT / 2u); i += rstep) {
        const uint32_t x = row[i], key = a * kT + 2u * i;
        uint32_t e0 = 0, e1 = 0;
        const uint32_t d0 = (uint32_t)(m - (int32_t)(int16_t)x), d1 = (uint32_t)(m - ((int32_t)x >> 16));
        if (key >= klo && key < khi) e0 = cs >= 8u ? smx_e(d0, sc, tab) : smx_e_wide(d0, cm, cs, tab);
        if (key + 1u >= klo && key + 1u < khi) e1 = cs >= 8u ? smx_e(d1, sc, tab) : smx_e_wide(d1, cm, cs, tab);
        sum += e0 + e1;
        if (keep) row[i] = e_pack(e0) | (e_pack(e1) << 16);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0 && sum) atomicAdd(&s_s[r], sum);
    }
  };
  // pass 3: P of the window in place, from e (one window) or from the scores
  auto p_pass = [&](uint32_t a, uint32_t e, bool from_e) {
    for (uint32_t r = rw; r < nr; r += wgr) {
      uint32_t* row = (uint32_t*)(S + r * pitch);
      const uint32_t cm = s_cm[r], cs = s_cs[r], fp = s_fp[r], R = s_R[r], klo = s_lo[r], khi = s_hi[r];
      const int32_t m = s_gm[r];
      const SmxScale sc = smx_scale(cm, max(cs, 8u));
      for (uint32_t i = rl; i < (e - a) * (kT / 2u); i += rstep) {
        const uint32_t x = row[i], key = a * kT + 2u * i;
        const bool v0 = key >= klo && key < khi, v1 = key + 1u >= klo && key + 1u < khi;
        uint32_t e0 = e_unpack(x & 0xFFFFu), e1 = e_unpack(x >> 16);
        if (!from_e) {
          const uint32_t d0 = (uint32_t)(m - (int32_t)(int16_t)x), d1 = (uint32_t)(m - ((int32_t)x >> 16));
          e0 = cs >= 8u ? smx_e(d0 & 0xFFFFu, sc, tab) : smx_e_wide(d0 & 0xFFFFu, cm, cs, tab);
          e1 = cs >= 8u ? smx_e(d1 & 0xFFFFu, sc, tab) : smx_e_wide(d1 & 0xFFFFu, cm, cs, tab);
        }
        row[i] = (v0 ? smx_p(e0, R, fp) : 0u) | ((v1 ? smx_p(e1, R, fp) : 0u) << 16);
      }
    }
  };
  for (uint32_t a = t0; a < t1; a += A.win) {
    const uint32_t e = min(a + A.win, t1);
    if (nwin > 1) {
      consumer_sync();  // the window before is read
      for (uint32_t t = a; t < e; t++) scores(t, a);
      consumer_sync();
    }
    e_pass(a, e, nwin == 1);
  }
  cluster_meet();
  if (tid < kRows) {
    unsigned long long sum = 0;
    if (X > 1)
      for (uint32_t i = 0; i < X; i++) sum += cluster_ld64(cluster_addr(&s_s[tid], i));
    else
      sum = s_s[tid];
    s_R[tid] = smx_r(sum);
  }
  consumer_sync();

  const uint32_t dg = warp % DG, kg = warp / DG;
  uint32_t acc[NT][3][4];
#pragma unroll
  for (uint32_t j = 0; j < NT; j++)
#pragma unroll
    for (int k = 0; k < 3; k++)
#pragma unroll
      for (int x = 0; x < 4; x++) acc[j][k][x] = 0;
  for (uint32_t a = t0; a < t1; a += A.win) {
    const uint32_t e = min(a + A.win, t1);
    if (nwin > 1) {
      consumer_sync();
      for (uint32_t t = a; t < e; t++) scores(t, a);
      consumer_sync();
    }
    p_pass(a, e, nwin == 1);
    consumer_sync();
    for (uint32_t t = a; t < e; t++) {
      const uint32_t s = gi % NST;
      // every warp takes and leaves every tile, its own 32-key blocks or not: a slot is
      // not filled again before all have seen it, so no wait falls a phase behind
      if (ok) ok = wait_for(&full[s], (gi / NST) & 1u, A.err, 304);
      __syncwarp();
      gi++;
#pragma unroll
      for (uint32_t half = 0; half < 2; half++) {
        const uint32_t u = 2u * (t - a) + half;
        if (u % KG != kg) continue;
        const uint8_t* vr = ring + s * STB + (32u * half + 4u * qt) * RB + (DW == 32 ? 32u * dg + 4u * qn : 2u * qn);
        uint32_t vh[2][4], vl[2][4];
#pragma unroll
        for (int p = 0; p < 2; p++) {
          uint32_t x[4], y[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint8_t* q = vr + (16u * p + i) * RB;
            if (DW == 32) {
              // quarters alternate between the planes, as the scores' keys do
              if (BITS == 16) {
                const uint32_t f0 = *(const uint32_t*)(q + ((qt & 1u) ? HD : 0)), f1 = *(const uint32_t*)(q + ((qt & 1u) ? 0 : HD));
                x[i] = (qt & 1u) ? f1 : f0;
                y[i] = (qt & 1u) ? f0 : f1;
              } else {
                x[i] = *(const uint32_t*)q;
              }
            } else {
              x[i] = *(const uint16_t*)q;
              if (BITS == 16) y[i] = *(const uint16_t*)(q + HD);
            }
          }
          transpose4(x[0], x[1], x[2], x[3], vh[p]);
          if (BITS == 16) transpose4(y[0], y[1], y[2], y[3], vl[p]);
        }
        const int16_t* pr = S + u * 32u + 4u * qt;
        uint32_t p0[4], p1[4], p2[4];
        uint32_t shw[2] = {0, 0};
        if (BITS == 8) {
          const uint8_t* sv = ring + s * STB + kT * RB + 32u * half + 4u * qt;
          shw[0] = *(const uint32_t*)sv;
          shw[1] = *(const uint32_t*)(sv + 16);
        }
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const uint32_t row = qn + 8u * (x & 1);
          uint2 v = make_uint2(0, 0);
          if (row < nr) v = *(const uint2*)(pr + row * pitch + 16u * (x >> 1));
          if (BITS == 16) {
            p0[x] = __byte_perm(v.x, v.y, 0x6420);
            p1[x] = __byte_perm(v.x, v.y, 0x7531);
          } else {  // P << shift: 23 bits, three planes against the codes
            const uint32_t sw = shw[x >> 1];
            const uint32_t y0 = (v.x & 0xFFFFu) << (sw & 31u), y1 = (v.x >> 16) << ((sw >> 8) & 31u);
            const uint32_t y2 = (v.y & 0xFFFFu) << ((sw >> 16) & 31u), y3 = (v.y >> 16) << ((sw >> 24) & 31u);
            const uint32_t f = __byte_perm(y0, y1, 0x5140), h = __byte_perm(y2, y3, 0x5140);
            p0[x] = __byte_perm(f, h, 0x5410);
            p1[x] = __byte_perm(f, h, 0x7632);
            p2[x] = __byte_perm(__byte_perm(y0, y1, 0x0062), __byte_perm(y2, y3, 0x0062), 0x5410);
          }
        }
#pragma unroll
        for (uint32_t j = 0; j < NT; j++) {
          if (BITS == 16) {
            mma_uu(acc[j][0], p0, vl[0][j], vl[1][j]);
            mma_us(acc[j][1], p0, vh[0][j], vh[1][j]);
            mma_uu(acc[j][1], p1, vl[0][j], vl[1][j]);
            mma_us(acc[j][2], p1, vh[0][j], vh[1][j]);
          } else {
            mma_us(acc[j][0], p0, vh[0][j], vh[1][j]);
            mma_us(acc[j][1], p1, vh[0][j], vh[1][j]);
            mma_us(acc[j][2], p2, vh[0][j], vh[1][j]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&empty[s]);
    }
  }
  // the key groups' sums (modulo 2^32: any order), then the cluster's
  if (t1 > t0) {
#pragma unroll
    for (uint32_t j = 0; j < NT; j++)
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const uint32_t row = qn + 8u * (x >> 1), col = 2u * qt + (x & 1);
        const uint32_t dim = DW == 32 ? 32u * dg + 4u * col + j : 2u * col + j;
        const uint32_t v = acc[j][0][x] + (acc[j][1][x] << 8) + (acc[j][2][x] << 16);
        if (row < nr) atomicAdd(&s_O[row * HD + dim], v);
      }
  }
  cluster_meet();
  for (uint32_t i = rank * 256u + tid; i < nr * HD; i += X * 256u) {
    uint32_t v = 0;
    if (X > 1)
      for (uint32_t k = 0; k < X; k++) v += cluster_ld32(cluster_addr(&s_O[i], k));
    else
      v = s_O[i];
    const uint32_t rr = r0 + i / HD;
    A.d.o[(uint64_t)(sq.lo + rr / G) * A.d.ldo + (uint64_t)(g * G + rr % G) * HD + i % HD] = (int16_t)out16(v);
  }
  if (X > 1) cluster_sync();  // no CTA leaves while another reads its sums
}

template <int HD, int BITS>
int launch_split(SplitArgs A, uint32_t tiles, cudaStream_t st) {
  using Sh = SplitShape<HD, BITS>;
  const corm_paged_cache& c = A.d.c;
  // two CTAs an SM up to 128 dimensions: about 112 KB each
  const uint32_t budget = HD <= 128 ? 110u * 1024u : 220u * 1024u;
  uint32_t stages = 48u * 1024u / Sh::STB;
  A.stages = stages = stages < 3u ? 3u : (stages > 8u ? 8u : stages);
  const uint64_t blocks = (uint64_t)c.B * c.KV * tiles;
  const uint32_t cap = c.table_width * c.page, keys = A.d.max_keys < cap ? A.d.max_keys : cap;
  uint32_t X = 1;
  while (X < kMaxCluster && blocks * X < 296u && keys / (2u * X) >= 128u) X *= 2u;
  A.X = X;
  const uint32_t fixed = stages * Sh::STB + A.rcap * HD * 4u + 8192u;
  const uint32_t room = (budget - fixed) / (A.rcap * 2u), most = (room - 16u) / kT;
  const uint32_t span = A.d.window && A.d.window < keys ? A.d.window + A.d.max_q : keys;
  const uint32_t need = ((span < keys ? span : keys) / kT + 2u + X - 1u) / X;
  A.win = need < 1u ? 1u : (need < most ? need : most);
  const size_t smem = stages * Sh::STB + (size_t)A.rcap * split_pitch(A.win) * 2u + A.rcap * HD * 4u + 8192u;
  auto kern = paged_attn_split_kernel<HD, BITS>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return corm::cuda_status("llm_paged_attn");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * X, c.KV, c.B);
  cfg.blockDim = dim3(288);
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
  A.vec = !(((uintptr_t)d->q0 | (uintptr_t)d->k0 | (uintptr_t)d->v0 | (uintptr_t)d->q) & 7u) &&
          !((d->ldq0 | d->ldk | d->ldv | d->ldq) & 3u) && !((uintptr_t)d->rope & 15u) && d->rot % 8u == 0;
  cudaStream_t st = (cudaStream_t)stream;
  const uint32_t slots = d->H + 2u * c.KV, spb = 256u / (c.HD / 8u);
  // a grid whose step is a whole number of rows: every thread keeps its head
  uint32_t g = slots, r = spb;
  while (r) {
    const uint32_t t = g % r;
    g = r;
    r = t;
  }
  const uint64_t unit = slots / g;  // blocks
  const uint64_t want = ((uint64_t)c.rows * slots + spb - 1) / spb, most = 148u * 16u;
  uint64_t grid = ((want < most ? want : most) + unit - 1) / unit * unit;
  auto launch = [&](auto kern) { corm_launch_pdl(kern, dim3((unsigned)grid), dim3(256), 0, st, A); };
  {
    corm::ProfScope prof_("paged_prep_kernel", st);
    auto pick = [&](auto hd) {
      constexpr int W = decltype(hd)::value;
      if (d->nq || d->nk) {
        if (A.vec) launch(paged_prep_kernel<W, true, true>);
        else launch(paged_prep_kernel<W, false, true>);
      } else {
        if (A.vec) launch(paged_prep_kernel<W, true, false>);
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
  const uint32_t vec = !(((uintptr_t)d->k | (uintptr_t)d->v) & 15u) && !((d->k ? d->ldk : 0) & 7u) &&
                       !((d->v ? d->ldv : 0) & 7u);
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = corm_blocks((size_t)c.rows * 2u * c.KV * (c.HD / 8u), 256, 148u * 16u);
  auto launch = [&](auto kern) { corm_launch_pdl(kern, dim3(grid), dim3(256), 0, st, *d, vec); };
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
  A.G = d->H / c.KV;
  const uint64_t rows = (uint64_t)A.d.max_q * A.G;
  A.rcap = rows < kRows ? (uint32_t)rows : kRows;
  const uint64_t tiles = (rows + kRows - 1u) / kRows;
  if (tiles > (1ull << 27)) return corm::fail(CORM_ELIMIT, "corm_llm_paged_attn: max_q %u", d->max_q);
  cudaStream_t st = (cudaStream_t)stream;
  if (rows > kSplitRows && paged::tile_takes(A.d)) return paged::launch_tiles(A.d, A.tab, A.err, st);
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
