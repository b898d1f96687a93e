// corm_llm_paged_attn on 128-row tiles (prompts and chunks): tcgen05 kind::i8
// on the cache's byte planes.
//
// A CTA per (sequence, KV head, 128 rows), a row being (token, head of the
// group), token-major; with few tiles a cluster of CTAs shares the keys.  As in
// the 16-row kernel, the unit's e(d) is a table of d = m - score, so nothing can
// be rescaled as a running maximum moves: three phases over the scores, which
// stay in shared memory (int16, then e in place) where the CTA's keys fit, and
// are formed again in windows where they do not.
//   warps 0..15  rows: thread = (row = TMEM lane, 32 of a tile's 128 keys).  Its
//                scores, e and P are its own, so the phases meet only at the
//                row's maximum and sum.  q goes to TMEM as the A operand.
//     phase 1    tcgen05.ld of the three accumulators (HH, MID, LL), the score
//                rule, the maximum
//     phase 2    e by the unit's table, its sum
//     phase 3    P's bytes into TMEM as the A operand of P.V; at the end the
//                output rule on P.V's accumulators
//   warp 16      TMA: per 128 keys the pages' rows (a box per page piece) into a
//                ring, K tiles then V tiles, running ahead across the phases
//   warp 17      owns TMEM, issues the MMAs: q.K^T (B K-major, N = 128 keys) and
//                P.V (the V rows as they are: B MN-major, N = HD)
// 16 bits: 2 x 2 planes, sums HH 2^16 + MID 2^8 + LL.  8 bits: the codes are one
// plane; a K row's shift applies to the score, a V row's to P (three planes).
// Every sum is modulo 2^32, the rule's own wrap.
#include <cudaTypedefs.h>

#include <mutex>

#include "gemm_i8x4.h"
#include "paged.cuh"
#include "paged_tile.h"

namespace paged {
namespace {

constexpr uint32_t BMR = 128, BK = 128;  // rows and keys of a tile
constexpr uint32_t ROW_WARPS = 16, ROW_THREADS = 512, THREADS = 576;

template <int HD, int BITS>
struct Shape {
  static constexpr uint32_t RB = HD * (BITS / 8);       // bytes of a cached row
  static constexpr uint32_t XB = RB < 128 ? RB : 128;   // bytes of a box row
  static constexpr uint32_t HALVES = RB / XB;           // 128 dimensions at 16 bits: the planes apart
  static constexpr uint32_t HALF_BYTES = BK * XB;
  static constexpr uint32_t STAGE = BK * RB;
  static constexpr uint32_t LO = HALVES == 2 ? HALF_BYTES : HD;  // the low plane's offset in a stage
  static constexpr uint32_t SW = XB;                    // swizzle span
  static constexpr uint32_t NP = BITS == 16 ? 2 : 3;    // planes of P
  // TMEM columns: scores at 0 (128 each); P.V sums at 0 (HD each), P after them, q last
  static constexpr uint32_t PCH = HD == 64 ? 128 : 64;  // keys of a P buffer
  static constexpr uint32_t PCOLS = NP * PCH / 4;
  static constexpr uint32_t P0 = 3 * HD;
  static constexpr uint32_t QC = HD / 4;                // columns of a q plane
  static constexpr uint32_t Q0 = 512 - 2 * QC;
  static constexpr bool Q_OVER = P0 + 2 * PCOLS > Q0;   // P lies over q: q again before scores are formed again
  static constexpr uint32_t PW = HD == 64 ? ROW_WARPS : ROW_WARPS / 2;  // warps that fill a P buffer
};

struct TileArgs {
  corm_llm_paged_attn_desc d;
  const int32_t* tab;
  int* err;
  uint32_t G, X, stages, win;  // win: tiles of a window
};

__device__ __forceinline__ void rows_sync() { asm volatile("bar.sync 1, 512;" ::: "memory"); }
__device__ __forceinline__ uint32_t shr_clamp(uint32_t x, uint32_t s) {  // 0 from 32 up
  uint32_t r;
  asm("shr.u32 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(s));
  return r;
}
// two values saturated to 16 bits in a word (lo in the low half)
__device__ __forceinline__ uint32_t pack_s16(uint32_t lo, uint32_t hi) {
  uint32_t r;
  asm("cvt.pack.sat.s16.s32 %0, %1, %2;" : "=r"(r) : "r"(hi), "r"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_u16(uint32_t lo, uint32_t hi) {
  uint32_t r;
  asm("cvt.pack.sat.u16.s32 %0, %1, %2;" : "=r"(r) : "r"(hi), "r"(lo));
  return r;
}
// any registers, out of line
__device__ __noinline__ uint32_t e_any(uint32_t d, uint32_t cm, uint32_t cs, const uint32_t* tab) {
  const uint64_t y = ((uint64_t)d * (cm & 0xFFFFFFu)) >> cs;
  return (y >> 12) > 16u ? 0u : tab[y & 4095u] >> (uint32_t)(y >> 12);
}
__device__ __noinline__ uint32_t p_any(uint32_t e, uint32_t R, uint32_t fp) { return smx_p(e, R, fp); }

// A row's softmax registers and maximum as e of a packed score pair wants them
struct RowE {
  uint32_t mode;       // 0: 10 <= Cs <= 26; 1: Cs >= 27; 2: any (alike over the warp)
  uint32_t cm8, cm, cs;
  int32_t mul;         // mode 0: -2^(26 - Cs)
  uint32_t m0;         // mode 0: m 2^(26 - Cs); 1: m 2^16; 2: m
};
// e of 8 scores (4 packed words).  t = floor(d Cm / 2^(Cs - 2)) = 4 y and two bits:
// the table's byte offset is t mod 2^14 without them, the octave t / 2^14.  Mode 0
// brings d to 2^(26 - Cs) as it subtracts, so the product's high word is t itself;
// mode 1 shifts it down (from Cs = 40 on Cm counts as 0: y is 0)
__device__ __forceinline__ void e_of8(const RowE& r, const uint32_t* x, uint32_t* e, const uint32_t* tab) {
  if (r.mode == 2u) {
#pragma unroll
    for (int k = 0; k < 8; k++)
      e[k] = e_any((r.m0 - (k & 1 ? x[k >> 1] >> 16 : x[k >> 1])) & 0xFFFFu, r.cm, r.cs, tab);
    return;
  }
  uint32_t t[8];
  if (r.mode == 0u) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      t[2 * k] = __umulhi((uint32_t)((int32_t)(int16_t)x[k] * r.mul) + r.m0, r.cm8);
      t[2 * k + 1] = __umulhi((uint32_t)(((int32_t)x[k] >> 16) * r.mul) + r.m0, r.cm8);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      t[2 * k] = __umulhi(r.m0 - (x[k] << 16), r.cm8) >> (r.cs - 10u);
      t[2 * k + 1] = __umulhi(r.m0 - (x[k] & 0xFFFF0000u), r.cm8) >> (r.cs - 10u);
    }
  }
#pragma unroll
  for (int k = 0; k < 8; k++)
    e[k] = shr_clamp(*(const uint32_t*)((const uint8_t*)tab + (t[k] & 0x3FFCu)), t[k] >> 14);
}

template <int HD, int BITS>
__global__ void __launch_bounds__(THREADS, 1)
    paged_attn_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           const __grid_constant__ TileArgs A) {
  using Sh = Shape<HD, BITS>;
  extern __shared__ uint8_t pt_sm[];
  __shared__ uint64_t kv_full[8], kv_empty[8], acc_full, tmem_free, p_full[2], p_empty[2], mma_done, cbar;
  __shared__ uint32_t tmem_slot;
  __shared__ int32_t s_pm[4][BMR], s_m[BMR];
  __shared__ unsigned long long s_s[BMR];
  __shared__ __align__(16) uint32_t tab[4096];  // the softmax unit's table
  const corm_paged_cache& c = A.d.c;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t X = A.X, G = A.G, g = blockIdx.y, b = blockIdx.z, rank = blockIdx.x % X;
  const uint32_t tile = gridDim.x / X - 1u - blockIdx.x / X;  // the last rows see most: first
  const uint32_t NST = A.stages, WIN = A.win;
  uint8_t* ring = (uint8_t*)(((uintptr_t)pt_sm + 1023) & ~(uintptr_t)1023);
  uint8_t* s_S = ring + NST * Sh::STAGE;                    // [tile of the window][4][512] 16-byte words
  uint8_t* s_kshift = s_S + WIN * (BMR * BK * 2u);          // 8 bits: shifts of the window's K and V rows
  uint8_t* s_vshift = s_kshift + WIN * BK;

  corm_pdl_wait();
  corm_pdl_trigger();
  const SeqRows sq = seq_rows(c, b, c.rows);
  const uint32_t n = min(sq.n, A.d.max_q);
  const uint64_t all = (uint64_t)n * G, first = (uint64_t)tile * BMR;
  if (first >= all) return;  // the cluster's CTAs alike
  const uint32_t r0 = (uint32_t)first, nr = (uint32_t)min((uint64_t)BMR, all - first);
  const uint32_t i0 = r0 / G, i1 = (r0 + nr - 1u) / G, w = A.d.window;
  const uint32_t hi = min(sq.pos + i1 + 1u, sq.cap);
  const uint32_t lo = (w && sq.pos + i0 + 1u > w) ? sq.pos + i0 + 1u - w : 0u;
  const uint32_t tile0 = lo / BK, ntile = hi > lo ? (hi + BK - 1u) / BK - tile0 : 0u;
  const uint32_t per = (ntile + X - 1u) / X;
  const uint32_t t0 = tile0 + min(rank * per, ntile), t1 = tile0 + min(rank * per + per, ntile);
  const bool again = t1 - t0 > WIN;  // more than a window
  // the keys every row of the tile sees: no element is masked there
  const uint32_t all_lo = (w && sq.pos + i1 + 1u > w) ? sq.pos + i1 + 1u - w : 0u;
  const uint32_t all_hi = nr == BMR ? min(sq.pos + i0 + 1u, sq.cap) : 0u;

  if (tid == 0) {
    for (uint32_t i = 0; i < NST; i++) {
      sm100::mbar_init(&kv_full[i], 1);
      sm100::mbar_init(&kv_empty[i], 1);
    }
    sm100::mbar_init(&acc_full, 1);
    sm100::mbar_init(&tmem_free, ROW_WARPS);
    for (int i = 0; i < 2; i++) {
      sm100::mbar_init(&p_full[i], Sh::PW);
      sm100::mbar_init(&p_empty[i], 1);
    }
    sm100::mbar_init(&mma_done, 1);
    sm100::mbar_init(&cbar, X);
    sm100::fence_mbar_init();
  }
  if (warp == 17) sm100::tmem_alloc<512>(&tmem_slot);
  sm100::tc_fence_before();
  __syncthreads();
  if (X > 1) cluster_sync();
  sm100::tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 16) {
    // ---------------- the copies
    if (lane == 0) {
      sm100::prefetch_tmap(&map_k);
      sm100::prefetch_tmap(&map_v);
    }
    const uint32_t sub = min(c.page, BK), pieces = BK / sub, psh = 31u - __clz(c.page);
    const int32_t* tb = c.table + (uint64_t)b * c.table_width;
    uint32_t gi = 0, base = 0xFFFFFF00u;
    int32_t ids = -1;
    bool ok = true;
    auto emit = [&](bool is_v, uint32_t t) {
      const uint32_t s = gi % NST;
      if (gi >= NST && ok) ok = sm100::mbar_wait(&kv_empty[s], ((gi / NST) - 1u) & 1u, A.err, 311);
      ok = __all_sync(0xffffffffu, ok);
      gi++;
      if (!ok) return;
      const uint32_t b0 = (t * BK) >> psh, b1 = (t * BK + BK - 1u) >> psh;
      if (b0 < base || b1 >= base + 32u) {  // 32 table entries at a time
        base = b0;
        ids = base + lane < c.table_width ? tb[base + lane] : -1;
      }
      const uint32_t key = t * BK + lane * sub;
      const bool in = lane < pieces && key < hi;
      const int32_t id = __shfl_sync(0xffffffffu, ids, in ? (key >> psh) - base : 0u);
      const bool good = in && (uint32_t)id < c.pages;
      uint8_t* dst = ring + s * Sh::STAGE + lane * sub * Sh::XB;
      if (in && !good) {  // a page of zeros
        for (uint32_t h = 0; h < Sh::HALVES; h++)
          for (uint32_t i = 0; i < sub * Sh::XB; i += 16u)
            *(int4*)(dst + h * Sh::HALF_BYTES + i) = make_int4(0, 0, 0, 0);
        sm100::fence_proxy_async_smem();
      }
      const uint32_t cnt = __popc(__ballot_sync(0xffffffffu, good));
      if (lane == 0) sm100::mbar_expect_tx(&kv_full[s], cnt * sub * Sh::RB);
      __syncwarp();
      if (good) {
        const uint32_t line = ((uint32_t)id * c.KV + g) * c.page + (key & (c.page - 1u));  // < 2^31 (the host checks)
        for (uint32_t h = 0; h < Sh::HALVES; h++)
          sm100::tma_load_2d(dst + h * Sh::HALF_BYTES, is_v ? &map_v : &map_k, &kv_full[s], (int)(h * 128u), (int)line);
      }
    };
    for (uint32_t t = t0; t < t1; t++) emit(false, t);
    if (again)
      for (uint32_t t = t0; t < t1; t++) emit(false, t);
    for (uint32_t a = t0; a < t1; a += WIN) {
      const uint32_t e = min(a + WIN, t1);
      if (again)
        for (uint32_t t = a; t < e; t++) emit(false, t);
      for (uint32_t t = a; t < e; t++) emit(true, t);
    }
    // every copy lands before the CTA's shared memory goes away
    for (uint32_t q = gi > NST ? gi - NST : 0u; ok && q < gi; q++)
      sm100::mbar_wait(&kv_full[q % NST], (q / NST) & 1u, nullptr, 0);
    __syncwarp();
  } else if (warp == 17) {
    // ---------------- the MMAs (one thread)
    if (lane == 0) {
      constexpr uint32_t MN = 1u << 16;  // B MN-major
      const uint32_t KSS = sm100::idesc_i8(BMR, BK, 1, 1), KSU = sm100::idesc_i8(BMR, BK, 1, 0);
      const uint32_t KUS = sm100::idesc_i8(BMR, BK, 0, 1), KUU = sm100::idesc_i8(BMR, BK, 0, 0);
      const uint32_t VUS = sm100::idesc_i8(BMR, HD, 0, 1) | MN, VUU = sm100::idesc_i8(BMR, HD, 0, 0) | MN;
      const uint32_t qh = tmem + Sh::Q0, ql = qh + Sh::QC;
      uint32_t gi = 0, unit = 0, pt = 0;
      bool ok = true;
      auto desc_k = [&](uint32_t a) { return Sh::SW == 128 ? sm100::sdesc_sw128(a) : sm100::sdesc_sw64(a); };
      auto desc_v = [&](uint32_t a) { return Sh::SW == 128 ? sm100::sdesc_sw128_mn(a) : sm100::sdesc_sw64(a); };
      auto stage_in = [&]() -> uint32_t {
        const uint32_t s = gi % NST;
        if (ok) ok = sm100::mbar_wait(&kv_full[s], (gi / NST) & 1u, A.err, 312);
        gi++;
        return s;
      };
      auto scores = [&]() {  // one tile's q.K^T
        const uint32_t s = stage_in();
        if (ok) ok = sm100::mbar_wait(&tmem_free, unit & 1u, A.err, 313);
        unit++;
        if (!ok) return;
        sm100::tc_fence_after();
        const uint32_t base = sm100::smem_u32(ring + s * Sh::STAGE);
#pragma unroll
        for (uint32_t ks = 0; ks < HD / 32; ks++) {
          const uint64_t kh = desc_k(base + 32u * ks);
          const uint32_t acc = ks ? 1u : 0u;
          if (BITS == 16) {
            const uint64_t kl = desc_k(base + Sh::LO + 32u * ks);
            sm100::mma_i8_ta(tmem, qh + 8u * ks, kh, KSS, acc);
            sm100::mma_i8_ta(tmem + 128u, qh + 8u * ks, kl, KSU, acc);
            sm100::mma_i8_ta(tmem + 128u, ql + 8u * ks, kh, KUS, 1u);
            sm100::mma_i8_ta(tmem + 256u, ql + 8u * ks, kl, KUU, acc);
          } else {
            sm100::mma_i8_ta(tmem, qh + 8u * ks, kh, KSS, acc);
            sm100::mma_i8_ta(tmem + 128u, ql + 8u * ks, kh, KUS, acc);
          }
        }
        sm100::mma_commit(&kv_empty[s]);
        sm100::mma_commit(&acc_full);
      };
      for (uint32_t t = t0; t < t1; t++) scores();
      if (again)
        for (uint32_t t = t0; t < t1; t++) scores();
      for (uint32_t a = t0; a < t1; a += WIN) {
        const uint32_t e = min(a + WIN, t1);
        if (again)
          for (uint32_t t = a; t < e; t++) scores();
        if (ok) ok = sm100::mbar_wait(&tmem_free, unit & 1u, A.err, 314);
        unit++;
        for (uint32_t t = a; t < e; t++, pt++) {
          const uint32_t s = stage_in();
          const uint32_t base = sm100::smem_u32(ring + s * Sh::STAGE);
#pragma unroll
          for (uint32_t ch = 0; ch < BK / Sh::PCH; ch++) {
            const uint32_t buf = HD == 64 ? (pt & 1u) : ch;
            if (ok) ok = sm100::mbar_wait(&p_full[buf], (HD == 64 ? pt >> 1 : pt) & 1u, A.err, 315);
            if (!ok) continue;
            sm100::tc_fence_after();
            const uint32_t p = tmem + Sh::P0 + buf * Sh::PCOLS;
#pragma unroll
            for (uint32_t ks = 0; ks < Sh::PCH / 32; ks++) {
              const uint32_t k = ch * (Sh::PCH / 32) + ks;  // 32 V rows
              const uint64_t vh = desc_v(base + k * 32u * Sh::XB);
              const uint32_t acc = (t != a || k) ? 1u : 0u;
              const uint32_t p0 = p + 8u * ks, p1 = p0 + Sh::PCH / 4, p2 = p1 + Sh::PCH / 4;
              if (BITS == 16) {  // P low, P high against V's planes
                const uint64_t vl = desc_v(base + Sh::LO + k * 32u * Sh::XB);
                sm100::mma_i8_ta(tmem, p1, vh, VUS, acc);
                sm100::mma_i8_ta(tmem + HD, p0, vh, VUS, acc);
                sm100::mma_i8_ta(tmem + HD, p1, vl, VUU, 1u);
                sm100::mma_i8_ta(tmem + 2 * HD, p0, vl, VUU, acc);
              } else {
                sm100::mma_i8_ta(tmem, p2, vh, VUS, acc);
                sm100::mma_i8_ta(tmem + HD, p1, vh, VUS, acc);
                sm100::mma_i8_ta(tmem + 2 * HD, p0, vh, VUS, acc);
              }
            }
            sm100::mma_commit(&p_empty[buf]);
          }
          if (ok) sm100::mma_commit(&kv_empty[s]);
        }
        if (ok) sm100::mma_commit(&acc_full);
      }
      // every MMA issued has completed before TMEM is freed
      sm100::mma_commit(&mma_done);
      sm100::mbar_wait(&mma_done, 0, nullptr, 0, 200000000ll);
    }
    __syncwarp();
  } else {
    // ---------------- the rows
    const uint32_t quarter = warp & 3u, part = warp >> 2, row = quarter * 32u + lane;  // part: 32 of a tile's keys
    const uint32_t lane_base = tmem + ((quarter * 32u) << 16);
    const uint32_t rr = r0 + min(row, nr - 1u), tok = rr / G, head = g * G + rr % G;
    const uint32_t pp = sq.pos + tok;
    const uint32_t khi = row < nr ? min(pp + 1u, sq.cap) : 0u, klo = (w && pp + 1u > w) ? pp + 1u - w : 0u;
    const uint32_t cm = A.d.smx[2u * head], cfg = A.d.smx[2u * head + 1u], cs = cfg & 63u, fp = (cfg >> 8) & 31u;
    const int16_t* qrow = A.d.q + (uint64_t)(sq.lo + tok) * A.d.ldq + (uint64_t)head * HD;
    const bool q16 = !(((uintptr_t)A.d.q & 15u) | (A.d.ldq & 7u));
    // q's bytes into TMEM: this warp's quarter of the dimensions of its 32 rows
    auto load_q = [&]() {
      constexpr uint32_t D = HD / 4, W = D / 4;  // dimensions and plane words of a part
      uint32_t h[8], l[8];
#pragma unroll
      for (uint32_t k = 0; k < W; k += 2) {
        uint4 v = make_uint4(0, 0, 0, 0);
        const int16_t* q = qrow + part * D + 4u * k;
        if (row < nr) {
          if (q16)
            v = *(const uint4*)q;
          else
            v = make_uint4(pack16(q[0], q[1]), pack16(q[2], q[3]), pack16(q[4], q[5]), pack16(q[6], q[7]));
        }
        h[k] = __byte_perm(v.x, v.y, 0x7531), h[k + 1] = __byte_perm(v.z, v.w, 0x7531);
        l[k] = __byte_perm(v.x, v.y, 0x6420), l[k + 1] = __byte_perm(v.z, v.w, 0x6420);
      }
      const uint32_t ta = lane_base + Sh::Q0 + part * W;
      __syncwarp();
      if (W == 8) {
        sm100::tmem_st8(ta, h);
        sm100::tmem_st8(ta + Sh::QC, l);
      } else {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(ta), "r"(h[0]), "r"(h[1]),
                     "r"(h[2]), "r"(h[3])
                     : "memory");
        asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(ta + Sh::QC), "r"(l[0]),
                     "r"(l[1]), "r"(l[2]), "r"(l[3])
                     : "memory");
      }
      sm100::tmem_st_wait();
    };
    bool ok = true;
    uint32_t unit = 0;
    auto release = [&]() {  // TMEM's accumulators (and q) are the MMAs' again
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&tmem_free);
    };
    auto acc_wait = [&]() {
      if (ok) ok = sm100::mbar_wait(&acc_full, unit & 1u, A.err, 316);
      unit++;
      __syncwarp();
      sm100::tc_fence_after();
    };
    // the shifts of the window's cached rows (8 bits)
    auto load_shifts = [&](uint32_t a, uint32_t e) {
      if (BITS == 16) return;
      rows_sync();
      for (uint32_t i = tid; i < (e - a) * BK; i += ROW_THREADS) {
        const uint32_t key = a * BK + i;
        const int32_t id = key < hi ? c.table[(uint64_t)b * c.table_width + key / c.page] : -1;
        const bool good = (uint32_t)id < c.pages;
        const uint64_t line = good ? ((uint64_t)(uint32_t)id * c.KV + g) * c.page + key % c.page : 0u;
        s_kshift[i] = good ? c.ks[line] & 31u : 0u;
        s_vshift[i] = good ? c.vs[line] & 31u : 0u;
      }
      rows_sync();
    };
    load_q();
    release();
    for (uint32_t i = tid; i < 1024u; i += ROW_THREADS) ((int4*)tab)[i] = ((const int4*)A.tab)[i];
    if (tid < BMR) s_s[tid] = 0;
    if (!again) load_shifts(t0, t1);

    // 16 scores of this thread's keys (half j of its 32) in tile t: 8 packed words
    auto scores16 = [&](uint32_t t, uint32_t a, uint32_t j, uint32_t (&out)[8], bool last) {
      uint32_t hh[16], mid[16], ll[16];
      const uint32_t col = lane_base + part * 32u + j * 16u;
      __syncwarp();
      sm100::tmem_ld16(col, hh);
      sm100::tmem_ld16(col + 128u, mid);
      if (BITS == 16) sm100::tmem_ld16(col + 256u, ll);
      sm100::tmem_ld_wait();
      if (last) release();
      uint32_t shw[4];
      if (BITS == 8) {
        const uint4 v = *(const uint4*)(s_kshift + (t - a) * BK + part * 32u + j * 16u);
        shw[0] = v.x, shw[1] = v.y, shw[2] = v.z, shw[3] = v.w;
      }
#pragma unroll
      for (uint32_t k = 0; k < 16; k += 2) {
        int32_t y[2];
#pragma unroll
        for (uint32_t x = 0; x < 2; x++) {
          uint32_t acc;
          if (BITS == 16)
            acc = (hh[k + x] << 16) + (mid[k + x] << 8) + ll[k + x];
          else
            acc = ((hh[k + x] << 8) + mid[k + x]) << ((shw[k / 4] >> (8u * ((k + x) & 3u))) & 31u);
          y[x] = (int32_t)acc >> 8;
        }
        out[k / 2] = pack_s16((uint32_t)y[0], (uint32_t)y[1]);
      }
    };
    auto masked = [&](uint32_t t) { return t * BK < all_lo || t * BK + BK > all_hi; };
    // this thread's keys of tile t that the row sees, a bit each
    auto seen = [&](uint32_t t) -> uint32_t {
      const uint32_t kb = t * BK + part * 32u;
      const uint32_t h = khi > kb ? min(khi - kb, 32u) : 0u, l = klo > kb ? min(klo - kb, 32u) : 0u;
      return (h ? 0xFFFFFFFFu >> (32u - h) : 0u) & (l < 32u ? 0xFFFFFFFFu << l : 0u);
    };
    uint4* S4 = (uint4*)s_S + tid;  // word j of tile i of the window: [(4 i + j) 512]

    // phase 1
    uint32_t mx = 0x80008000u;
    for (uint32_t a = t0; a < t1; a += WIN) {
      const uint32_t e = min(a + WIN, t1);
      if (again) load_shifts(a, e);
      for (uint32_t t = a; t < e; t++) {
        acc_wait();
#pragma unroll
        for (uint32_t j = 0; j < 2; j++) {
          uint32_t o[8];
          scores16(t, a, j, o, j == 1);
          if (!again) {
            S4[((t - a) * 4u + 2u * j) * ROW_THREADS] = make_uint4(o[0], o[1], o[2], o[3]);
            S4[((t - a) * 4u + 2u * j + 1u) * ROW_THREADS] = make_uint4(o[4], o[5], o[6], o[7]);
          }
          if (masked(t)) {
            const uint32_t sk = seen(t) >> (16u * j);
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) {
              const uint32_t lo16 = (sk >> (2u * k)) & 1u ? o[k] : 0x8000u, hi16 = (sk >> (2u * k)) & 2u ? o[k] : 0x80000000u;
              o[k] = __byte_perm(lo16, hi16, 0x7610);
            }
          }
#pragma unroll
          for (uint32_t k = 0; k < 8; k++) mx = __vmaxs2(mx, o[k]);
        }
      }
    }
    uint32_t cphase = 0;
    // every CTA of the cluster is here, and what it wrote before is visible
    auto meet = [&]() {
      rows_sync();
      if (X > 1) {
        if (tid < X) mbar_arrive_remote(&cbar, tid);
        if (ok) ok = mbar_wait_cluster(&cbar, cphase, A.err, 317);
        cphase ^= 1u;
      }
    };
    s_pm[part][row] = max((int32_t)(int16_t)(mx & 0xFFFFu), (int32_t)mx >> 16);
    rows_sync();
    int32_t m = max(max(s_pm[0][row], s_pm[1][row]), max(s_pm[2][row], s_pm[3][row]));
    if (X > 1) {
      if (part == 0) s_m[row] = m;
      meet();
      for (uint32_t i = 0; i < X; i++) m = max(m, (int32_t)cluster_ld32(cluster_addr(&s_m[row], i)));
    }
    RowE re;
    re.cm = cm, re.cs = cs;
    re.cm8 = cs >= 40u ? 0u : (cm & 0xFFFFFFu) << 8;
    re.mode = __reduce_max_sync(0xffffffffu, cs < 10u ? 2u : (cs > 26u ? 1u : 0u));
    re.mul = -(int32_t)(1u << ((26u - min(cs, 26u)) & 31u));
    re.m0 = re.mode == 0u ? (uint32_t)(-m * re.mul) : (re.mode == 1u ? (uint32_t)m << 16 : (uint32_t)m);
    if (re.mode == 1u) re.cs = cs >= 40u ? 10u : cs;
    // e of keys 8 j .. 8 j + 7 of this thread's 32, those unseen 0; their sum
    auto e_seen = [&](const uint32_t* x, uint32_t* e, bool mk, uint32_t sk) -> uint32_t {
      e_of8(re, x, e, tab);
      if (mk) {
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) e[k] = (sk >> k) & 1u ? e[k] : 0u;
      }
      return ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
    };
    // phase 2: e in place (one window), the row's sum
    unsigned long long sum = 0;
    if (!again) {
      rows_sync();  // the table is there
      for (uint32_t t = t0; t < t1; t++) {
        const bool mk = masked(t);
        const uint32_t sk = mk ? seen(t) : 0u;
        uint32_t part_sum = 0;
#pragma unroll 2
        for (uint32_t j = 0; j < 4; j++) {
          uint4& v = S4[((t - t0) * 4u + j) * ROW_THREADS];
          const uint4 x4 = v;
          const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w};
          uint32_t ev[8];
          part_sum += e_seen(x, ev, mk, sk >> (8u * j));
          v = make_uint4(pack_u16(ev[0], ev[1]), pack_u16(ev[2], ev[3]), pack_u16(ev[4], ev[5]), pack_u16(ev[6], ev[7]));
        }
        sum += part_sum;
      }
    } else {
      for (uint32_t a = t0; a < t1; a += WIN) {
        const uint32_t e = min(a + WIN, t1);
        load_shifts(a, e);
        if (BITS == 16) rows_sync();
        for (uint32_t t = a; t < e; t++) {
          acc_wait();
          const bool mk = masked(t);
          const uint32_t sk = mk ? seen(t) : 0u;
          uint32_t part_sum = 0;
#pragma unroll
          for (uint32_t j = 0; j < 2; j++) {
            uint32_t o[8], ev[8];
            scores16(t, a, j, o, j == 1);
            part_sum += e_seen(o, ev, mk, sk >> (16u * j));
            part_sum += e_seen(o + 4, ev, mk, sk >> (16u * j + 8u));
          }
          sum += part_sum;
        }
      }
    }
    atomicAdd(&s_s[row], sum);
    meet();
    unsigned long long total = 0;
    if (X > 1)
      for (uint32_t i = 0; i < X; i++) total += cluster_ld64(cluster_addr(&s_s[row], i));
    else
      total = s_s[row];
    const uint32_t R = smx_r(total);
    // P of a packed e: with 8 <= f_p <= 15 the high word of e R 2^(f_p - 8) + 2^31
    const bool pfast = __all_sync(0xffffffffu, fp >= 8u && fp <= 15u);
    const uint32_t Rp = pfast ? R << (fp - 8u) : R;
    auto p_of = [&](uint32_t h) -> uint32_t {
      const uint32_t e = h + ((h + 1u) >> 16);
      if (pfast) return (uint32_t)(((uint64_t)e * Rp + (1ull << 31)) >> 32);
      return p_any(e, R, fp);
    };

    // phase 3
    uint32_t oacc[HD / 4];
#pragma unroll
    for (uint32_t k = 0; k < HD / 4; k++) oacc[k] = 0;
    uint32_t pt = 0;
    for (uint32_t a = t0; a < t1; a += WIN) {
      const uint32_t e = min(a + WIN, t1);
      if (again) {
        load_shifts(a, e);
        for (uint32_t t = a; t < e; t++) {
          acc_wait();
          const bool mk = masked(t);
          const uint32_t sk = mk ? seen(t) : 0u;
#pragma unroll
          for (uint32_t j = 0; j < 2; j++) {
            uint32_t o[8], ev[8];
            scores16(t, a, j, o, j == 1);
#pragma unroll
            for (uint32_t h = 0; h < 2; h++) {
              e_seen(o + 4 * h, ev, mk, sk >> (16u * j + 8u * h));
              S4[((t - a) * 4u + 2u * j + h) * ROW_THREADS] =
                  make_uint4(pack_u16(ev[0], ev[1]), pack_u16(ev[2], ev[3]), pack_u16(ev[4], ev[5]), pack_u16(ev[6], ev[7]));
            }
          }
        }
        rows_sync();  // every warp has read the scores: P goes over their columns
      }
      for (uint32_t t = a; t < e; t++, pt++) {
        const uint32_t buf = HD == 64 ? (pt & 1u) : part >> 1;
        const uint32_t uses = HD == 64 ? pt >> 1 : pt;  // of this buffer, before
        if (uses && ok) ok = sm100::mbar_wait(&p_empty[buf], (uses - 1u) & 1u, A.err, 318);
        sm100::tc_fence_after();
        uint32_t pl[3][8];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
          const uint4 v = S4[((t - a) * 4u + j) * ROW_THREADS];
          const uint32_t xw[4] = {v.x, v.y, v.z, v.w};
          uint32_t p[8];
#pragma unroll
          for (uint32_t k = 0; k < 4; k++) {
            p[2 * k] = p_of(xw[k] & 0xFFFFu);
            p[2 * k + 1] = p_of(xw[k] >> 16);
          }
#pragma unroll
          for (uint32_t h = 0; h < 2; h++) {
            if (BITS == 16) {
              // saturated to 32767 as signed halves
              const uint32_t w0 = pack_s16(p[4 * h], p[4 * h + 1]), w1 = pack_s16(p[4 * h + 2], p[4 * h + 3]);
              pl[0][2 * j + h] = __byte_perm(w0, w1, 0x6420);
              pl[1][2 * j + h] = __byte_perm(w0, w1, 0x7531);
            } else {
              const uint32_t sw = *(const uint32_t*)(s_vshift + (t - a) * BK + part * 32u + j * 8u + 4u * h);
              uint32_t y[4];
#pragma unroll
              for (uint32_t x = 0; x < 4; x++) y[x] = min(p[4 * h + x], 32767u) << ((sw >> (8u * x)) & 31u);
              const uint32_t f = __byte_perm(y[0], y[1], 0x5140), q = __byte_perm(y[2], y[3], 0x5140);
              pl[0][2 * j + h] = __byte_perm(f, q, 0x5410);
              pl[1][2 * j + h] = __byte_perm(f, q, 0x7632);
              pl[2][2 * j + h] = __byte_perm(__byte_perm(y[0], y[1], 0x0062), __byte_perm(y[2], y[3], 0x0062), 0x5410);
            }
          }
        }
        const uint32_t ta = lane_base + Sh::P0 + buf * Sh::PCOLS + (HD == 64 ? part : part & 1u) * 8u;
        __syncwarp();
#pragma unroll
        for (uint32_t k = 0; k < Sh::NP; k++) sm100::tmem_st8(ta + k * (Sh::PCH / 4), pl[k]);
        sm100::tmem_st_wait();
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&p_full[buf]);
      }
      // the window's P.V: this warp's quarter of the dimensions
      acc_wait();
#pragma unroll
      for (uint32_t k = 0; k < HD / 4; k += 16) {
        uint32_t hh[16], mid[16], ll[16];
        const uint32_t col = lane_base + part * (HD / 4) + k;
        sm100::tmem_ld16(col, hh);
        sm100::tmem_ld16(col + HD, mid);
        sm100::tmem_ld16(col + 2 * HD, ll);
        sm100::tmem_ld_wait();
#pragma unroll
        for (uint32_t x = 0; x < 16; x++) oacc[k + x] += (hh[x] << 16) + (mid[x] << 8) + ll[x];
      }
      if (Sh::Q_OVER && e < t1) load_q();
      release();
    }
    constexpr uint32_t D = HD / 4;  // this thread's dimensions
    if (X > 1) {
      // the cluster's sums: every CTA leaves its own in shared memory, and adds up a slice
      rows_sync();
      uint4* so = (uint4*)s_S;  // [D / 4][512]
#pragma unroll
      for (uint32_t k = 0; k < D; k += 4)
        so[(k / 4u) * ROW_THREADS + tid] = make_uint4(oacc[k], oacc[k + 1], oacc[k + 2], oacc[k + 3]);
      meet();
      // words of (thread's place, 4 dimensions): rank r takes every X-th
      for (uint32_t i = rank * ROW_THREADS + tid; i < D / 4u * ROW_THREADS; i += X * ROW_THREADS) {
        uint32_t v[4] = {0, 0, 0, 0};
        for (uint32_t q = 0; q < X; q++) {
          const uint32_t ad = cluster_addr(so + i, q);
#pragma unroll
          for (uint32_t x = 0; x < 4; x++) v[x] += cluster_ld32(ad + 4u * x);
        }
        const uint32_t th = i % ROW_THREADS, orow = ((th >> 5) & 3u) * 32u + (th & 31u);
        if (orow < nr) {
          const uint32_t o_r = r0 + orow, dim = (th >> 7) * D + 4u * (i / ROW_THREADS);
          int16_t* o = A.d.o + (uint64_t)(sq.lo + o_r / G) * A.d.ldo + (uint64_t)(g * G + o_r % G) * HD + dim;
#pragma unroll
          for (uint32_t x = 0; x < 4; x++) o[x] = (int16_t)out16(v[x]);
        }
      }
    } else if (row < nr) {
      int16_t* o = A.d.o + (uint64_t)(sq.lo + tok) * A.d.ldo + (uint64_t)head * HD + part * D;
      uint32_t ow[D / 2];
#pragma unroll
      for (uint32_t k = 0; k < D / 2; k++) ow[k] = pack16(out16(oacc[2 * k]), out16(oacc[2 * k + 1]));
      if (!(((uintptr_t)A.d.o & 15u) | (A.d.ldo & 7u))) {
#pragma unroll
        for (uint32_t k = 0; k < D / 8; k++)
          ((uint4*)o)[k] = make_uint4(ow[4 * k], ow[4 * k + 1], ow[4 * k + 2], ow[4 * k + 3]);
      } else {
#pragma unroll
        for (uint32_t k = 0; k < D / 2; k++) {
          o[2 * k] = (int16_t)ow[k];
          o[2 * k + 1] = (int16_t)(ow[k] >> 16);
        }
      }
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (X > 1) cluster_sync();  // no CTA leaves while another reads its shared memory
  if (warp == 17) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc<512>(tmem);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
  });
  return fn;
}

// the cached rows [lines][rb] bytes; a box: rows of up to 128 bytes of a page piece
bool make_row_map(CUtensorMap* map, const void* base, uint32_t rb, uint64_t lines, uint32_t sub) {
  auto fn = encode_fn();
  if (!fn) return false;
  const uint32_t xb = rb < 128u ? rb : 128u;
  cuuint64_t dims[2] = {rb, lines};
  cuuint64_t strides[1] = {rb};
  cuuint32_t box[2] = {xb, sub};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, xb == 128u ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, int BITS>
int launch(TileArgs A, uint32_t tiles, cudaStream_t st) {
  using Sh = Shape<HD, BITS>;
  const corm_paged_cache& c = A.d.c;
  CUtensorMap mk, mv;
  const uint64_t lines = (uint64_t)c.pages * c.KV * c.page;
  const uint32_t sub = c.page < BK ? c.page : BK;
  if (!make_row_map(&mk, c.kc, Sh::RB, lines, sub) || !make_row_map(&mv, c.vc, Sh::RB, lines, sub))
    return corm::fail(CORM_ECUDA, "corm_llm_paged_attn: cuTensorMapEncodeTiled failed");
  const uint32_t cap = c.table_width * c.page, keys = A.d.max_keys < cap ? A.d.max_keys : cap;
  const uint32_t span = A.d.window && A.d.window < keys ? A.d.window + BMR : keys;
  const uint32_t ktiles = ((span < keys ? span : keys) + BK - 1u) / BK + 1u;
  const uint64_t blocks = (uint64_t)c.B * c.KV * tiles;
  uint32_t X = 1;
  while (X < 8u && blocks * 2u * X <= 148u && ktiles >= 4u * X) X *= 2u;
  A.X = X;
  A.stages = 3u * 16384u / Sh::STAGE < 2u ? 2u : (3u * 16384u / Sh::STAGE > 6u ? 6u : 3u * 16384u / Sh::STAGE);
  const uint32_t tile_bytes = BMR * BK * 2u + (BITS == 8 ? 2u * BK : 0u);
  const uint32_t room = 206u * 1024u - 1024u - A.stages * Sh::STAGE;  // beside 20 KB of static arrays
  const uint32_t most = room / tile_bytes, need = (ktiles + X - 1u) / X;
  // a cluster's sums use the scores' memory: HD KB / 2
  const uint32_t least = (HD * 512u + BMR * BK * 2u - 1u) / (BMR * BK * 2u);
  A.win = need < least ? least : (need < most ? need : most);
  const size_t smem = 1024u + A.stages * Sh::STAGE + (size_t)A.win * tile_bytes;
  auto kern = paged_attn_tile_kernel<HD, BITS>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return corm::cuda_status("llm_paged_attn");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * X, c.KV, c.B);
  cfg.blockDim = dim3(THREADS);
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
    corm::ProfScope prof_("paged_attn_tile_kernel", st);
    cudaLaunchKernelEx(&cfg, kern, mk, mv, A);
  }
  return corm::cuda_status("llm_paged_attn");
}

}  // namespace

bool tile_takes(const corm_llm_paged_attn_desc& d) {
  return (d.c.HD == 64u || d.c.HD == 128u) && (uint64_t)d.c.pages * d.c.KV * d.c.page < (1ull << 31);
}

int launch_tiles(const corm_llm_paged_attn_desc& d, const int32_t* tab, int* err, cudaStream_t st) {
  TileArgs A{};
  A.d = d;
  A.tab = tab;
  A.err = err;
  A.G = d.H / d.c.KV;
  const uint32_t tiles = (uint32_t)(((uint64_t)d.max_q * A.G + BMR - 1u) / BMR);
  switch (d.c.HD * 2u + (d.c.bits == 8u)) {
    case 128: return launch<64, 16>(A, tiles, st);
    case 129: return launch<64, 8>(A, tiles, st);
    case 256: return launch<128, 16>(A, tiles, st);
    default: return launch<128, 8>(A, tiles, st);
  }
}

}  // namespace paged
