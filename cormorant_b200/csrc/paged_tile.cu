// corm_llm_paged_attn on 128-row tiles (prompts and chunks): tcgen05 kind::i8
// on the cache's byte planes.
//
// Persistent: a CTA an SM takes items = (128-row tile, sequence, KV head), the ones that
// see most keys first, a row being (token, head of the group), token-major; with few items a
// cluster of CTAs shares an item's keys.  As in the 8-row kernel, the unit's e(d) is a
// table of d = m - score, so nothing can be rescaled as a running maximum moves: three
// phases over the scores, which stay in shared memory (int16, then e in place) where the
// CTA's keys fit, and are formed again in windows where they do not.
//   row warps    thread = (row = TMEM lane, 32 of a tile's 128 keys).  Its scores, e and
//                P are its own, so the phases meet only at the row's maximum and sum.
//                q goes to TMEM as the A operand.
//     phase 0    tcgen05.ld of the three accumulators (HH, MID, LL), the score rule,
//                the maximum
//     phase 1    e by the unit's table, its sum
//     phase 2    P's bytes into TMEM as the A operand of P.V; at the end the output
//                rule on P.V's accumulators, while the next item's first scores form
//   a copy warp  TMA: per tile of keys the pages' rows (a box per page piece) into a
//                ring, K tiles then V tiles, running ahead across phases and items
//   an MMA warp  owns TMEM, issues the MMAs: q.K^T (B K-major, N = 128 keys: N = 64 takes
//                58 cycles against 65, so halves of a tile would double its time) and P.V
//                (the V rows as they are: B MN-major, N = HD)
// 16 bits: 2 x 2 planes, sums HH 2^16 + MID 2^8 + LL.  8 bits: the codes are one
// plane; a K row's shift applies to the score, a V row's to P (three planes).
// Every sum is modulo 2^32, the rule's own wrap.
//
// Bound by the row warps' integer work, phase by phase (cycles of a 128 x 128 tile of 64
// dimensions at 16 bits): scores 1800 (the MMAs, 65 cycles each and twice that between
// issues beside 16 busy warps, do not overlap the loads of their one set of sums: three
// sums of 128 columns and P fill TMEM), e 2500 (16384 table lookups at random banks: 1700
// at the least), P 2000, and about 7500 an item around them.  In windows the scores are
// formed three times and e twice: 11600 a tile.  64 prompts of 97 to 512 rows, 15 heads
// of 64: 189 us; one of 8192: 1257 us; 4 chunks of 257 over 1k to 8k, 16 heads of 128:
// 364 us.  Tried and slower: tiles of 64 keys, two CTAs an SM (332 us for the prompts);
// more score columns a load (spills); one CTA an item, not persistent (266 us); the low
// planes made signed, so that one MMA takes both (204 us: two instructions a score more).
#include <cudaTypedefs.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "gemm_i8x4.h"
#include "paged.cuh"
#include "paged_tile.h"

namespace paged {
namespace {

constexpr uint32_t BMR = 128, BK = 128;              // rows and keys of a tile
constexpr uint32_t PARTS = 4;                        // row warps a TMEM quarter: 32 keys of a tile a thread
constexpr uint32_t RW = 4 * PARTS, RT = 32 * RW, THREADS = RT + 64;
constexpr uint32_t TILE_BYTES = BMR * BK * 2;        // a tile's scores
constexpr uint32_t ITEMS = 4;                        // items known ahead

template <int HD, int BITS>
struct Shape {
  static constexpr uint32_t RB = HD * (BITS / 8);       // bytes of a cached row
  static constexpr uint32_t XB = RB < 128 ? RB : 128;   // bytes of a box row, the swizzle's span
  static constexpr uint32_t HALVES = RB / XB;           // 128 dimensions at 16 bits: the planes apart
  static constexpr uint32_t HALF_BYTES = BK * XB;
  static constexpr uint32_t STAGE = BK * RB;
  static constexpr uint32_t LO = HALVES == 2 ? HALF_BYTES : HD;  // the low plane's offset in a stage
  static constexpr uint32_t NP = BITS == 16 ? 2 : 3;    // planes of P
  static constexpr uint32_t D = HD / PARTS;             // a thread's dimensions of q and of the output
  // TMEM columns: the scores' sums at 0 (BK each); P.V's sums at 0 (HD each), P's
  // buffers of PCH keys after them, q last
  static constexpr uint32_t PCH = HD == 64 ? 128 : 64;  // keys of a P buffer (two buffers)
  static constexpr uint32_t CH = BK / PCH;              // buffers a tile fills
  static constexpr uint32_t PCOLS = NP * PCH / 4;
  static constexpr uint32_t P0 = 3 * HD;
  static constexpr uint32_t QC = HD / 4;                // columns of a q plane
  static constexpr uint32_t Q0 = 512 - 2 * QC;
  static constexpr bool Q_OVER = P0 + 2 * PCOLS > Q0;   // P lies over q: q again before scores are formed again
};

struct TileArgs {
  corm_llm_paged_attn_desc d;
  const int32_t* tab;
  int* err;
  Waits waits;
  uint32_t G, X, stages, win;  // win: tiles of a window
  uint32_t tiles;              // row tiles of the longest sequence
  uint32_t by_seq;             // items in the order of the sequences' lengths
  uint32_t k8, k16;            // 2^8 and 2^16, as operands (shifts would go to the busier pipe)
};

__device__ __forceinline__ void rows_sync() { asm volatile("bar.sync 1, %0;" ::"n"(RT) : "memory"); }
// A row's softmax registers and maximum as e of a packed score pair wants them.
// t = floor(d Cm / 2^(Cs - 2)) = 4 y and two bits: the table's byte offset is t mod
// 2^14 without them, the octave t / 2^14.
//   mode 0  19 <= Cs <= 26 (scales of 2^-3 to 2^4): a two-way dot product picks a half
//           of the pair, multiplies it by -2^(26 - Cs) and adds m 2^(26 - Cs); the
//           product with Cm 2^8 has t as its high word
//   mode 1  10 <= Cs: the product of d 2^16 and Cm 2^8, shifted down (from Cs = 40 on
//           Cm counts as 0: y is 0)
//   mode 2  any: a Cs below 10 as 10 with Cm 2^(10 - Cs).  Past 24 bits that is a
//           scale of 2^14 and more, where e is 0 from d = 5 on: d up to 31 is enough,
//           and Cm up to 2^27 (e is 0 for every d > 0 there)
struct RowE {
  uint32_t mode;  // alike over the warp
  uint32_t cm, sh;
  int32_t mul;
  uint32_t m0;
};
__device__ __forceinline__ RowE row_e(uint32_t cm, uint32_t cs, int32_t m) {
  RowE r;
  const uint32_t want = cs < 10u ? 2u : ((cs > 26u || cs < 19u) ? 1u : 0u);
  r.mode = __reduce_max_sync(0xffffffffu, want);
  r.cm = cs >= 40u ? 0u : cm << 8;
  r.sh = cs >= 40u ? 0u : max(cs, 10u) - 10u;
  r.mul = 0;
  if (r.mode == 0u) {
    const uint32_t k = 26u - cs;  // up to 7
    const uint32_t c8 = (0u - (1u << k)) & 0xFFu;
    r.mul = (int32_t)(c8 | c8 << 24);
    r.m0 = (uint32_t)m << k;
  } else if (r.mode == 1u) {
    r.m0 = (uint32_t)m << 16;
  } else {
    // narrow: 16 bits of d at 2^16 by 24 of Cm at 2^8, down by sh; wide: 5 at 2^19 by 27 at 2^5
    const uint64_t wide = cs < 10u ? (uint64_t)cm << (10u - cs) : cm;
    const bool w = wide >> 24;
    r.m0 = (uint32_t)m;
    r.mul = w ? 19 : 16;
    r.cm = w ? (uint32_t)(wide < (1ull << 27) ? wide : (1ull << 27) - 1u) << 5 : (cs >= 40u ? 0u : (uint32_t)wide << 8);
  }
  return r;
}
__device__ __forceinline__ void e_of8(const RowE& r, const uint32_t* x, uint32_t* e, const uint32_t* tab) {
  uint32_t t[8];
  if (r.mode == 0u) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      t[2 * k] = __umulhi((uint32_t)__dp2a_lo((int)x[k], r.mul, (int)r.m0), r.cm);
      t[2 * k + 1] = __umulhi((uint32_t)__dp2a_hi((int)x[k], r.mul, (int)r.m0), r.cm);
    }
  } else if (r.mode == 1u) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      t[2 * k] = __umulhi(r.m0 - (x[k] << 16), r.cm) >> r.sh;
      t[2 * k + 1] = __umulhi(r.m0 - (x[k] & 0xFFFF0000u), r.cm) >> r.sh;
    }
  } else {
    const uint32_t top = r.mul == 19 ? 31u : 65535u;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const uint32_t d = (r.m0 - (k & 1 ? x[k >> 1] >> 16 : x[k >> 1])) & 0xFFFFu;
      t[k] = __umulhi(min(d, top) << r.mul, r.cm) >> r.sh;
    }
  }
#pragma unroll
  for (int k = 0; k < 8; k++)
    e[k] = shr_clamp(*(const uint32_t*)((const uint8_t*)tab + (t[k] & 0x3FFCu)), t[k] >> 14);
}

// An item: a tile of rows of one sequence and KV head, and this CTA's keys of it
struct Item {
  uint32_t b, g, r0, nr, lo_row;  // rows r0 .. r0 + nr - 1 of the sequence, whose first packed row is lo_row
  uint32_t pos, cap, hi;          // the first row's position; positions of the table; keys seen end before hi
  uint32_t t0, t1;                // key tiles
};
// Item i (tiles of the last rows first, as they see most); false: its tile has no rows.
__device__ __forceinline__ bool item_at(const TileArgs& A, uint32_t i, uint32_t rank, uint32_t order, Item& o) {
  const corm_paged_cache& c = A.d.c;
  const uint32_t G = A.G, w = A.d.window;
  uint32_t tile;
  if (A.by_seq) {
    const uint32_t per = A.tiles * c.KV, rem = i % per;
    o.b = __shfl_sync(0xffffffffu, order, i / per);
    tile = A.tiles - 1u - rem / c.KV;
    o.g = rem % c.KV;
  } else {
    const uint32_t per = c.B * c.KV, rem = i % per;
    tile = A.tiles - 1u - i / per;
    o.b = rem / c.KV;
    o.g = rem % c.KV;
  }
  const SeqRows s = seq_rows(c, o.b, c.rows);
  const uint32_t all = min(s.n, A.d.max_q) * G;  // < 2^31 (the host checks)
  o.r0 = tile * BMR;
  if (o.r0 >= all) return false;
  o.nr = min(BMR, all - o.r0);
  o.lo_row = s.lo;
  o.pos = s.pos;
  o.cap = s.cap;
  const uint32_t i0 = o.r0 / G, i1 = (o.r0 + o.nr - 1u) / G;
  o.hi = min(s.pos + i1 + 1u, s.cap);
  const uint32_t lo = (w && s.pos + i0 + 1u > w) ? s.pos + i0 + 1u - w : 0u;
  const uint32_t tile0 = lo / BK, n = o.hi > lo ? (o.hi + BK - 1u) / BK - tile0 : 0u, per = (n + A.X - 1u) / A.X;
  o.t0 = tile0 + min(rank * per, n);
  o.t1 = tile0 + min(rank * per + per, n);
  return true;
}

// Lane k's sequence is the one with the k-th most keys (B <= 32)
__device__ __forceinline__ uint32_t order_of(const TileArgs& A, uint32_t lane) {
  const corm_paged_cache& c = A.d.c;
  uint32_t keys = 0;
  if (lane < c.B) {
    const SeqRows s = seq_rows(c, lane, c.rows);
    keys = s.n ? min(s.pos + min(s.n, A.d.max_q), s.cap) : 0u;
  }
  uint32_t rank = 0, order = 0;
  for (uint32_t i = 0; i < c.B; i++) {
    const uint32_t k = __shfl_sync(0xffffffffu, keys, i);
    rank += k > keys || (k == keys && i < lane);
  }
  for (uint32_t i = 0; i < c.B; i++)
    if (__shfl_sync(0xffffffffu, rank, i) == lane) order = i;
  return order;
}

// The grid has a CTA (cluster) an item; those that run take over the ones not yet
// launched, one at a time (cluster launch control): no counter in memory, none shared
// by two launches, and whoever is free takes the next.
__device__ __forceinline__ void ask_next(uint4* answer, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
          sm100::smem_u32(answer)),
      "r"(sm100::smem_u32(bar))
      : "memory");
}
// the CTA index taken over, or -1: none is left (and none may be asked for again)
__device__ __forceinline__ int32_t next_taken(const uint4* answer) {
  uint32_t some, x;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t.reg .b32 y, z, u;\n\t"
      "mov.u32 %1, 0;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, u}, r;\n\t}"
      : "=&r"(some), "=&r"(x)
      : "r"(sm100::smem_u32(answer))
      : "memory");
  return some ? (int32_t)x : -1;
}

template <int HD, int BITS>
__global__ void __launch_bounds__(THREADS, 1)
    paged_attn_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           const __grid_constant__ TileArgs A) {
  using Sh = Shape<HD, BITS>;
  extern __shared__ uint8_t pt_sm[];
  __shared__ uint64_t kv_full[8], kv_empty[8], s_full, s_free, o_full, p_full[2], p_empty[2], mma_done, cbar;
  __shared__ uint32_t tmem_slot;
  __shared__ int32_t s_pm[PARTS][BMR], s_m[BMR];
  __shared__ unsigned long long s_ps[PARTS][BMR], s_s[BMR];
  __shared__ __align__(16) uint32_t tab[4096];  // the softmax unit's table
  __shared__ Item s_item[ITEMS];                // written by the copy warp
  __shared__ uint32_t s_more[ITEMS];            // 0: the end
  __shared__ uint64_t item_full[ITEMS], item_free[ITEMS], taken_bar;
  __shared__ uint32_t s_go;                     // the rows go on with the next item
  __shared__ __align__(16) uint4 s_taken;
  const corm_paged_cache& c = A.d.c;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t X = A.X, G = A.G, rank = blockIdx.x % X, NST = A.stages, WIN = A.win;
  uint8_t* ring = (uint8_t*)(((uintptr_t)pt_sm + 1023) & ~(uintptr_t)1023);
  uint8_t* s_S = ring + NST * Sh::STAGE;           // [tile of the window][4][row threads] 16-byte words
  uint8_t* s_kshift = s_S + WIN * TILE_BYTES;      // 8 bits: shifts of the window's K and V rows
  uint8_t* s_vshift = s_kshift + WIN * BK;

  if (tid == 0) {
    for (uint32_t i = 0; i < NST; i++) {
      sm100::mbar_init(&kv_full[i], 1);
      sm100::mbar_init(&kv_empty[i], 1);
    }
    sm100::mbar_init(&s_full, 1);
    sm100::mbar_init(&s_free, RW);
    sm100::mbar_init(&o_full, 1);
    for (int i = 0; i < 2; i++) {
      sm100::mbar_init(&p_full[i], RW / Sh::CH);
      sm100::mbar_init(&p_empty[i], 1);
    }
    for (uint32_t i = 0; i < ITEMS; i++) {
      sm100::mbar_init(&item_full[i], 1);
      sm100::mbar_init(&item_free[i], RW + 1);
    }
    sm100::mbar_init(&taken_bar, 1);
    sm100::mbar_init(&mma_done, 1);
    sm100::mbar_init(&cbar, X);
    sm100::fence_mbar_init();
  }
  if (warp == RW + 1u) sm100::tmem_alloc<512>(&tmem_slot);
  sm100::tc_fence_before();
  __syncthreads();
  if (X > 1) cluster_sync();
  sm100::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // the prologue above overlaps the kernel before; global memory only after it
  corm_pdl_wait();
  corm_pdl_trigger();
  uint32_t islot = 0, ipar = 0;  // the next item's slot and its parity

  if (warp == RW) {
    // ---------------- the copies
    if (lane == 0) {
      sm100::prefetch_tmap(&map_k);
      sm100::prefetch_tmap(&map_v);
    }
    const uint32_t sub = min(c.page, BK), pieces = BK / sub, psh = 31u - __clz(c.page);
    const uint32_t order = A.by_seq ? order_of(A, lane) : 0u;
    uint32_t gi = 0, asked = 0, answered = 0;
    bool ok = true;
    auto item_slot = [&]() {  // the slot's readers of ITEMS items ago are done
      if (ok) ok = wait_for(&item_free[islot], ipar ^ 1u, A.err, 321, A.waits);
      ok = __all_sync(0xffffffffu, ok);
    };
    auto publish = [&](const Item* o) {
      if (lane == 0) {
        s_more[islot] = o != nullptr;
        if (o) s_item[islot] = *o;
        sm100::mbar_arrive(&item_full[islot]);
      }
      __syncwarp();
      if (++islot == ITEMS) islot = 0, ipar ^= 1u;
    };
    auto ask = [&]() {
      if (X > 1) return;
      if (lane == 0) {
        sm100::mbar_expect_tx(&taken_bar, 16);
        ask_next(&s_taken, &taken_bar);
      }
      asked++;
    };
    auto taken = [&]() -> int32_t {
      if (asked == answered) return -1;
      if (!__all_sync(0xffffffffu, wait_for(&taken_bar, answered & 1u, A.err, 322, A.waits))) {
        ok = false;  // (the answer is waited for at the end)
        return -1;
      }
      answered++;
      const int32_t at = ok ? next_taken(&s_taken) : -1;
      __syncwarp();
      sm100::fence_proxy_async_smem();
      return at;
    };
    // publishes the first item with rows from number `at` on, or the end
    auto find = [&](int32_t at, Item& o) {
      while (at >= 0 && !item_at(A, (uint32_t)at, rank, order, o)) {
        ask();
        at = taken();
      }
      item_slot();
      const bool some = at >= 0 && ok;
      publish(some ? &o : nullptr);
      return some;
    };
    Item it;
    bool more = find((int32_t)(blockIdx.x / X), it);
    while (more) {
      ask();
      const int32_t* tb = c.table + (uint64_t)it.b * c.table_width;
      uint32_t base = 0xFFFFFF00u;
      int32_t ids = -1;
      auto emit = [&](bool is_v, uint32_t t) {
        const uint32_t s = gi % NST;
        if (gi >= NST && ok) ok = wait_for(&kv_empty[s], ((gi / NST) - 1u) & 1u, A.err, 311, A.waits);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        gi++;
        const uint32_t b0 = (t * BK) >> psh, b1 = (t * BK + BK - 1u) >> psh;
        if (b0 < base || b1 >= base + 32u) {  // 32 table entries at a time
          base = b0;
          ids = base + lane < c.table_width ? tb[base + lane] : -1;
        }
        const uint32_t key = t * BK + lane * sub;
        const bool in = lane < pieces && key < it.hi;
        const int32_t id = __shfl_sync(0xffffffffu, ids, in ? (key >> psh) - base : 0u);
        const bool good = in && (uint32_t)id < c.pages;
        uint8_t* dst = ring + s * Sh::STAGE + lane * sub * Sh::XB;
        if (in && !good) {  // a page of zeros
          for (uint32_t h = 0; h < Sh::HALVES; h++)
            for (uint32_t i = 0; i < sub * Sh::XB; i += 16u)
              *(int4*)(dst + h * Sh::HALF_BYTES + i) = make_int4(0, 0, 0, 0);
          sm100::fence_proxy_async_smem();
        }
        __syncwarp();  // every lane's zeros come before the arrival (a vote orders no memory)
        const uint32_t cnt = __popc(__ballot_sync(0xffffffffu, good));
        if (lane == 0) sm100::mbar_expect_tx(&kv_full[s], cnt * sub * Sh::RB);
        __syncwarp();
        if (good) {
          const uint32_t line = ((uint32_t)id * c.KV + it.g) * c.page + (key & (c.page - 1u));  // < 2^31 (the host checks)
          for (uint32_t h = 0; h < Sh::HALVES; h++)
            sm100::tma_load_2d(dst + h * Sh::HALF_BYTES, is_v ? &map_v : &map_k, &kv_full[s], (int)(h * 128u), (int)line);
        }
      };
      const bool again = it.t1 - it.t0 > WIN;
      // K (v = 0) for the first phase and, in windows, again for the other two; V (v = 1)
      // behind each window's K of the last
#pragma unroll 1
      for (uint32_t t = it.t0; t < it.t1; t++) emit(false, t);
      // the next item is known before this one's values are read: the rows look for it then
      Item nx;
      const bool some = find(taken(), nx);
#pragma unroll 1
      for (uint32_t phase = 1; phase < 3; phase++)
#pragma unroll 1
        for (uint32_t a = it.t0; a < it.t1; a += WIN)
#pragma unroll 1
          for (uint32_t v = again ? 0u : 1u; v < phase; v++)
#pragma unroll 1
            for (uint32_t t = a; t < min(a + WIN, it.t1); t++) emit(v == 1u, t);
      it = nx;
      more = some;
    }
    // every copy made, and the last answer, lands before the CTA's shared memory goes
    // away, whoever gave up before (they need nobody: no diagnostic limit)
    for (uint32_t q = gi > NST ? gi - NST : 0u; q < gi; q++) wait_for(&kv_full[q % NST], (q / NST) & 1u, nullptr, 0, kWaits);
    if (asked != answered) wait_for(&taken_bar, answered & 1u, nullptr, 0, kWaits);
    __syncwarp();
  } else if (warp == RW + 1u) {
    // ---------------- the MMAs (one lane)
    if (lane == 0) {
      constexpr uint32_t MN = 1u << 16;  // B MN-major
      constexpr uint32_t KSS = sm100::idesc_i8(BMR, BK, 1, 1), KSU = sm100::idesc_i8(BMR, BK, 1, 0);
      constexpr uint32_t KUS = sm100::idesc_i8(BMR, BK, 0, 1), KUU = sm100::idesc_i8(BMR, BK, 0, 0);
      constexpr uint32_t VUS = sm100::idesc_i8(BMR, HD, 0, 1) | MN, VUU = sm100::idesc_i8(BMR, HD, 0, 0) | MN;
      const uint32_t qh = tmem + Sh::Q0, ql = qh + Sh::QC;
      // a stage's descriptors: the words of its address 0, K-major and MN-major, then
      // every operand a constant away (16-byte units)
      const uint64_t k0 = Sh::XB == 128 ? sm100::sdesc_sw128(0) : sm100::sdesc_sw64(0);
      const uint64_t v0 = Sh::XB == 128 ? sm100::sdesc_sw128_mn(0) : sm100::sdesc_sw64(0);
      const uint32_t khi = (uint32_t)(k0 >> 32), vhi = (uint32_t)(v0 >> 32);
      const uint32_t ring_a = sm100::smem_u32(ring);
      uint32_t s = 0, sp = 0;            // the next ring stage and its parity
      uint32_t use = 0, pu = 0;          // uses of the scores' columns; P buffers
      bool ok = true;
      auto stage_in = [&]() -> uint32_t {  // the next stage, full: its address / 16
        if (ok) ok = wait_for(&kv_full[s], sp, A.err, 312, A.waits);
        return (ring_a + s * Sh::STAGE) >> 4;
      };
      auto stage_out = [&]() {
        if (ok) sm100::mma_commit(&kv_empty[s]);
        if (++s == NST) s = 0, sp ^= 1u;
      };
      auto scores = [&]() {  // one tile's q.K^T
        const uint32_t b = (uint32_t)k0 + stage_in();
        if (ok) ok = wait_for(&s_free, use & 1u, A.err, 313, A.waits);
        use++;
        if (ok) {
          sm100::tc_fence_after();
          auto step = [&](auto ks, auto keep) {
            constexpr uint32_t K = decltype(ks)::value;
            constexpr bool KEEP = decltype(keep)::value;
            const uint32_t bh = b + 2u * K;
            sm100::mma_i8_tb<KEEP>(tmem, qh + 8u * K, bh, khi, KSS);
            if constexpr (BITS == 16) {
              const uint32_t bl = bh + Sh::LO / 16;
              sm100::mma_i8_tb<KEEP>(tmem + BK, qh + 8u * K, bl, khi, KSU);
              sm100::mma_i8_tb<true>(tmem + BK, ql + 8u * K, bh, khi, KUS);
              sm100::mma_i8_tb<KEEP>(tmem + 2 * BK, ql + 8u * K, bl, khi, KUU);
            } else {
              sm100::mma_i8_tb<KEEP>(tmem + BK, ql + 8u * K, bh, khi, KUS);
            }
          };
          using std::integral_constant;
          step(integral_constant<uint32_t, 0>(), std::false_type());
          step(integral_constant<uint32_t, 1>(), std::true_type());
          if constexpr (HD == 128) {
            step(integral_constant<uint32_t, 2>(), std::true_type());
            step(integral_constant<uint32_t, 3>(), std::true_type());
          }
          sm100::mma_commit(&s_full);
        }
        stage_out();
      };
      auto values = [&](auto first) {  // one tile's P.V, into new sums or the ones there are
        const uint32_t b = (uint32_t)v0 + stage_in();
#pragma unroll
        for (uint32_t ch = 0; ch < Sh::CH; ch++, pu++) {
          const uint32_t buf = pu & 1u;
          if (ok) ok = wait_for(&p_full[buf], (pu >> 1) & 1u, A.err, 315, A.waits);
          if (!ok) continue;
          sm100::tc_fence_after();
          const uint32_t p = tmem + Sh::P0 + buf * Sh::PCOLS;
          auto step = [&](auto k32, auto keep) {
            constexpr uint32_t K = decltype(k32)::value;  // 32 V rows
            constexpr bool KEEP = decltype(keep)::value;
            const uint32_t bh = b + (ch * Sh::PCH + K * 32u) * Sh::XB / 16u;
            const uint32_t p0 = p + 8u * K, p1 = p0 + Sh::PCH / 4, p2 = p1 + Sh::PCH / 4;
            if constexpr (BITS == 16) {  // P low, P high against V's planes
              const uint32_t bl = bh + Sh::LO / 16;
              sm100::mma_i8_tb<KEEP>(tmem, p1, bh, vhi, VUS);
              sm100::mma_i8_tb<KEEP>(tmem + HD, p0, bh, vhi, VUS);
              sm100::mma_i8_tb<true>(tmem + HD, p1, bl, vhi, VUU);
              sm100::mma_i8_tb<KEEP>(tmem + 2 * HD, p0, bl, vhi, VUU);
            } else {
              sm100::mma_i8_tb<KEEP>(tmem, p2, bh, vhi, VUS);
              sm100::mma_i8_tb<KEEP>(tmem + HD, p1, bh, vhi, VUS);
              sm100::mma_i8_tb<KEEP>(tmem + 2 * HD, p0, bh, vhi, VUS);
            }
          };
          using std::integral_constant;
          if (ch == 0)
            step(integral_constant<uint32_t, 0>(), std::integral_constant<bool, !decltype(first)::value>());
          else
            step(integral_constant<uint32_t, 0>(), std::true_type());
          step(integral_constant<uint32_t, 1>(), std::true_type());
          if constexpr (Sh::PCH == 128) {
            step(integral_constant<uint32_t, 2>(), std::true_type());
            step(integral_constant<uint32_t, 3>(), std::true_type());
          }
          sm100::mma_commit(&p_empty[buf]);
        }
        stage_out();
      };
      // (one lane walks the items: the others' candidates by itself)
      while (true) {
        if (ok) ok = wait_for(&item_full[islot], ipar, A.err, 320, A.waits);
        const Item& it = s_item[islot];
        const bool end = !ok || !s_more[islot];
        const uint32_t t0 = it.t0, t1 = it.t1;
        if (end) break;
        sm100::mbar_arrive(&item_free[islot]);
        if (++islot == ITEMS) islot = 0, ipar ^= 1u;
        const bool again = t1 - t0 > WIN;
        auto taken = [&]() {
          if (ok) ok = wait_for(&s_free, use & 1u, A.err, 314, A.waits);
          use++;
        };
        if (t0 == t1) taken();  // no key is seen: the next item's q comes with the next release
#pragma unroll 1
        for (uint32_t phase = 0; phase < 3; phase++)
#pragma unroll 1
          for (uint32_t a = t0; a < t1; a += WIN) {
            const uint32_t e = min(a + WIN, t1);
            if (phase == 0 || again)
#pragma unroll 1
              for (uint32_t t = a; t < e; t++) scores();
            if (phase < 2) continue;
            taken();  // P.V's sums go over the scores'
            values(std::true_type());
#pragma unroll 1
            for (uint32_t t = a + 1u; t < e; t++) values(std::false_type());
            if (ok) sm100::mma_commit(&o_full);
          }
      }
      // every MMA issued has completed before TMEM is freed
      sm100::mma_commit(&mma_done);
      sm100::mbar_wait(&mma_done, 0, nullptr, 0, 200000000ll);
    }
    __syncwarp();
  } else {
    // ---------------- the rows
    const uint32_t quarter = warp & 3u, part = warp >> 2, row = quarter * 32u + lane;
    const uint32_t lane_base = tmem + ((quarter * 32u) << 16);
    constexpr uint32_t D = Sh::D;
    const bool q16 = !(((uintptr_t)A.d.q & 15u) | (A.d.ldq & 7u));
    const bool o16 = !(((uintptr_t)A.d.o & 15u) | (A.d.ldo & 7u));
    uint4* S4 = (uint4*)s_S + tid;  // word j of tile i of the window: [(4 i + j) RT]
    bool ok = true;
    uint32_t su = 0, ou = 0, pt = 0;  // tiles scored, P.V sums taken, tiles of P handed over
    // q: this part's dimensions of an item's row, from memory and into TMEM
    auto fetch_q = [&](const Item& o, uint4 (&v)[D / 8]) {
#pragma unroll
      for (uint32_t k = 0; k < D / 8; k++) v[k] = make_uint4(0, 0, 0, 0);
      if (row >= o.nr) return;
      const uint32_t rr = o.r0 + row;
      const int16_t* q = A.d.q + (uint64_t)(o.lo_row + rr / G) * A.d.ldq + (uint64_t)(o.g * G + rr % G) * HD + part * D;
#pragma unroll
      for (uint32_t k = 0; k < D / 8; k++, q += 8) {
        if (q16)
          v[k] = *(const uint4*)q;
        else
          v[k] = make_uint4(pack16(q[0], q[1]), pack16(q[2], q[3]), pack16(q[4], q[5]), pack16(q[6], q[7]));
      }
    };
    auto store_q = [&](const uint4 (&v)[D / 8]) {
      uint32_t h[D / 4], l[D / 4];
#pragma unroll
      for (uint32_t k = 0; k < D / 8; k++) {
        h[2 * k] = __byte_perm(v[k].x, v[k].y, 0x7531), h[2 * k + 1] = __byte_perm(v[k].z, v[k].w, 0x7531);
        l[2 * k] = __byte_perm(v[k].x, v[k].y, 0x6420), l[2 * k + 1] = __byte_perm(v[k].z, v[k].w, 0x6420);
      }
      const uint32_t ta = lane_base + Sh::Q0 + part * (D / 4);
      __syncwarp();
      if constexpr (D == 32) {
        sm100::tmem_st8(ta, h);
        sm100::tmem_st8(ta + Sh::QC, l);
      } else {
        sm100::tmem_st4(ta, h);
        sm100::tmem_st4(ta + Sh::QC, l);
      }
      sm100::tmem_st_wait();
    };
    auto release = [&]() {  // the scores' columns (and q) are the MMAs' again
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&s_free);
    };
    for (uint32_t i = tid; i < 1024u; i += RT) ((int4*)tab)[i] = ((const int4*)A.tab)[i];
    // whether a slot holds an item: the first row warp waits for it and tells the others
    // across a barrier, so that all leave together whatever ran out
    auto look = [&](uint32_t slot, uint32_t par) {
      if (warp != 0) return;
      if (ok) ok = wait_for(&item_full[slot], par, A.err, 323, A.waits);
      const bool some = __all_sync(0xffffffffu, ok && s_more[slot] != 0u);
      if (lane == 0) s_go = some;
    };
    look(0, 0);
    rows_sync();
    bool more = s_go != 0u;
    if (more) {
      uint4 v[D / 8];
      fetch_q(s_item[0], v);
      store_q(v);
    }
    release();
    uint32_t cphase = 0;
    // every CTA of the cluster is here, and what it wrote before is visible
    auto meet = [&]() {
      rows_sync();
      if (X > 1) {
        if (tid < X) mbar_arrive_remote(&cbar, tid);
        if (ok) ok = mbar_wait_cluster(&cbar, cphase, A.err, 317, A.waits);
        cphase ^= 1u;
      }
    };
#pragma unroll 1
    while (more) {
      const uint32_t cur = islot;
      if (++islot == ITEMS) islot = 0, ipar ^= 1u;
      const Item& it = s_item[cur];
      const uint32_t t0 = it.t0, t1 = it.t1;
      const bool again = t1 - t0 > WIN;  // more than a window
      const uint32_t rr = it.r0 + min(row, it.nr - 1u), head = it.g * G + rr % G, pp = it.pos + rr / G, w = A.d.window;
      const uint32_t khi = row < it.nr ? min(pp + 1u, it.cap) : 0u, klo = (w && pp + 1u > w) ? pp + 1u - w : 0u;
      // the rows of this warp see all, or none, of its 32 keys: known without a look at the elements
      auto unseen = [&](uint32_t key) { return __all_sync(0xffffffffu, key >= khi || key + 32u <= klo); };
      auto whole = [&](uint32_t key) { return __all_sync(0xffffffffu, key + 32u <= khi && key >= klo); };
      // the keys of [key, key + 32) that this row sees, a bit each
      auto seen = [&](uint32_t key) -> uint32_t {
        const uint32_t h = khi > key ? min(khi - key, 32u) : 0u, l = klo > key ? min(klo - key, 32u) : 0u;
        return (h ? 0xFFFFFFFFu >> (32u - h) : 0u) & (l < 32u ? 0xFFFFFFFFu << l : 0u);
      };
      // the shifts of the window's cached rows (8 bits)
      auto load_shifts = [&](uint32_t a, uint32_t e) {
        if (BITS == 16) return;
        rows_sync();
        for (uint32_t i = tid; i < (e - a) * BK; i += RT) {
          const uint32_t key = a * BK + i;
          const int32_t id = key < it.hi ? c.table[(uint64_t)it.b * c.table_width + key / c.page] : -1;
          const bool good = (uint32_t)id < c.pages;
          const uint64_t line = good ? ((uint64_t)(uint32_t)id * c.KV + it.g) * c.page + key % c.page : 0u;
          s_kshift[i] = good ? c.ks[line] & 31u : 0u;
          s_vshift[i] = good ? c.vs[line] & 31u : 0u;
        }
        rows_sync();
      };
      if (!again) load_shifts(t0, t1);

      RowE re{};
      uint32_t mx = 0x80008000u;
      unsigned long long sum = 0;
      auto packed_e = [&](const uint32_t* e) {
        return make_uint4(pack_u16(e[0], e[1]), pack_u16(e[2], e[3]), pack_u16(e[4], e[5]), pack_u16(e[6], e[7]));
      };
      // tile t's scores.  Phase 0: their maximum, and the scores into the window where it
      // holds all; in windows, phase 1: the sum of e, 2: e into the window
      auto score_pass = [&](uint32_t t, uint32_t a, const uint32_t phase) {
        if (ok) ok = wait_for(&s_full, su & 1u, A.err, 316, A.waits);
        su++;
        __syncwarp();
        sm100::tc_fence_after();
        const uint32_t key = t * BK + part * 32u;
        if (unseen(key)) {
          release();
          return;
        }
        const bool mk = !whole(key);
        const uint32_t sk = mk ? seen(key) : 0u;
        uint32_t tile_sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < 2; j++) {
          uint32_t hh[16], mid[16], ll[16], o[8];
          const uint32_t col = lane_base + part * 32u + j * 16u;
          sm100::tmem_ld16(col, hh);
          sm100::tmem_ld16(col + BK, mid);
          if (BITS == 16) sm100::tmem_ld16(col + 2 * BK, ll);
          sm100::tmem_ld_wait();
          if (j == 1) release();
          uint32_t shw[4];
          if (BITS == 8) {
            const uint4 v = *(const uint4*)(s_kshift + (key - a * BK) + j * 16u);
            shw[0] = v.x, shw[1] = v.y, shw[2] = v.z, shw[3] = v.w;
          }
#pragma unroll
          for (uint32_t k = 0; k < 16; k += 2) {
            uint32_t y[2];
#pragma unroll
            for (uint32_t x = 0; x < 2; x++) {
              uint32_t acc;
              if (BITS == 16)
                acc = hh[k + x] * A.k16 + (mid[k + x] * A.k8 + ll[k + x]);
              else
                acc = (hh[k + x] * A.k8 + mid[k + x]) << ((shw[k / 4] >> (8u * ((k + x) & 3u))) & 31u);
              y[x] = (uint32_t)((int32_t)acc >> 8);
            }
            o[k / 2] = pack_s16(y[0], y[1]);
          }
          uint4* dst = S4 + ((t - a) * 4u + 2u * j) * RT;
          if (phase == 0) {
            if (!again) {
              dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
              dst[RT] = make_uint4(o[4], o[5], o[6], o[7]);
            }
            if (mk) {
#pragma unroll
              for (uint32_t k = 0; k < 8; k++) {
                const uint32_t two = sk >> (16u * j + 2u * k);
                o[k] = __byte_perm((two & 1u) ? o[k] : 0x8000u, (two & 2u) ? o[k] : 0x80000000u, 0x7610);
              }
            }
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) mx = __vmaxs2(mx, o[k]);
          } else {
#pragma unroll
            for (uint32_t i = 0; i < 2; i++) {
              uint32_t ev[8];
              e_of8(re, o + 4 * i, ev, tab);
              if (mk) {
#pragma unroll
                for (uint32_t k = 0; k < 8; k++) ev[k] = (sk >> (16u * j + 8u * i + k)) & 1u ? ev[k] : 0u;
              }
              if (phase == 1) {
#pragma unroll
                for (uint32_t k = 0; k < 8; k++) tile_sum += ev[k];
              } else {
                dst[i * RT] = packed_e(ev);
              }
            }
          }
        }
        sum += tile_sum;
      };
      // one window: tile t's scores to e in place (0 where unseen), their sum
      auto e_pass = [&](uint32_t t, uint32_t a) {
        const uint32_t key = t * BK + part * 32u;
        uint4* w4 = S4 + (t - a) * 4u * RT;
        if (unseen(key)) return;
        const bool mk = !whole(key);
        const uint32_t sk = mk ? seen(key) : 0u;
        uint32_t tile_sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
          uint32_t ev[8];
          const uint4 v = w4[j * RT];
          e_of8(re, (const uint32_t*)&v, ev, tab);
          if (mk) {
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) ev[k] = (sk >> (8u * j + k)) & 1u ? ev[k] : 0u;
          }
#pragma unroll
          for (uint32_t k = 0; k < 8; k++) tile_sum += ev[k];
          w4[j * RT] = packed_e(ev);
        }
        sum += tile_sum;
      };
      uint32_t R = 0, Rp = 0;
      bool pfast = true;
      // tile t's e to the bytes of P, into the MMAs' operand.  With 8 <= f_p <= 15 P is
      // the high word of e R 2^(f_p - 8) + 2^31; with any other f_p P is formed in place
      // before, and taken as it is
      auto p_any = [&](uint32_t t, uint32_t a, uint32_t fp) {
        uint32_t* w = (uint32_t*)(S4 + (t - a) * 4u * RT);
#pragma unroll 1
        for (uint32_t i = 0; i < 16 && !unseen(t * BK + part * 32u); i++) {
          uint32_t& x = w[(i >> 2) * 4u * RT + (i & 3u)];
          x = smx_p(e_unpack(x & 0xFFFFu), R, fp) | smx_p(e_unpack(x >> 16), R, fp) << 16;
        }
      };
      auto p_pass = [&](uint32_t t, uint32_t a) {
        const uint32_t pu = pt * Sh::CH + part / (Sh::PCH / 32u), buf = pu & 1u, uses = pu >> 1, key = t * BK + part * 32u;
        pt++;
        uint32_t pl[3][8];
        if (unseen(key)) {
#pragma unroll
          for (uint32_t k = 0; k < 24; k++) pl[k / 8][k % 8] = 0;
        } else {
#pragma unroll
          for (uint32_t j = 0; j < 4; j++) {
            const uint4 v = S4[((t - a) * 4u + j) * RT];
            const uint32_t xw[4] = {v.x, v.y, v.z, v.w};
            uint32_t p[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) {
              const uint32_t u = k & 1u ? xw[k / 2] >> 16 : xw[k / 2] & 0xFFFFu, ee = u + ((u + 1u) >> 16);
              p[k] = pfast ? (uint32_t)(((uint64_t)ee * Rp + (1ull << 31)) >> 32) : u;
            }
#pragma unroll
            for (uint32_t q = 0; q < 2; q++) {
              if (BITS == 16) {
                // saturated to 32767 as signed halves
                const uint32_t w0 = pack_s16(p[4 * q], p[4 * q + 1]), w1 = pack_s16(p[4 * q + 2], p[4 * q + 3]);
                pl[0][2 * j + q] = __byte_perm(w0, w1, 0x6420);
                pl[1][2 * j + q] = __byte_perm(w0, w1, 0x7531);
              } else {
                const uint32_t sw = *(const uint32_t*)(s_vshift + (key - a * BK) + j * 8u + 4u * q);
                uint32_t y[4];
#pragma unroll
                for (uint32_t x = 0; x < 4; x++) y[x] = min(p[4 * q + x], 32767u) << ((sw >> (8u * x)) & 31u);
                const uint32_t f = __byte_perm(y[0], y[1], 0x5140), z = __byte_perm(y[2], y[3], 0x5140);
                pl[0][2 * j + q] = __byte_perm(f, z, 0x5410);
                pl[1][2 * j + q] = __byte_perm(f, z, 0x7632);
                pl[2][2 * j + q] = __byte_perm(__byte_perm(y[0], y[1], 0x0062), __byte_perm(y[2], y[3], 0x0062), 0x5410);
              }
            }
          }
        }
        if (uses && ok) ok = wait_for(&p_empty[buf], (uses - 1u) & 1u, A.err, 318, A.waits);
        __syncwarp();
        sm100::tc_fence_after();
        const uint32_t ta = lane_base + Sh::P0 + buf * Sh::PCOLS + (part % (Sh::PCH / 32u)) * 8u;
#pragma unroll
        for (uint32_t k = 0; k < Sh::NP; k++) sm100::tmem_st8(ta + k * (Sh::PCH / 4), pl[k]);
        sm100::tmem_st_wait();
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&p_full[buf]);
      };

#pragma unroll 1
      for (uint32_t phase = 0; phase < 2; phase++) {
#pragma unroll 1
        for (uint32_t a = t0; a < t1; a += WIN) {
          const uint32_t e = min(a + WIN, t1);
          if (again) load_shifts(a, e);
          if (phase == 0 || again)
#pragma unroll 1
            for (uint32_t t = a; t < e; t++) score_pass(t, a, phase);
          else
#pragma unroll 1
            for (uint32_t t = a; t < e; t++) e_pass(t, a);
        }
        if (phase == 0) {
          s_pm[part][row] = max((int32_t)(int16_t)(mx & 0xFFFFu), (int32_t)mx >> 16);
          rows_sync();
          int32_t m = s_pm[0][row];
#pragma unroll
          for (uint32_t i = 1; i < PARTS; i++) m = max(m, s_pm[i][row]);
          if (X > 1) {
            if (part == 0) s_m[row] = m;
            meet();
            for (uint32_t i = 0; i < X; i++) m = max(m, (int32_t)cluster_ld32(cluster_addr(&s_m[row], i)));
          }
          re = row_e(A.d.smx[2u * head] & 0xFFFFFFu, A.d.smx[2u * head + 1u] & 63u, m);
        }
      }
      look(islot, ipar);
      s_ps[part][row] = sum;
      rows_sync();
      {
        unsigned long long total = s_ps[0][row];
#pragma unroll
        for (uint32_t i = 1; i < PARTS; i++) total += s_ps[i][row];
        if (X > 1) {
          if (part == 0) s_s[row] = total;
          meet();
          total = 0;
          for (uint32_t i = 0; i < X; i++) total += cluster_ld64(cluster_addr(&s_s[row], i));
        }
        R = smx_r(total);
      }
      const uint32_t fp = (A.d.smx[2u * head + 1u] >> 8) & 31u;
      pfast = __all_sync(0xffffffffu, fp >= 8u && fp <= 15u);
      Rp = pfast ? R << (fp - 8u) : R;
      more = s_go != 0u;
      uint32_t oacc[D];
#pragma unroll
      for (uint32_t k = 0; k < D; k++) oacc[k] = 0;
      uint4 qn[D / 8];  // the q that the next scores take
#pragma unroll 1
      for (uint32_t a = t0; a < t1; a += WIN) {
        const uint32_t e = min(a + WIN, t1);
        if (again) {
          load_shifts(a, e);
#pragma unroll 1
          for (uint32_t t = a; t < e; t++) score_pass(t, a, 2u);
        }
        if (!pfast)
#pragma unroll 1
          for (uint32_t t = a; t < e; t++) p_any(t, a, fp);
        if (again) rows_sync();  // every warp has read the scores: P goes over their columns
#pragma unroll 1
        for (uint32_t t = a; t < e; t++) p_pass(t, a);
        const bool last = e == t1;
        if (last ? more : Sh::Q_OVER) fetch_q(s_item[last ? islot : cur], qn);  // (its latency under the wait)
        // the window's P.V: this part's dimensions
        if (ok) ok = wait_for(&o_full, ou & 1u, A.err, 319, A.waits);
        ou++;
        __syncwarp();
        sm100::tc_fence_after();
#pragma unroll
        for (uint32_t k = 0; k < D; k += 16) {
          uint32_t hh[16], mid[16], ll[16];
          const uint32_t col = lane_base + part * D + k;
          sm100::tmem_ld16(col, hh);
          sm100::tmem_ld16(col + HD, mid);
          sm100::tmem_ld16(col + 2 * HD, ll);
          sm100::tmem_ld_wait();
#pragma unroll
          for (uint32_t x = 0; x < 16; x++) oacc[k + x] += hh[x] * A.k16 + (mid[x] * A.k8 + ll[x]);
        }
        if (last ? more : Sh::Q_OVER) store_q(qn);
        release();
      }
      if (t0 == t1) {  // no key is seen: no P.V to wait for, the next q takes its place here
        if (more) {
          fetch_q(s_item[islot], qn);
          store_q(qn);
        }
        release();
      }
      if (X > 1) {
        // the cluster's sums: every CTA leaves its own in shared memory, and adds up a slice
        rows_sync();
        uint4* so = (uint4*)s_S;  // [D / 4][RT]
#pragma unroll
        for (uint32_t k = 0; k < D; k += 4)
          so[(k / 4u) * RT + tid] = make_uint4(oacc[k], oacc[k + 1], oacc[k + 2], oacc[k + 3]);
        meet();
        // words of (thread's place, 4 dimensions): rank r takes every X-th
        for (uint32_t i = rank * RT + tid; i < D / 4u * RT; i += X * RT) {
          uint32_t v[4] = {0, 0, 0, 0};
          for (uint32_t q = 0; q < X; q++) {
            const uint32_t ad = cluster_addr(so + i, q);
#pragma unroll
            for (uint32_t x = 0; x < 4; x++) v[x] += cluster_ld32(ad + 4u * x);
          }
          const uint32_t th = i % RT, orow = ((th >> 5) & 3u) * 32u + (th & 31u);
          if (orow < it.nr) {
            const uint32_t o_r = it.r0 + orow, dim = (th >> 7) * D + 4u * (i / RT);
            int16_t* o = A.d.o + (uint64_t)(it.lo_row + o_r / G) * A.d.ldo + (uint64_t)(it.g * G + o_r % G) * HD + dim;
#pragma unroll
            for (uint32_t x = 0; x < 4; x++) o[x] = (int16_t)out16(v[x]);
          }
        }
      } else {
        // a row's D dimensions are W 16-byte words: W lanes trade them, so that each
        // store writes whole rows' parts (W lanes a row) instead of a word of 32 rows
        constexpr uint32_t W = D / 8;
        uint4 ow[W];
#pragma unroll
        for (uint32_t k = 0; k < W; k++) {
          uint32_t x[4];
#pragma unroll
          for (uint32_t i = 0; i < 4; i++)
            x[i] = pack_s16((uint32_t)((int32_t)oacc[8 * k + 2 * i] >> 8), (uint32_t)((int32_t)oacc[8 * k + 2 * i + 1] >> 8));
          ow[k] = make_uint4(x[0], x[1], x[2], x[3]);
        }
        int16_t* const o = A.d.o + (uint64_t)(it.lo_row + rr / G) * A.d.ldo + (uint64_t)head * HD + part * D;
        if (o16) {
#pragma unroll
          for (uint32_t st = W / 2; st > 0; st >>= 1) {  // after it, word k of lane l is word l % W of row l - l % W + k
            const bool up = lane & st;
#pragma unroll
            for (uint32_t k = 0; k < W; k++) {
              if (k & st) continue;
              const uint4 give = up ? ow[k] : ow[k | st];
              uint4 take;
              take.x = __shfl_xor_sync(0xffffffffu, give.x, st);
              take.y = __shfl_xor_sync(0xffffffffu, give.y, st);
              take.z = __shfl_xor_sync(0xffffffffu, give.z, st);
              take.w = __shfl_xor_sync(0xffffffffu, give.w, st);
              if (up) ow[k] = take;
              else ow[k | st] = take;
            }
          }
          const uint32_t first = row - lane % W;
#pragma unroll
          for (uint32_t k = 0; k < W; k++) {
            int16_t* const p = (int16_t*)__shfl_sync(0xffffffffu, (unsigned long long)o, (lane & ~(W - 1u)) + k);
            if (first + k < it.nr) *(uint4*)(p + 8u * (lane % W)) = ow[k];
          }
        } else if (row < it.nr) {
#pragma unroll
          for (uint32_t k = 0; k < W; k++) {
            const uint32_t x[4] = {ow[k].x, ow[k].y, ow[k].z, ow[k].w};
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
              o[8 * k + 2 * i] = (int16_t)x[i];
              o[8 * k + 2 * i + 1] = (int16_t)(x[i] >> 16);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&item_free[cur]);
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (X > 1) cluster_sync();  // no CTA leaves while another reads its shared memory
  if (warp == RW + 1u) {
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

constexpr uint32_t kTileSmem = 203u * 1024u;  // dynamic, of the 227 KB: the static arrays take 24

// how many clusters of X CTAs the current device holds at once (asked for once)
template <int HD, int BITS>
uint32_t resident_clusters(uint32_t X) {
  static std::atomic<int> known[16][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 16)
    if (const int n = known[dev][X].load(std::memory_order_relaxed)) return (uint32_t)n - 1u;
  auto kern = paged_attn_tile_kernel<HD, BITS>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(X * 1024u);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = kTileSmem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = X;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kTileSmem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  if (dev < 16) known[dev][X].store(n + 1, std::memory_order_relaxed);
  return (uint32_t)n;
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
  A.tiles = tiles;
  A.k8 = 1u << 8;
  A.k16 = 1u << 16;
  const uint32_t cap = c.table_width * c.page, keys = A.d.max_keys < cap ? A.d.max_keys : cap;
  const uint32_t span = A.d.window && A.d.window < keys ? A.d.window + BMR : keys;
  const uint32_t ktiles = ((span < keys ? span : keys) + BK - 1u) / BK + 1u;
  const uint64_t blocks = (uint64_t)c.B * c.KV * tiles;
  if (blocks > (1ull << 27)) return corm::fail(CORM_ELIMIT, "corm_llm_paged_attn: max_q %u over %u sequences", A.d.max_q, c.B);
  // two stages of at most 32 KB (a tile's copies are short beside its integer work); the
  // rest for scores
  A.stages = Sh::STAGE > 16384u ? 2u : 32768u / Sh::STAGE;
  const uint32_t tile_bytes = TILE_BYTES + (BITS == 8 ? 2u * BK : 0u);
  const uint32_t most = (kTileSmem - 1024u - A.stages * Sh::STAGE) / tile_bytes;
  // Shares of an item's keys.  A cluster's items cost its tiles of keys and the time of
  // about 3.5 more, a round of those at once resident or (unlike lengths overlap) a little
  // less than the items by those; without clusters a CTA goes from item to item.  8k keys
  // of 128 dimensions: 16 items 466 us with 1, 257 with 2, 144 with 4, 185 with 8; 36 items
  // 484, 257, 287, 279; 144 items of unlike lengths 489, 364; one prompt of 8192 1267, 1441
  const uint64_t live = live_tiles(A.d, BMR, tiles);
  uint32_t X = 1;
  float best = 0.0f;
  for (uint32_t x = 1; x <= 8u && (x == 1u || ktiles >= 4u * x); x *= 2u) {
    const float at_once = x == 1u ? 148.0f : (float)resident_clusters<HD, BITS>(x);
    if (at_once < 1.0f) continue;
    const float rounds = (float)live / at_once, least = c.B == 1u ? 2.0f : 1.5f;
    const float cost = (rounds <= 1.0f ? 1.0f : (0.9f * rounds > least ? 0.9f * rounds : least)) * ((float)ktiles / (float)x + 3.5f);
    if (x == 1u || cost < best) X = x, best = cost;
  }
  A.X = X;
  // the rows that see most first: a prompt's last tiles, or, where most keys were there
  // before the rows, the tiles of the sequences with most
  A.by_seq = c.B <= 32u && keys / 2u >= A.d.max_q;
  const uint32_t need = (ktiles + X - 1u) / X;
  A.win = need < 2u ? 2u : (need < most ? need : most);  // (a cluster's sums take up to two tiles' memory)
  const size_t smem = 1024u + A.stages * Sh::STAGE + (size_t)A.win * tile_bytes;
  auto kern = paged_attn_tile_kernel<HD, BITS>;
  // (one limit for every launch: another thread's may be between its limit and its launch)
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kTileSmem) != cudaSuccess)
    return corm::cuda_status("llm_paged_attn");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks * X);
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
  A.waits = waits();
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
