// Shared pieces of the paged KV-cache operators (paged.cu, paged_tile.cu):
// the geometry checks, a row's place in the batch, the softmax unit's integers
// and the warp-level byte shuffles.
//
// The cache: [pages][KV][page][row] bytes, a row of 16-bit words as two byte
// planes side by side (hi = v >> 8 signed, HD bytes; lo = v & 255, HD bytes) —
// the operands of the int8 tensor cores, so attention splits no word — or of
// 8-bit codes (HD bytes) with one shift per (page, KV head, row) in a second
// array: the word is code << shift.
#pragma once

#include "corm_common.cuh"
#include "corm_sm100.cuh"
#include "gemm_i8x4.h"

namespace paged {

// The descriptor's host checks every entry shares; what: the entry's name.
int check_cache(const corm_paged_cache* c, const char* what);

struct SeqRows {
  uint32_t lo, n;    // first packed row and rows of the sequence
  uint32_t pos, cap; // position of its first row; positions the table covers
};

// Sequence b, with the device arrays' values brought into range: cu within
// [0, rows] and not descending, pos not negative.
__device__ __forceinline__ SeqRows seq_rows(const corm_paged_cache& c, uint32_t b, uint32_t rows) {
  const int32_t a = c.cu[b], e = c.cu[b + 1], p = c.pos[b];
  SeqRows s;
  s.lo = min((uint32_t)max(a, 0), rows);
  const uint32_t hi = min((uint32_t)max(e, 0), rows);
  s.n = hi > s.lo ? hi - s.lo : 0u;
  s.cap = c.table_width * c.page;
  s.pos = (uint32_t)max(p, 0);
  return s;
}

// ---------------------------------------------------------------- the softmax unit's integers
// e of a score d below the row's maximum: y = (d Cm) >> Cs, TAB[y mod 4096] >>
// (y / 4096); the form for any Cs (below 8 y may pass 32 bits), the table held less
// one in 16 bits (TAB is 32774 .. 65536)
__device__ __forceinline__ uint32_t smx_e_wide(uint32_t d, uint32_t cm, uint32_t cs, const uint16_t* tab) {
  const uint64_t y = ((uint64_t)d * (cm & 0xFFFFFFu)) >> cs;
  return (y >> 12) > 16u ? 0u : ((uint32_t)tab[y & 4095u] + 1u) >> (uint32_t)(y >> 12);
}
// e in 16 bits: TAB[0] = 65536 is the only value past 65535, and no entry is 65535
__device__ __forceinline__ uint32_t e_unpack(uint32_t h) { return h + (h == 65535u ? 1u : 0u); }

// P = min((e R + 2^(39 - f_p)) >> (40 - f_p), 32767); e R < 2^41
__device__ __forceinline__ uint32_t smx_p(uint32_t e, uint32_t R, uint32_t fp) {
  const uint64_t v = ((uint64_t)e * R + (1ull << (39u - fp))) >> (40u - fp);
  return v > 32767ull ? 32767u : (uint32_t)v;
}
// R = floor(2^40 / S) for 2^16 <= S <= 2^40 (S >= 2^16 wherever a row sees a key).  The
// single-precision reciprocal is within 2^-22: R0 is within 5 of the quotient (below
// 2^24), and the exact remainder corrects it: first by its own quotient, then by one
__device__ __forceinline__ uint32_t smx_r(unsigned long long S) {
  if (S < 65536ull || S > (1ull << 40)) return 0u;
  const float inv = __frcp_rn((float)S);
  uint32_t r = (uint32_t)(1099511627776.0f * inv);
  long long rem = (1ll << 40) - (long long)(r * S);
  const int q = (int)((float)rem * inv);  // (towards zero)
  r += (uint32_t)q;
  rem -= q * (long long)S;
  if (rem < 0) r--;
  else if (rem >= (long long)S) r++;
  return r;
}

// an exact sum modulo 2^32 as the kernels round it: floor / 2^8, saturated
__device__ __forceinline__ int32_t out16(uint32_t acc) {
  const int32_t y = (int32_t)acc >> 8;
  return min(max(y, -32768), 32767);
}
// two values saturated to 16 bits in a word (lo in the low half)
__device__ __forceinline__ uint32_t pack_s16(uint32_t lo, uint32_t hi) {
  uint32_t r;
  asm("cvt.pack.sat.s16.s32 %0, %1, %2;" : "=r"(r) : "r"(hi), "r"(lo));
  return r;
}
__device__ __forceinline__ uint32_t shr_clamp(uint32_t x, uint32_t s) {  // 0 from 32 up
  uint32_t r;
  asm("shr.u32 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(s));
  return r;
}
__device__ __forceinline__ uint32_t pack_u16(uint32_t lo, uint32_t hi) {
  uint32_t r;
  asm("cvt.pack.sat.u16.s32 %0, %1, %2;" : "=r"(r) : "r"(hi), "r"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack16(int32_t lo, int32_t hi) {  // both already in int16
  return ((uint32_t)hi << 16) | ((uint32_t)lo & 0xFFFFu);
}

// C[16 x 8] += A[16 x 32] B[32 x 8] on 8-bit operands, int32 sums modulo 2^32
// (warp-level; for tiles of 8 query rows)
#define CORM_MMA_I8(NAME, TA, TB)                                                                                      \
  __device__ __forceinline__ void NAME(uint32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {           \
    asm("mma.sync.aligned.m16n8k32.row.col.s32." TA "." TB                                                    \
                 ".s32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"                                             \
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])                                                      \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));                                      \
  }                                                                                                                    \
  /* C = A B */                                                                                                        \
  __device__ __forceinline__ void NAME##_first(uint32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {   \
    asm("mma.sync.aligned.m16n8k32.row.col.s32." TA "." TB                                                    \
                 ".s32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%10,%10,%10,%10};"                                         \
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])                                                      \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));                              \
  }
CORM_MMA_I8(mma_ss, "s8", "s8")
CORM_MMA_I8(mma_su, "s8", "u8")
CORM_MMA_I8(mma_us, "u8", "s8")
CORM_MMA_I8(mma_uu, "u8", "u8")
#undef CORM_MMA_I8

// 8-bit operand fragments from shared memory, a row of 16 bytes a lane: a 16 x 32 (or
// 16 x 16) A operand as it lies, and one of 32 rows whose columns become A's rows (two
// 16 x 16 byte matrices transposed: lane l gets column l / 4, then l / 4 + 8, of rows
// 4 (l mod 4) .. + 3, then of those 16 on)
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x2(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix_t8(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}

// ---------------------------------------------------------------- waits
// How long a kernel's waits may take: clock cycles, about 2 s unless the host set
// another limit (corm_set_wait_limit).  nap: each look may suspend the warp for so many
// nanoseconds (20 us, so that the many warps that wait leave the issue slots to those that
// work; 0 with a short limit, so that it counts).
struct Waits {
  long long limit;
  uint32_t nap;
};
constexpr Waits kWaits = {4000000000ll, 20000u};
inline Waits waits() {
  const long long limit = corm::wait_limit();
  return {limit, limit < sm100::kShortWaitLimit ? 0u : kWaits.nap};
}
__device__ __forceinline__ bool try_wait_nap(uint64_t* bar, uint32_t parity, uint32_t nap) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(sm100::smem_u32(bar)), "r"(parity), "r"(nap)
      : "memory");
  return ok != 0;
}
// Bounded like sm100::mbar_wait
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int* err, int code, Waits w) {
  if (try_wait_nap(bar, parity, w.nap)) return true;
  const long long t0 = clock64();
  while (!try_wait_nap(bar, parity, w.nap)) {
    if (clock64() - t0 > w.limit) {
      if (err) atomicCAS(err, 0, code);
      return false;
    }
  }
  return true;
}

// ---------------------------------------------------------------- copies and clusters
// 16 bytes, the first n of them from memory (n = 0: zeros)
__device__ __forceinline__ void cp_async16(void* dst, const void* src, uint32_t n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sm100::smem_u32(dst)), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of this CTA's shared variable p in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(sm100::smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ uint32_t cluster_ld32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long cluster_ld64(uint32_t a) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
// bounded, acquiring what the cluster's CTAs released by their arrivals (a look that
// suspends the warp as long as the hardware likes; with a short limit one look that does not)
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, int* err, int code, const Waits& w) {
  const long long t0 = clock64();
  do {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %3, 0;\n\t"
        "@q mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "@!q mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(sm100::smem_u32(bar)), "r"(parity), "r"(w.nap)
        : "memory");
    if (ok) return true;
  } while (clock64() - t0 <= w.limit);
  atomicCAS(err, 0, code);
  return false;
}
__device__ __forceinline__ void mbar_arrive_remote(const uint64_t* bar, uint32_t rank) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr(bar, rank)) : "memory");
}

}  // namespace paged
