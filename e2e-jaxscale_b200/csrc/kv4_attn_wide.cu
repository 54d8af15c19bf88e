// Attention over the 4-bit key/value pages for many query rows per kv head (several tokens
// per sequence): items of 128 rows on the tcgen05 tensor cores, head_dim 128.
//
// The kernel of 16-row items (kv4_attn.cu) converts every cache row again for each 16 query
// rows, and its MMA, conversions and multiplications share the issue slots; here a cache row
// is converted once for 128 query rows and each product is issued by one thread.  Per step of
// 64 cache rows:
//   warps 10..17 codes -> f16 operands in shared memory, 128-byte swizzled, three steps ahead:
//                K [64][128] as it is (four warps), V transposed to [128][64] (four; the nibbles
//                of two rows interleaved before the conversion give a pair along the summed
//                axis).  Which 16 bytes of a row a lane reads moves with the lane: rows are 64
//                bytes apart, read straight they met in two bank groups (365 of 741 wavefronts
//                a step were conflicts, now 69 of 424);
//   warp 9       S = Q K^T (M 128, N 64, K 128) into one of four TMEM accumulators;
//   warp 18      O += P V (M 128, N 128, K 64) once P is there.  Two warps, and elect.sync rather
//                than a lane's branch, because issuing the twelve products is itself long
//                (64 tokens x 16 sequences of 8191: 235 -> 205 us by elect, 198 by two warps);
//   warps 0..3   a thread per query row, for even steps: tcgen05.ld of its 64 scores, mask,
//                running reference, weights as f16 into P; O stays in TMEM and is rescaled there
//                on the rare occasions that a row's reference moves;
//   warps 4..7   the same for odd steps, with a reference and an O of their own; the two meet at
//                an item's end (with one group of four every scheduler waited for one warp);
//   warp 8       places and pages (cp.async.bulk), running ahead.
// A stored value is exact in f16, q is scaled by a power of two per row, P has 11 bits: the
// same roundings as the 16-row kernel's.
//
// Bound: the two groups of softmax warps, two warps per scheduler, not the products.  A group's
// step takes 2700 cycles, 1300 of them for 64 exponentials, their conversions and sums, and shares
// the issue slots (55% taken) with the conversions of codes; an item's first rows and its end cost about 6 us a CTA, the
// joining launch 7.  32 heads on 2, 16 sequences of up to 8191 rows: 41 us for 5 tokens, 64 for
// 16, 198 for 64 (the 16-row kernel: 48, 130, 490), which is 0.45 PFLOP/s at 64; a prompt of
// 8192 tokens with a window of 4096: 980 us, 0.42 PFLOP/s.
//
// NaN: a row's NaN scale enters V as 0 (it would reach every query row through weights of
// 0) and is noted; the query rows that see it get their NaN when they are written.
//
// Items that several CTAs share leave (output, maximum, sum) records, which a second launch
// joins, 16 rows per CTA, in part order: a record is 64 KB, and more CTAs than there are
// items read them.
#include "kv4_attn.cuh"
#include "launch.cuh"

namespace jsx {

constexpr int kKwRows = 128;
constexpr int kKwStep = 64;  // cache rows per product
constexpr int kKwD = 128;
constexpr int kKwStages = 3;
constexpr int kKwBufs = 3;  // steps of operands ahead
constexpr int kKwThreads = 19 * 32;
constexpr int kKwCopyWarp = 8, kKwMmaWarp = 9, kKwKWarp = 10, kKwVWarp = 14, kKwPvWarp = 18;
constexpr int kKwStage = kv4_block_bytes(kKaChunk, kKwD);
constexpr int kKwQBytes = kKwRows * kKwD * 2;       // two blocks of [128 rows][64]
constexpr int kKwKBytes = kKwStep * kKwD * 2;       // two blocks of [64 rows][64]
constexpr int kKwVBytes = kKwD * kKwStep * 2;       // [128 dimensions][64 rows]
constexpr int kKwPBytes = kKwRows * kKwStep * 2;    // [128 query rows][64 rows]
constexpr int kKwOffK = kKwQBytes, kKwOffV = kKwOffK + kKwBufs * kKwKBytes, kKwOffP = kKwOffV + kKwBufs * kKwVBytes;
constexpr int kKwOffRing = kKwOffP + 2 * kKwPBytes;
constexpr int kKwSmem = kKwOffRing + kKwStages * kKwStage + 1024 /* align */;
constexpr uint32_t kKwTmemCols = 512, kKwTmemO = 256;  // S four times 64, O of even steps, O of odd ones
constexpr int kKwRecord = kKwRows * kKwD + 2 * kKwRows;  // floats: output [dimensions / 4][row][4], maxima, sums
// f16 x f16 -> f32, both operands K-major
constexpr uint32_t kw_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

int read_clear_kv4_wide_error(uint32_t* out) {
  const uint32_t zero = 0;
  JSX_CUDA(cudaMemcpyFromSymbol(out, g_kv4_error, sizeof(*out)));
  if (*out) JSX_CUDA(cudaMemcpyToSymbol(g_kv4_error, &zero, sizeof(zero)));
  return JSX_OK;
}

__device__ __forceinline__ void kw_sts128(uint32_t p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(p), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void kw_sts32(uint32_t p, uint32_t a) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(p), "r"(a) : "memory"); }
// One thread of a converged warp; operands of what it issues stay in uniform registers.
__device__ __forceinline__ bool kw_elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n selp.u32 %0, 1, 0, e;\n}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void kw_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// O's next 16 columns of this thread's lane, times f.
__device__ __forceinline__ void kw_scale16(uint32_t taddr, float f) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// 16-byte piece c of row r of a 128-byte-swizzled operand block
__device__ __forceinline__ uint32_t kw_at(uint32_t base, int r, int c) { return base + r * 128 + ((c ^ (r & 7)) << 4); }

struct KwInfo {
  int first, parts, odd, pad;  // CTAs of an item: first .. first + parts - 1; odd: the first one's second record
};

__global__ void __launch_bounds__(kKwThreads, 1) k_kv4_attn_wide(const __grid_constant__ KaArgs a, KwInfo* info) {
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ int cum[kKaListMax + 1];
  __shared__ KaPos place[2];
  __shared__ uint64_t full[kKwStages], empty[kKwStages], k_full[kKwBufs], k_free[kKwBufs], v_full[kKwBufs],
      v_free[kKwBufs], s_full[4], s_free[4], p_full[2], pv_done[2], begun[2], ended[2], q_ready, drained, met;
  __shared__ uint32_t present[kKwStages];  // pages of the stage that were copied
  __shared__ uint32_t step_rows[8];        // by step % 8: its 16-row pieces that are there (operands are made at most 5 steps
                                   // ahead of the last P, so no slot is written before it was read)
  __shared__ uint32_t nan_any[kKwBufs];          // a byte per V warp
  __shared__ __align__(16) uint8_t nan_row[kKwBufs][4][kKwStep];  // per 32 dimensions (a bit per group of 16) and cache row
  __shared__ float4 row_state[2][kKwRows];  // per group of softmax warps and query row: maximum, sum, NaN groups
  __shared__ uint32_t flags[2], tmem_at;
  volatile uint32_t* abort = flags;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = s_u32(smem);

  if (tid == 0) {
    for (int s = 0; s < kKwStages; ++s) {
      tc_mbar_init(&full[s], 1);
      tc_mbar_init(&empty[s], 8);
    }
    for (int s = 0; s < 2; ++s) {
      tc_mbar_init(&p_full[s], 4);
      tc_mbar_init(&pv_done[s], 1);
      tc_mbar_init(&begun[s], 1);
      tc_mbar_init(&ended[s], 18);
    }
    for (int s = 0; s < 4; ++s) {
      tc_mbar_init(&s_full[s], 2);
      tc_mbar_init(&s_free[s], 4);
    }
    for (int s = 0; s < kKwBufs; ++s) {
      tc_mbar_init(&k_full[s], 4);
      tc_mbar_init(&k_free[s], 1);
      tc_mbar_init(&v_full[s], 4);
      tc_mbar_init(&v_free[s], 1);
      nan_any[s] = 0;
    }
    tc_mbar_init(&q_ready, 8);
    tc_mbar_init(&met, 8);
    tc_mbar_init(&drained, 2);
    flags[0] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < kKwBufs * 4 * kKwStep / 4) reinterpret_cast<uint32_t*>(nan_row)[tid] = 0;
  // rows of P that no thread writes are zero for good
  for (int e = tid; e < 2 * kKwPBytes / 16; e += kKwThreads) kw_sts128(base + kKwOffP + e * 16, 0, 0, 0, 0);
  kw_proxy_fence();
  if (warp == kKwMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(&tmem_at)), "r"(kKwTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  pdl_wait();
  const uint32_t block = kv4_block_bytes(a.pt, kKwD);

  if (warp == kKwCopyWarp) {
    // ---- places and pages ----
    const int pages = kKaChunk >> a.pt_log;
    uint32_t f = 0, k = 0;
    const KaPos first = ka_first(a, cum, lane);
    if (lane == 0) place[0] = first;
    __syncwarp();
    bool ok = true;
    for (;; ++k) {
      KaPos& p = place[k & 1];
      if (lane == 0) tc_arrive(&begun[k & 1]);
      __syncwarp();
      if (!p.live) break;
      const int c0 = p.c0, c1 = p.c1, lo_chunk = p.x.lo_chunk, sink_chunks = p.x.sink_chunks, hi = p.x.hi;
      const int sinks = min(a.sinks, hi);
      const int32_t* table = a.table + (int64_t)p.b * a.slots;
      const int64_t head = p.h;
      auto look_up = [&](int c) {
        const int chunk = c < sink_chunks ? c : lo_chunk + c - sink_chunks;
        const int slot = chunk * pages + lane;
        return lane < pages && (slot << a.pt_log) < (c < sink_chunks ? sinks : hi) && slot < a.slots ? table[slot] : -1;
      };
      int soon = c0 < c1 ? look_up(c0) : -1;
      for (int c = c0; c < c1 && ok; ++c) {
        const uint32_t s = f % kKwStages;
        const int page = soon;
        if (c + 1 < c1) soon = look_up(c + 1);
        if (f >= kKwStages && !ka_wait(&empty[s], (f / kKwStages - 1) & 1, abort)) {
          ok = false;
          break;
        }
        const uint32_t have = __ballot_sync(0xffffffffu, page >= 0 && page < a.num_pages);
        if (lane == 0) {
          present[s] = have;
          tc_expect_tx(&full[s], __popc(have) * block);
        }
        __syncwarp();
        if (have >> lane & 1u)
          ka_copy(smem + kKwOffRing + s * kKwStage + lane * block, a.pool + ((int64_t)page * a.nkv + head) * block, block,
                  &full[s]);
        ++f;
      }
      if (ok && k >= 1) ok = ka_wait(&ended[(k + 1) & 1], ((k + 1) / 2 - 1) & 1, abort);
      if (!ok) break;
      if (lane == 0) {
        place[(k + 1) & 1] = p;
        ka_next(a, cum, &place[(k + 1) & 1]);
      }
      __syncwarp();
    }
    // the copies in flight land before this CTA's shared memory is given away, also when a wait gave up
    for (uint32_t x = f > kKwStages ? f - kKwStages : 0; x < f; ++x)
      tc_wait_err(&full[x % kKwStages], (x / kKwStages) & 1, nullptr, &g_kv4_error);

  } else if (warp == kKwMmaWarp || warp == kKwPvWarp) {
    // ---- products: S by one warp, O += P V by another (issuing is what they spend time on) ----
    uint32_t st = 0, asked = 0;  // steps and items with steps so far
    bool ok = true;
    for (uint32_t item = 0; ok; ++item) {
      ok = ka_wait(&begun[item & 1], (item / 2) & 1, abort);
      if (!ok || !place[item & 1].live) break;
      const int steps = (place[item & 1].c1 - place[item & 1].c0) * (kKaChunk / kKwStep);
      if (warp == kKwMmaWarp) {
        if (steps) {
          ok = ka_wait(&q_ready, asked & 1, abort);
          ++asked;
        }
        for (int n = 0; n < steps && ok; ++n) {
          const uint32_t x = st + n, buf = x % 4, kb = x % kKwBufs;
          if (x >= 4) ok = ka_wait(&s_free[buf], (x / 4 - 1) & 1, abort);
          if (ok) ok = ka_wait(&k_full[kb], (x / kKwBufs) & 1, abort);
          if (!ok) break;
          tc_fence_after();
          if (kw_elect()) {
#pragma unroll
            for (int kk = 0; kk < kKwD / 16; ++kk)
              tc_mma(tmem + buf * kKwStep,
                     umma_desc_sw128(base + (kk / 4) * (kKwQBytes / 2) + (kk % 4) * 32),
                     umma_desc_sw128(base + kKwOffK + kb * kKwKBytes + (kk / 4) * (kKwKBytes / 2) + (kk % 4) * 32),
                     kw_idesc(kKwRows, kKwStep), kk > 0);
            tc_commit(&s_full[buf]);
            tc_arrive(&s_full[buf]);  // (step_rows, seen by this thread, with it)
            tc_commit(&k_free[kb]);
          }
          __syncwarp();
        }
      } else {
        for (int n = 0; n < steps && ok; ++n) {
          const uint32_t x = st + n, buf = x & 1, kb = x % kKwBufs;
          ok = ka_wait(&v_full[kb], (x / kKwBufs) & 1, abort) && ka_wait(&p_full[buf], (x >> 1) & 1, abort);
          if (!ok) break;
          tc_fence_after();
          if (kw_elect()) {
#pragma unroll
            for (int kk = 0; kk < kKwStep / 16; ++kk)
              tc_mma(tmem + kKwTmemO + buf * kKwD, umma_desc_sw128(base + kKwOffP + buf * kKwPBytes + kk * 32),
                     umma_desc_sw128(base + kKwOffV + kb * kKwVBytes + kk * 32), kw_idesc(kKwRows, kKwD), n > 1 || kk > 0);
            tc_commit(&pv_done[buf]);
            tc_commit(&v_free[kb]);
          }
          __syncwarp();
        }
      }
      st += steps;
      __syncwarp();
      if (lane == 0) tc_arrive(&ended[item & 1]);
    }
    // products in flight end before TMEM is given back (only after a wait gave up are there any)
    if (lane == 0) tc_commit(&drained);
    __syncwarp();
    tc_wait_err(&drained, 0, nullptr, &g_kv4_error);

  } else if (warp >= kKwKWarp) {
    // ---- codes to operands ----
    const bool is_v = warp >= kKwVWarp;
    const int w = warp - (is_v ? kKwVWarp : kKwKWarp);
    uint32_t st = 0, f = 0;
    bool ok = true;
    for (uint32_t item = 0; ok; ++item) {
      ok = ka_wait(&begun[item & 1], (item / 2) & 1, abort);
      if (!ok || !place[item & 1].live) break;
      const int chunks = place[item & 1].c1 - place[item & 1].c0;
      for (int c = 0; c < chunks && ok; ++c, ++f) {
        const uint32_t s = f % kKwStages;
        ok = ka_wait(&full[s], (f / kKwStages) & 1, abort);
        if (!ok) break;
        const uint32_t ring = base + kKwOffRing + s * kKwStage, have = present[s];
        for (int half = 0; half < kKaChunk / kKwStep && ok; ++half, ++st) {
          const uint32_t buf = st % kKwBufs;
          if (st >= kKwBufs) ok = ka_wait(is_v ? &v_free[buf] : &k_free[buf], (st / kKwBufs - 1) & 1, abort);
          if (!ok) break;
          if (!is_v) {
            // two rows x 32 dimensions per thread; eight lanes of a phase read eight 16-byte pieces
            // of different banks: rows are 64 bytes apart, so the piece moves with the row
            const int c = (w + (lane >> 1)) & 3;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int key = lane + 32 * j, r = half * kKwStep + key, page = r >> a.pt_log, in = r & (a.pt - 1);
              const uint32_t at = ring + page * block;
              const uint4 code = ka_lds128(at + in * (kKwD / 2) + c * 16);
              const uint32_t sc = ka_lds16(at + kv4_off_ks(a.pt, kKwD) + in * (kKwD / 16) + c * 2);
              const uint32_t dst = base + kKwOffK + buf * kKwKBytes + (c >> 1) * (kKwKBytes / 2);
              const uint32_t both = e4m3x2_to_h2(sc), f2[2] = {__byte_perm(both, 0, 0x1010), __byte_perm(both, 0, 0x3232)};
              const uint32_t words[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t h[4];
                e2m1x8_to_h2(words[k], h);
                const uint32_t f = f2[k / 2];
                kw_sts128(kw_at(dst, key, (c & 1) * 4 + k), hmul2_u(h[0], f), hmul2_u(h[1], f), hmul2_u(h[2], f), hmul2_u(h[3], f));
              }
            }
            if (w == 0 && lane == 0) {
              uint32_t rows = 0;
              for (int u = 0; u < kKwStep / 16; ++u) rows |= (have >> ((half * kKwStep + u * 16) >> a.pt_log) & 1u) << u;
              step_rows[st % 8] = rows;
            }
          } else {
            // a pair of rows x 32 dimensions per thread, transposed a pair at a time; the pieces and
            // which row of the pair is read first move with the lane, for the banks' sake as above
            const int c = (w + lane) & 3, swap = lane >> 2 & 1;
            const int r = half * kKwStep + 2 * lane, page = r >> a.pt_log, in = r & (a.pt - 1);
            const uint32_t at = ring + page * block, codes = at + kv4_off_v(a.pt, kKwD) + in * (kKwD / 2) + c * 16;
            const uint4 one = ka_lds128(codes + swap * (kKwD / 2)), two = ka_lds128(codes + (swap ^ 1) * (kKwD / 2));
            const uint32_t scales = at + kv4_off_vs(a.pt, kKwD) + in * (kKwD / 16) + c * 2;
            uint32_t s0 = ka_lds16(scales), s1 = ka_lds16(scales + kKwD / 16);
            if (!(have >> page & 1u)) s0 = s1 = 0;
            const bool odd = ka_nan_scale(s0 & 0xff) || ka_nan_scale(s0 >> 8) || ka_nan_scale(s1 & 0xff) || ka_nan_scale(s1 >> 8);
            uint8_t* any = reinterpret_cast<uint8_t*>(&nan_any[buf]) + w;
            const bool before = *any != 0, now = __any_sync(0xffffffffu, odd);
            if (before || now) {  // note the rows
              nan_row[buf][c][2 * lane] = (uint8_t)(ka_nan_scale(s0 & 0xff) | ka_nan_scale(s0 >> 8) << 1);
              nan_row[buf][c][2 * lane + 1] = (uint8_t)(ka_nan_scale(s1 & 0xff) | ka_nan_scale(s1 >> 8) << 1);
              if (ka_nan_scale(s0 & 0xff)) s0 &= 0xff00;
              if (ka_nan_scale(s0 >> 8)) s0 &= 0xff;
              if (ka_nan_scale(s1 & 0xff)) s1 &= 0xff00;
              if (ka_nan_scale(s1 >> 8)) s1 &= 0xff;
              __syncwarp();
              if (lane == 0) *any = now;
            }
            // a factor per row of the pair, for each of the two groups
            const uint32_t fx = e4m3x2_to_h2(s0), fy = e4m3x2_to_h2(s1);
            const uint32_t f2[2] = {__byte_perm(fx, fy, 0x5410), __byte_perm(fx, fy, 0x7632)};
            const uint32_t first[4] = {one.x, one.y, one.z, one.w}, second[4] = {two.x, two.y, two.z, two.w};
            const uint32_t dst = base + kKwOffV + buf * kKwVBytes + c * 32 * 128 + (lane & 3) * 4;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t x = swap ? second[k] : first[k], y = swap ? first[k] : second[k];
              uint32_t h[2][4];
              e2m1x8_to_h2((x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u), h[0]);  // even dimensions
              e2m1x8_to_h2(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), h[1]);  // odd ones
#pragma unroll
              for (int d = 0; d < 8; ++d) kw_sts32(kw_at(dst, k * 8 + d, lane >> 2), hmul2_u(h[d & 1][d >> 1], f2[k / 2]));
            }
          }
          kw_proxy_fence();
          __syncwarp();
          if (lane == 0) tc_arrive(is_v ? &v_full[buf] : &k_full[buf]);
        }
        __syncwarp();
        if (ok && lane == 0) tc_arrive(&empty[s]);
      }
      __syncwarp();
      if (ok && lane == 0) tc_arrive(&ended[item & 1]);
    }

  } else {
    // ---- a query row per thread, even steps by warps 0..3 and odd ones by warps 4..7 ----
    const int grp = warp >> 2, r = tid & (kKwRows - 1);
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    uint32_t st = 0, meetings = 0;  // steps and meetings of the two groups so far
    bool ok = true;
    for (uint32_t item = 0; ok; ++item) {
      ok = ka_wait(&begun[item & 1], (item / 2) & 1, abort);
      if (!ok || !place[item & 1].live) break;
      const KaPos& it = place[item & 1];
      const int c0 = it.c0, c1 = it.c1, row = it.tile * kKwRows + r;
      const bool live = row < a.G * a.T;
      const bool busy = __any_sync(0xffffffffu, live);  // rows of this warp are someone's
      const int i = live ? ka_div_g(a, row) : 0, rowpos = it.x.pos + i;
      bf16* out = a.out + ((int64_t)it.b * a.T + i) * a.out_stride + (int64_t)(it.h * a.G + row - i * a.G) * kKwD;
      const bool on = live && i < it.x.used;
      float sc = 1e-37f;
      if (c0 < c1) {
        // q as f16, scaled per row by a power of two
        const uint4* q = reinterpret_cast<const uint4*>(a.q + ((int64_t)it.b * a.T + i) * a.q_stride +
                                                        (int64_t)(it.h * a.G + row - i * a.G) * kKwD);
        uint4 v[kKwD / 8];
#pragma unroll
        for (int c = 0; c < kKwD / 8; ++c) v[c] = live ? q[c ^ (8 * grp)] : make_uint4(0, 0, 0, 0);  // own half first
        uint32_t mx = 0;
#pragma unroll
        for (int c = 0; c < kKwD / 8; ++c)
          mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(v[c].x & 0x7fff7fffu, v[c].y & 0x7fff7fffu),
                                     __vmaxu2(v[c].z & 0x7fff7fffu, v[c].w & 0x7fff7fffu)));
        float undo;
        float mul = ka_q_scale(max(mx & 0xffffu, mx >> 16), &undo);
        sc = fmaxf(a.scale_log2 * undo, 1e-37f);  // never 0: 0 x -inf
        if (a.negate) mul = -mul;
#pragma unroll
        for (int c = 0; c < kKwD / 16; ++c)
          kw_sts128(kw_at(base + grp * (kKwQBytes / 2), r, c), ka_h2(bf_lo(v[c].x) * mul, bf_hi(v[c].x) * mul),
                    ka_h2(bf_lo(v[c].y) * mul, bf_hi(v[c].y) * mul), ka_h2(bf_lo(v[c].z) * mul, bf_hi(v[c].z) * mul),
                    ka_h2(bf_lo(v[c].w) * mul, bf_hi(v[c].w) * mul));
        kw_proxy_fence();
        __syncwarp();
        if (lane == 0) tc_arrive(&q_ready);
      }
      float m = -INFINITY, l = 0.f;
      uint32_t nan_groups = 0;
      const int all_hi = it.x.pos + it.x.t0, all_lo = a.window > 0 ? it.x.pos + it.x.t1 - a.window + 1 : 0;
      const int sink_chunks = it.x.sink_chunks, lo_chunk = it.x.lo_chunk;
      const int steps = (c1 - c0) * (kKaChunk / kKwStep);
      // (an item has an even number of steps, so a group's steps use one buffer: its own)
      for (int n = grp; n < steps && ok; n += 2) {
        const uint32_t x = st + n, buf = grp, kb = x % kKwBufs;
        ok = ka_wait(&s_full[x % 4], (x >> 2) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        if (busy) {
          const uint32_t rows = step_rows[x % 8];
          float s[kKwStep];
          tc_ld32(lanes + x % 4 * kKwStep, reinterpret_cast<float(&)[32]>(s[0]));
          tc_ld32(lanes + x % 4 * kKwStep + 32, reinterpret_cast<float(&)[32]>(s[32]));
          tc_fence_before();
          __syncwarp();
          if (lane == 0) tc_arrive(&s_free[x % 4]);
          const int c = c0 + n / 2;
          const int key0 = (c < sink_chunks ? c : lo_chunk + c - sink_chunks) * kKaChunk + (n & 1) * kKwStep;
          auto see = [&](int e) {
            const int key = key0 + e;
            return key <= rowpos && (a.window == 0 || key > rowpos - a.window || key < a.sinks) && (rows >> (e / 16) & 1u);
          };
          if (rows != 0xfu || key0 + kKwStep - 1 > all_hi || (key0 < all_lo && key0 + kKwStep > a.sinks)) {
#pragma unroll
            for (int e = 0; e < kKwStep; ++e)
              if (!see(e)) s[e] = -INFINITY;
          }
          float tops[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) tops[e] = s[e];
#pragma unroll
          for (int e = 8; e < kKwStep; ++e) tops[e % 8] = fmaxf(tops[e % 8], s[e]);
          const float top = sc * fmaxf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])),
                                       fmaxf(fmaxf(tops[4], tops[5]), fmaxf(tops[6], tops[7])));
          const bool move = top > m + kKaLazy;
          if (__any_sync(0xffffffffu, move)) {
            const float f = !move ? 1.f : m == -INFINITY ? 0.f : ka_exp2(m - top);
            if (move) m = top;
            l *= f;
            if (n > 1) {  // this group's O is complete, and nothing adds to it until P is handed over
              ok = ka_wait(&pv_done[buf], ((x >> 1) - 1) & 1, abort);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int y = 0; y < kKwD; y += 16) kw_scale16(lanes + kKwTmemO + buf * kKwD + y, f);
            }
          }
          const float ref = m == -INFINITY ? 0.f : kKaOff - m;
          if (x >= 2) ok = ka_wait(&pv_done[buf], ((x >> 1) - 1) & 1, abort);
          if (!ok) break;
          float sum[2] = {0.f, 0.f};
#pragma unroll
          for (int y = 0; y < kKwStep / 8; ++y) {
            uint32_t p2[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w0 = ka_exp2(__fmaf_rn(s[8 * y + 2 * e], sc, ref)), w1 = ka_exp2(__fmaf_rn(s[8 * y + 2 * e + 1], sc, ref));
              sum[0] += w0;
              sum[1] += w1;
              p2[e] = ka_h2(w0, w1);
            }
            kw_sts128(kw_at(base + kKwOffP + buf * kKwPBytes, r, y), p2[0], p2[1], p2[2], p2[3]);
          }
          l += sum[0] + sum[1];
          ok = ka_wait(&v_full[kb], (x / kKwBufs) & 1, abort);
          if (!ok) break;
          if (nan_any[kb] != 0) {
            for (int e = 0; e < kKwStep; ++e)
              if (see(e))
                for (int y = 0; y < 4; ++y) nan_groups |= (uint32_t)nan_row[kb][y][e] << (2 * y);
          }
          kw_proxy_fence();
        } else {
          if (lane == 0) tc_arrive(&s_free[x % 4]);
          if (x >= 2) ok = ka_wait(&pv_done[buf], ((x >> 1) - 1) & 1, abort);  // (or P's arrival could count for the step before)
          if (!ok) break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) tc_arrive(&p_full[buf]);
      }
      st += steps;
      if (!ok) break;
      // ---- the item's end: the groups' states meet, O out of TMEM, half of the dimensions each ----
      const bool whole = c1 - c0 == it.x.n;
      const int u0 = it.w - c0;
      int first = blockIdx.x, parts = 1;
      if (!whole) {
        first = ka_owner(it, u0);
        parts = ka_owner(it, u0 + it.x.n - 1) - first + 1;
      }
      const int odd = !whole && ka_range(it, first) < u0;
      if (tid == 0 && c0 == 0) info[((int64_t)it.b * a.nkv + it.h) * a.tiles + it.tile] = {first, parts, odd, 0};
      float weight[2] = {0.f, 0.f};
      if (steps) {
        row_state[grp][r] = make_float4(m, l, __uint_as_float(nan_groups), 0.f);
        __syncwarp();
        if (lane == 0) tc_arrive(&met);
        ok = ka_wait(&met, meetings++ & 1, abort) && ka_wait(&pv_done[0], ((st - 2) >> 1) & 1, abort) &&
             ka_wait(&pv_done[1], ((st - 1) >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const float4 other = row_state[grp ^ 1][r];
        const float to = fmaxf(m, other.x);
        weight[grp] = m == -INFINITY ? 0.f : ka_exp2(m - to);
        weight[grp ^ 1] = other.x == -INFINITY ? 0.f : ka_exp2(other.x - to);
        l = l * weight[grp] + other.y * weight[grp ^ 1];
        m = to;
        nan_groups |= __float_as_uint(other.z);
      }
      float* rec = a.parts + (size_t)(2 * blockIdx.x + (blockIdx.x == (unsigned)first ? odd : 0)) * kKwRecord;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (busy) {
#pragma unroll 1
        for (int x = 2 * grp; x < 2 * grp + 2; ++x) {
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.f;
          if (steps) {
#pragma unroll 1
            for (int y = 0; y < 2; ++y) {
              float o[32];
              tc_ld32(lanes + kKwTmemO + y * kKwD + x * 32, o);
              const float f = weight[y];
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] += o[e] * f;
            }
          }
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (nan_groups >> (2 * x + e / 16) & 1u) v[e] = NAN;
          if (live && whole) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = on ? v[e] * inv : 0.f;
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              *reinterpret_cast<uint4*>(out + x * 32 + e) =
                  make_uint4(pack2(v[e], v[e + 1]), pack2(v[e + 2], v[e + 3]), pack2(v[e + 4], v[e + 5]), pack2(v[e + 6], v[e + 7]));
          } else if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(rec + ((x * 32 + e) / 4 * kKwRows + r) * 4) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
          __syncwarp();
        }
        if (!whole && live && grp == 0) {
          rec[kKwRows * kKwD + r] = m;
          rec[kKwRows * kKwD + kKwRows + r] = l;
        }
      }
      // both groups have read both halves of O before either hands over the next item's first P
      tc_fence_before();
      __syncwarp();
      if (steps) {
        if (lane == 0) tc_arrive(&met);
        ok = ka_wait(&met, meetings++ & 1, abort);
        if (!ok) break;
      }
      if (lane == 0) tc_arrive(&ended[item & 1]);
      __syncwarp();
    }
    // rows of items without a chunk
    if (a.listed) {
      const int items = a.B * a.nkv * a.tiles;
      for (int k = blockIdx.x; k < items; k += gridDim.x) {
        const int tile = k % a.tiles, h = k / a.tiles % a.nkv, b = k / a.tiles / a.nkv;
        if (ka_tile(a, b, tile).n) continue;
        if (tid == 0) info[k] = {0, 1, 0, 0};
        const int row = tile * kKwRows + r, i = ka_div_g(a, row);
        if (row < a.G * a.T && grp == 0)
          for (int d = 0; d < kKwD; d += 8)
            *reinterpret_cast<uint4*>(a.out + ((int64_t)b * a.T + i) * a.out_stride + (int64_t)(h * a.G + row - i * a.G) * kKwD + d) =
                make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kKwMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kKwTmemCols));
  }
}

constexpr int kKjRows = 16, kKjThreads = 128, kKjMost = 160;  // (parts of an item: at most the SMs)

// grid (items, row groups of 16): joins the records of items that several CTAs shared.
__global__ void __launch_bounds__(kKjThreads) k_kv4_join(const __grid_constant__ KaArgs a, const KwInfo* info, int ctas) {
  __shared__ float wgt[kKjMost * kKjRows], part_sum[kKjThreads];
  pdl_wait();
  const int item = blockIdx.x, r0 = blockIdx.y * kKjRows, tid = threadIdx.x;
  const KwInfo x = info[item];
  const int tile = item % a.tiles, h = item / a.tiles % a.nkv, b = item / a.tiles / a.nkv;
  // (the bounds hold unless the first launch gave up before it wrote this)
  if (x.parts <= 1 || x.first < 0 || x.parts > ctas || x.first > ctas - x.parts || tile * kKwRows + r0 >= a.G * a.T) return;
  auto record = [&](int p) { return a.parts + (size_t)(2 * (x.first + p) + (p == 0 && x.odd ? 1 : 0)) * kKwRecord; };
  const int row = tid % kKjRows, p0 = tid / kKjRows, step = kKjThreads / kKjRows;
  constexpr int kMine = kKjRows * kKwD / 4 / kKjThreads;
  float4 v[kMine][4];
  auto load = [&](int q) {  // four parts of this thread's pieces (the last one again where there are fewer)
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float4* rec = reinterpret_cast<const float4*>(record(min(q + p, x.parts - 1))) + r0 + row;
#pragma unroll
      for (int k = 0; k < kMine; ++k) v[k][p] = rec[(p0 + k * step) * kKwRows];
    }
  };
  load(0);
  float top = -INFINITY;
  for (int p = p0; p < x.parts; p += step) {
    const float m = record(p)[kKwRows * kKwD + r0 + row];
    wgt[p * kKjRows + row] = m;
    top = fmaxf(top, m);
  }
  part_sum[tid] = top;
  __syncthreads();
#pragma unroll
  for (int y = 0; y < kKjThreads / kKjRows; ++y) top = fmaxf(top, part_sum[y * kKjRows + row]);
  __syncthreads();
  float sum = 0.f;
  for (int p = p0; p < x.parts; p += step) {
    const float m = wgt[p * kKjRows + row], f = m == -INFINITY ? 0.f : ka_exp2(m - top);
    wgt[p * kKjRows + row] = f;
    sum += record(p)[kKwRows * kKwD + kKwRows + r0 + row] * f;
  }
  part_sum[tid] = sum;
  __syncthreads();
  float4 acc[kMine];
#pragma unroll
  for (int k = 0; k < kMine; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int q = 0; q < x.parts; q += 4) {
    if (q) load(q);
#pragma unroll
    for (int p = 0; p < 4; ++p)
      if (q + p < x.parts)
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
          const float f = wgt[(q + p) * kKjRows + row];
          acc[k] = make_float4(acc[k].x + v[k][p].x * f, acc[k].y + v[k][p].y * f, acc[k].z + v[k][p].z * f, acc[k].w + v[k][p].w * f);
        }
  }
  const int used = a.n_tokens ? min(max(a.n_tokens[b], 0), a.T) : a.T;
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int d = (p0 + k * step) * 4, query = tile * kKwRows + r0 + row, i = ka_div_g(a, query);
    if (query >= a.G * a.T) continue;
    float l = 0.f;
#pragma unroll
    for (int y = 0; y < kKjThreads / kKjRows; ++y) l += part_sum[y * kKjRows + row];
    const float f = l == 0.f || i >= used ? 0.f : 1.f / l;
    uint2 o = make_uint2(pack2(acc[k].x * f, acc[k].y * f), pack2(acc[k].z * f, acc[k].w * f));
    if (i >= used) o = make_uint2(0u, 0u);
    *reinterpret_cast<uint2*>(a.out + ((int64_t)b * a.T + i) * a.out_stride + (int64_t)(h * a.G + query - i * a.G) * kKwD + d) = o;
  }
}

static size_t kw_info_bytes(int64_t items) { return ((size_t)items * sizeof(KwInfo) + 255) / 256 * 256; }
size_t kv4_wide_workspace(int B, int T, int nq, int nkv) {
  const int64_t items = (int64_t)B * nkv * ((nq / nkv * (int64_t)T + kKwRows - 1) / kKwRows);
  return kw_info_bytes(items) + 2 * (size_t)sm_count() * kKwRecord * 4;
}

// a: all but rows, tiles, listed and the workspace
int kv4_wide_launch(KaArgs a, void* workspace, cudaStream_t s) {
  static bool done[128] = {};
  int dev = 0;
  JSX_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 128 || !done[dev]) {
    JSX_CUDA(cudaFuncSetAttribute(k_kv4_attn_wide, cudaFuncAttributeMaxDynamicSharedMemorySize, kKwSmem));
    if (dev >= 0 && dev < 128) done[dev] = true;
  }
  a.rows = kKwRows;
  a.tiles = (a.G * a.T + kKwRows - 1) / kKwRows;
  const int64_t items = (int64_t)a.B * a.nkv * a.tiles;
  const int64_t chunks = items * (((int64_t)a.slots * a.pt + kKaChunk - 1) / kKaChunk);
  a.listed = (int64_t)a.B * a.tiles <= kKaListMax && chunks < (1 << 30);
  const int64_t units = a.listed ? chunks : items;
  const int most = sm_count() < kKjMost ? sm_count() : kKjMost;
  KwInfo* info = (KwInfo*)workspace;
  a.parts = (float*)((char*)workspace + kw_info_bytes(items));
  a.arrived = nullptr;
  const int ctas = (int)(units < most ? units : most);
  JSX_CUDA(launch_kernel(k_kv4_attn_wide, dim3(ctas), dim3(kKwThreads), kKwSmem, s, a, info));
  if (a.listed) {
    const int rows = a.G * a.T < kKwRows ? a.G * a.T : kKwRows;
    JSX_CUDA(launch_kernel(k_kv4_join, dim3((unsigned)items, (rows + kKjRows - 1) / kKjRows), dim3(kKjThreads), 0, s, a,
                           (const KwInfo*)info, ctas));
  }
  return JSX_OK;
}

}  // namespace jsx
