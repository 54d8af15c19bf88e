// What the two kernels of attention over the 4-bit pages share (kv4_attn.cu: items of 16 query
// rows, kv4_attn_wide.cu: items of 128): arguments, the list of chunks and its places, waits.
#pragma once

#include <math.h>

#include "common.cuh"
#include "kv4.cuh"
#include "tc_core.cuh"

namespace jsx {

constexpr int kKaChunk = 128;     // cache rows per stage
constexpr int kKaListMax = 512;   // (sequence, row tile) pairs up to which the chunk list is cut into ranges
constexpr float kKaOff = 10.f;    // weights are 2^(s - m + 10): f16 holds them down to 2^-34 of the largest
constexpr float kKaLazy = 4.f;    // the reference m moves when the maximum exceeds it by this much

static __device__ uint32_t g_kv4_error;

struct KaArgs {
  const bf16* q;
  bf16* out;
  int64_t q_stride, out_stride;  // per token, elements
  const uint8_t* pool;
  const int32_t* table;
  const int32_t* positions;
  const int32_t* n_tokens;
  float* parts;       // [2 x CTAs] records
  uint32_t* arrived;  // [kKaLevels][2 x CTAs], zero between calls
  int num_pages, slots, B, T, nkv, G, tiles, pt, pt_log, window, sinks;
  uint32_t per_g;  // 2^32 / G rounded up: x / G = umulhi(x, per_g) for x G < 2^32 (G > 1)
  int rows;    // query rows per item
  int listed;  // chunk list cut into ranges; else whole items per CTA
  int negate;        // the scale is negative
  float scale_log2;  // its magnitude x log2(e)
};

__device__ __forceinline__ int ka_div_g(const KaArgs& a, int x) { return a.G == 1 ? x : (int)__umulhi((uint32_t)x, a.per_g); }

// Rows of one (sequence, row tile): tokens t0..t1, cache rows below `hi`, chunks.
struct KaTile {
  int pos, t0, t1, used, hi, lo_chunk, sink_chunks, n;
};

__device__ __forceinline__ KaTile ka_tile(const KaArgs& a, int b, int tile) {
  KaTile x;
  x.pos = min(a.positions[b], 1 << 30);
  x.used = a.n_tokens ? min(max(a.n_tokens[b], 0), a.T) : a.T;
  x.t0 = ka_div_g(a, tile * a.rows);
  x.t1 = min(ka_div_g(a, min(tile * a.rows + a.rows, a.G * a.T) - 1), x.used - 1);
  x.hi = min(max(x.pos + x.t1 + 1, 0), a.slots * a.pt);
  x.n = x.lo_chunk = x.sink_chunks = 0;
  if (x.t0 > x.t1 || x.hi == 0) return x;
  const int lo = a.window > 0 ? max(x.pos + x.t0 - a.window + 1, 0) : 0;
  x.lo_chunk = lo / kKaChunk;
  const int end = (x.hi + kKaChunk - 1) / kKaChunk;
  x.sink_chunks = min((min(a.sinks, x.hi) + kKaChunk - 1) / kKaChunk, x.lo_chunk);
  x.n = x.sink_chunks + max(end - x.lo_chunk, 0);
  return x;
}

// A place in the list: an item, with the chunks [c0, c1) of it that are this CTA's.  Kept
// in shared memory, one for the copying warp and one for the computing ones.
struct KaPos {
  int live;
  int b, h, tile, c0, c1;
  int w, w1;         // place and end in the list
  int share, extra;  // how the list is cut
  KaTile x;
};

// The list is cut into ranges of `share` + 1 places (the first `extra` CTAs) and `share`:
// where CTA `cta`'s range begins, and the CTA whose range holds place u.
__device__ __forceinline__ int ka_range(const KaPos& p, int cta) { return cta * p.share + min(cta, p.extra); }
__device__ __forceinline__ int ka_owner(const KaPos& p, int u) {
  const uint32_t big = (uint32_t)p.share + 1u, edge = (uint32_t)p.extra * big;
  return (uint32_t)u < edge ? (uint32_t)u / big : p.extra + ((uint32_t)u - edge) / (uint32_t)p.share;
}

// The place after *p; cum[b]: chunks before sequence b.  Called by one thread: out of
// line, so that its code is there once.
static __device__ __noinline__ void ka_next(const KaArgs& a, const int* cum, KaPos* p) {
  KaPos q = *p;
  if (!a.listed) {
    q.w += gridDim.x;
    q.live = q.w < a.B * a.nkv * a.tiles;
    if (q.live) {
      q.tile = q.w % a.tiles;
      q.h = q.w / a.tiles % a.nkv;
      q.b = q.w / a.tiles / a.nkv;
      q.x = ka_tile(a, q.b, q.tile);
    }
  } else {
    q.w += q.c1 - q.c0;
    q.live = q.w < q.w1;
    if (q.live) do {
        if (++q.tile == a.tiles) {
          q.tile = 0;
          if (++q.h == a.nkv) {
            q.h = 0;
            do ++q.b;
            while (cum[q.b + 1] == cum[q.b]);
          }
        }
        q.x = ka_tile(a, q.b, q.tile);
      } while (q.x.n == 0);
  }
  q.c0 = 0;
  q.c1 = a.listed ? min(q.x.n, q.w1 - q.w) : q.x.n;
  *p = q;
}

// The CTA's first place, by one warp; in the listed form cum is filled on the way.
__device__ __forceinline__ KaPos ka_first(const KaArgs& a, int* cum, int lane) {
  KaPos q;
  if (!a.listed) {
    q.w = blockIdx.x;
    q.live = 1;
    q.tile = q.w % a.tiles;
    q.h = q.w / a.tiles % a.nkv;
    q.b = q.w / a.tiles / a.nkv;
    q.x = ka_tile(a, q.b, q.tile);
    q.c0 = 0;
    q.c1 = q.x.n;
    q.w1 = q.share = q.extra = 0;
    return q;
  }
  uint32_t total = 0;
#pragma unroll 2
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane;
    int n = 0;
    if (b < a.B)
      for (int t = 0; t < a.tiles; ++t) n += ka_tile(a, b, t).n;
    int v = n * a.nkv;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    if (b < a.B) cum[b + 1] = total + v;
    total += __shfl_sync(0xffffffffu, v, 31);
  }
  if (lane == 0) cum[0] = 0;
  __syncwarp();
  // CTAs with a range have a chunk at least
  q.share = total <= gridDim.x ? 1 : total / gridDim.x;
  q.extra = total <= gridDim.x ? 0 : total - q.share * gridDim.x;
  q.live = blockIdx.x < total;
  q.w = ka_range(q, blockIdx.x);
  q.w1 = ka_range(q, blockIdx.x + 1);
  q.b = q.h = q.tile = q.c0 = q.c1 = 0;
  if (!q.live) return q;
  int n = 0;  // sequences whose chunks begin at or before w: the last of them is it
  for (int b0 = 0; b0 < a.B; b0 += 32) n += __popc(__ballot_sync(0xffffffffu, b0 + lane < a.B && cum[b0 + lane] <= q.w));
  q.b = n - 1;
  int off = q.w - cum[q.b];
  if (a.tiles == 1) {
    q.x = ka_tile(a, q.b, 0);
    while (off >= q.x.n) {
      off -= q.x.n;
      ++q.h;
    }
  } else {
    int per = 0;
    for (int t = 0; t < a.tiles; ++t) per += ka_tile(a, q.b, t).n;
    while (off >= per) {
      off -= per;
      ++q.h;
    }
    for (;; ++q.tile) {
      q.x = ka_tile(a, q.b, q.tile);
      if (off < q.x.n) break;
      off -= q.x.n;
    }
  }
  q.c0 = off;
  q.c1 = min(q.x.n, off + q.w1 - q.w);
  return q;
}

__device__ __forceinline__ void ka_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(s_u32(dst)),
               "l"(src), "r"(bytes), "r"(s_u32(bar))
               : "memory");
}
__device__ __forceinline__ void ka_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ka_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t ka_h2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
// Shared-memory loads by 32-bit address.  Volatile: the copies that fill the stages are
// ordered by the barriers alone.
__device__ __forceinline__ uint4 ka_lds128(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p));
  return v;
}
__device__ __forceinline__ uint2 ka_lds64(uint32_t p) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p));
  return v;
}
__device__ __forceinline__ uint32_t ka_lds32(uint32_t p) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(p));
  return v;
}
__device__ __forceinline__ uint32_t ka_lds16(uint32_t p) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(p));
  return v;
}
__device__ __forceinline__ uint32_t ka_lds8(uint32_t p) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(p));
  return v;
}
// Bounded wait of a warp, false when it gave up; the waiting loop is out of line.
static __device__ __noinline__ bool ka_wait_slow(uint64_t* b, uint32_t parity, volatile uint32_t* abort) {
  return __all_sync(0xffffffffu, tc_wait_err(b, parity, abort, &g_kv4_error));
}
__device__ __forceinline__ bool ka_wait(uint64_t* b, uint32_t parity, volatile uint32_t* abort) {
  return __all_sync(0xffffffffu, tc_try_wait<false>(b, parity)) || ka_wait_slow(b, parity, abort);
}
__device__ __forceinline__ bool ka_nan_scale(uint32_t s) { return (s & 0x7fu) == 0x7fu; }

// The power of two that brings a row of q, whose largest magnitude has the bf16 bits `top`,
// to 2^8 .. 2^9, and the one that undoes it.
__device__ __forceinline__ float ka_q_scale(uint32_t top, float* undo) {
  const int e = (int)(top >> 7);  // exponent field of the largest
  const int f = e == 255 ? 127 : min(262 - e, 254);
  *undo = f == 254 ? 0x1p-127f : __uint_as_float((uint32_t)(254 - f) << 23);
  return __uint_as_float((uint32_t)f << 23);
}

}  // namespace jsx
