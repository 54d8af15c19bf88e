// Sharing, growing, shrinking and compacting the pages of a paged cache, on the
// device: which sequence holds which page is a table [S][slots] of page numbers,
// held[S] says how many slots of a row are in use and refs[P] how many rows (and
// other holders) have a page; refs 0 is a free page.  Nothing is read back to
// the host, so scheduling steps chain with the model's on one stream.
//
//   fork     row b becomes row parent[b]: integer updates only, no page moves;
//   resize   keep the first tokens of every row and make room for more: pages
//            that will be written and that others hold too are replaced
//            (copy-on-write), missing ones are taken from the free pages, the
//            rest is given back;
//   compact  live pages move into the free ones below, so that the pool's upper
//            part becomes free.
//
// The bookkeeping of a call is one CTA, or one cluster of 8 (8192 threads) for large pools:
// its phases depend on one another (count, rank, assign) and the barrier orders
// them without further launches.  Ranks are prefix sums over page and sequence
// order, so the pages chosen do not depend on the order of execution.  Page
// bytes move in a second launch, one (page, layer) unit per CTA at a time,
// reading the page list that the first one wrote.  Bound: the copy by memory once there is
// more than a few megabytes to move (500 pages of 40 layers, 737 MB read and written: 128 us
// with the bookkeeping, 0.88 of the copy rate; one load of a page in flight at a time: 147 us),
// the bookkeeping by its chain of barriers and loads (forking one row into 4: 8.6 us,
// 8 into 64 with growth and the copies: 27 us).
#include "common.cuh"
#include "launch.cuh"

namespace jsx {

constexpr int kPgCtas = 8;
constexpr int kPgThreads = 1024;
constexpr int kPgCopyThreads = 288;  // pages are multiples of 72 vectors of 16 bytes; 1152 (2 kv heads, 64 x 128) are four each

// workspace (int32): header [16], cnt [S], base [S], src [cap], dst [cap], ref [cap]
constexpr int kPgHeader = 16;  // [0] pages in the list
static size_t pages_cap(int S, int slots, int P) {
  const long long most = (long long)S * slots;
  const long long grow = most < P ? most : P, moves = (P + 1) / 2;
  return (size_t)(grow > moves ? grow : moves);
}
static size_t pages_ws_bytes(int S, int slots, int P) {
  return 4 * ((size_t)kPgHeader + 2 * (size_t)S + 3 * pages_cap(S, slots, P));
}

struct PgWs {
  int32_t *head, *cnt, *base, *src, *dst, *ref;
};
static PgWs pages_ws(void* w, int S, int slots, int P) {
  PgWs x;
  x.head = (int32_t*)w;
  x.cnt = x.head + kPgHeader;
  x.base = x.cnt + S;
  x.src = x.base + S;
  x.dst = x.src + pages_cap(S, slots, P);
  x.ref = x.dst + pages_cap(S, slots, P);
  return x;
}

__device__ __forceinline__ uint32_t pg_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// barrier over the kCtas CTAs; global and shared writes before it are visible after it
template <int kCtas>
__device__ __forceinline__ void pg_sync() {
  if constexpr (kCtas == 1) {
    __syncthreads();
    return;
  }
  __threadfence();
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int kCtas>
__device__ __forceinline__ int pg_peer(const int* p, uint32_t rank) {
  if constexpr (kCtas == 1) return *p;
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return (int)v;
}
// exclusive prefix sum over the CTA's threads; the sum of all in *total
__device__ __forceinline__ int pg_scan(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the previous use of warp_sums is over
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *total = warp_sums[31];
  return x - v + (warp > 0 ? warp_sums[warp - 1] : 0);
}
// this thread's pages [lo, hi) of the CTAs' partition of [0, P)
template <int kCtas>
__device__ __forceinline__ void pg_range(int P, uint32_t cta, int* lo, int* hi) {
  const int per = (P + kCtas * kPgThreads - 1) / (kCtas * kPgThreads);
  const long long l = (long long)(cta * kPgThreads + threadIdx.x) * per;
  *lo = (int)(l < P ? l : P);
  *hi = (int)(l + per < P ? l + per : P);
}
__device__ __forceinline__ int pg_held(const int32_t* held, int s, int slots) {
  const int h = held[s];
  return h < 0 ? 0 : h > slots ? slots : h;
}

struct PgForkArgs {
  const int32_t *table, *held, *refs, *parent;
  int32_t *table_out, *held_out, *refs_out;
  int S, slots, P;
};

template <int kCtas>
__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kPgThreads) k_pages_fork(PgForkArgs a) {
  pdl_wait();
  const uint32_t cta = pg_rank();
  const int lane = threadIdx.x & 31, w0 = cta * (kPgThreads / 32) + (threadIdx.x >> 5);
  for (int p = cta * kPgThreads + threadIdx.x; p < a.P; p += kCtas * kPgThreads) a.refs_out[p] = a.refs[p];
  for (int s = w0; s < a.S; s += kCtas * kPgThreads / 32) {
    const int par = a.parent[s];
    const int h = par >= 0 && par < a.S ? pg_held(a.held, par, a.slots) : 0;
    for (int i = lane; i < a.slots; i += 32)
      a.table_out[(size_t)s * a.slots + i] = i < h ? a.table[(size_t)par * a.slots + i] : -1;
    if (lane == 0) a.held_out[s] = h;
  }
  pg_sync<kCtas>();  // refs_out holds the old counts
  for (int s = w0; s < a.S; s += kCtas * kPgThreads / 32) {
    const int par = a.parent[s];
    if (par == s) continue;
    const int h0 = pg_held(a.held, s, a.slots);
    const int h1 = par >= 0 && par < a.S ? pg_held(a.held, par, a.slots) : 0;
    for (int i = lane; i < h0; i += 32) {
      const int p = a.table[(size_t)s * a.slots + i];
      if (p >= 0 && p < a.P) atomicSub(&a.refs_out[p], 1);
    }
    for (int i = lane; i < h1; i += 32) {
      const int p = a.table[(size_t)par * a.slots + i];
      if (p >= 0 && p < a.P) atomicAdd(&a.refs_out[p], 1);
    }
  }
}

struct PgResizeArgs {
  int32_t *table, *held, *refs;
  const int32_t *keep, *need;
  int32_t* missing;
  PgWs ws;
  int S, slots, P, pt;
};

// Slots of sequence s: in use before, in use after, and the first that will be written.  A row
// keeps no more than its pages hold, so first <= before: the slots from `before` on that are
// counted as taken are the ones that are assigned, and no entry of the list is left unwritten.
struct PgRow {
  int before, after, first, over;  // over: pages beyond the table's slots
  int keep;
};
__device__ __forceinline__ PgRow pg_row(const PgResizeArgs& a, int s) {
  PgRow r;
  const int need = max(a.need[s], 0);
  const int n = need / a.pt + (need % a.pt != 0);
  r.before = pg_held(a.held, s, a.slots);
  r.keep = (int)min((long long)min(max(a.keep[s], 0), need), (long long)r.before * a.pt);
  r.after = min(n, a.slots);
  r.over = min(n - r.after, 1 << 15);  // (a sum over 2^15 rows stays in 31 bits)
  r.first = r.keep / a.pt;
  return r;
}

template <int kCtas>
__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kPgThreads) k_pages_resize(PgResizeArgs a) {
  __shared__ int warp_sums[32];
  __shared__ int mine;
  pdl_wait();
  const uint32_t cta = pg_rank();
  const int tid = threadIdx.x, lane = tid & 31, w0 = cta * (kPgThreads / 32) + (tid >> 5);
  auto writable = [&](int page) { return page >= 0 && page < a.P && a.refs[page] <= 1; };

  // pages that every sequence takes
  for (int s = w0; s < a.S; s += kCtas * kPgThreads / 32) {
    const PgRow r = pg_row(a, s);
    int n = 0;
    for (int i = r.first + lane; i < min(r.before, r.after); i += 32) n += !writable(a.table[(size_t)s * a.slots + i]);
    n = __reduce_add_sync(0xffffffffu, n);
    // a row that needs more slots than the table has cannot be served
    if (lane == 0) {
      a.ws.cnt[s] = n + max(r.after - r.before, 0);
      a.ws.base[s] = r.over;
    }
  }
  // free pages of this thread's range
  int lo, hi, total_free;
  pg_range<kCtas>(a.P, cta, &lo, &hi);
  int nfree = 0;
  for (int p = lo; p < hi; ++p) nfree += a.refs[p] == 0;
  int rank = pg_scan(nfree, warp_sums, &total_free);
  if (tid == 0) mine = total_free;
  pg_sync<kCtas>();
  int found = 0;
  for (int r = 0; r < kCtas; ++r) {
    const int n = pg_peer<kCtas>(&mine, r);
    if (r < (int)cta) rank += n;
    found += n;
  }
  // where every sequence's pages begin in the list of free ones (each CTA computes it, the first keeps it)
  const int per = (a.S + kPgThreads - 1) / kPgThreads;
  const int s0 = min(tid * per, a.S), s1 = min(s0 + per, a.S);
  int n = 0, over = 0, total, total_over;
  for (int s = s0; s < s1; ++s) {
    n += a.ws.cnt[s];
    over += a.ws.base[s];
  }
  int base = pg_scan(n, warp_sums, &total);
  pg_scan(over, warp_sums, &total_over);
  const int missing = max(total - found, 0) + total_over;
  pg_sync<kCtas>();  // everyone has read cnt and base
  if (missing == 0) {
    for (int p = lo; p < hi && rank < total; ++p)
      if (a.refs[p] == 0) a.ws.dst[rank++] = p;
    if (cta == 0)
      for (int s = s0; s < s1; ++s) {
        a.ws.base[s] = base;
        base += a.ws.cnt[s];
      }
  }
  if (cta == 0 && tid == 0) {
    a.ws.head[0] = missing ? 0 : total;
    *a.missing = missing;
  }
  pg_sync<kCtas>();
  if (missing) return;  // all or nothing

  // Whether a page is shared is asked of the counts before this call: they are
  // changed only after every warp of the cluster has its answers.
  for (int s = w0; s < a.S; s += kCtas * kPgThreads / 32) {
    const PgRow r = pg_row(a, s);
    int at = a.ws.base[s];
    for (int i0 = r.first; i0 < r.after; i0 += 32) {
      const int i = i0 + lane;
      int old = -1;
      bool take = false;
      if (i < r.after) {
        if (i < r.before) old = a.table[(size_t)s * a.slots + i];
        take = i >= r.before || !writable(old);
      }
      const uint32_t m = __ballot_sync(0xffffffffu, take);
      if (take) {
        const int k = at + __popc(m & ((1u << lane) - 1u));
        const bool was = old >= 0 && old < a.P;
        a.ws.src[k] = was && (long long)i * a.pt < r.keep ? old : -1;
        a.ws.ref[k] = was ? old : -1;  // gives its hold back
        a.table[(size_t)s * a.slots + i] = a.ws.dst[k];
      }
      at += __popc(m);
    }
  }
  pg_sync<kCtas>();
  for (int k = cta * kPgThreads + tid; k < total; k += kCtas * kPgThreads) {
    a.refs[a.ws.dst[k]] = 1;
    if (a.ws.ref[k] >= 0) atomicSub(&a.refs[a.ws.ref[k]], 1);
  }
  for (int s = w0; s < a.S; s += kCtas * kPgThreads / 32) {
    const PgRow r = pg_row(a, s);
    for (int i = r.after + lane; i < r.before; i += 32) {
      int32_t* e = &a.table[(size_t)s * a.slots + i];
      if (*e >= 0 && *e < a.P) atomicSub(&a.refs[*e], 1);
      *e = -1;
    }
    __syncwarp();
    if (lane == 0) a.held[s] = r.after;
  }
}

struct PgCompactArgs {
  const int32_t *table, *held, *refs;
  int32_t *refs_out, *remap;
  PgWs ws;
  int S, slots, P;
};

// refs_out may be refs: every count is read before the last barrier, written after it.
template <int kCtas>
__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kPgThreads) k_pages_plan(PgCompactArgs a) {
  __shared__ int warp_sums[32];
  __shared__ int mine[3];
  pdl_wait();
  const uint32_t cta = pg_rank();
  const int tid = threadIdx.x;
  int lo, hi, n = 0, total;
  pg_range<kCtas>(a.P, cta, &lo, &hi);
  for (int p = lo; p < hi; ++p) n += a.refs[p] > 0;
  pg_scan(n, warp_sums, &total);
  if (tid == 0) mine[0] = total;
  pg_sync<kCtas>();
  int live = 0;
  for (int r = 0; r < kCtas; ++r) live += pg_peer<kCtas>(&mine[0], r);
  int holes = 0, movers = 0;
  for (int p = lo; p < hi; ++p) {
    const bool on = a.refs[p] > 0;
    holes += !on && p < live;
    movers += on && p >= live;
  }
  int hole_rank = pg_scan(holes, warp_sums, &total);
  if (tid == 0) mine[1] = total;
  int mover_rank = pg_scan(movers, warp_sums, &total);
  if (tid == 0) mine[2] = total;
  pg_sync<kCtas>();
  int moved = 0;
  for (int r = 0; r < kCtas; ++r) {
    const int h = pg_peer<kCtas>(&mine[1], r), m = pg_peer<kCtas>(&mine[2], r);
    if (r < (int)cta) {
      hole_rank += h;
      mover_rank += m;
    }
    moved += m;
  }
  for (int p = lo; p < hi; ++p) {
    const int r = a.refs[p];
    if (r <= 0 && p < live) a.ws.dst[hole_rank++] = p;
    if (r > 0 && p >= live) {
      a.ws.src[mover_rank] = p;
      a.ws.ref[mover_rank++] = r;
    }
  }
  if (cta == 0 && tid == 0) a.ws.head[0] = moved;
  pg_sync<kCtas>();
  for (int p = lo; p < hi; ++p) {
    const int r = a.refs[p];
    if (p >= live) {
      a.refs_out[p] = 0;
      if (r <= 0) a.remap[p] = -1;
    } else if (r > 0) {
      a.refs_out[p] = r;
      a.remap[p] = p;
    } else {
      a.remap[p] = -1;
    }
  }
  pg_sync<kCtas>();  // with refs_out == refs, a hole's count is read above and written below
  for (int k = cta * kPgThreads + tid; k < moved; k += kCtas * kPgThreads) {
    a.refs_out[a.ws.dst[k]] = a.ws.ref[k];
    a.remap[a.ws.src[k]] = a.ws.dst[k];
  }
}

struct PgCopyArgs {
  uint4* pool;
  size_t page_vecs, layer_vecs;  // 16-byte units of a page and of a layer's pool
  int layers;
  PgWs ws;
  // compaction: entries of the table renamed on the way (table_out null: none)
  const int32_t *table, *held, *remap;
  int32_t* table_out;
  int S, slots, P;
};

__global__ void __launch_bounds__(kPgCopyThreads) k_pages_copy(PgCopyArgs a) {
  pdl_wait();
  const int tid = threadIdx.x;
  if (a.table_out) {
    const long long n = (long long)a.S * a.slots;
    for (long long e = (long long)blockIdx.x * kPgCopyThreads + tid; e < n; e += (long long)gridDim.x * kPgCopyThreads) {
      const int s = (int)(e / a.slots), i = (int)(e % a.slots);
      const int p = a.table[e];
      a.table_out[e] = i < pg_held(a.held, s, a.slots) && p >= 0 && p < a.P ? a.remap[p] : -1;
    }
  }
  // a CTA takes as many (page, layer) units at once as its threads cover; all of a
  // thread's loads are in flight before its first store
  const int together = a.page_vecs < kPgCopyThreads ? kPgCopyThreads / (int)a.page_vecs : 1;
  const int mine = together > 1 ? tid / (int)a.page_vecs : 0, v0 = tid - mine * (int)a.page_vecs;
  const long long units = (long long)a.ws.head[0] * a.layers;
  if (mine >= together) return;
  for (long long u = (long long)blockIdx.x * together + mine; u < units; u += (long long)gridDim.x * together) {
    const int k = (int)(u / a.layers), l = (int)(u % a.layers);
    const int from = a.ws.src[k];
    if (from < 0) continue;
    const uint4* s = a.pool + (size_t)l * a.layer_vecs + (size_t)from * a.page_vecs;
    uint4* d = a.pool + (size_t)l * a.layer_vecs + (size_t)a.ws.dst[k] * a.page_vecs;
    for (size_t v = v0; v < a.page_vecs; v += 4 * kPgCopyThreads) {
      uint4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + i * kPgCopyThreads < a.page_vecs) x[i] = ld_stream(s + v + i * kPgCopyThreads);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + i * kPgCopyThreads < a.page_vecs) d[v + i * kPgCopyThreads] = x[i];
    }
  }
}

// One CTA where it has at most 8 pages and 8 table entries a thread to look at: a CTA's
// barrier is then cheaper than a cluster's.
static int pages_ctas(int S, int slots, int P) {
  return P <= 8 * kPgThreads && (long long)S * slots <= 8 * kPgThreads ? 1 : kPgCtas;
}

static int pages_check(const void* table, const void* held, const void* refs, int S, int slots, int P) {
  JSX_REQUIRE(table && held && refs, "null table, held or refs");
  JSX_REQUIRE(S >= 1 && slots >= 1 && P >= 1, "sequences=%d slots=%d num_pages=%d", S, slots, P);
  JSX_REQUIRE(S <= (1 << 15) && (long long)S * slots <= (1ll << 30), "more than 2^15 sequences or 2^30 table entries");
  JSX_REQUIRE(aligned4(table) && aligned4(held) && aligned4(refs), "table, held and refs must be 4-byte aligned");
  return JSX_OK;
}
static int pages_check_pool(const void* pool, int layers, size_t page_bytes, const void* ws, size_t ws_bytes, int S,
                            int slots, int P) {
  JSX_REQUIRE(pool && aligned16(pool) && layers >= 1, "null or unaligned pool, or layers=%d", layers);
  JSX_REQUIRE(page_bytes >= 16 && page_bytes % 16 == 0, "page_bytes=%zu must be a positive multiple of 16", page_bytes);
  JSX_REQUIRE(ws && aligned16(ws) && ws_bytes >= pages_ws_bytes(S, slots, P), "workspace of %zu bytes, %zu needed",
              ws_bytes, pages_ws_bytes(S, slots, P));
  return JSX_OK;
}
static int pages_copy(PgCopyArgs& c, void* pool, int layers, size_t page_bytes, int P, cudaStream_t s) {
  c.pool = (uint4*)pool;
  c.page_vecs = page_bytes / 16;
  c.layer_vecs = c.page_vecs * P;
  c.layers = layers;
  c.P = P;
  JSX_CUDA(launch_kernel(k_pages_copy, dim3(8 * sm_count()), dim3(kPgCopyThreads), 0, s, c));
  return JSX_OK;
}

}  // namespace jsx

using namespace jsx;

extern "C" int jsx_pages_workspace_size(int sequences, int slots, int num_pages, size_t* bytes) {
  JSX_REQUIRE(bytes && sequences >= 1 && slots >= 1 && num_pages >= 1, "bad arguments");
  *bytes = pages_ws_bytes(sequences, slots, num_pages);
  return JSX_OK;
}

extern "C" int jsx_pages_fork(const int32_t* table, const int32_t* held, const int32_t* refs, const int32_t* parent,
                              int32_t* table_out, int32_t* held_out, int32_t* refs_out, int sequences, int slots,
                              int num_pages, void* stream) {
  const int st = pages_check(table, held, refs, sequences, slots, num_pages);
  if (st) return st;
  JSX_REQUIRE(parent && table_out && held_out && refs_out, "null pointer argument");
  JSX_REQUIRE(table_out != table && held_out != held, "table_out and held_out must not be table and held");
  PgForkArgs a = {table, held, refs, parent, table_out, held_out, refs_out, sequences, slots, num_pages};
  const int n = pages_ctas(sequences, slots, num_pages);
  JSX_CUDA(launch_kernel(n == 1 ? k_pages_fork<1> : k_pages_fork<kPgCtas>, dim3(n), dim3(kPgThreads), 0,
                         (cudaStream_t)stream, a));
  return JSX_OK;
}

extern "C" int jsx_pages_resize(int32_t* table, int32_t* held, int32_t* refs, const int32_t* keep, const int32_t* need,
                                void* pool, int layers, size_t page_bytes, int sequences, int slots, int num_pages,
                                int page_tokens, int32_t* missing, void* workspace, size_t workspace_bytes,
                                void* stream) {
  int st = pages_check(table, held, refs, sequences, slots, num_pages);
  if (st) return st;
  JSX_REQUIRE(keep && need && missing && page_tokens >= 1, "null keep, need or missing, or page_tokens=%d", page_tokens);
  st = pages_check_pool(pool, layers, page_bytes, workspace, workspace_bytes, sequences, slots, num_pages);
  if (st) return st;
  PgResizeArgs a;
  a.table = table;
  a.held = held;
  a.refs = refs;
  a.keep = keep;
  a.need = need;
  a.missing = missing;
  a.ws = pages_ws(workspace, sequences, slots, num_pages);
  a.S = sequences;
  a.slots = slots;
  a.P = num_pages;
  a.pt = page_tokens;
  const int n = pages_ctas(sequences, slots, num_pages);
  JSX_CUDA(launch_kernel(n == 1 ? k_pages_resize<1> : k_pages_resize<kPgCtas>, dim3(n), dim3(kPgThreads), 0,
                         (cudaStream_t)stream, a));
  PgCopyArgs c = {};
  c.ws = a.ws;
  return pages_copy(c, pool, layers, page_bytes, num_pages, (cudaStream_t)stream);
}

extern "C" int jsx_pages_compact(const int32_t* table, const int32_t* held, const int32_t* refs, void* pool, int layers,
                                 size_t page_bytes, int32_t* table_out, int32_t* refs_out, int32_t* remap,
                                 int sequences, int slots, int num_pages, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  int st = pages_check(table, held, refs, sequences, slots, num_pages);
  if (st) return st;
  JSX_REQUIRE(table_out && refs_out && remap, "null pointer argument");
  st = pages_check_pool(pool, layers, page_bytes, workspace, workspace_bytes, sequences, slots, num_pages);
  if (st) return st;
  PgCompactArgs a;
  a.table = table;
  a.held = held;
  a.refs = refs;
  a.refs_out = refs_out;
  a.remap = remap;
  a.ws = pages_ws(workspace, sequences, slots, num_pages);
  a.S = sequences;
  a.slots = slots;
  a.P = num_pages;
  const int n = pages_ctas(sequences, slots, num_pages);
  JSX_CUDA(launch_kernel(n == 1 ? k_pages_plan<1> : k_pages_plan<kPgCtas>, dim3(n), dim3(kPgThreads), 0,
                         (cudaStream_t)stream, a));
  PgCopyArgs c = {};
  c.ws = a.ws;
  c.table = table;
  c.held = held;
  c.remap = remap;
  c.table_out = table_out;
  c.S = sequences;
  c.slots = slots;
  return pages_copy(c, pool, layers, page_bytes, num_pages, (cudaStream_t)stream);
}
