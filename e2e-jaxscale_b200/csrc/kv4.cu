// Rows written to and read back from the 4-bit key/value pages (kv4.cuh).
//
// Append, per 16 values x of a row: s = e4m3(min(max |x| / 6, 448)), code =
// e2m1(x / s) (0 where s is 0), both rounded to nearest even.  A bf16 value has
// 8 significant bits and a scale 4, so a quotient is either exactly on a code's
// rounding boundary or at least 2^-10 from it; x (1/s) is within 2^-21 of x / s, 1/s within
// 2^-22.  The scale too comes from a product, max |x| (1/6): over all 32640 bf16 magnitudes it
// rounds to the same e4m3 as the quotient.
// Rounding it to multiples of 2^-13 (one fused multiply-add against 1536 and a
// subtraction) therefore gives the codes of the exact quotient, without 16
// divisions per group.  The largest magnitude is an integer maximum over the
// bf16 bit patterns, where NaN is above infinity: a group with a NaN gets a NaN
// scale and reads back as NaN; infinities saturate at 6 x 448.
//
// Both kernels move 32 bytes of bf16 per 9 bytes of page.  One thread handles a group of a K row
// and the same of its V row: two 16-byte accesses each on the bf16 side (dealt to pairs of
// lanes, kv4_swap), 8 bytes of codes and one scale byte on the page side; the threads of a row
// are adjacent.  (8 values a thread would make every access whole, but doubles the index
// arithmetic: 30 against 23 us for 32 x 1024 rows of 2 heads there and back.)
//
// Bound: memory for many rows (32 x 1024 rows of 2 heads there and back: 18.0 us, 86 MB of
// rows and pages, 4.8 TB/s, much of it in L2; 21.6 us while a lane's accesses were 16 bytes of
// every 32), the launch for few (32 x 1: 3.1 us on the device).
#include "common.cuh"
#include "kv4.cuh"
#include "launch.cuh"

namespace jsx {

constexpr int kKv4Threads = 256;

struct Kv4RowArgs {
  bf16* k;  // append: read; read: written
  bf16* v;
  int64_t seq_stride, token_stride, head_stride;  // elements
  int cache_rows;  // > 0: rows of a static cache, indexed by position; 0: one row per token of the call
  uint8_t* pool;
  const int32_t* table;
  const int32_t* positions;
  const int32_t* n_tokens;
  int num_pages, slots, nkv, pt, pt_log;
  uint32_t units;  // of a sequence: T * nkv * (D / 16)
};

// Where unit u of sequence b, 16 values of a K row and the same of its V row, lies: in the
// rows (row), and in its block of the pool.  (32-bit indexes inside a sequence, and K and V
// together: finding the place is what these kernels spend most instructions on.)
struct Kv4Unit {
  int64_t row;     // elements from k and from v
  uint8_t* codes;  // of K; V's are kv4_off_v further
  uint8_t* scale;  // of K; V's pt * D / 16 further
  bool inside;     // the row exists (token used, position inside the static cache)
  bool paged;      // ... and has a page
};

template <int D>
__device__ __forceinline__ Kv4Unit kv4_unit(const Kv4RowArgs& a, int b, uint32_t u, int first, int used) {
  constexpr int NG = D / kKv4Group;
  const int g = (int)(u % NG);
  const uint32_t mh = u / NG;
  const int i = (int)(mh / (uint32_t)a.nkv), h = (int)(mh - (uint32_t)i * a.nkv);
  const int pos = first + i;
  Kv4Unit x;
  x.inside = u < a.units && i < used && pos >= 0 && (a.cache_rows == 0 || pos < a.cache_rows);
  x.row = b * a.seq_stride + (int64_t)(a.cache_rows ? pos : i) * a.token_stride + h * a.head_stride + g * kKv4Group;
  const int slot = pos >> a.pt_log;
  int page = -1;
  if (x.inside && slot < a.slots) page = a.table[(int64_t)b * a.slots + slot];
  x.paged = page >= 0 && page < a.num_pages;
  const int t = pos & (a.pt - 1);
  uint8_t* block = a.pool + ((int64_t)page * a.nkv + h) * kv4_block_bytes(a.pt, D);
  x.codes = block + t * (D / 2) + g * 8;
  x.scale = block + kv4_off_ks(a.pt, D) + t * NG + g;
  return x;
}

// Two lanes access 32 bytes side by side, the even one's group and then the odd one's, so that
// every access is of whole 32-byte sectors; this takes them to the lanes' own groups and back.
// (A row has an even number of groups: both lanes have one or neither.)
__device__ __forceinline__ void kv4_swap(uint4& lo, uint4& hi, bool odd) {
  uint32_t x[4] = {lo.x, lo.y, lo.z, lo.w}, y[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t z = __shfl_xor_sync(3u << (threadIdx.x & 30), odd ? x[i] : y[i], 1);
    x[i] = odd ? z : x[i];
    y[i] = odd ? y[i] : z;
  }
  lo = make_uint4(x[0], x[1], x[2], x[3]);
  hi = make_uint4(y[0], y[1], y[2], y[3]);
}

template <int D>
__global__ void __launch_bounds__(kKv4Threads) k_kv4_append(Kv4RowArgs a) {
  pdl_wait();
  const int b = blockIdx.y, first = a.positions[b], used = a.n_tokens ? a.n_tokens[b] : INT32_MAX;
  for (uint32_t u = blockIdx.x * kKv4Threads + threadIdx.x; u < a.units; u += gridDim.x * kKv4Threads) {
    const Kv4Unit x = kv4_unit<D>(a, b, u, first, used);
    if (!x.inside) continue;
    const bool odd = threadIdx.x & 1;
    uint4 p[2][2];  // in flight together with the page number
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const bf16* row = (k ? a.v : a.k) + x.row - (odd ? 8 : 0);
      p[k][0] = *reinterpret_cast<const uint4*>(row);
      p[k][1] = *reinterpret_cast<const uint4*>(row + 16);
    }
    if (!x.paged) continue;
#pragma unroll
    for (int k = 0; k < 2; ++k) kv4_swap(p[k][0], p[k][1], odd);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t w[8] = {p[k][0].x, p[k][0].y, p[k][0].z, p[k][0].w, p[k][1].x, p[k][1].y, p[k][1].z, p[k][1].w};
      uint32_t mx = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = __vmaxu2(mx, w[i] & 0x7fff7fffu);
      const float top = __uint_as_float(max(mx & 0xffffu, mx >> 16) << 16);
      const uint32_t sc = f32_to_e4m3(top * (1.f / 6.f));
      const float s = __half2float(__ushort_as_half((unsigned short)(e4m3x2_to_h2(sc) & 0xffffu)));
      const float inv = s == 0.f ? 0.f : __fdividef(1.f, s);
      float q[2][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q[i >> 2][2 * (i & 3)] = __fmaf_rn(bf_lo(w[i]), inv, 1536.f) - 1536.f;
        q[i >> 2][2 * (i & 3) + 1] = __fmaf_rn(bf_hi(w[i]), inv, 1536.f) - 1536.f;
      }
      *reinterpret_cast<uint2*>(x.codes + k * kv4_off_v(a.pt, D)) = make_uint2(f32x8_to_e2m1(q[0]), f32x8_to_e2m1(q[1]));
      x.scale[k * a.pt * (D / kKv4Group)] = (uint8_t)sc;
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kKv4Threads) k_kv4_read(Kv4RowArgs a) {
  pdl_wait();
  const int b = blockIdx.y, first = a.positions[b], used = a.n_tokens ? a.n_tokens[b] : INT32_MAX;
  for (uint32_t u = blockIdx.x * kKv4Threads + threadIdx.x; u < a.units; u += gridDim.x * kKv4Threads) {
    const Kv4Unit x = kv4_unit<D>(a, b, u, first, used);
    if (!x.inside) continue;
    uint2 c[2] = {};
    uint32_t sc[2] = {};
    if (x.paged) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        c[k] = *reinterpret_cast<const uint2*>(x.codes + k * kv4_off_v(a.pt, D));
        sc[k] = x.scale[k * a.pt * (D / kKv4Group)];
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t s2 = e4m3x2_to_h2(sc[k] | (sc[k] << 8));
      uint32_t h[8], o[8];
      e2m1x8_to_h2(c[k].x, reinterpret_cast<uint32_t(&)[4]>(h[0]));
      e2m1x8_to_h2(c[k].y, reinterpret_cast<uint32_t(&)[4]>(h[4]));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t y = hmul2_u(h[i], s2);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&y));
        o[i] = pack2(f.x, f.y);
      }
      const bool odd = threadIdx.x & 1;
      uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
      kv4_swap(lo, hi, odd);
      bf16* row = (k ? a.v : a.k) + x.row - (odd ? 8 : 0);
      *reinterpret_cast<uint4*>(row) = lo;
      *reinterpret_cast<uint4*>(row + 16) = hi;
    }
  }
}

static int kv4_rows(bool append, const void* k, const void* v, int64_t seq_stride, int64_t token_stride,
                    int64_t head_stride, int cache_rows, const void* pool, int num_pages, const int32_t* table,
                    int table_slots, const int32_t* positions, const int32_t* n_tokens, int B, int T, int nkv,
                    int head_dim, int page_tokens, void* stream) {
  JSX_REQUIRE(k && v && positions, "null pointer argument");
  JSX_KV4_REQUIRE(pool, num_pages, table, table_slots, nkv, head_dim, page_tokens);
  JSX_REQUIRE(B >= 1 && B <= 65535 && T >= 1 && cache_rows >= 0, "B=%d (1..65535) T=%d cache_rows=%d", B, T, cache_rows);
  JSX_REQUIRE((int64_t)T * nkv * (head_dim / kKv4Group) < (1ll << 30), "%d tokens of %d kv heads per sequence", T, nkv);
  JSX_REQUIRE(aligned16(k) && aligned16(v) && seq_stride % 8 == 0 && token_stride % 8 == 0 && head_stride % 8 == 0,
              "rows must be 16-byte aligned");
  JSX_REQUIRE(seq_stride >= 0 && token_stride >= 0 && head_stride >= 0, "negative stride");
  Kv4RowArgs a;
  a.k = (bf16*)const_cast<void*>(k);
  a.v = (bf16*)const_cast<void*>(v);
  a.seq_stride = seq_stride;
  a.token_stride = token_stride;
  a.head_stride = head_stride;
  a.cache_rows = cache_rows;
  a.pool = (uint8_t*)const_cast<void*>(pool);
  a.table = table;
  a.positions = positions;
  a.n_tokens = n_tokens;
  a.num_pages = num_pages;
  a.slots = table_slots;
  a.nkv = nkv;
  a.pt = page_tokens;
  a.pt_log = page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : 7;
  a.units = (uint32_t)T * nkv * (head_dim / kKv4Group);
  const uint32_t blocks = (a.units + kKv4Threads - 1) / kKv4Threads, most = (16u * sm_count() + B - 1) / B;
  const dim3 grid(blocks < most ? blocks : most, B);
  auto kern = append ? (head_dim == 128 ? k_kv4_append<128> : k_kv4_append<64>)
                     : (head_dim == 128 ? k_kv4_read<128> : k_kv4_read<64>);
  JSX_CUDA(launch_kernel(kern, grid, dim3(kKv4Threads), 0, (cudaStream_t)stream, a));
  return JSX_OK;
}

}  // namespace jsx

using namespace jsx;

extern "C" int jsx_kv4_page_bytes(int nkv, int head_dim, int page_tokens, size_t* bytes) {
  JSX_REQUIRE(bytes && nkv >= 1, "bad arguments");
  JSX_REQUIRE(kv4_page_tokens_ok(page_tokens), "page_tokens=%d is not 16, 32, 64 or 128", page_tokens);
  if (head_dim != 64 && head_dim != 128) {
    set_error("head_dim=%d (the 4-bit cache takes 64 and 128)", head_dim);
    return JSX_ENOTSUP;
  }
  *bytes = (size_t)nkv * kv4_block_bytes(page_tokens, head_dim);
  return JSX_OK;
}

extern "C" int jsx_kv4_append(const void* k, const void* v, int64_t seq_stride, int64_t token_stride,
                              int64_t head_stride, int cache_rows, void* pool, int num_pages, const int32_t* table,
                              int table_slots, const int32_t* positions, const int32_t* n_tokens, int B, int T,
                              int nkv, int head_dim, int page_tokens, void* stream) {
  return kv4_rows(true, k, v, seq_stride, token_stride, head_stride, cache_rows, pool, num_pages, table, table_slots,
                  positions, n_tokens, B, T, nkv, head_dim, page_tokens, stream);
}

extern "C" int jsx_kv4_read(const void* pool, int num_pages, const int32_t* table, int table_slots,
                            const int32_t* positions, const int32_t* n_tokens, void* k, void* v, int64_t seq_stride,
                            int64_t token_stride, int64_t head_stride, int cache_rows, int B, int T, int nkv,
                            int head_dim, int page_tokens, void* stream) {
  return kv4_rows(false, k, v, seq_stride, token_stride, head_stride, cache_rows, pool, num_pages, table, table_slots,
                  positions, n_tokens, B, T, nkv, head_dim, page_tokens, stream);
}
