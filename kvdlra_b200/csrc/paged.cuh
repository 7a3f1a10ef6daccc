// Shared pieces of the 8-bit paged KV cache's kernels: the pool as kernels see
// it, the two code formats, and the division of attention work over CTAs.
//
// A pool holds, per (page, KV head), page_size slots of head_dim 8-bit codes
// for the keys and for the values, and one fp32 scale each: x = code * scale.
#pragma once

#include <cuda_fp16.h>

#include "kernels.cuh"

namespace kvd {

constexpr int kStoreE4M3 = KVD_STORE_E4M3, kStoreInt8 = KVD_STORE_INT8;
constexpr int kPagedBadSlot = 1, kPagedBadPage = 2, kPagedNonFinite = 1;  // status bits

struct PagedPool {
  unsigned char* k;
  unsigned char* v;
  float* ks;
  float* vs;                             // [num_pages][H], pages scale_stride apart
  long page_stride, head_stride, slot_stride;  // bytes
  long scale_stride;                     // elements
  int num_pages, lg_page, H;
  int* status;                           // may be null
  KVD_DEVICE int page() const { return 1 << lg_page; }
  KVD_DEVICE void flag(int word, int bits) const {
    if (status) atomicOr(status + word, bits);
  }
};

template <> struct IO<__half> {
  static KVD_DEVICE float load(const __half* p) { return __half2float(*p); }
  static KVD_DEVICE void store(__half* p, float v) { *p = __float2half_rn(v); }
};

// Four codes (the bytes of w) as two f16 pairs, exactly: both formats have at
// most 8 significant bits and stay within f16's normal and subnormal range.
template <int STORE>
KVD_DEVICE void codes_to_f16(uint32_t w, uint32_t* lo, uint32_t* hi) {
  if constexpr (STORE == kStoreE4M3) {
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(*lo), "=r"(*hi) : "r"(w));
  } else {
    // byte u = code + 128 under the exponent of 1024: the half is 1024 + u
    const uint32_t u = w ^ 0x80808080u, bias = 0x64806480u;  // 1024 + 128
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
    *lo = *reinterpret_cast<const uint32_t*>(&x);
    *hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

template <int STORE>
KVD_DEVICE void codes_to_f32(uint32_t w, float (&x)[4]) {
  uint32_t a, b;
  codes_to_f16<STORE>(w, &a, &b);
  const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&a));
  const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&b));
  x[0] = p.x; x[1] = p.y; x[2] = q.x; x[3] = q.y;
}

// Four values as codes: round to nearest, ties to even, saturating.
template <int STORE>
KVD_DEVICE uint32_t f32_to_codes(float a, float b, float c, float d) {
  if constexpr (STORE == kStoreE4M3) {
    uint32_t r;
    asm("{\n .reg .b16 p, q;\n cvt.rn.satfinite.e4m3x2.f32 p, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 q, %4, %3;\n"
        " mov.b32 %0, {p, q};\n}"
        : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
  } else {
    auto one = [](float x) { return (uint32_t)max(-127, min(127, __float2int_rn(x))) & 0xffu; };
    return one(a) | (one(b) << 8) | (one(c) << 16) | (one(d) << 24);
  }
}

// The least power of two s (2^-100 at the least) with amax <= M s, M = 448 or
// 127: M = f 2^t with f in [1, 2), so s = 2^(E - t), or twice that where
// amax's significand is above f.  A power of two makes x / s exact, so a code
// is one rounding of the value, and a page's codes can follow a growing scale
// (e4m3: without loss, but for subnormals).
template <int STORE>
KVD_DEVICE float code_scale(float amax) {
  constexpr int t = STORE == kStoreE4M3 ? 8 : 6;
  constexpr uint32_t f = STORE == kStoreE4M3 ? 0x600000u : 0x7e0000u;  // 1.75, 1.984375
  const uint32_t b = __float_as_uint(amax);
  const int e = max((int)(b >> 23) - 127 - t + ((b & 0x7fffffu) > f ? 1 : 0), -100);
  return amax > 0.f ? __uint_as_float((uint32_t)(e + 127) << 23) : __uint_as_float(27u << 23);
}

// ------------------------------------------------------------ attention work

// Requests of one attention call.  Request b answers q_len(b) query tokens
// over its first len(b) cached tokens; query token i sees tokens
// (i + len - q_len - window, i + len - q_len] (window 0: from starts[b] on).
// A query row is (token, head of the group): row = i * G + head.
struct PagedReqs {
  int batch, H, G, q_tokens, window, max_len;
  const int* lens;
  const int* cu_q;    // null: every request has q_tokens query tokens
  const int* starts;  // null: 0
  int min_rows, max_rows;  // requests with rows in [min_rows, max_rows] belong to this launch
  KVD_DEVICE int q0(int b) const { return cu_q ? cu_q[b] : 0; }
  // query tokens of request b, whatever cu_q holds: within [0, q_tokens]
  KVD_DEVICE int q_len(int b) const {
    if (!cu_q) return q_tokens;
    const int lo = cu_q[b], hi = cu_q[b + 1];
    return lo < 0 || hi > q_tokens || hi < lo ? 0 : hi - lo;
  }
  KVD_DEVICE int len(int b) const { return max(0, min(lens[b], max_len)); }
  KVD_DEVICE int start(int b) const { return starts ? max(0, starts[b]) : 0; }
  KVD_DEVICE bool mine(int q) const { return (long)q * G >= min_rows && (long)q * G <= max_rows; }
};

// Tokens that row tile `rt` (of RT rows) of a request sees: [lo, hi), and the
// tiles of TT tokens that cover them (one at least: an empty row is written too).
template <int RT, int TT>
KVD_DEVICE int row_tile_span(const PagedReqs& a, int len, int q, int start, int rt, int* lo, int* hi) {
  const int i0 = rt * RT / a.G, i1 = min(q * a.G - 1, rt * RT + RT - 1) / a.G;
  *hi = max(0, min(len, len - q + i1 + 1));
  int l = start;
  if (a.window > 0) l = max(l, len - q + i0 - a.window + 1);
  *lo = min(l, *hi);
  return max(1, (*hi + TT - 1) / TT - *lo / TT);
}

// Where a CTA's share of the flattened (request, KV head, row tile, token
// tile) list begins.
struct WorkAt {
  long total;   // token tiles of all units
  long chunk;   // tiles per CTA
  int b;        // request; its units start `off` tiles before the CTA's first
  long off;
};

// All threads of the CTA call it (NTHR of them).  Every CTA counts the whole
// list itself: lengths live on the device and the counts cost a few reads.
template <int RT, int TT, int NTHR>
KVD_DEVICE WorkAt find_work(const PagedReqs& a, int cta, int nctas) {
  __shared__ long wsum[NTHR / 32 + 1];
  __shared__ long found_off;
  __shared__ int found_b;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.batch + NTHR - 1) / NTHR;
  const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
  auto tiles = [&](int b) -> long {
    const int q = a.q_len(b);
    if (q == 0 || !a.mine(q)) return 0;
    const int len = a.len(b), st = a.start(b), nrt = (int)(((long)q * a.G + RT - 1) / RT);
    long s = 0;
    for (int rt = 0; rt < nrt; ++rt) {
      int lo, hi;
      s += row_tile_span<RT, TT>(a, len, q, st, rt, &lo, &hi);
    }
    return s * a.H;
  };
  long mine = 0;
  for (int b = b0; b < b1; ++b) mine += tiles(b);
  long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) wsum[warp] = incl;
  if (tid == 0) found_b = -1;
  __syncthreads();
  long before = 0, total = 0;
  for (int w = 0; w < NTHR / 32; ++w) {
    if (w < warp) before += wsum[w];
    total += wsum[w];
  }
  WorkAt r;
  r.total = total;
  r.chunk = max(1L, (total + nctas - 1) / nctas);
  const long first = cta * r.chunk;
  long at = before + incl - mine;
  if (first >= at && first < at + mine) {
    for (int b = b0; b < b1; ++b) {
      const long n = tiles(b);
      if (first < at + n) {
        found_b = b;
        found_off = first - at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  r.b = found_b;
  r.off = found_off;
  __syncthreads();
  return r;
}

// Partial results of a unit that several CTAs share: CTA c's record 0 is the
// piece of the unit that it continues, record 1 the piece of the unit that it
// begins and does not finish.  head[c] says what c begins.
struct PagedPart {
  float* rec;          // [ctas][2][rows][D + 2]: O (unnormalised), m, l
  int4* head;          // [ctas]: request, KV head, row tile, pieces (0: none)
};

struct PagedOut {
  void* out;           // (tokens, Hq, D)
  float* lse;          // (tokens, Hq) or null
  int Hq;
};

}  // namespace kvd

namespace kvd_host {
// Checks of a pool's description; fills the kernels' view of it.
int paged_pool_view(const kvd_paged_pool* p, kvd::PagedPool* out);
int paged_sm_count();
// Attention over the pages on tcgen05 for requests of many rows; the workspace
// it needs, 0 where it has no kernel for the shape.
size_t paged_chunk_ws_bytes(const kvd_paged_pool& p, int dtype, int G);
int launch_paged_chunk(const kvd_paged_pool& p, const kvd::PagedPool& pool, const kvd::PagedReqs& reqs, const int* table,
                       long table_stride, int dtype, const void* q, long q_sb, long q_sh, long q_st,
                       float scaling, const kvd::PagedOut& out, void* ws, cudaStream_t s);
}  // namespace kvd_host
