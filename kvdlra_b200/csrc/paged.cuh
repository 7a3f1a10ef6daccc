// Shared pieces of the 8-bit paged KV cache's kernels: the pool as kernels see
// it, the two code formats, and the division of attention work over CTAs.
//
// A pool holds, per (page, KV head), page_size slots of head_dim 8-bit codes
// for the keys and for the values, and one fp32 scale each: x = code * scale.
#pragma once

#include <algorithm>

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

// Values read back, and averages of them, held to their type's range: a code may
// round up past it (65504 in f16 is 256 x 256 in e4m3).  NaN stays.
KVD_DEVICE void store_held(float* p, float v) { *p = fabsf(v) == INFINITY ? copysignf(3.402823466e38f, v) : v; }
KVD_DEVICE void store_held(__nv_bfloat16* p, float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
  *reinterpret_cast<uint16_t*>(p) = r;
}
KVD_DEVICE void store_held(__half* p, float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.f16.f32 %0, %1;" : "=h"(r) : "f"(v));
  *reinterpret_cast<uint16_t*>(p) = r;
}

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
  KVD_DEVICE int q_len(int b) const { return !cu_q ? q_tokens : in_rows(b) ? cu_q[b + 1] - cu_q[b] : 0; }
  KVD_DEVICE bool in_rows(int b) const { return cu_q[b] >= 0 && cu_q[b + 1] <= q_tokens && cu_q[b + 1] >= cu_q[b]; }
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

// One CTA's pieces of units, in order: `next` moves to the next one.  Every
// thread that walks them sees the same.
template <int RT, int TT>
struct Pieces {
  const PagedReqs& rq;
  long left, off_next;
  int b_next, h_next, rt_next, nrt;
  bool inside;                    // the next piece is of the same request
  // the current piece: tiles [tile, tile + n) of unit (b, h, rt), whose own are
  // [lo / TT, lo / TT + span); `off` of them lie before the piece
  int b, h, rt, q_len, len, start, rows, lo, hi, span, off, tile, n;
  KVD_DEVICE Pieces(const PagedReqs& r, const WorkAt& at, int cta) : rq(r) {
    left = min(at.chunk, at.total - (long)cta * at.chunk);
    b_next = at.b;
    off_next = at.off;
    inside = false;
  }
  KVD_DEVICE bool next() {
    if (left <= 0) return false;
    if (!inside) {
      while (true) {
        if (b_next >= rq.batch) return false;
        q_len = rq.q_len(b_next);
        if (q_len > 0 && rq.mine(q_len)) break;
        ++b_next;
      }
      len = rq.len(b_next);
      start = rq.start(b_next);
      rows = q_len * rq.G;
      nrt = (rows + RT - 1) / RT;
      h_next = rt_next = 0;
      if (off_next > 0) {
        long per_head = 0;
        int l, u;
        for (int r = 0; r < nrt; ++r) per_head += row_tile_span<RT, TT>(rq, len, q_len, start, r, &l, &u);
        h_next = (int)(off_next / per_head);
        off_next -= h_next * per_head;
        int s;
        while (off_next >= (s = row_tile_span<RT, TT>(rq, len, q_len, start, rt_next, &l, &u))) { off_next -= s; ++rt_next; }
      }
      inside = true;
    }
    b = b_next; h = h_next; rt = rt_next;
    span = row_tile_span<RT, TT>(rq, len, q_len, start, rt, &lo, &hi);
    off = (int)off_next;
    tile = lo / TT + off;
    n = (int)min((long)span - off, left);
    left -= n;
    off_next = 0;
    if (++rt_next == nrt) {
      rt_next = 0;
      if (++h_next == rq.H) {
        inside = false;
        ++b_next;
      }
    }
    return true;
  }
  KVD_DEVICE bool whole() const { return off == 0 && n == span; }
  // pieces of the unit when the current one begins it and does not finish it
  KVD_DEVICE int pieces(long chunk) const { return off == 0 && n < span ? 1 + (int)((span - n + chunk - 1) / chunk) : 0; }
  KVD_DEVICE long out_row(int R) const { return (rq.cu_q ? rq.q0(b) : (long)b * rq.q_tokens) + R / rq.G; }
  // the tokens that row R sees
  KVD_DEVICE int row_hi(int R) const { return min(len, len - q_len + R / rq.G + 1); }
  KVD_DEVICE int row_lo(int R) const {
    return rq.window > 0 ? max(start, len - q_len + R / rq.G - rq.window + 1) : start;
  }
};

// Partial results of a unit that several CTAs share: CTA c's record 0 is the
// piece of the unit that it continues, record 1 the piece of the unit that it
// begins and does not finish.  head[c] says what c begins.
struct PagedPart {
  float* rec;          // [ctas][2][rows][D + 2]: O (unnormalised), m, l
  int4* head;          // [ctas]: request, KV head, row tile, pieces (0: none)
};

// A row's weights before their rounding to f16: P = p vs / 2^mv.  The reference
// mv is kPBias under the largest p vs when it is set and moves when P would pass
// 2^kPTop: P's subnormals, spaced 2^-24, are 2^-30 of the row's largest weight or
// less, and the move, which rescales O, is rare after the first tiles.
constexpr float kPBias = 6.f, kPTop = 15.f;
constexpr float kLTop = 14.f;  // log2 of the largest weight in l, over its own reference m

KVD_DEVICE float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
KVD_DEVICE uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
KVD_DEVICE float2 unpack_f16(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }

struct PagedOut {
  void* out;           // (tokens, Hq, D)
  float* lse;          // (tokens, Hq) or null
  int Hq;
};

// Joins a split unit's records: M = max m_i, out = sum 2^(m_i - M) O_i / sum
// 2^(m_i - M) l_i.  blockIdx.x is the CTA of the kernel before that began the
// unit (most began none that others finish); the rows go over blockIdx.y and the
// warps.  A row is a warp's, or the four warps' where there are many records (a
// long context split over the SMs): the lanes find the records' factors, two
// each, then every lane sums its columns over them.  Bound by the latency of a
// few dependent reads: the head, the maxima and sums, the records.
template <int D, int RT, typename T>
__global__ void __launch_bounds__(128) paged_merge_kernel(PagedReqs rq, PagedPart part, PagedOut out, int fill_tail) {
  constexpr int V = D < 128 ? D / 32 : 4;      // columns per lane and step
  constexpr int C = D / (32 * V);              // steps
  __shared__ float sums[4][D];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 u = part.head[blockIdx.x];
  if (fill_tail && rq.cu_q) {  // rows that no request answers: zeros
    bool odd = false;            // offsets that are none into the rows
    for (int b = threadIdx.x; b < rq.batch; b += 128) odd |= !rq.in_rows(b);
    odd = __syncthreads_or(odd);
    const long ctas = (long)gridDim.x * gridDim.y, cta = (long)blockIdx.y * gridDim.x + blockIdx.x;
    auto clear = [&](long from, long to, long at, long stride) {  // rows [from, to)
      for (long e = from * out.Hq * D + at; e < to * out.Hq * D; e += stride) store_f(reinterpret_cast<T*>(out.out) + e, 0.f);
      if (out.lse)
        for (long e = from * out.Hq + at; e < to * out.Hq; e += stride) out.lse[e] = -INFINITY;
    };
    if (!odd) {
      clear(0, rq.cu_q[0], cta * 128 + threadIdx.x, ctas * 128);
      clear(rq.cu_q[rq.batch], rq.q_tokens, cta * 128 + threadIdx.x, ctas * 128);
    } else {
      for (long r = cta; r < rq.q_tokens; r += ctas) {
        bool answered = false;
        for (int b = threadIdx.x; b < rq.batch; b += 128) answered |= rq.in_rows(b) && r >= rq.cu_q[b] && r < rq.cu_q[b + 1];
        if (!__syncthreads_or(answered)) clear(r, r + 1, threadIdx.x, 128);
      }
    }
  }
  if (u.w == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = u.x, h = u.y, rt = u.z, n = u.w;
  const int rows = min(RT, rq.q_len(b) * rq.G - rt * RT);
  const long step = 2L * RT * (D + 2);
  // record 1 of the CTA that began the unit, then record 0 of those after it
  const float* first = part.rec + (long)blockIdx.x * step + (long)RT * (D + 2);
  const float* rest = part.rec + (long)blockIdx.x * step;
  auto record = [&](int i) { return i == 0 ? first : rest + i * step; };
  const bool many = n >= 12;
  const int per = many ? 1 : 4, stride = many ? 4 : 1, part0 = many ? warp : 0;
  for (int r = blockIdx.y * per + (many ? 0 : warp); r < rows; r += gridDim.y * per) {
    float M = -INFINITY, L = 0.f, o[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) o[c][k] = 0.f;
    for (int i0 = 0; i0 < n; i0 += 64) {  // two records a lane
      float m2[2], l2[2], f2[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = i0 + 32 * k + lane;
        const float* p = record(min(i, n - 1)) + RT * D + r;
        m2[k] = i < n ? p[0] : -INFINITY;
        l2[k] = i < n ? p[RT] : 0.f;
      }
      const float top = fmaxf(M, warp_max(fmaxf(m2[0], m2[1])));
      const float old = M == -INFINITY ? 1.f : exp2_fast(M - top);
      M = top;
      L *= old;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f2[k] = M == -INFINITY ? 1.f : exp2_fast(m2[k] - M);
        L = fmaf(f2[k], l2[k], L);
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < V; ++k) o[c][k] *= old;
      const int m = min(64, n - i0);
#pragma unroll 8
      for (int i = part0; i < m; i += stride) {
        const float w = __shfl_sync(0xffffffffu, i < 32 ? f2[0] : f2[1], i & 31);
        const float* p = record(i0 + i) + r * D + V * lane;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float x[V];
          if constexpr (V == 4) {
            const float4 y = *reinterpret_cast<const float4*>(p + 128 * c);
            x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
          } else if constexpr (V == 2) {
            const float2 y = *reinterpret_cast<const float2*>(p);
            x[0] = y.x; x[1] = y.y;
          } else {
            x[0] = *p;
          }
#pragma unroll
          for (int k = 0; k < V; ++k) o[c][k] = fmaf(w, x[k], o[c][k]);
        }
      }
    }
    L = warp_sum(L);
    if (many) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < V; ++k) sums[warp][32 * V * c + V * lane + k] = o[c][k];
      __syncthreads();
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const int d = 32 * V * c + V * lane + k;
          o[c][k] = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
        }
      __syncthreads();
      if (warp != 0) continue;
    }
    const int R = rt * RT + r;
    const long row = (rq.cu_q ? rq.q0(b) : (long)b * rq.q_tokens) + R / rq.G;
    const int hq = h * rq.G + R % rq.G;
    T* dst = reinterpret_cast<T*>(out.out) + (row * out.Hq + hq) * D + V * lane;
    const float f = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) store_held(dst + 32 * V * c + k, o[c][k] * f);
    if (lane == 0 && out.lse) out.lse[row * out.Hq + hq] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
  }
}

}  // namespace kvd

namespace kvd_host {
using kvd::PagedOut; using kvd::PagedPart; using kvd::PagedReqs;
// Checks of a pool's description; fills the kernels' view of it.
int paged_pool_view(const kvd_paged_pool* p, kvd::PagedPool* out);
int paged_sm_count();
// Attention over the pages on tcgen05, for requests of many rows: whether it
// takes the shape, its workspace, its launch.
bool paged_chunk_takes(int head_dim, int dtype);
size_t paged_chunk_ws_bytes(int head_dim);
int launch_paged_chunk(const kvd::PagedPool& pool, int D, int store, const PagedReqs& reqs, const int* table, long table_stride,
                       int dtype, const void* q, long q_sb, long q_sh, long q_st, float scaling_log2, const PagedOut& out,
                       int fill_tail, void* ws, cudaStream_t s);

inline size_t part_bytes(int ctas, int rt, int D) {
  return (size_t)ctas * sizeof(int4) + (size_t)ctas * 2 * rt * (D + 2) * sizeof(float);
}
inline PagedPart part_at(void* ws, int ctas) {
  PagedPart p;
  p.head = (int4*)ws;
  p.rec = (float*)((char*)ws + (size_t)ctas * sizeof(int4));
  return p;
}

template <int D, int RT, typename T>
int launch_merge(const PagedReqs& rq, const PagedPart& part, const PagedOut& out, int fill_tail, int ctas,
                        cudaStream_t s) {
  // starts while the kernel before it drains, and waits for it in the kernel
  cudaLaunchConfig_t cfg = {};
  const long rows = std::min((long)RT, (long)rq.q_tokens * rq.G);
  cfg.gridDim = dim3(ctas, (unsigned)std::min(32L, rows));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  KTimerScope kts_("paged_merge_kernel", s);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kvd::paged_merge_kernel<D, RT, T>, rq, part, out, fill_tail);
  if (e != cudaSuccess) { set_error("paged_merge_kernel: %s", cudaGetErrorString(e)); return KVD_ERR_CUDA; }
  return KVD_OK;
}

}  // namespace kvd_host
