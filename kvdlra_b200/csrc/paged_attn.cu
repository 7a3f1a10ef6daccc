// Attention over 8-bit pages for requests of few query rows (single tokens,
// a few drafted ones), and of any number of rows where no tensor-memory kernel
// takes the shape (sm_100a).
//
// o = sum_t softmax_t(scale * ks_t (q . kc_t)) vs_t vc_t over the tokens a row
// sees; kc, vc are codes and ks, vs the scales of the token's page.  One pass:
// running maximum m, sum l and accumulator O, in base 2.
//
// A decode reads 2 len H D bytes and computes 4 len Hq D flops, so HBM bounds
// it.  Every code is used by one warp only, so codes go from global memory
// straight into the registers of the matrix fragments, without shared memory:
//   scores   S^T = K Q^T with m16n8k16 f16: 16 tokens x 8 query rows.  Lane
//            (g, j) loads 16 contiguous bytes of token g's row; which of the
//            head's dims a fragment slot stands for is free as long as Q's
//            fragments follow it, so the bytes are used in the order they come.
//   values   O^T = V^T P^T: 16 dims x 8 rows.  Lane (g, j) loads contiguous
//            bytes of tokens 2j, 2j+1, 2j+8, 2j+9; a byte permute pairs two
//            tokens of a dim before the conversion, which is all the transpose
//            that V needs.  P^T comes from S^T's accumulators by movmatrix.
// The next tile's keys are loaded as soon as this tile's are used up, its
// values likewise: 4 to 8 KB in flight per warp.
//
// Codes are exact in f16.  Q rows are scaled by a power of two to below 2 and
// rounded to f16 (exact for bf16 and f16 but for elements 2^-13 of the row's
// largest); an fp32 call splits Q and P into two f16 parts, about 22 bits.
// P is rounded to f16 (2^-11); m, l and O are fp32.
//
// Two references per row, in base 2: m for the sum l of the weights, and mv
// for O, whose weights carry the page's value scale: p vs = 2^(x - m) (vs
// 2^(m - mv)), so P's rounding is relative to the largest p vs.  They follow
// the running maxima only when these pass them by kLTop and kPTop: a tile costs
// one vote instead of reductions over the lanes.
//
// Measured: 64 requests of 1 to 32768 tokens, 32 heads over 8 of 128, int8: 424 us,
// 5.1 TB/s, 78 % of the copy rate; one of 131072 tokens, e4m3: 63 us, 4.2 TB/s; 64
// ragged ones by form: fp32 of 128 517 us where the bytes take 319, bf16 of 64, 32 and
// 256 241, 197 and 451 where they take 159, 80 and 319.  The
// conversions' and the softmax's instructions bound it (half of all issue slots at
// three warps a scheduler): a prefetch of the tile after next into L2 gained nothing.
//
// Work: (request, KV head, row tile, 128-token tile) is one list, every CTA
// takes an equal run of it; a unit that spans CTAs leaves records that
// paged_merge_kernel joins.  Lengths stay on the device.
#include <algorithm>
#include <new>

#include "paged.cuh"

namespace kvd {

constexpr int kRowThreads = 128;  // 4 warps, each its own tokens of a tile
constexpr int kSegPages = 256;    // pages whose ids and scales are staged at a time

struct RowArgs {
  PagedPool pool;
  PagedReqs reqs;
  const int* table;
  long table_stride;
  const void* q;
  long q_sb, q_sh, q_st;
  float scaling;  // times log2(e)
  PagedOut out;
  PagedPart part;
  int fill_tail;
};

KVD_DEVICE void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
KVD_DEVICE uint32_t transpose_f16x2(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// CTAs of the few-row kernel per SM: as many as its accumulators and the codes
// in flight leave registers for without spills
__host__ __device__ constexpr int rows_per_sm(int D, int nt, bool fp32) {
  return D <= 64 ? (fp32 ? 3 : nt == 1 ? 4 : 3) : D == 128 && nt == 1 && !fp32 ? 3 : 2;
}

// W words from global memory, read once
template <int W>
KVD_DEVICE void load_words(const unsigned char* p, uint32_t* w) {
  if constexpr (W == 1) {
    asm volatile("ld.global.nc.L1::no_allocate.b32 %0, [%1];" : "=r"(w[0]) : "l"(p));
  } else if constexpr (W == 2) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4)
      asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "l"(p + 4 * i));
  }
}

// D: head dim; NT: query rows / 8; ST: 16-token subtiles per warp and tile
template <int D, int NT, int ST>
struct RowShape {
  static constexpr int RT = 8 * NT;         // rows of a unit
  static constexpr int WT = 16 * ST;        // tokens per warp and tile
  static constexpr int TT = 4 * WT;         // tokens per CTA and tile
  static constexpr int KW = D / 16;         // words per lane of a key row, and k-steps
  static constexpr int VW = D / 32;         // words per lane of a value row
  static constexpr int smem = 4 * RT * D * 4;
};

template <int D, int NT, int ST, int STORE, typename T>
__global__ void __launch_bounds__(kRowThreads, rows_per_sm(D, NT, sizeof(T) == 4))
    paged_rows_kernel(const __grid_constant__ RowArgs a) {
  using Sh = RowShape<D, NT, ST>;
  constexpr int RT = Sh::RT, WT = Sh::WT, TT = Sh::TT, KW = Sh::KW, VW = Sh::VW;
  constexpr bool SPLIT = sizeof(T) == 4;
  extern __shared__ __align__(16) float osm[];  // [4 warps][RT][D]
  __shared__ float4 seg[kSegPages];  // of a page: keys' scale, values' scale, log2 of that, id (as bits; < 0: none)
  __shared__ float sm_m[4][RT], sm_l[4][RT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j = lane & 3;
  const PagedPool& pool = a.pool;
  const PagedReqs& rq = a.reqs;
  const int lg = pool.lg_page, page_mask = pool.page() - 1;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge waits for this grid's end itself
  const WorkAt at = find_work<RT, TT, kRowThreads>(rq, blockIdx.x, gridDim.x);
  // The walk over the pieces lies in shared memory and is taken by one thread:
  // the registers have no room for it beside the codes and the accumulators.
  __shared__ alignas(16) unsigned char walk[sizeof(Pieces<RT, TT>)];
  __shared__ int walk_more;
  __shared__ int4 begun;
  Pieces<RT, TT>& pc = *reinterpret_cast<Pieces<RT, TT>*>(walk);
  if (tid == 0) {
    new (&pc) Pieces<RT, TT>(rq, at, blockIdx.x);
    begun = make_int4(0, 0, 0, 0);
  }
  const long chunk = at.chunk;
  while (true) {
    if (tid == 0) walk_more = pc.next();
    __syncthreads();
    if (!walk_more) break;
    const int b = pc.b, h = pc.h, row0 = pc.rt * RT, rows = pc.rows, lo = pc.lo, hi = pc.hi;
    const int t_begin = pc.tile * TT, t_end = min(hi, t_begin + pc.n * TT);
    // every row sees [lo_all, hi_all)
    const int hi_all = pc.row_hi(row0), lo_all = pc.row_lo(min(rows - 1, row0 + RT - 1));

    // ---- Q fragments (B operand: k = dims, n = rows), scaled by a power of two per row
    uint32_t qf[NT][KW][2], ql[SPLIT ? NT : 1][SPLIT ? KW : 1][2];
    float cq[NT][2];   // this lane's score columns: rows 8 nt + 2j + {0, 1}
    int lim_lo[NT][2], lim_hi[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int R = row0 + 8 * nt + g;
      const bool live = R < rows;
      const int qi = live ? R / rq.G : 0;
      const T* src = reinterpret_cast<const T*>(a.q) + (rq.cu_q ? 0 : (long)b * a.q_sb) +
                     (long)(h * rq.G + (live ? R % rq.G : 0)) * a.q_sh + (long)(rq.q0(b) + qi) * a.q_st;
      float x[KW][4];
      float amax = 0.f;
#pragma unroll
      for (int kk = 0; kk < KW; ++kk) {
        const int d = D == 32 ? 8 * j + 4 * kk : 64 * (kk >> 2) + 16 * j + 4 * (kk & 3);
        if constexpr (sizeof(T) == 4) {
          const float4 f = live ? *reinterpret_cast<const float4*>(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
          x[kk][0] = f.x; x[kk][1] = f.y; x[kk][2] = f.z; x[kk][3] = f.w;
        } else {
          const uint2 u = live ? *reinterpret_cast<const uint2*>(src + d) : make_uint2(0u, 0u);
          const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[kk][i] = load_f(e + i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(x[kk][i]));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      int e = (int)(__float_as_uint(amax) >> 23) - 127;
      e = e > 127 ? 0 : max(-100, min(126, e));  // an infinite row keeps its values
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int kk = 0; kk < KW; ++kk) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const float u = x[kk][2 * p] * down, w = x[kk][2 * p + 1] * down;
          qf[nt][kk][p] = pack_f16(u, w);
          if constexpr (SPLIT) {
            const float2 r = unpack_f16(qf[nt][kk][p]);
            ql[nt][kk][p] = pack_f16(u - r.x, w - r.y);
          }
        }
      }
      const float up = __uint_as_float((uint32_t)(127 + e) << 23) * a.scaling;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        cq[nt][c] = __shfl_sync(0xffffffffu, up, (2 * j + c) * 4);
        const int Rc = min(rows - 1, row0 + 8 * nt + 2 * j + c);
        lim_hi[nt][c] = pc.row_hi(Rc);
        lim_lo[nt][c] = pc.row_lo(Rc);
      }
    }

    float acc[D / 16][NT][4];
    float m[NT][2], mv[NT][2], l[NT][2];  // references of l and of O, see the top
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[dt][nt][i] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = mv[nt][0] = mv[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;

    const int pg_end = (t_end + page_mask) >> lg;  // pages of the piece
    for (int pg0 = t_begin >> lg; pg0 < pg_end; ) {
      // ---- page ids and scales of the next pages (whole tiles)
      const int t_seg0 = max(t_begin, pg0 << lg);
      int t_seg1 = t_seg0 + (((pg0 + kSegPages) << lg) - t_seg0) / TT * TT;
      t_seg1 = min(t_seg1, t_end);
      const int np = ((t_seg1 + page_mask) >> lg) - pg0;
      __syncthreads();  // the previous segment's (or unit's) readers are done
      for (int i = tid; i < np; i += kRowThreads) {
        int id = -1;  // of a page that no row of the piece sees: the tile begins before the window, or in the padding
        if (pg0 + i >= lo >> lg && ((pg0 + i) << lg) < hi) {
          id = a.table[(long)b * a.table_stride + pg0 + i];
          if (id < 0 || id >= pool.num_pages) {
            pool.flag(kStatusBounds, kPagedBadPage);
            id = -1;
          }
        }
        const float vs = id < 0 ? 0.f : pool.vs[(long)id * pool.scale_stride + h];
        seg[i] = make_float4(id < 0 ? 0.f : pool.ks[(long)id * pool.scale_stride + h], vs, log2f(vs), __int_as_float(id));
      }
      __syncthreads();

      // ---- this warp's tiles
      const int w_off = warp * WT;
      auto key_words = [&](int t, uint32_t (&kw)[ST][2][KW]) {
#pragma unroll
        for (int s = 0; s < ST; ++s) {
          const int tb = t + 16 * s, pi = (tb >> lg) - pg0;
          const int id = pi < np ? __float_as_int(seg[pi].w) : -1;
          const unsigned char* p = pool.k + (long)id * pool.page_stride + (long)h * pool.head_stride +
                                   (long)((tb & page_mask) + g) * pool.slot_stride + (D == 32 ? 8 : 16) * j;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (id >= 0) {
              constexpr int W = KW < 4 ? KW : 4;
#pragma unroll
              for (int c = 0; c < KW / W; ++c) load_words<W>(p + 8L * r * pool.slot_stride + 64 * c, &kw[s][r][W * c]);
            } else {
#pragma unroll
              for (int c = 0; c < KW; ++c) kw[s][r][c] = 0u;
            }
          }
        }
      };
      auto value_words = [&](int t, uint32_t (&vw)[ST][4][VW]) {
#pragma unroll
        for (int s = 0; s < ST; ++s) {
          const int tb = t + 16 * s, pi = (tb >> lg) - pg0;
          const int id = pi < np ? __float_as_int(seg[pi].w) : -1;
          const unsigned char* p = pool.v + (long)id * pool.page_stride + (long)h * pool.head_stride +
                                   (long)((tb & page_mask) + 2 * j) * pool.slot_stride + (D / 8) * g;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = (r & 1) + 8 * (r >> 1);  // tokens 2j, 2j + 1, 2j + 8, 2j + 9
            if (id >= 0) {
              load_words<VW>(p + (long)row * pool.slot_stride, vw[s][r]);
            } else {
#pragma unroll
              for (int c = 0; c < VW; ++c) vw[s][r][c] = 0u;
            }
          }
        }
      };
      uint32_t kw[ST][2][KW], vw[ST][4][VW];
      int t = t_seg0 + w_off;
      if (t < t_seg1) {
        key_words(t, kw);
        value_words(t, vw);
      }
      for (; t < t_seg1; t += TT) {
        // scores of WT tokens x RT rows
        float s[ST][NT][4];
#pragma unroll
        for (int u = 0; u < ST; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][nt][i] = 0.f;
#pragma unroll
        for (int u = 0; u < ST; ++u) {
#pragma unroll
          for (int kk = 0; kk < KW; ++kk) {
            uint32_t f[4];
            codes_to_f16<STORE>(kw[u][0][kk], &f[0], &f[2]);
            codes_to_f16<STORE>(kw[u][1][kk], &f[1], &f[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(s[u][nt], f, qf[nt][kk][0], qf[nt][kk][1]);
              if constexpr (SPLIT) mma_f16(s[u][nt], f, ql[nt][kk][0], ql[nt][kk][1]);
            }
          }
        }
        float ksc[ST], vsc[ST], lvs[ST];
        bool whole = t >= lo_all && t + WT <= hi_all;  // every row sees every token of the tile
        bool bad[ST];
#pragma unroll
        for (int u = 0; u < ST; ++u) {
          const int pi = ((t + 16 * u) >> lg) - pg0;
          const float4 e = seg[min(pi, np - 1)];
          ksc[u] = e.x;
          vsc[u] = e.y;
          lvs[u] = e.z;
          bad[u] = pi >= np || __float_as_int(e.w) < 0;
          whole = whole && !bad[u];
        }
        if (t + TT < t_seg1) key_words(t + TT, kw);
        // maxima of x and of x + log2(vs), of this lane's tokens
        float mt[NT][2], vt[NT][2];
        bool grew = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mt[nt][0] = mt[nt][1] = vt[nt][0] = vt[nt][1] = -INFINITY;
#pragma unroll
        for (int u = 0; u < ST; ++u) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float f = fmaxf(ksc[u] * cq[nt][c], 0x1p-126f);
              s[u][nt][c] *= f;
              s[u][nt][2 + c] *= f;
              if (!whole) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                  const int tok = t + 16 * u + g + 8 * hf;
                  if (bad[u] || tok < lim_lo[nt][c] || tok >= lim_hi[nt][c]) s[u][nt][2 * hf + c] = -INFINITY;
                }
              }
              const float x = fmaxf(s[u][nt][c], s[u][nt][2 + c]);
              mt[nt][c] = fmaxf(mt[nt][c], x);
              vt[nt][c] = fmaxf(vt[nt][c], x + lvs[u]);
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) grew |= mt[nt][c] > m[nt][c] + kLTop || vt[nt][c] > mv[nt][c] + kPTop;
        if (__any_sync(0xffffffffu, grew)) {  // rare after the first tiles
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float al[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = fmaxf(m[nt][c], mt[nt][c]), y = fmaxf(mv[nt][c], vt[nt][c] - kPBias);
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) {
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
                y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, o));
              }
              if (m[nt][c] != -INFINITY) l[nt][c] *= exp2_fast(m[nt][c] - x);
              al[c] = mv[nt][c] == -INFINITY ? 1.f : exp2_fast(mv[nt][c] - y);
              m[nt][c] = x;
              mv[nt][c] = y;
            }
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[dt][nt][i] *= al[i & 1];
          }
        }
        // weights p vs / 2^(mv - m), rounded to f16, as the B operand
        uint32_t pf[ST][NT][2], pl[SPLIT ? ST : 1][SPLIT ? NT : 1][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float base[2], fr[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            base[c] = m[nt][c] == -INFINITY ? 0.f : m[nt][c];
            fr[c] = mv[nt][c] == -INFINITY ? 0.f : exp2_fast(m[nt][c] - mv[nt][c]);
          }
#pragma unroll
          for (int u = 0; u < ST; ++u)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              float p[2];
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                p[c] = exp2_fast(s[u][nt][2 * hf + c] - base[c]);
                l[nt][c] += p[c];
                p[c] *= fminf(vsc[u] * fr[c], 0x1p100f);
              }
              const uint32_t w = pack_f16(p[0], p[1]);
              pf[u][nt][hf] = transpose_f16x2(w);
              if constexpr (SPLIT) {
                const float2 r = unpack_f16(w);
                pl[u][nt][hf] = transpose_f16x2(pack_f16(p[0] - r.x, p[1] - r.y));
              }
            }
        }
        if (!whole) {  // codes of tokens outside [lo, hi) may be anything
#pragma unroll
          for (int u = 0; u < ST; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int tok = t + 16 * u + 2 * j + (r & 1) + 8 * (r >> 1);
              if (tok < lo || tok >= hi) {
#pragma unroll
                for (int c = 0; c < VW; ++c) vw[u][r][c] = 0u;
              }
            }
        }
#pragma unroll
        for (int u = 0; u < ST; ++u)
#pragma unroll
          for (int c = 0; c < VW; ++c) {
            // words c of tokens 2j, 2j+1 (then 2j+8, 2j+9): dims 4c .. 4c+3 of the lane's chunk
            const uint32_t p01 = __byte_perm(vw[u][0][c], vw[u][1][c], 0x5140);
            const uint32_t p23 = __byte_perm(vw[u][0][c], vw[u][1][c], 0x7362);
            const uint32_t r01 = __byte_perm(vw[u][2][c], vw[u][3][c], 0x5140);
            const uint32_t r23 = __byte_perm(vw[u][2][c], vw[u][3][c], 0x7362);
            uint32_t f[4], e[4];
            codes_to_f16<STORE>(p01, &f[0], &f[1]);
            codes_to_f16<STORE>(r01, &f[2], &f[3]);
            codes_to_f16<STORE>(p23, &e[0], &e[1]);
            codes_to_f16<STORE>(r23, &e[2], &e[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(acc[2 * c][nt], f, pf[u][nt][0], pf[u][nt][1]);
              mma_f16(acc[2 * c + 1][nt], e, pf[u][nt][0], pf[u][nt][1]);
              if constexpr (SPLIT) {
                mma_f16(acc[2 * c][nt], f, pl[u][nt][0], pl[u][nt][1]);
                mma_f16(acc[2 * c + 1][nt], e, pl[u][nt][0], pl[u][nt][1]);
              }
            }
          }
        if (t + TT < t_seg1) value_words(t + TT, vw);
      }
      pg0 = t_seg1 >> lg;  // a tile border is a page border, or the end of the piece
      if (t_seg1 >= t_end) break;
    }

    // ---- the four warps' shares: one maximum, summed accumulators
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], o);
        if (g == 0) {
          sm_m[warp][8 * nt + 2 * j + c] = m[nt][c];
          sm_l[warp][8 * nt + 2 * j + c] = l[nt][c];
        }
      }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 8 * nt + 2 * j + c;
        const float M = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r]));
        // a warp that saw nothing has O = 0 (or NaN, from a NaN query)
        const float f = mv[nt][c] == -INFINITY ? 1.f : exp2_fast(mv[nt][c] - M);
        float* dst = osm + ((long)warp * RT + r) * D + (D / 8) * g;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          dst[2 * dt] = acc[dt][nt][c] * f;
          dst[2 * dt + 1] = acc[dt][nt][2 + c] * f;
        }
      }
    __syncthreads();
    const bool whole_unit = pc.whole();
    float* rec = a.part.rec + ((long)blockIdx.x * 2 + (pc.off == 0 ? 1 : 0)) * RT * (D + 2);
    for (int e = tid; e < RT * D; e += kRowThreads) {
      const int r = e / D, d = e % D, R = row0 + r;
      if (R >= rows) break;
      const float M = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r]));
      float L = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        L += sm_l[w][r] * (sm_m[w][r] == -INFINITY ? 1.f : exp2_fast(sm_m[w][r] - M));
        o += osm[(w * RT + r) * D + d];
      }
      if (whole_unit) {
        const long row = pc.out_row(R);
        const int hq = h * rq.G + R % rq.G;
        store_held(reinterpret_cast<T*>(a.out.out) + (row * a.out.Hq + hq) * D + d, L == 0.f ? 0.f : o / L);
        if (d == 0 && a.out.lse)
          a.out.lse[row * a.out.Hq + hq] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
      } else {
        rec[r * D + d] = o;
        if (d == 0) {
          rec[RT * D + r] = M;
          rec[RT * D + RT + r] = L;
        }
      }
    }
    if (tid == 0)
      if (const int n = pc.pieces(chunk)) begun = make_int4(b, h, pc.rt, n);
    __syncthreads();  // the output's readers, and the piece's, are done
  }
  if (tid == 0) a.part.head[blockIdx.x] = begun;
}

}  // namespace kvd

namespace kvd_host {
using namespace kvd;

int paged_sm_count() {
  static int sms[kMaxDevices] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 148;
  if (!sms[dev]) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  return sms[dev] > 0 ? sms[dev] : 148;
}

int paged_pool_view(const kvd_paged_pool* p, PagedPool* out) {
  if (!p || !p->k || !p->v || !p->k_scale || !p->v_scale) { set_error("paged pool: null pointer"); return KVD_ERR_ARG; }
  if (p->store != KVD_STORE_E4M3 && p->store != KVD_STORE_INT8) { set_error("paged pool: unknown store %d", p->store); return KVD_ERR_DTYPE; }
  const int s = p->page_size;
  if (s != 16 && s != 32 && s != 64 && s != 128) { set_error("paged pool: page_size %d is none of 16, 32, 64, 128", s); return KVD_ERR_ARG; }
  const int d = p->head_dim;
  if (d != 32 && d != 64 && d != 128 && d != 256) { set_error("paged pool: head_dim %d is none of 32, 64, 128, 256", d); return KVD_ERR_ARG; }
  if (p->num_pages < 1 || p->num_heads < 1 || p->num_heads > 1024 || (int64_t)p->num_pages * s > INT32_MAX) {
    set_error("paged pool: %d pages of %d tokens, %d heads", p->num_pages, s, p->num_heads);
    return KVD_ERR_ARG;
  }
  if (p->page_stride % 16 || p->head_stride % 16 || p->slot_stride % 16 || p->slot_stride < d ||
      ((uintptr_t)p->k | (uintptr_t)p->v) % 16) {
    set_error("paged pool: codes and their strides must be multiples of 16 bytes");
    return KVD_ERR_ARG;
  }
  out->k = (unsigned char*)p->k; out->v = (unsigned char*)p->v;
  out->ks = p->k_scale; out->vs = p->v_scale;
  out->page_stride = p->page_stride; out->head_stride = p->head_stride; out->slot_stride = p->slot_stride;
  if (p->scale_stride < p->num_heads) { set_error("paged pool: scale_stride %lld below %d heads", (long long)p->scale_stride, p->num_heads); return KVD_ERR_ARG; }
  out->scale_stride = p->scale_stride;
  out->num_pages = p->num_pages; out->H = p->num_heads; out->status = p->status;
  out->lg_page = s == 16 ? 4 : s == 32 ? 5 : s == 64 ? 6 : 7;
  return KVD_OK;
}

// A request of at most this many rows goes to the few-row kernel: its codes are
// read once per 8 or 16 rows, the tensor-memory kernel's once per 256, whose tile
// costs the same however few rows it has.  The first and the other, in us:
//   head_dim 64   96 requests of 100 to 4099 tokens, 4 KV heads: 140 and 178 at 17
//                 rows, 164 and 189 at 32, 212 and 191 at 33, 312 and 195 at 64;
//                 one of 32768, 8 KV heads: 36 and 52 at 17, 38 and 54 at 32, 44 and
//                 55 at 33, 52 and 57 at 64
//   head_dim 128  96 requests of 100 to 4099: 192 and 194 at 32 rows; 512 of 300 to
//                 899: 319 and 353 at 17, 385 and 428 at 32, 499 and 428 at 33; one of
//                 32768: 49 and 58 at 17, 52 and 61 at 32, 65 and 62 at 33
constexpr int kFewRows = 32;

// Rows of a unit / 8: one, or two where a request has more than eight rows.  64
// requests of 1 to 32768 tokens, 8 KV heads of 128, bf16: 442 us in units of 8 rows
// and 632 in units of 16 at 8 rows, 799 and 707 at 9, 856 and 726 at 16; fp32: 569 and
// 781, 1021 and 799, 1092 and 888 (head_dim 256: sixteen rows' accumulators would not
// fit the registers; thirty-two rows at head_dim 64 fit, but took 237 us where sixteen
// take 211, for 24 fp32 requests of 1 to 257 rows).
static int rows_nt(long max_rows, int D) { return max_rows <= 8 || D == 256 ? 1 : 2; }
// CTAs that fit an SM (the kernel's launch bounds)
static int rows_ctas(int D, int nt, bool fp32) { return paged_sm_count() * rows_per_sm(D, nt, fp32); }

template <int D, int NT, int STORE, typename T>
static int launch_rows(RowArgs& a, void* ws, cudaStream_t s) {
  constexpr int ST = D == 256 ? 1 : 2;
  using Sh = RowShape<D, NT, ST>;
  auto kern = paged_rows_kernel<D, NT, ST, STORE, T>;
  if (int rc = ensure_smem((const void*)kern, Sh::smem, "paged_rows_kernel")) return rc;
  const int ctas = rows_ctas(D, NT, sizeof(T) == 4);
  a.part = part_at(ws, ctas);
  {
    KTimerScope kts_("paged_rows_kernel", s);
    kern<<<ctas, kRowThreads, Sh::smem, s>>>(a);
  }
  if (int rc = check_launch("paged_rows_kernel")) return rc;
  return launch_merge<D, Sh::RT, T>(a.reqs, a.part, a.out, a.fill_tail, ctas, s);
}

template <int D, typename T>
static int launch_rows_d(RowArgs& a, int nt, int store, void* ws, cudaStream_t s) {
  if (D == 256 || nt == 1) return store == KVD_STORE_E4M3 ? launch_rows<D, 1, kStoreE4M3, T>(a, ws, s) : launch_rows<D, 1, kStoreInt8, T>(a, ws, s);
  if constexpr (D != 256)
    return store == KVD_STORE_E4M3 ? launch_rows<D, 2, kStoreE4M3, T>(a, ws, s) : launch_rows<D, 2, kStoreInt8, T>(a, ws, s);
  return KVD_ERR_ARG;
}

template <typename T>
static int launch_rows_t(RowArgs& a, int D, int nt, int store, void* ws, cudaStream_t s) {
  switch (D) {
    case 32: return launch_rows_d<32, T>(a, nt, store, ws, s);
    case 64: return launch_rows_d<64, T>(a, nt, store, ws, s);
    case 128: return launch_rows_d<128, T>(a, nt, store, ws, s);
    default: return launch_rows_d<256, T>(a, nt, store, ws, s);
  }
}

}  // namespace kvd_host

using namespace kvd_host;

extern "C" size_t kvd_paged_attention_workspace_bytes(const kvd_paged_pool* pool, int32_t dtype, int32_t num_q_heads) {
  kvd::PagedPool v;
  if (paged_pool_view(pool, &v)) return 0;
  if (num_q_heads < 1 || num_q_heads % pool->num_heads) { set_error("%d query heads over %d KV heads", num_q_heads, pool->num_heads); return 0; }
  const int D = pool->head_dim;
  size_t need = 0;
  for (int nt = 1; nt <= 2; ++nt) need = std::max(need, part_bytes(rows_ctas(D, nt, dtype == KVD_DTYPE_F32), 8 * nt, D));
  if (paged_chunk_takes(D, dtype)) need = std::max(need, paged_chunk_ws_bytes(D));
  return need;
}

extern "C" int kvd_paged_attention(const kvd_paged_pool* pool, int32_t batch, const int32_t* table, int64_t table_stride,
                                   int32_t max_pages, const int32_t* lens, const int32_t* starts, const int32_t* cu_q,
                                   int32_t dtype, const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st,
                                   int32_t q_tokens, int32_t max_q, int32_t num_q_heads, float scaling, int32_t window,
                                   void* out, float* lse, int32_t fill_tail, void* workspace, size_t ws_bytes, kvd_stream_t stream) try {
  RowArgs a;
  if (int rc = paged_pool_view(pool, &a.pool)) return rc;
  const int H = pool->num_heads, D = pool->head_dim;
  if (dtype != KVD_DTYPE_F32 && dtype != KVD_DTYPE_BF16 && dtype != KVD_DTYPE_F16) { set_error("paged attention: unsupported dtype %d", dtype); return KVD_ERR_DTYPE; }
  if (batch < 0 || q_tokens < 0 || max_q < 0 || max_pages < 0 || window < 0 || table_stride < max_pages) { set_error("paged attention: negative size, or a table stride below its width"); return KVD_ERR_ARG; }
  if (num_q_heads < H || num_q_heads % H) { set_error("paged attention: %d query heads over %d KV heads", num_q_heads, H); return KVD_ERR_ARG; }
  if (!(scaling > 0.f) || scaling > 1e30f) { set_error("paged attention: scaling must be positive and finite, got %g", scaling); return KVD_ERR_ARG; }
  if (batch == 0 || q_tokens == 0) return KVD_OK;
  const int G = num_q_heads / H;
  if ((int64_t)q_tokens * G > INT32_MAX / 2 || (int64_t)max_pages * pool->page_size > INT32_MAX / 2) { set_error("paged attention: too many rows or cached tokens for one request"); return KVD_ERR_ARG; }
  if ((!table && max_pages) || !lens || !q || !out) { set_error("paged attention: null pointer"); return KVD_ERR_ARG; }
  const int size = dtype == KVD_DTYPE_F32 ? 4 : 2;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)(q_sb * size) | (uintptr_t)(q_sh * size) | (uintptr_t)(q_st * size)) % 16) {
    set_error("paged attention: queries, their strides and the output must be multiples of 16 bytes");
    return KVD_ERR_ARG;
  }
  if (!workspace || (uintptr_t)workspace % 16 || ws_bytes < kvd_paged_attention_workspace_bytes(pool, dtype, num_q_heads)) {
    set_error("paged attention: workspace of %zu bytes, 16-byte aligned, is needed", kvd_paged_attention_workspace_bytes(pool, dtype, num_q_heads));
    return KVD_ERR_WORKSPACE;
  }
  PagedReqs& r = a.reqs;
  r.batch = batch; r.H = H; r.G = G; r.q_tokens = q_tokens;
  r.window = std::min(window, 1 << 30);  // more than any request holds: place and window stay within 32 bits
  r.max_len = max_pages * pool->page_size;
  r.lens = lens; r.cu_q = cu_q; r.starts = starts;
  r.min_rows = 1; r.max_rows = INT32_MAX;
  a.table = table; a.table_stride = table_stride;
  a.q = q; a.q_sb = q_sb; a.q_sh = q_sh; a.q_st = q_st;
  a.fill_tail = fill_tail;
  a.scaling = scaling * 1.4426950408889634f;
  a.out.out = out; a.out.lse = lse; a.out.Hq = num_q_heads;
  const int most = cu_q ? std::min(max_q > 0 ? max_q : q_tokens, q_tokens) : q_tokens;
  // Requests of more rows than kFewRows go to the tensor-memory kernel, where it
  // takes the shape; a packed batch may hold both kinds, and each kernel passes
  // over the other's requests.  One workspace serves both: they run in turn.
  const bool chunks = paged_chunk_takes(D, dtype) && (long)most * G > kFewRows;
  const bool few = !chunks || cu_q;
  if (chunks) {
    PagedReqs rc_ = r;
    rc_.min_rows = kFewRows + 1;
    if (int rc = launch_paged_chunk(a.pool, D, pool->store, rc_, table, table_stride, dtype, q, q_sb, q_sh, q_st, a.scaling, a.out,
                                    few ? 0 : fill_tail, workspace, (cudaStream_t)stream))
      return rc;
    r.max_rows = kFewRows;
  }
  if (!few) return KVD_OK;
  const int nt = rows_nt(std::min((long)most * G, (long)r.max_rows), D);
  if (dtype == KVD_DTYPE_F32) return launch_rows_t<float>(a, D, nt, pool->store, workspace, (cudaStream_t)stream);
  if (dtype == KVD_DTYPE_BF16) return launch_rows_t<__nv_bfloat16>(a, D, nt, pool->store, workspace, (cudaStream_t)stream);
  return launch_rows_t<__half>(a, D, nt, pool->store, workspace, (cudaStream_t)stream);
} catch (...) {
  set_error("paged attention: host error");
  return KVD_ERR_CUDA;
}
