// Attention over 8-bit pages for requests of many query rows (chunks of a
// prompt) on tcgen05 (sm_100a): bf16 and f16 queries, head_dim 64 and 128.
//
// One CTA of 13 warps per SM walks its run of the work list; a unit is
// (request, KV head, 256 query rows), a row (token, head of the group).  Per
// 128-token tile:
//   loaders (4 warps)  the page's codes from global memory, a tile ahead in
//                      registers, converted exactly to f16 and written to shared
//                      memory as rows of 64 dims with the 128-byte swizzle: the
//                      same image is a K-major operand of the scores and an
//                      MN-major one of the values.
//   issuer (1 thread)  S_w = Q_w K^T for the two row tiles w of 128 rows, and
//                      O_w += P_w V with P_w in TMEM; while one row tile's
//                      softmax runs, the tensor core works for the other.
//   softmax (2 x 4 warps)  a thread owns a row (a TMEM lane): the row's maxima
//                      and sums need no other thread.  P_w (f16) goes over the
//                      columns of S_w.
// TMEM: S_0, S_1 (128 columns each), O_0, O_1 (head_dim each).
//
// Two references per row, in base 2: m for the sum l of the weights, and mv
// for O, whose weights carry the page's value scale: p vs = 2^(x - m) (vs 2^(m -
// mv)), so the f16 rounding of P is relative to the largest p vs.  They follow
// the running maxima only when these pass them by 8 (P <= 2^8): rescaling O,
// which lies in TMEM, is rare after the first tiles.
//
// Q is scaled per row by a power of two and rounded to f16 (exact but for
// elements 2^-13 of the row's largest); S, O, m, l are fp32; P is rounded to
// f16 (2^-11).
//
// Bound, per tile of 256 rows x 128 tokens at head_dim 128 and clock: tensor
// core 2048, exponentials 2048 (16 a clock), shared memory about 2048 (Q, K and
// V operands, and the converted tiles).
#include "paged.cuh"
#include "umma.cuh"

namespace kvd {

constexpr int kPcRows = 256, kPcTok = 128;
constexpr int kPcThreads = 512;            // 8 softmax warps, 4 loaders, issuer, planner (and 2 that wait)
// registers per thread of the four warpgroups: a softmax thread holds its row
// of S, a loader a tile's codes; their sum is what the CTA is launched with
constexpr int kPcRegsSoftmax = 168, kPcRegsLoad = 128, kPcRegsIssue = 48;
static_assert(2 * kPcRegsSoftmax + kPcRegsLoad + kPcRegsIssue == 4 * (65536 / kPcThreads), "register split");
constexpr int kPcLoad0 = 256, kPcIssue0 = 384, kPcPlan0 = 416;
constexpr int kPcBlock = kPcTok * 128;     // bytes of 64 columns of a 128-row f16 operand
constexpr long kPcPolls = 1L << 20;

struct ChunkArgs {
  PagedPool pool;
  PagedReqs reqs;
  const int* table;
  long table_stride;
  const void* q;
  long q_sb, q_sh, q_st;
  float scaling;  // times log2(e)
  PagedOut out;
  PagedPart part;
};

struct ChunkScales {  // of one tile, per 16 tokens
  float ks[8], vs[8], lv[8];  // lv = log2(vs)
  int bad[8];                 // page id out of range
};

// A piece of the CTA's work, as the planner hands it to the other roles (their
// registers have no room for the walk over the requests).
struct ChunkPiece {
  int n, tile;            // its token tiles; 0: there are no more pieces
  int b, h, row0, rows;   // request, KV head, the unit's first row, rows of the request
  int lo, hi;             // tokens that any of the unit's rows sees
  int len, q_len, start, q0;
  int whole, begins;      // covers its unit; begins it
};
constexpr int kPcPieces = 4;  // pieces planned ahead

template <int D>
struct ChunkSmem {
  static constexpr int NS = D == 64 ? 4 : 2;   // stages of keys, and of values
  static constexpr int tile = kPcTok * D * 2;  // f16 bytes of a 128-row operand
  static constexpr int q = 0, v = q + 2 * tile, k = v + NS * tile, sc = k + NS * tile;
  static constexpr int ring = 8;               // tiles whose scales are held: NS + 1 at least
  static constexpr int bars = sc + ring * (int)sizeof(ChunkScales);
  static constexpr int nbars = 4 * NS + 8 + 2 * kPcPieces;
  static constexpr int total = bars + nbars * 8 + 1024;  // room to align
};

KVD_DEVICE uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
KVD_DEVICE void unpack2(uint64_t x, float* a, float* b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(x)); }
KVD_DEVICE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
KVD_DEVICE uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
KVD_DEVICE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int D, int STORE, typename T>
__global__ void __launch_bounds__(kPcThreads, 1) paged_chunk_kernel(const __grid_constant__ ChunkArgs a) {
  using L = ChunkSmem<D>;
  constexpr int NS = L::NS;
  extern __shared__ unsigned char psm_raw[];
  unsigned char* psm = psm_raw + (-(int)(uint32_t)__cvta_generic_to_shared(psm_raw) & 1023);  // swizzle atoms are aligned
  __shared__ uint32_t tmem_base;
  __shared__ volatile int dead;  // a wait gave up
  __shared__ ChunkPiece pieces[kPcPieces];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const PagedPool& pool = a.pool;
  const PagedReqs& rq = a.reqs;
  uint64_t* bars = reinterpret_cast<uint64_t*>(psm + L::bars);
  uint64_t *kf = bars, *ke = kf + NS, *vf = ke + NS, *ve = vf + NS, *sf = ve + NS, *pf = sf + 2, *of = pf + 2, *qf = of + 2, *drain = qf + 1,
           *nf = drain + 1, *ne = nf + kPcPieces;
  ChunkScales* scales = reinterpret_cast<ChunkScales*>(psm + L::sc);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 0) {
    umma::tmem_alloc(&tmem_base, 512);
    umma::tmem_relinquish();
  }
  if (tid == 0) {
    dead = 0;
    for (int i = 0; i < NS; ++i) {
      umma::mbar_init(kf + i, 128);
      umma::mbar_init(ke + i, 1);
      umma::mbar_init(vf + i, 128);
      umma::mbar_init(ve + i, 1);
    }
    for (int w = 0; w < 2; ++w) {
      umma::mbar_init(sf + w, 1);
      umma::mbar_init(pf + w, 128);
      umma::mbar_init(of + w, 1);
    }
    for (int i = 0; i < kPcPieces; ++i) {
      umma::mbar_init(nf + i, 1);
      umma::mbar_init(ne + i, 256 + 128 + 1);
    }
    umma::mbar_init(qf, 256);
    umma::mbar_init(drain, 1);
    umma::mbar_fence_init();
  }
  umma::fence_before_sync();
  const WorkAt at = find_work<kPcRows, kPcTok, kPcThreads>(rq, blockIdx.x, gridDim.x);  // has barriers
  umma::fence_after_sync();
  const uint32_t tmem = tmem_base;
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    for (long i = 0; i < kPcPolls; ++i) {
      if (umma::mbar_try_wait(bar, parity)) return true;
      if (dead) return false;
    }
    dead = 1;
    pool.flag(kStatusTimeout, 1);
    return false;
  };

  if (tid >= kPcIssue0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPcRegsIssue));
    if (warp == kPcPlan0 / 32 && lane == 0) {
      // ---------------------------------------------------------- planner
      Pieces<kPcRows, kPcTok> pc(rq, at, blockIdx.x);
      int4 begun = make_int4(0, 0, 0, 0);
      for (int k = 0;; ++k) {
        const bool more = pc.next();
        const int sl = k % kPcPieces;
        if (!wait(ne + sl, ((k / kPcPieces) & 1) ^ 1)) break;
        ChunkPiece& p = pieces[sl];
        p.n = more ? pc.n : 0;
        if (more) {
          p.tile = pc.tile; p.b = pc.b; p.h = pc.h; p.row0 = pc.rt * kPcRows; p.rows = pc.rows;
          p.lo = pc.lo; p.hi = pc.hi; p.len = pc.len; p.q_len = pc.q_len; p.start = pc.start; p.q0 = rq.q0(pc.b);
          p.whole = pc.whole(); p.begins = pc.off == 0;
          if (const int n = pc.pieces(at.chunk)) begun = make_int4(pc.b, pc.h, pc.rt, n);
        }
        umma::mbar_arrive(nf + sl);
        if (!more) break;
      }
      a.part.head[blockIdx.x] = begun;
    } else if (warp == kPcIssue0 / 32) {
      // ----------------------------------------------------------- issuer
      // the whole warp walks, one lane issues: descriptors stay in uniform registers
      const uint64_t q_d = umma::smem_desc_sw128((uint32_t)__cvta_generic_to_shared(psm + L::q), 16, 1024);
      const uint64_t k_d = umma::smem_desc_sw128((uint32_t)__cvta_generic_to_shared(psm + L::k), 16, 1024);
      const uint64_t v_d = umma::smem_desc_sw128((uint32_t)__cvta_generic_to_shared(psm + L::v), kPcBlock, 1024);
      constexpr uint32_t id_s = umma::idesc_f16(128, kPcTok, false), id_o = umma::idesc_f16(128, D, true);
      // a descriptor's address field counts 16 bytes
      auto scores = [&](int w, int stage) {
        const uint64_t q_w = q_d + w * (L::tile >> 4), k_s = k_d + stage * (L::tile >> 4);
        if (umma::elect_one()) {
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            const uint64_t at_j = ((j >> 2) * kPcBlock + 32 * (j & 3)) >> 4;
            umma::mma_bf16(tmem + 128 * w, q_w + at_j, k_s + at_j, id_s, j > 0);
          }
          umma::commit(sf + w);
        }
        __syncwarp();
      };
      auto values = [&](int w, int stage, bool acc) {
        const uint64_t v_s = v_d + stage * (L::tile >> 4);
        if (umma::elect_one()) {
#pragma unroll
          for (int j = 0; j < kPcTok / 16; ++j)
            umma::mma_f16_ts(tmem + 256 + D * w, tmem + 128 * w + 8 * j, v_s + ((2048 * j) >> 4), id_o, acc || j > 0);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (umma::elect_one()) umma::commit(bar);
        __syncwarp();
      };
      auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(bar, parity)); };
      int it = 0, tc0 = 0, tc1 = 0;
      bool ok = true;
      for (int un = 0;; ++un) {
        const int sl = un % kPcPieces;
        ok = wait_all(nf + sl, (un / kPcPieces) & 1);
        if (!ok) break;
        const int n = __shfl_sync(0xffffffffu, pieces[sl].n, 0);
        const bool two = __shfl_sync(0xffffffffu, pieces[sl].rows - pieces[sl].row0 > 128, 0);
        if (lane == 0) umma::mbar_arrive(ne + sl);
        if (n == 0) break;
        ok = wait_all(qf, un & 1) && wait_all(kf + it % NS, (it / NS) & 1);
        if (!ok) break;
        umma::fence_after_sync();
        scores(0, it % NS);
        if (two) scores(1, it % NS);
        commit(ke + it % NS);
        for (int i = 0; i < n; ++i) {
          const int g = it + i, st = g % NS, nx = (g + 1) % NS;
          const bool more = i + 1 < n;
          ok = wait_all(vf + st, (g / NS) & 1) && wait_all(pf, tc0++ & 1);
          if (!ok) break;
          umma::fence_after_sync();
          values(0, st, i > 0);
          if (!two) commit(ve + st);
          if (more) {
            ok = wait_all(kf + nx, ((g + 1) / NS) & 1);
            if (!ok) break;
            umma::fence_after_sync();
            scores(0, nx);  // S over P: the tensor core takes one thread's products in order
            if (!two) commit(ke + nx);
          } else {
            commit(of);
          }
          if (!two) continue;
          ok = wait_all(pf + 1, tc1++ & 1);
          if (!ok) break;
          umma::fence_after_sync();
          values(1, st, i > 0);
          commit(ve + st);
          if (more) {
            scores(1, nx);
            commit(ke + nx);
          } else {
            commit(of + 1);
          }
        }
        if (!ok) break;
        it += n;
      }
      if (!ok) {  // nothing may be in flight when TMEM is freed
        commit(drain);
        umma::mbar_wait_bounded(drain, 0, kPcPolls);
      }
    }
  } else if (tid >= kPcLoad0) {
    // ----------------------------------------------------------- loaders
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPcRegsLoad));
    const int lw = warp - kPcLoad0 / 32;
    constexpr int QC = D / 64;  // 64-byte column blocks of a row
    const int tr = lane & 7, cl = lane >> 3;
    const int lg = pool.lg_page, mask = pool.page() - 1;
    struct Tile { int b, h, tok0, lo, hi; bool any; };
    Tile cur, nxt;
    nxt.any = false;
    int left = 0, un = 0;
    bool ok = true;
    auto step = [&](Tile* t) {  // the tile after *t
      if (left > 0) {
        --left;
        t->tok0 += kPcTok;
        return;
      }
      const int sl = un % kPcPieces;
      ok = wait(nf + sl, (un / kPcPieces) & 1);
      ok = __all_sync(0xffffffffu, ok);
      t->any = false;
      if (!ok) return;
      const ChunkPiece& p = pieces[sl];
      left = p.n - 1;
      t->any = p.n > 0;
      t->b = p.b; t->h = p.h; t->tok0 = p.tile * kPcTok; t->lo = p.lo; t->hi = p.hi;
      umma::mbar_arrive(ne + sl);
      ++un;
    };
    // lane l (mod 8) knows the page of the tile's l-th 16 tokens: -1 outside [lo, hi), -2 a bad id
    auto page_id = [&](const Tile& t) -> int {
      const int tok = t.tok0 + 16 * tr;
      if (!t.any || tok >= t.hi || tok + 16 <= t.lo) return -1;
      const int id = a.table[(long)t.b * a.table_stride + (tok >> lg)];
      return id < 0 || id >= pool.num_pages ? -2 : id;
    };
    uint4 kr[4][QC], vr[4][QC];
    auto fetch = [&](const Tile& t, int ids, const unsigned char* codes, uint4 (&r)[4][QC]) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int tg = 4 * k + lw, tok = t.tok0 + 8 * tg + tr;
        const int id = __shfl_sync(0xffffffffu, ids, tg >> 1);
        const bool live = t.any && id >= 0 && tok >= t.lo && tok < t.hi;
        const unsigned char* p = codes + (long)id * pool.page_stride + (long)t.h * pool.head_stride +
                                 (long)(tok & mask) * pool.slot_stride + 16 * cl;
#pragma unroll
        for (int c = 0; c < QC; ++c) {
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (live) asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p + 64 * c));
          r[k][c] = x;
        }
      }
    };
    auto put = [&](unsigned char* dst, const uint4 (&r)[4][QC]) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int tg = 4 * k + lw;
#pragma unroll
        for (int c = 0; c < QC; ++c) {
          const uint32_t w[4] = {r[k][c].x, r[k][c].y, r[k][c].z, r[k][c].w};
          uint32_t o[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) codes_to_f16<STORE>(w[e], &o[2 * e], &o[2 * e + 1]);
          unsigned char* p = dst + c * kPcBlock + tg * 1024 + tr * 128;
          *reinterpret_cast<uint4*>(p + 16 * ((2 * cl) ^ tr)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(p + 16 * ((2 * cl + 1) ^ tr)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
    };
    step(&nxt);
    cur = nxt;
    int ids = page_id(cur);
    fetch(cur, ids, pool.k, kr);
    fetch(cur, ids, pool.v, vr);
    for (int it = 0; cur.any && ok; ++it) {
      step(&nxt);
      if (!ok) break;
      const int ids_n = page_id(nxt);
      const int st = it % NS;
      float ks = 0.f, vs = 0.f;
      if (lw == 0 && lane < 8 && ids >= 0) {
        ks = pool.ks[(long)ids * pool.scale_stride + cur.h];
        vs = pool.vs[(long)ids * pool.scale_stride + cur.h];
      }
      ok = wait(ke + st, ((it / NS) & 1) ^ 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      put(psm + L::k + st * L::tile, kr);
      if (lw == 0 && lane < 8) {
        ChunkScales& s = scales[it % L::ring];
        s.ks[lane] = ks;
        s.vs[lane] = vs;
        s.lv[lane] = log2f(vs);
        s.bad[lane] = ids == -2;
        if (ids == -2) pool.flag(kStatusBounds, kPagedBadPage);
      }
      umma::fence_proxy_async_smem();
      umma::mbar_arrive(kf + st);
      fetch(nxt, ids_n, pool.k, kr);
      ok = wait(ve + st, ((it / NS) & 1) ^ 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      put(psm + L::v + st * L::tile, vr);
      umma::fence_proxy_async_smem();
      umma::mbar_arrive(vf + st);
      fetch(nxt, ids_n, pool.v, vr);
      cur = nxt;
      ids = ids_n;
    }
  } else {
    // ----------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPcRegsSoftmax));
    const int w = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t t_s = tmem + 128 * w + lanes, t_o = tmem + 256 + D * w + lanes;
    int it = 0, tc = 0, uc = 0;
    bool ok = true;
    for (int un = 0;; ++un) {
      const int sl = un % kPcPieces;
      ok = wait(nf + sl, (un / kPcPieces) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const ChunkPiece pc = pieces[sl];
      umma::mbar_arrive(ne + sl);
      if (pc.n == 0) break;
      const int R = pc.row0 + 128 * w + r;
      const bool two = pc.rows - pc.row0 > 128, active = w == 0 || two;
      const bool live = R < pc.rows;
      const int Rl = live ? R : pc.rows - 1, tok_q = Rl / rq.G, head = pc.h * rq.G + Rl % rq.G;
      float cq = 0.f;
      if (active) {
        // ---- this thread's query row, scaled by a power of two, as f16
        const T* src = reinterpret_cast<const T*>(a.q) + (rq.cu_q ? 0 : (long)pc.b * a.q_sb) + (long)head * a.q_sh +
                       (long)(pc.q0 + tok_q) * a.q_st;
        uint4 x[D / 8];
        float amax = 0.f;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          x[c] = *reinterpret_cast<const uint4*>(src + 8 * c);
          const T* e = reinterpret_cast<const T*>(&x[c]);
#pragma unroll
          for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(load_f(e + k)));
        }
        int e2 = (int)(__float_as_uint(amax) >> 23) - 127;
        e2 = e2 > 127 ? 0 : max(-100, min(100, e2));  // an infinite row keeps its values
        const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
        cq = __uint_as_float((uint32_t)(127 + e2) << 23) * a.scaling;
        unsigned char* dst = psm + L::q + w * L::tile + (r >> 3) * 1024 + (r & 7) * 128;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const T* e = reinterpret_cast<const T*>(&x[c]);
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = pack_f16(load_f(e + 2 * k) * down, load_f(e + 2 * k + 1) * down);
          *reinterpret_cast<uint4*>(dst + (c >> 3) * kPcBlock + 16 * ((c & 7) ^ (r & 7))) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        umma::fence_proxy_async_smem();
      }
      umma::mbar_arrive(qf);
      if (!active) {
        it += pc.n;
        continue;
      }
      // the row sees [lim_lo, lim_hi)
      const int last = pc.len - pc.q_len + tok_q;
      const int lim_hi = live ? min(pc.len, last + 1) : 0;
      const int lim_lo = !live ? 0 : rq.window > 0 ? max(pc.start, last - rq.window + 1) : pc.start;
      float m = -INFINITY, mv = -INFINITY, l = 0.f;
      for (int i = 0; i < pc.n; ++i) {
        const ChunkScales& sc = scales[(it + i) % L::ring];
        ok = wait(sf + w, tc & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++tc;
        umma::fence_after_sync();
        const int tok0 = (pc.tile + i) * kPcTok;
        const int e_lo = lim_lo - tok0, e_hi = lim_hi - tok0;  // visible columns
        int bad = 0;
#pragma unroll
        for (int g = 0; g < 8; ++g) bad |= sc.bad[g];
        const bool plain = __all_sync(0xffffffffu, e_lo <= 0 && e_hi >= kPcTok && !bad);
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) umma::tmem_ld32(t_s + 32 * c, s[c]);
        umma::tmem_wait_ld();
        if (!plain) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const int col = 32 * c + e;
              if (col < e_lo || col >= e_hi || sc.bad[col >> 4]) s[c][e] = 0xff800000u;  // -inf
            }
        }
        // ---- the tile's maxima of x and of x + log2(vs)
        float tm = -INFINITY, tv = -INFINITY;
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const uint32_t* v = s[g >> 1] + 16 * (g & 1);
          float bm = __uint_as_float(v[0]);
#pragma unroll
          for (int e = 1; e < 15; e += 2) bm = fmaxf(fmaxf(bm, __uint_as_float(v[e])), __uint_as_float(v[e + 1]));
          bm = fmaxf(bm, __uint_as_float(v[15]));
          const float x = bm * fmaxf(sc.ks[g] * cq, 0x1p-126f);  // above zero: a masked -inf stays
          tm = fmaxf(tm, x);
          tv = fmaxf(tv, x + sc.lv[g]);
        }
        const bool grew = tm > m + 8.f || tv > mv + 8.f;
        if (__any_sync(0xffffffffu, grew)) {
          const float nm = grew ? fmaxf(m, tm) : m, nv = grew ? fmaxf(mv, tv) : mv;
          if (m != -INFINITY) l *= exp2_fast(m - nm);
          const float f = mv == -INFINITY ? 1.f : exp2_fast(mv - nv);
          m = nm;
          mv = nv;
          if (i > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {  // few registers: S is held meanwhile
              float o[16];
              uint32_t u[16];
              umma::tmem_ld16(t_o + 16 * c, o);
              umma::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * f);
              umma::tmem_st16(t_o + 16 * c, u);
            }
            umma::tmem_wait_st();
          }
        }
        // ---- weights
        const float base = m == -INFINITY ? 0.f : -m;
        const float fr = mv == -INFINITY ? 0.f : exp2_fast(m - mv);
        uint64_t l2 = pack2(0.f, 0.f);
        const uint64_t base2 = pack2(base, base);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t p16[16];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float cg = fmaxf(sc.ks[2 * c + g] * cq, 0x1p-126f), wg = fminf(sc.vs[2 * c + g] * fr, 0x1p100f);
            const uint64_t c2 = pack2(cg, cg), w2 = pack2(wg, wg);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const uint64_t x2 = fma2(pack2(__uint_as_float(s[c][16 * g + e]), __uint_as_float(s[c][16 * g + e + 1])), c2, base2);
              float x0, x1;
              unpack2(x2, &x0, &x1);
              const uint64_t p2 = pack2(exp2_fast(x0), exp2_fast(x1));
              l2 = add2(l2, p2);
              float y0, y1;
              unpack2(mul2(p2, w2), &y0, &y1);
              p16[8 * g + e / 2] = pack_f16(y0, y1);
            }
          }
          umma::tmem_st16(t_s + 16 * c, p16);
        }
        float l0, l1;
        unpack2(l2, &l0, &l1);
        l += l0 + l1;
        umma::tmem_wait_st();
        umma::fence_before_sync();
        umma::mbar_arrive(pf + w);
      }
      it += pc.n;
      if (!ok) break;
      // ---- the row's result, or this CTA's record of it
      ok = wait(of + w, uc & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ++uc;
      umma::fence_after_sync();
      const bool whole = pc.whole;
      const float back = mv == -INFINITY ? 1.f : exp2_fast(mv - m);
      const float f = whole ? (l == 0.f ? 0.f : back / l) : back;
      const int row = 128 * w + r;
      float* rec = a.part.rec + ((long)blockIdx.x * 2 + (pc.begins ? 1 : 0)) * kPcRows * (D + 2);
      const long orow = ((rq.cu_q ? pc.q0 : (long)pc.b * rq.q_tokens) + tok_q) * a.out.Hq + head;
      T* dst = reinterpret_cast<T*>(a.out.out) + orow * D;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        umma::tmem_ld32(t_o + 32 * c, o);
        umma::tmem_wait_ld();
        if (live) {
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 v;
              T* t = reinterpret_cast<T*>(&v);
#pragma unroll
              for (int k = 0; k < 8; ++k) store_f(t + k, __uint_as_float(o[e + k]) * f);
              *reinterpret_cast<uint4*>(dst + 32 * c + e) = v;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(rec + row * D + 32 * c + e) =
                  make_float4(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f, __uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f);
          }
        }
      }
      umma::fence_before_sync();  // O is read: the next unit's products may follow (through qf)
      if (live) {
        if (whole) {
          if (a.out.lse) a.out.lse[orow] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
        } else {
          rec[kPcRows * D + row] = m;
          rec[kPcRows * D + kPcRows + row] = l;
        }
      }
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (warp == 0) umma::tmem_dealloc(tmem, 512);
}

}  // namespace kvd

namespace kvd_host {
using namespace kvd;

bool paged_chunk_takes(int head_dim, int dtype) { return (head_dim == 64 || head_dim == 128) && dtype != KVD_DTYPE_F32; }

size_t paged_chunk_ws_bytes(int head_dim) { return part_bytes(paged_sm_count(), kPcRows, head_dim); }

template <int D, int STORE, typename T>
static int launch_chunk(ChunkArgs& a, int fill_tail, void* ws, cudaStream_t s) {
  auto kern = paged_chunk_kernel<D, STORE, T>;
  if (int rc = ensure_smem((const void*)kern, ChunkSmem<D>::total, "paged_chunk_kernel")) return rc;
  const int ctas = paged_sm_count();
  a.part = part_at(ws, ctas);
  {
    KTimerScope kts_("paged_chunk_kernel", s);
    kern<<<ctas, kPcThreads, ChunkSmem<D>::total, s>>>(a);
  }
  if (int rc = check_launch("paged_chunk_kernel")) return rc;
  return launch_merge<D, kPcRows, T>(a.reqs, a.part, a.out, fill_tail, ctas, s);
}

template <int D, typename T>
static int launch_chunk_d(ChunkArgs& a, int store, int fill_tail, void* ws, cudaStream_t s) {
  return store == KVD_STORE_E4M3 ? launch_chunk<D, kStoreE4M3, T>(a, fill_tail, ws, s) : launch_chunk<D, kStoreInt8, T>(a, fill_tail, ws, s);
}

int launch_paged_chunk(const PagedPool& pool, int D, int store, const PagedReqs& reqs, const int* table, long table_stride,
                       int dtype, const void* q, long q_sb, long q_sh, long q_st, float scaling_log2, const PagedOut& out,
                       int fill_tail, void* ws, cudaStream_t s) {
  ChunkArgs a{pool, reqs, table, table_stride, q, q_sb, q_sh, q_st, scaling_log2, out, {}};
  if (dtype == KVD_DTYPE_BF16)
    return D == 64 ? launch_chunk_d<64, __nv_bfloat16>(a, store, fill_tail, ws, s) : launch_chunk_d<128, __nv_bfloat16>(a, store, fill_tail, ws, s);
  return D == 64 ? launch_chunk_d<64, __half>(a, store, fill_tail, ws, s) : launch_chunk_d<128, __half>(a, store, fill_tail, ws, s);
}

}  // namespace kvd_host
