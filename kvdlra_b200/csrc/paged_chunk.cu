// Attention over 8-bit pages for requests of many query rows (chunks of a
// prompt) on tcgen05 (sm_100a): bf16 and f16 queries, head_dim 64 and 128.
//
// One CTA of 20 warps per SM walks its run of the work list; a unit is
// (request, KV head, 256 query rows), a row (token, head of the group).  Per
// 128-token tile:
//   loaders (4 warps for keys, 4 for values)  the page's codes from global
//                      memory, a tile ahead in registers, converted exactly to
//                      f16 and written to shared memory as rows of 64 dims with
//                      the 128-byte swizzle: the same image is a K-major operand
//                      of the scores and an MN-major one of the values.
//   issuers (a warp for each row tile w of 128 rows)  S_w = Q_w K^T, and O_w +=
//                      P_w V with P_w in TMEM, by subtiles of 64 tokens.  S has two
//                      buffers per row tile: the next scores are there while this
//                      subtile's weights are computed.  P lies over S's columns, so
//                      the next scores wait for the product that reads it: products
//                      of different accumulators are in no order otherwise.  One
//                      issuer for both row tiles, waiting for each in turn, took
//                      1.40 ms where two take 1.25 (below); with one row tile, 96
//                      requests of 32 rows, head_dim 128, 196 us and 194 to 220.
//   softmax (2 x 4 warps)  a thread owns a row (a TMEM lane): the row's maxima
//                      and sums need no other thread.  S is read once, in one wait
//                      (TMEM reads are slow beside the tensor core); P_w (f16) goes
//                      over the columns of S_w.
//   planner (1 thread) the walk over the requests, handed on piece by piece.
// TMEM: S_0, S_1 (two buffers of 64 columns each), O_0, O_1 (head_dim each).
//
// Two references per row, in base 2: m for the sum l of the weights, and mv
// for O, whose weights carry the page's value scale: p vs = 2^(x - m) (vs 2^(m -
// mv)), so the f16 rounding of P is relative to the largest p vs.  They follow
// the running maxima only when these pass them by kLTop and kPTop: rescaling O,
// which lies in TMEM, is rare after the first tiles.
//
// Q is scaled per row by a power of two and rounded to f16 (exact but for
// elements 2^-13 of the row's largest); S, O, m, l are fp32; P is rounded to
// f16 (2^-11).
//
// Bound, per tile of 256 rows x 128 tokens at head_dim 128, in clocks: tensor
// core 2048, exponentials 2176 (8 a warp), shared memory 2500 (Q and K once per
// subtile, V, the converted tiles).  Measured: 4700, 1.25 ms and 850 TFLOP/s for
// 2048 queries of 32768 tokens with 32 heads over 8 (int8 pages, bf16).  S of 128
// tokens in one buffer (fewer reads of Q, the softmax waits for it) took as long;
// the exponentials' share, or the count of the softmax's instructions, made no
// difference.  Loaders of one warpgroup, and 16 softmax warps with half a row each,
// ran out of registers.
#include <atomic>
#include <climits>
#include <type_traits>

#include "paged.cuh"
#include "umma.cuh"

namespace kvd {

constexpr int kPcRows = 256, kPcTok = 128;  // rows of a unit, tokens of a tile
constexpr int kPcSub = 64;                  // tokens of a subtile: S has two buffers of them
constexpr int kPcThreads = 640;            // 8 softmax warps, 8 loaders, 2 issuers, planner (and 1 that waits)
// registers per thread of the five warpgroups: a softmax thread holds a subtile's
// row of S, a loader its share of a tile's codes; their sum is what the CTA is
// launched with (96 a thread)
constexpr int kPcRegsLaunch = 65536 / kPcThreads / 8 * 8;
constexpr int kPcRegsSoftmax = 128, kPcRegsLoad = 80, kPcRegsIssue = 64;
static_assert(2 * kPcRegsSoftmax + 2 * kPcRegsLoad + kPcRegsIssue <= 5 * kPcRegsLaunch, "register split");
constexpr int kPcLoad0 = 256, kPcIssue0 = 512, kPcPlan0 = 544, kPcIssue1 = 576;
constexpr int kPcBlock = kPcTok * 128;     // bytes of 64 columns of a 128-row f16 operand
// A wait gives up after a second's clocks and 70 us for each tile of the CTA's share
// (which the planner and an idle row tile may have to wait for whole; a tile takes 3
// to 4): time, counted in steps of 2^16 clocks.
constexpr int kPcClockShift = 16, kPcWaitBase = 1 << 15, kPcWaitTile = 2;
constexpr long kPcPolls = 1L << 20;  // of the last wait, for products that are on their way

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
  int wait_limit;  // steps of the clock, < 0: none at all, 0: by the work
};

struct alignas(16) ChunkScales {  // of one tile, per 16 tokens
  float ks[8], lv[8];  // keys' scale, log2 of the values'
  int bad;             // bit g: the g-th page id is out of range
  int pad[3];
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
constexpr int kPcPieces = 8;  // pieces planned ahead

template <int D>
struct ChunkSmem {
  static constexpr int NS = D == 64 ? 4 : 2;   // stages of keys, and of values
  static constexpr int tile = kPcTok * D * 2;  // f16 bytes of a 128-row operand
  static constexpr int q = 0, v = q + 2 * tile, k = v + NS * tile;
  static constexpr int total = k + NS * tile + 1024;  // room to align
  static constexpr int ring = NS == 2 ? 4 : 8;        // tiles whose scales are held: NS + 1 at least
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
KVD_DEVICE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

KVD_DEVICE float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
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
  __shared__ int wait_limit;     // steps of the clock
  __shared__ ChunkPiece pieces[kPcPieces];
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be warp-uniform
  const PagedPool& pool = a.pool;
  const PagedReqs& rq = a.reqs;
  __shared__ ChunkScales scales[L::ring];
  __shared__ uint64_t kf[NS], ke[NS], vf[NS], ve[NS];  // a stage of keys, of values: full, empty
  __shared__ uint64_t sf[2][2], pf[2][2];              // scores, weights of (row tile, S buffer)
  __shared__ uint64_t of[2], od[2], qf[2], drain[2];   // a subtile's product into O, a unit's last one; queries
  __shared__ uint64_t nf[kPcPieces], ne[kPcPieces];    // pieces
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 0) {
    umma::tmem_alloc(&tmem_base, 512);
    umma::tmem_relinquish();
  }
  if (tid == 0) {
    dead = 0;
    for (int i = 0; i < NS; ++i) {
      umma::mbar_init(kf + i, 128);
      umma::mbar_init(ke + i, 2);
      umma::mbar_init(vf + i, 128);
      umma::mbar_init(ve + i, 2);
    }
    for (int w = 0; w < 2; ++w) {
      for (int b = 0; b < 2; ++b) {
        umma::mbar_init(&sf[w][b], 1);
        umma::mbar_init(&pf[w][b], 128);
      }
      umma::mbar_init(of + w, 1);
      umma::mbar_init(od + w, 1);
      umma::mbar_init(qf + w, 128);
      umma::mbar_init(drain + w, 1);
    }
    for (int i = 0; i < kPcPieces; ++i) {
      umma::mbar_init(nf + i, 1);
      umma::mbar_init(ne + i, 256 + 256 + 2);
    }
    umma::mbar_fence_init();
  }
  umma::fence_before_sync();
  const WorkAt at = find_work<kPcRows, kPcTok, kPcThreads>(rq, blockIdx.x, gridDim.x);  // has barriers
  if (tid == 0) wait_limit = a.wait_limit ? (int)a.wait_limit : (int)min((long)INT_MAX, kPcWaitBase + kPcWaitTile * at.chunk);
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = tmem_base;
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (umma::mbar_try_wait(bar, parity)) return true;
    const uint32_t since = (uint32_t)(clock64() >> kPcClockShift);
    while (!dead && (int)((uint32_t)(clock64() >> kPcClockShift) - since) <= wait_limit) {
      for (int i = 0; i < 32; ++i)
        if (umma::mbar_try_wait(bar, parity)) return true;
    }
    if (dead) return false;
    dead = 1;
    pool.flag(kStatusTimeout, 1);
    return false;
  };

  if (warp >= kPcIssue0 / 32) {
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
    } else if (warp == kPcIssue0 / 32 || warp == kPcIssue1 / 32) {
      // ---------------------------------------------------------- issuers
      // The whole warp walks, one lane issues: descriptors stay in uniform registers.
      // A row tile that has no rows takes no part (its softmax threads may be units
      // ahead); its issuer then gives the stages back and nothing else.
      const int w = warp == kPcIssue0 / 32 ? 0 : 1;
      const uint64_t k_d = umma::smem_desc_sw128((uint32_t)__cvta_generic_to_shared(psm + L::k), 16, 1024);
      const uint32_t hi = (uint32_t)(k_d >> 32), k_lo = (uint32_t)k_d;
      const uint32_t q_w = k_lo - ((L::k - L::q) >> 4) + w * (L::tile >> 4);  // an address counts 16 bytes
      const uint32_t v_lo = (uint32_t)umma::smem_desc_sw128((uint32_t)__cvta_generic_to_shared(psm + L::v), kPcBlock, 1024);
      constexpr uint32_t id_s = umma::idesc_f16(128, kPcSub, false), id_o = umma::idesc_f16(128, D, true);
      // subtile b of a stage, S buffer b
      auto scores = [&](int stage, int b) {
        const uint32_t k_s = k_lo + stage * (L::tile >> 4) + b * (kPcSub * 128 >> 4);
        if (umma::elect_one()) {
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            const uint32_t at_j = ((j >> 2) * kPcBlock + 32 * (j & 3)) >> 4;
            umma::mma_f16_ss_lo(tmem + 128 * w + 64 * b, q_w + at_j, k_s + at_j, hi, id_s, j > 0);
          }
          umma::commit(&sf[w][b]);
        }
        __syncwarp();
      };
      auto values = [&](int stage, int b, bool acc) {
        const uint32_t v_s = v_lo + stage * (L::tile >> 4) + b * (kPcSub * 128 >> 4);
        if (umma::elect_one()) {
#pragma unroll
          for (int j = 0; j < kPcSub / 16; ++j)
            umma::mma_f16_ts_lo(tmem + 256 + D * w, tmem + 128 * w + 64 * b + 8 * j, v_s + ((2048 * j) >> 4), hi, id_o, acc || j > 0);
          umma::commit(&of[w]);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (umma::elect_one()) umma::commit(bar);
        __syncwarp();
      };
      auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(bar, parity)); };
      int it = 0, t = 0, uq = 0;  // tiles of all units and of this row tile's, units of it
      bool ok = true;
      for (int un = 0;; ++un) {
        const int sl = un % kPcPieces;
        ok = wait_all(nf + sl, (un / kPcPieces) & 1);
        if (!ok) break;
        const int n = __shfl_sync(0xffffffffu, pieces[sl].n, 0);
        const bool active = __shfl_sync(0xffffffffu, w == 0 || pieces[sl].rows - pieces[sl].row0 > 128, 0);
        if (lane == 0) umma::mbar_arrive(ne + sl);
        if (n == 0) break;
        if (!active) {
          for (int i = 0; i < n && ok; ++i) {
            const int g = it + i, st = g % NS;
            ok = wait_all(kf + st, (g / NS) & 1) && wait_all(vf + st, (g / NS) & 1);
            if (ok && lane == 0) {
              umma::mbar_arrive(ke + st);
              umma::mbar_arrive(ve + st);
            }
          }
          if (!ok) break;
          it += n;
          continue;
        }
        ok = wait_all(qf + w, uq++ & 1) && wait_all(kf + it % NS, (it / NS) & 1);
        if (!ok) break;
        umma::fence_after_sync();
        scores(it % NS, 0);
        scores(it % NS, 1);
        commit(ke + it % NS);
        for (int i = 0; i < n && ok; ++i) {
          const int g = it + i, st = g % NS, nx = (g + 1) % NS;
          const bool more = i + 1 < n;
          ok = wait_all(vf + st, (g / NS) & 1);
          for (int b = 0; b < 2 && ok; ++b) {
            // O += P V of this subtile, then S of the next tile's over its P.  The two
            // have accumulators of their own, so nothing but the wait for the first
            // keeps the second from P's columns while they are read.
            ok = wait_all(&pf[w][b], t & 1);
            if (!ok) break;
            umma::fence_after_sync();
            values(st, b, i > 0 || b > 0);
            if (b == 0 && more) {
              ok = wait_all(kf + nx, ((g + 1) / NS) & 1);
              if (!ok) break;
            }
            ok = wait_all(of + w, b);  // two products a tile: the parity is the subtile's
            if (!ok) break;
            umma::fence_after_sync();
            if (more) scores(nx, b);
          }
          if (!ok) break;
          ++t;
          commit(ve + st);
          if (more) commit(ke + nx);
        }
        if (!ok) break;
        commit(od + w);
        it += n;
      }
      if (!ok) {  // nothing may be in flight when TMEM is freed
        commit(drain + w);
        umma::mbar_wait_bounded(drain + w, 0, kPcPolls);
      }
    }
  } else if (warp >= kPcLoad0 / 32) {
    // ----------------------------------------------------------- loaders
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPcRegsLoad));
    // keys by the first warpgroup, values by the second
    const bool keys = warp < kPcLoad0 / 32 + 4;
    const int lw = (warp - kPcLoad0 / 32) & 3;
    const unsigned char* codes = keys ? pool.k : pool.v;
    unsigned char* stages = psm + (keys ? L::k : L::v);
    uint64_t *full = keys ? kf : vf, *empty = keys ? ke : ve;
    constexpr int QC = D / 64;  // 64-byte column blocks of a row
    // A lane's token of eight, and its 16 bytes of a 64-byte block.  At head_dim
    // 128 odd tokens take the blocks in the other order: the eight lanes of a
    // memory cycle then touch every bank once, in the load and in the store.
    const int tr = lane >> 2, cl = lane & 3;
    const int lg = pool.lg_page, mask = pool.page() - 1;
    // A tile is a piece's slot and a token; the piece stays in its slot until the
    // tile after it is current.  Three are under way: the current one (converted),
    // the next (codes and scales on their way) and the one after (page ids).
    struct Tile { int sl, tok0; };  // sl < 0: none
    Tile cur, nxt, aft = {0, 0};
    int left = 0, un = 0;
    bool ok = true;
    auto step = [&](Tile* t) {  // the tile after *t
      if (left > 0) {
        --left;
        t->tok0 += kPcTok;
        return;
      }
      if (t->sl < 0) return;
      const int sl = un % kPcPieces;
      ok = wait(nf + sl, (un / kPcPieces) & 1);
      ok = __all_sync(0xffffffffu, ok);
      const int n = ok ? pieces[sl].n : 0;
      if (n == 0) {
        t->sl = -1;
        return;
      }
      left = n - 1;
      t->sl = sl;
      t->tok0 = pieces[sl].tile * kPcTok;
      ++un;
    };
    // lane l (mod 8) knows the page of the tile's l-th 16 tokens: -1 outside [lo, hi), -2 a bad id
    auto page_id = [&](const Tile& t) -> int {
      if (t.sl < 0) return -1;
      const ChunkPiece& p = pieces[t.sl];
      const int tok = t.tok0 + 16 * (lane & 7);
      if (tok >= p.hi || tok + 16 <= p.lo) return -1;
      const int id = a.table[(long)p.b * a.table_stride + (tok >> lg)];
      return id < 0 || id >= pool.num_pages ? -2 : id;
    };
    uint4 raw[4][QC];  // tokens 8 (4k + lw) + tr, block c
    // Converts what is there to `dst` (unless null) and starts the loads of tile
    // t, a quarter at a time: a load then has the rest of this tile's conversion
    // and the wait for a stage to arrive in.
    auto turn = [&](unsigned char* dst, const Tile& t, int ids) {
      const int sl = max(0, t.sl), lo = pieces[sl].lo, hi = t.sl < 0 ? 0 : pieces[sl].hi;
      const unsigned char* base = codes + (long)pieces[sl].h * pool.head_stride + 16 * cl;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int tg = 4 * k + lw, tok = t.tok0 + 8 * tg + tr;
        if (dst) {
#pragma unroll
          for (int c = 0; c < QC; ++c) {
            const uint32_t w[4] = {raw[k][c].x, raw[k][c].y, raw[k][c].z, raw[k][c].w};
            uint32_t o[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) codes_to_f16<STORE>(w[e], &o[2 * e], &o[2 * e + 1]);
            unsigned char* p = dst + (c ^ (QC - 1 & tr)) * kPcBlock + tg * 1024 + tr * 128;
            *reinterpret_cast<uint4*>(p + 16 * ((2 * cl) ^ tr)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(p + 16 * ((2 * cl + 1) ^ tr)) = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
        const int id = __shfl_sync(0xffffffffu, ids, tg >> 1);
        const bool live = id >= 0 && tok >= lo && tok < hi;
        const unsigned char* p = base + (long)id * pool.page_stride + (long)(tok & mask) * pool.slot_stride;
#pragma unroll
        for (int c = 0; c < QC; ++c) {
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (live) asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p + 64 * (c ^ (QC - 1 & tr))));
          raw[k][c] = x;
        }
      }
    };
    float ks = 0.f, vs = 0.f, ks_n = 0.f, vs_n = 0.f;
    auto scale = [&](const Tile& t, int ids, float* k, float* v) {
      *k = *v = 0.f;
      if (keys && lw == 0 && lane < 8 && ids >= 0) {
        const long at_s = (long)ids * pool.scale_stride + pieces[t.sl].h;
        *k = pool.ks[at_s];
        *v = pool.vs[at_s];
      }
    };
    step(&aft);
    cur = aft;
    int ids = page_id(cur);
    step(&aft);
    nxt = aft;
    int ids_n = page_id(nxt);
    turn(nullptr, cur, ids);
    scale(cur, ids, &ks, &vs);
    for (int it = 0; cur.sl >= 0 && ok; ++it) {
      step(&aft);
      if (!ok) break;
      const int ids_a = page_id(aft);
      scale(nxt, ids_n, &ks_n, &vs_n);
      const int st = it % NS;
      ok = wait(empty + st, ((it / NS) & 1) ^ 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      turn(stages + st * L::tile, nxt, ids_n);
      if (keys && lw == 0 && lane < 8) {
        ChunkScales& s = scales[it % L::ring];
        s.ks[lane] = ks;
        s.lv[lane] = log2f(vs);
        const uint32_t bad = __ballot_sync(0xffu, ids == -2);
        if (lane == 0) s.bad = (int)bad;
        if (ids == -2) pool.flag(kStatusBounds, kPagedBadPage);
      }
      umma::fence_proxy_async_smem();
      umma::mbar_arrive(full + st);
      if (nxt.sl != cur.sl) umma::mbar_arrive(ne + cur.sl);
      cur = nxt;
      nxt = aft;
      ids = ids_n;
      ids_n = ids_a;
      ks = ks_n;
      vs = vs_n;
    }
  } else {
    // ----------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPcRegsSoftmax));
    const int w = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t t_s = tmem + 128 * w + lanes, t_o = tmem + 256 + D * w + lanes;
    int it = 0, tc = 0, uc = 0;  // tiles of all units and of this row tile, units of it
    bool ok = true;
    for (int un = 0;; ++un) {
      const int sl = un % kPcPieces;
      ok = wait(nf + sl, (un / kPcPieces) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const ChunkPiece& pc = pieces[sl];  // stays until this thread has written the result
      const int n = pc.n;
      if (n == 0) break;
      const bool active = w == 0 || pc.rows - pc.row0 > 128;
      float cq = 0.f;
      int lim_lo = 0, lim_hi = 0;  // the row sees [lim_lo, lim_hi)
      if (active) {
        const int R = min(pc.rows - 1, pc.row0 + 128 * w + r), tok_q = R / rq.G, head = pc.h * rq.G + R % rq.G;
        if (pc.row0 + 128 * w + r < pc.rows) {
          const int last = pc.len - pc.q_len + tok_q;
          lim_hi = min(pc.len, last + 1);
          lim_lo = rq.window > 0 ? max(pc.start, last - rq.window + 1) : pc.start;
        }
        // ---- this thread's query row, scaled by a power of two, as f16
        const T* src = reinterpret_cast<const T*>(a.q) + (rq.cu_q ? 0 : (long)pc.b * a.q_sb) + (long)head * a.q_sh +
                       (long)(pc.q0 + tok_q) * a.q_st;
        float amax = 0.f;
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          const uint4 x = *reinterpret_cast<const uint4*>(src + 8 * c);
          const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
          for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(load_f(e + k)));
        }
        int e2 = (int)(__float_as_uint(amax) >> 23) - 127;
        e2 = e2 > 127 ? 0 : max(-100, min(126, e2));  // an infinite row keeps its values
        const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
        cq = __uint_as_float((uint32_t)(127 + e2) << 23) * a.scaling;
        unsigned char* dst = psm + L::q + w * L::tile + (r >> 3) * 1024 + (r & 7) * 128;
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          const uint4 x = *reinterpret_cast<const uint4*>(src + 8 * c);
          const T* e = reinterpret_cast<const T*>(&x);
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = pack_f16(load_f(e + 2 * k) * down, load_f(e + 2 * k + 1) * down);
          *reinterpret_cast<uint4*>(dst + (c >> 3) * kPcBlock + 16 * ((c & 7) ^ (r & 7))) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        umma::fence_proxy_async_smem();
        umma::mbar_arrive(qf + w);
      } else {
        umma::mbar_arrive(ne + sl);
        it += n;
        continue;
      }
      float m = -INFINITY, mv = -INFINITY, l = 0.f;
      for (int u = 0; u < 2 * n; ++u) {  // subtiles
        const ChunkScales& sc = scales[(it + (u >> 1)) % L::ring];
        const int b = u & 1, g0 = 4 * b;
        ok = wait(&sf[w][b], (tc + (u >> 1)) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        umma::fence_after_sync();
        const uint32_t t_b = t_s + 64 * b;
        const int tok0 = pc.tile * kPcTok + u * kPcSub;
        const int e_lo = lim_lo - tok0, e_hi = lim_hi - tok0;  // visible columns
        const int bad = sc.bad >> g0;
        const bool plain = __all_sync(0xffffffffu, e_lo <= 0 && e_hi >= kPcSub && !(bad & 15));
        // twice in the code, so that the usual subtile has no trace of the masks
        auto subtile = [&](auto masked) {
          // ---- the subtile's maxima of x and of x + log2(vs)
          uint32_t s[2][32];
          umma::tmem_ld32(t_b, s[0]);
          umma::tmem_ld32(t_b + 32, s[1]);
          // meanwhile the scales of the subtile's four 16 tokens
          const float4 ks4 = *reinterpret_cast<const float4*>(sc.ks + g0), lv4 = *reinterpret_cast<const float4*>(sc.lv + g0);
          // above zero: a masked -inf stays one
          const float cg[4] = {fmaxf(ks4.x * cq, 0x1p-126f), fmaxf(ks4.y * cq, 0x1p-126f), fmaxf(ks4.z * cq, 0x1p-126f), fmaxf(ks4.w * cq, 0x1p-126f)};
          const float lv[4] = {lv4.x, lv4.y, lv4.z, lv4.w};
          umma::tmem_wait_ld32(s[0]);
          umma::tmem_loaded32(s[1]);
          if constexpr (decltype(masked)::value) {
#pragma unroll
            for (int e = 0; e < kPcSub; ++e)
              if (e < e_lo || e >= e_hi || (bad >> (e >> 4) & 1)) s[e >> 5][e & 31] = 0xff800000u;  // -inf
          }
          float tm = -INFINITY, tv = -INFINITY;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t* v = s[g >> 1] + 16 * (g & 1);
            float b0 = __uint_as_float(v[0]), b1 = __uint_as_float(v[1]);
#pragma unroll
            for (int e = 2; e < 14; e += 4) {
              b0 = max3(b0, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
              b1 = max3(b1, __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
            }
            b0 = max3(b0, __uint_as_float(v[14]), __uint_as_float(v[15]));
            const float x = fmaxf(b0, b1) * cg[g];
            tm = fmaxf(tm, x);
            tv = fmaxf(tv, x + lv[g]);
          }
          const bool grew = tm > m + kLTop || tv > mv + kPTop;
          if (__any_sync(0xffffffffu, grew)) {
            const float nm = grew ? fmaxf(m, tm) : m, nv = grew ? fmaxf(mv, tv - kPBias) : mv;
            if (m != -INFINITY) l *= exp2_fast(m - nm);
            const float f = mv == -INFINITY ? 1.f : exp2_fast(mv - nv);
            m = nm;
            mv = nv;
            if (u > 0) {
              // The product before may still be under way.  The one before that is done
            // (S of this subtile came after it) and the next waits for this thread, so
            // the phase's parity says which it is.
            ok = wait(&of[w], (u - 1) & 1);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) return;
              umma::fence_after_sync();
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                umma::tmem_ld32(t_o + 32 * c, o);
                umma::tmem_wait_ld32(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                umma::tmem_st32(t_o + 32 * c, o);
              }
              umma::tmem_wait_st();
            }
          }
          // ---- weights: p vs 2^(m - mv) = 2^(x - m + d), d = log2(vs) + m - mv; their sum
          // over a page's tokens, times 2^-d, goes to l.  d ends at -40: x - m is 14 at
          // most, so P is 2^-26 or less there, 0 in f16, while l's share keeps weights
          // down to 2^-86
          const float base = m == -INFINITY ? 0.f : -m;
          const float dm = mv == -INFINITY ? 0.f : m - mv;
          uint32_t p16[32];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float d = fmaxf(lv[g] + dm, -40.f), bg = base + d;
            const uint64_t c2 = pack2(cg[g], cg[g]), b2 = pack2(bg, bg);
            uint64_t l2 = pack2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float x0, x1;
              const uint32_t* v = s[g >> 1] + 16 * (g & 1) + e;
              unpack2(fma2(pack2(__uint_as_float(v[0]), __uint_as_float(v[1])), c2, b2), &x0, &x1);
              x0 = exp2_fast(x0);
              x1 = exp2_fast(x1);
              l2 = add2(l2, pack2(x0, x1));
              p16[8 * g + e / 2] = pack_f16(x0, x1);
            }
            float l0, l1;
            unpack2(l2, &l0, &l1);
            l = fmaf(l0 + l1, exp2_fast(-d), l);
          }
          umma::tmem_st32(t_b, p16);  // one store: the exponentials of all 64 may overlap
          umma::tmem_wait_st();
          umma::fence_before_sync();
          umma::mbar_arrive(&pf[w][b]);
        };
        if (plain) subtile(std::false_type());
        else subtile(std::true_type());
        if (!ok) break;
      }
      it += n;
      tc += n;
      if (!ok) break;
      // ---- the row's result, or this CTA's record of it
      ok = wait(&od[w], uc & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ++uc;
      umma::fence_after_sync();
      const int R = pc.row0 + 128 * w + r, tok_q = R / rq.G, head = pc.h * rq.G + R % rq.G;
      const bool whole = pc.whole, live = R < pc.rows;
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
        umma::tmem_wait_ld32(o);
        if (live) {
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 v;
              T* t = reinterpret_cast<T*>(&v);
#pragma unroll
              for (int k = 0; k < 8; ++k) store_held(t + k, __uint_as_float(o[e + k]) * f);
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
      umma::mbar_arrive(ne + sl);
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

static std::atomic<int> paged_wait_limit{0};

bool paged_chunk_takes(int head_dim, int dtype) { return (head_dim == 64 || head_dim == 128) && dtype != KVD_DTYPE_F32; }

size_t paged_chunk_ws_bytes(int head_dim) { return part_bytes(paged_sm_count(), kPcRows, head_dim); }

template <int D, int STORE, typename T>
static int launch_chunk(ChunkArgs& a, int fill_tail, void* ws, cudaStream_t s) {
  auto kern = paged_chunk_kernel<D, STORE, T>;
  if (int rc = ensure_smem((const void*)kern, ChunkSmem<D>::total, "paged_chunk_kernel")) return rc;
  // The warpgroups' shares draw on what the CTA is launched with: fewer registers,
  // from another compiler, and they would wait for good.
  static int regs = 0;
  if (!regs) {
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, (const void*)kern) != cudaSuccess) { set_error("paged_chunk_kernel: no attributes"); return KVD_ERR_CUDA; }
    regs = attr.numRegs;
  }
  if (regs != kPcRegsLaunch) { set_error("paged_chunk_kernel was built with %d registers, not %d", regs, kPcRegsLaunch); return KVD_ERR_CUDA; }
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
  ChunkArgs a{pool, reqs, table, table_stride, q, q_sb, q_sh, q_st, scaling_log2, out, {}, paged_wait_limit.load()};
  if (dtype == KVD_DTYPE_BF16)
    return D == 64 ? launch_chunk_d<64, __nv_bfloat16>(a, store, fill_tail, ws, s) : launch_chunk_d<128, __nv_bfloat16>(a, store, fill_tail, ws, s);
  return D == 64 ? launch_chunk_d<64, __half>(a, store, fill_tail, ws, s) : launch_chunk_d<128, __half>(a, store, fill_tail, ws, s);
}

}  // namespace kvd_host

extern "C" int kvd_paged_wait_limit(int64_t clocks) {
  const int64_t steps = clocks >> kvd::kPcClockShift;
  kvd_host::paged_wait_limit = clocks < 0 ? -1 : clocks == 0 ? 0 : (int)std::max<int64_t>(1, std::min<int64_t>(INT_MAX, steps));
  return KVD_OK;
}
