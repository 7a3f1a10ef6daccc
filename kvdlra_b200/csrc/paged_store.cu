// Writing tokens into the 8-bit paged KV cache, and reading them back dense
// (sm_100a).
#include <algorithm>

#include "paged.cuh"

namespace kvd {

// ------------------------------------------------------------------ append
//
// Row i of the call goes to slots[i].  Rows that follow one another into
// consecutive slots of one page are a run, a page's only one in the call; a run's
// page gets, per KV head, the scale
//   s = code_scale(max |x| over the run), if the run begins at the page's first slot
//   s = max(that, the page's scale), otherwise; where the scale grew, the
//       codes of the slots before the run are rounded again to the new one
// and the run's codes x / s.  Infinities take the largest code and are left
// out of the maximum, NaN is stored as 0; both set the numeric status bit, so
// a cache holds finite values only.
//
// A group of W warps takes a (run, head, keys or values) item: the run's rows
// are read once, 16 bytes a load, and stay in registers between the maximum
// and the codes (W = page * D / 2048 warps hold a whole page, 8 or 16 loads of 16
// bytes a lane: 32 or 64 registers).  A prompt's floor is HBM's (2 or 4 bytes read
// and one written per value); four prompts of 8191 tokens, 8 heads of 128, take 60
// us in f16 and 95 in bf16 where that is 31, 93 in fp32 where it is 51: a CTA's reads
// wait in turn for its slots, and the 16-bit forms spill.  32 single tokens are
// latency, 3.6 us (times of calls in a row, without the host).
struct AppendArgs {
  PagedPool pool;
  const int* slots;
  long rows;           // batch * tokens
  int tokens;          // rows per batch entry
  const void* x[2];    // keys, values
  long sb[2], sh[2], st[2];  // strides of batch, head, token (elements)
  int per_cta;         // consecutive rows whose runs one CTA takes
  int most;            // rows of the longest run; 0: not known
  int head_groups;     // CTAs that share the heads
};

constexpr int kMaxPage = 128;

template <int D, int W, int STORE, typename T>
__global__ void __launch_bounds__(W < 4 ? 128 : 32 * W, (sizeof(T) == 2 ? 1024 : 512) / (W < 4 ? 128 : 32 * W))
    paged_append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int NTHR = W < 4 ? 128 : 32 * W;      // threads of the CTA
  constexpr int GT = 32 * W, GROUPS = NTHR / GT;  // threads of a group, groups (heads) of the CTA
  constexpr int VE = 16 / (int)sizeof(T);         // elements per load
  constexpr int CPR = D / VE;                     // loads per row
  constexpr int PER = (2048 * (int)sizeof(T)) / 512;  // loads per thread of a whole page: 8 or 16
  __shared__ int slot_sm[2 * kMaxPage + 1];
  __shared__ uint32_t brk[2 * kMaxPage / 32];     // row i does not continue row i - 1's run
  __shared__ float red[2][NTHR / 32];             // of every other reduction, so that one barrier does for each
  const PagedPool& pool = a.pool;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = tid / GT, gt = tid % GT;
  // neighbouring CTAs take neighbouring heads of the same rows, which lie together
  const int h = (int)(blockIdx.x % a.head_groups) * GROUPS + group, kv = blockIdx.y;
  const bool live_head = h < pool.H;
  const int lg = pool.lg_page, mask = pool.page() - 1;
  const long r0 = (long)(blockIdx.x / a.head_groups) * a.per_cta;
  const int span = a.per_cta + pool.page();       // a run of this CTA ends within it
  const int limit = pool.num_pages << lg;
  for (int i = tid; i <= span; i += NTHR) {
    const long r = r0 + i - 1;
    int s = r >= 0 && r < a.rows ? a.slots[r] : -1;
    if (s >= limit) {
      if (i > 0 && i <= a.per_cta) pool.flag(kStatusBounds, kPagedBadSlot);
      s = -1;
    }
    slot_sm[i] = s < 0 ? -1 : s;
  }
  __syncthreads();
  for (int i = tid; i < (span + 31) / 32 * 32; i += NTHR) {
    bool b = true;
    if (i < span) {
      const int s = slot_sm[i + 1], p = slot_sm[i];
      b = s < 0 || p < 0 || s != p + 1 || (s & mask) == 0;
    }
    const uint32_t w = __ballot_sync(0xffffffffu, b);
    if (lane == 0) brk[i >> 5] = w;
  }
  __syncthreads();
  unsigned char* codes = kv ? pool.v : pool.k;
  float* scales = kv ? pool.vs : pool.ks;
  int turn = 0;
  for (int i0 = 0; i0 < a.per_cta; ) {
    // the next run that begins at or after row i0 (and its end)
    int i = i0;
    while (i < a.per_cta) {
      const uint32_t w = brk[i >> 5] >> (i & 31);
      if (w) { i += __ffs(w) - 1; break; }
      i = (i | 31) + 1;
    }
    if (i >= a.per_cta) break;
    i0 = i + 1;
    const int slot = slot_sm[i + 1], prev = slot_sm[i];
    if (slot < 0) continue;
    if (prev >= 0 && (prev >> lg) == (slot >> lg)) {  // its page's run has ended: it would race with this one
      if (tid == 0) pool.flag(kStatusBounds, kPagedBadSlot);
      continue;
    }
    int n = 1;
    while (i + n < span) {
      const int k = i + n;
      const uint32_t w = brk[k >> 5] >> (k & 31);
      if (w) { n += __ffs(w) - 1; break; }
      n = (k | 31) + 1 - i;
    }
    n = min(n, (mask + 1) - (slot & mask));
    const int page = slot >> lg, o = slot & mask;
    unsigned char* base = codes + (long)page * pool.page_stride + (long)h * pool.head_stride;
    float* sp = scales + (long)page * pool.scale_stride + h;
    const float was = live_head && o > 0 ? *sp : 0.f;  // read before the barriers that stand before its write
    // ---- the run's rows, and their largest finite magnitude
    uint4 x[PER];
    const int b0 = (int)(r0 + i) / a.tokens, t0 = (int)(r0 + i) - b0 * a.tokens;  // one division a run
    float amax = 0.f, odd = 0.f;  // odd: 0, or NaN once a value is not finite
#pragma unroll
    for (int c = 0; c < PER; ++c) {
      const int e = gt + c * GT, row = e / CPR;
      x[c] = make_uint4(0u, 0u, 0u, 0u);
      if (live_head && row < n) {
        int bt = b0, t = t0 + row;
        while (t >= a.tokens) { t -= a.tokens; ++bt; }
        const T* src = reinterpret_cast<const T*>(a.x[kv]) + (long)bt * a.sb[kv] + (long)h * a.sh[kv] + (long)t * a.st[kv];
        x[c] = *reinterpret_cast<const uint4*>(src + (e % CPR) * VE);
      }
    }
#pragma unroll
    for (int c = 0; c < PER; ++c) {
      const T* v = reinterpret_cast<const T*>(&x[c]);
#pragma unroll
      for (int q = 0; q < VE; ++q) {
        const float f = load_f(v + q);
        amax = fmaxf(amax, fabsf(f));
        odd = fmaf(f, 0.f, odd);
      }
    }
    auto group_max = [&](float v) {
      v = warp_max(v);
      if constexpr (W > 1) {
        turn ^= 1;
        if (lane == 0) red[turn][warp] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) v = fmaxf(v, red[turn][group * W + w]);
      }
      return v;
    };
    // one number tells both: +inf where a value is not finite
    amax = group_max(odd == 0.f ? amax : INFINITY);
    bool again = amax == INFINITY;
    if constexpr (W > 1 && GROUPS > 1) again = __syncthreads_or(again);  // the groups of a CTA meet at the barriers
    if (again) {
      float fin = 0.f;
#pragma unroll
      for (int c = 0; c < PER; ++c) {
        const T* v = reinterpret_cast<const T*>(&x[c]);
#pragma unroll
        for (int q = 0; q < VE; ++q) {
          const float f = fabsf(load_f(v + q));
          if (f < INFINITY) fin = fmaxf(fin, f);
        }
      }
      if (amax == INFINITY && gt == 0) pool.flag(kStatusNumeric, kPagedNonFinite);
      amax = group_max(fin);
    }
    float s = code_scale<STORE>(amax);
    const bool grew = o > 0 && s > was;
    s = o > 0 ? fmaxf(s, was) : s;
    if (!live_head) continue;
    __syncwarp();
    if (gt == 0 && (o == 0 || grew)) *sp = s;
    if (grew) {
      const float ratio = was / s;
      for (int e = gt; e < o * (D / 16); e += GT) {
        uint4* p = reinterpret_cast<uint4*>(base + (long)(e / (D / 16)) * pool.slot_stride + 16 * (e % (D / 16)));
        uint4 w = *p;
        uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float f[4];
          codes_to_f32<STORE>(u[q], f);
          u[q] = f32_to_codes<STORE>(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
        }
        *p = w;
      }
    }
    const float inv = 1.f / s;  // a power of two: exact
#pragma unroll
    for (int c = 0; c < PER; ++c) {
      const int e = gt + c * GT, row = e / CPR;
      if (row >= n) break;
      const T* v = reinterpret_cast<const T*>(&x[c]);
      float f[VE];
#pragma unroll
      for (int q = 0; q < VE; ++q) {
        f[q] = load_f(v + q);
        f[q] = f[q] == f[q] ? f[q] * inv : 0.f;
      }
      unsigned char* dst = base + (long)(o + row) * pool.slot_stride + (e % CPR) * VE;
      if constexpr (VE == 8) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(f32_to_codes<STORE>(f[0], f[1], f[2], f[3]), f32_to_codes<STORE>(f[4], f[5], f[6], f[7]));
      } else {
        *reinterpret_cast<uint32_t*>(dst) = f32_to_codes<STORE>(f[0], f[1], f[2], f[3]);
      }
    }
  }
}

// -------------------------------------------------------------------- peek
//
// Dense keys and values of requests, (B, H, T, D) in the model's type: row t
// is code * scale, held to the type's range, zero from the request's length on.  One 16-byte store per
// thread and step, neighbouring threads on neighbouring bytes.  HBM bounds it:
// one byte read and 2 or 4 written per value (four prompts of 8191 tokens, 8 heads
// of 128, to f16: 33 us, 6.1 TB/s; to fp32: 55 us where the bytes take 51).
struct PeekArgs {
  PagedPool pool;
  const int* table;
  long table_stride;
  const int* lens;
  int max_len, tokens;
  void* out[2];
  long sb[2], sh[2], st[2];
};

template <int D, int STORE, typename T>
__global__ void __launch_bounds__(256) paged_peek_kernel(const __grid_constant__ PeekArgs a) {
  constexpr int VE = 16 / (int)sizeof(T), CPR = D / VE, STEPS = 4;
  const PagedPool& pool = a.pool;
  const int h = blockIdx.y, b = blockIdx.z >> 1, kv = blockIdx.z & 1;
  const int len = max(0, min(a.lens[b], a.max_len));
  const unsigned char* codes = (kv ? pool.v : pool.k) + (long)h * pool.head_stride;
  const float* scales = (kv ? pool.vs : pool.ks) + h;
  T* out = reinterpret_cast<T*>(a.out[kv]) + (long)b * a.sb[kv] + (long)h * a.sh[kv];
  const long e0 = (long)blockIdx.x * (256 * STEPS) + threadIdx.x;
  uint32_t w[STEPS][VE / 4];
  float sc[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const long e = e0 + 256 * i;
    const int t = (int)(e / CPR), c = (int)(e % CPR) * VE;
#pragma unroll
    for (int q = 0; q < VE / 4; ++q) w[i][q] = 0u;
    sc[i] = 0.f;
    if (t < len && t < a.tokens) {
      const int id = a.table[(long)b * a.table_stride + (t >> pool.lg_page)];
      if (id < 0 || id >= pool.num_pages) {
        pool.flag(kStatusBounds, kPagedBadPage);
      } else {
        sc[i] = scales[(long)id * pool.scale_stride];
        const unsigned char* p = codes + (long)id * pool.page_stride + (long)(t & (pool.page() - 1)) * pool.slot_stride + c;
        if constexpr (VE == 8) {
          const uint2 u = *reinterpret_cast<const uint2*>(p);
          w[i][0] = u.x; w[i][1] = u.y;
        } else {
          w[i][0] = *reinterpret_cast<const uint32_t*>(p);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const long e = e0 + 256 * i;
    const int t = (int)(e / CPR), c = (int)(e % CPR) * VE;
    if (t >= a.tokens) return;
    uint4 r;
    T* v = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int q = 0; q < VE / 4; ++q) {
      float f[4];
      codes_to_f32<STORE>(w[i][q], f);
#pragma unroll
      for (int k = 0; k < 4; ++k) store_held(v + 4 * q + k, f[k] * sc[i]);
    }
    *reinterpret_cast<uint4*>(out + (long)t * a.st[kv] + c) = r;
  }
}

}  // namespace kvd

namespace kvd_host {
using namespace kvd;

static bool view_ok(const kvd_hf_view& v, int size) {
  return v.ptr && (((uintptr_t)v.ptr | (uintptr_t)(v.stride_b * size) | (uintptr_t)(v.stride_h * size) | (uintptr_t)(v.stride_t * size)) % 16) == 0;
}

template <int D, int STORE, typename T>
static int launch_append(AppendArgs& a, cudaStream_t s) {
  const int page = 1 << a.pool.lg_page;
  const int W = std::max(1, page * D / 2048);
  const int groups = W < 4 ? 4 / W : 1;
  const int hy = (a.pool.H + groups - 1) / groups;
  // A page's worth of rows per CTA where runs are long: a CTA in which no run
  // begins is only a start (four prompts of 8191 tokens, pages of 128, 8 heads of
  // 128: 95 us; 151 at 16 rows per CTA).  Short runs are taken one after another, so
  // about two of the longest a CTA: 512 single tokens, the same pages: 74 us, 141 at
  // 64 rows; pages of 64: 36 and 121; pages of 16, 8 heads of 64: 12.6 and 28 at 16.
  // 512 runs of 5 (16 rows a CTA): 80 us, 117 at 64, 98 at two.  Fewer while the grid
  // would leave most SMs idle: 32 single tokens of 8 heads of 64 take 3.5 us at one row
  // per CTA, 5.1 at two, 28 at sixteen.
  a.per_cta = page;
  while (a.most > 0 && a.per_cta > 1 && a.per_cta / 2 >= 2L * a.most) a.per_cta >>= 1;
  while (a.per_cta > 1 && (a.rows + a.per_cta - 1) / a.per_cta * hy * 2 < paged_sm_count() / 2) a.per_cta >>= 1;
  a.head_groups = hy;
  const long ctas = (a.rows + a.per_cta - 1) / a.per_cta * hy;
  if (ctas > INT32_MAX) { set_error("paged append: %ld rows of %d heads", a.rows, a.pool.H); return KVD_ERR_ARG; }
  const dim3 grid((unsigned)ctas, 2);
  KTimerScope kts_("paged_append_kernel", s);
#define KVD_APPEND(w) \
  case w: paged_append_kernel<D, w, STORE, T><<<grid, w < 4 ? 128 : 32 * w, 0, s>>>(a); break;
  switch (W) {
    KVD_APPEND(1) KVD_APPEND(2) KVD_APPEND(4) KVD_APPEND(8)
    default: paged_append_kernel<D, 16, STORE, T><<<grid, 512, 0, s>>>(a);
  }
#undef KVD_APPEND
  return check_launch("paged_append_kernel");
}

template <int D, int STORE, typename T>
static int launch_peek8(const PeekArgs& a, int batch, cudaStream_t s) {
  constexpr int VE = 16 / (int)sizeof(T);
  const long per = (long)a.tokens * (D / VE);
  const dim3 grid((unsigned)((per + 1023) / 1024), a.pool.H, 2 * batch);
  KTimerScope kts_("paged_peek_kernel", s);
  paged_peek_kernel<D, STORE, T><<<grid, 256, 0, s>>>(a);
  return check_launch("paged_peek_kernel");
}

template <int STORE, typename T, typename A, typename F>
static int by_dim(int D, A& a, F f) {
  switch (D) {
    case 32: return f.template operator()<32, STORE, T>(a);
    case 64: return f.template operator()<64, STORE, T>(a);
    case 128: return f.template operator()<128, STORE, T>(a);
    default: return f.template operator()<256, STORE, T>(a);
  }
}
template <typename A, typename F>
static int by_shape(int D, int store, int dtype, A& a, F f) {
  const bool e4 = store == KVD_STORE_E4M3;
  if (dtype == KVD_DTYPE_F32) return e4 ? by_dim<kStoreE4M3, float>(D, a, f) : by_dim<kStoreInt8, float>(D, a, f);
  if (dtype == KVD_DTYPE_BF16) return e4 ? by_dim<kStoreE4M3, __nv_bfloat16>(D, a, f) : by_dim<kStoreInt8, __nv_bfloat16>(D, a, f);
  if (dtype == KVD_DTYPE_F16) return e4 ? by_dim<kStoreE4M3, __half>(D, a, f) : by_dim<kStoreInt8, __half>(D, a, f);
  set_error("paged cache: unsupported dtype %d", dtype);
  return KVD_ERR_DTYPE;
}
struct DoAppend {
  cudaStream_t s;
  template <int D, int STORE, typename T> int operator()(AppendArgs& a) const { return launch_append<D, STORE, T>(a, s); }
};
struct DoPeek {
  int batch;
  cudaStream_t s;
  template <int D, int STORE, typename T> int operator()(PeekArgs& a) const { return launch_peek8<D, STORE, T>(a, batch, s); }
};

}  // namespace kvd_host

using namespace kvd_host;

extern "C" int kvd_paged_append(const kvd_paged_pool* pool, const int32_t* slots, int32_t batch, int32_t dtype,
                                kvd_hf_view k, kvd_hf_view v, kvd_stream_t stream) {
  return kvd_paged_append_runs(pool, slots, batch, dtype, k, v, batch > 1 ? std::max(0, k.tokens) : 0, stream);
}

extern "C" int kvd_paged_append_runs(const kvd_paged_pool* pool, const int32_t* slots, int32_t batch, int32_t dtype,
                                     kvd_hf_view k, kvd_hf_view v, int32_t max_new, kvd_stream_t stream) try {
  kvd::AppendArgs a;
  if (int rc = paged_pool_view(pool, &a.pool)) return rc;
  if (batch < 0 || max_new < 0 || k.tokens < 0 || k.tokens != v.tokens) { set_error("paged append: keys of %d tokens, values of %d, batch %d", k.tokens, v.tokens, batch); return KVD_ERR_ARG; }
  if (batch == 0 || k.tokens == 0) return KVD_OK;
  const int size = dtype == KVD_DTYPE_F32 ? 4 : 2;
  if (!slots || !view_ok(k, size) || !view_ok(v, size)) { set_error("paged append: keys, values and their strides must be multiples of 16 bytes"); return KVD_ERR_ARG; }
  a.slots = slots;
  a.tokens = k.tokens;
  a.most = max_new;
  a.rows = (long)batch * k.tokens;
  if (a.rows > INT32_MAX) { set_error("paged append: %ld rows", a.rows); return KVD_ERR_ARG; }
  a.x[0] = k.ptr; a.sb[0] = k.stride_b; a.sh[0] = k.stride_h; a.st[0] = k.stride_t;
  a.x[1] = v.ptr; a.sb[1] = v.stride_b; a.sh[1] = v.stride_h; a.st[1] = v.stride_t;
  return by_shape(pool->head_dim, pool->store, dtype, a, DoAppend{(cudaStream_t)stream});
} catch (...) {
  set_error("paged append: host error");
  return KVD_ERR_CUDA;
}

extern "C" int kvd_paged_peek(const kvd_paged_pool* pool, int32_t batch, const int32_t* table, int64_t table_stride,
                              int32_t max_pages, const int32_t* lens, int32_t dtype, kvd_hf_view out_k,
                              kvd_hf_view out_v, kvd_stream_t stream) try {
  kvd::PeekArgs a;
  if (int rc = paged_pool_view(pool, &a.pool)) return rc;
  if (batch < 0 || batch > 32767 || max_pages < 0 || table_stride < max_pages || out_k.tokens < 0 || out_k.tokens != out_v.tokens ||
      (int64_t)max_pages * pool->page_size > INT32_MAX) {
    set_error("paged peek: batch %d, %d pages, outputs of %d and %d tokens", batch, max_pages, out_k.tokens, out_v.tokens);
    return KVD_ERR_ARG;
  }
  if (batch == 0 || out_k.tokens == 0) return KVD_OK;
  const int size = dtype == KVD_DTYPE_F32 ? 4 : 2;
  if (!table || !lens || !view_ok(out_k, size) || !view_ok(out_v, size)) { set_error("paged peek: outputs and their strides must be multiples of 16 bytes"); return KVD_ERR_ARG; }
  a.table = table; a.table_stride = table_stride; a.lens = lens;
  a.max_len = max_pages * pool->page_size;
  a.tokens = out_k.tokens;
  a.out[0] = out_k.ptr; a.sb[0] = out_k.stride_b; a.sh[0] = out_k.stride_h; a.st[0] = out_k.stride_t;
  a.out[1] = out_v.ptr; a.sb[1] = out_v.stride_b; a.sh[1] = out_v.stride_h; a.st[1] = out_v.stride_t;
  return by_shape(pool->head_dim, pool->store, dtype, a, DoPeek{batch, (cudaStream_t)stream});
} catch (...) {
  set_error("paged peek: host error");
  return KVD_ERR_CUDA;
}

extern "C" int kvd_paged_check_status(int32_t* status, kvd_stream_t stream) {
  int32_t h[4] = {0, 0, 0, 0};
  if (!status) { set_error("paged status: null pointer"); return KVD_ERR_ARG; }
  cudaError_t e = cudaMemcpyAsync(h, status, sizeof(h), cudaMemcpyDeviceToHost, (cudaStream_t)stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(status, 0, sizeof(h), (cudaStream_t)stream);
  if (e != cudaSuccess) { set_error("status read: %s", cudaGetErrorString(e)); return KVD_ERR_CUDA; }
  if (h[kvd::kStatusTimeout]) { set_error("paged cache: a device wait timed out (code %d)", h[kvd::kStatusTimeout]); return KVD_ERR_TIMEOUT; }
  if (h[kvd::kStatusBounds]) {
    set_error("paged cache: bad indices were skipped (flags %d: 1 slot, 2 page id, 4 the step's tables could not be built, 8 a captured step's attention mask)", h[kvd::kStatusBounds]);
    return KVD_ERR_ARG;
  }
  if (h[kvd::kStatusNumeric]) { set_error("paged cache: values that are not finite were stored (infinities saturated, NaN as 0)"); return KVD_ERR_NUMERIC; }
  return KVD_OK;
}
