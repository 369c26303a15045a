// Rotary positions, alone (altxs_rope) and on the way into a paged KV cache
// (altxs_paged_append).  (a, b) -> (a cos + b sin, b cos - a sin) for each pair
// of a head's first `rot` dims, the sign of the step's QKV epilogue
// (apply_rotary_emb, src/xsa_ttt/model.py:195-206).
//
// Both only move data (3 flops per element), so they are built to read and write
// every element once in 16-byte accesses: a head's row is cut into units -- one
// 16-byte vector of first and one of second elements (half layout), one vector
// of whole pairs (interleaved), or one vector of unrotated dims -- and a
// workgroup takes whole tokens, consecutive threads consecutive units.  Rows
// that 16-byte accesses do not fit (strides, alignment, rot) go by units of one
// pair or one element.
//
// Large calls are bound by memory: 65536 x 16 x 128 fp16 with its tables (571 MB) 92.5 us, 6.2
// TB/s (a large copy moves 5.1); 9973 x 8 x 64 fp32 (41 MB) 9.8 us; 16 segments' ragged chunks into
// their pages (8 + 2 x 4 heads of 64 bf16, 60 MB) 18.4 us.  Small ones are a chain of latencies: 64 rows
// 3.0 us, an append of 64 4.2 us (bounds, page entry, table row; the sources are read meanwhile).
// Four units a thread instead of one changed nothing.
#include <type_traits>

#include "common.h"
#include "paged.h"

namespace {

using namespace altxs_paged;

constexpr int THREADS = 256;
constexpr double CACHE = 256 << 20;  // bytes of the memory-side cache

template <class T> struct alignas(16) Vec { T v[16 / sizeof(T)]; };

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_f(_Float16 x) { return (float)x; }

// fp32 -> T in a rounding of its own: fused into the product before it (v_fma_mixlo_f16),
// it would give a kernel's fp16 rows other bits than another's.
template <class T> __device__ __forceinline__ T rounded(float x) {
  if constexpr (std::is_same_v<T, _Float16>) asm("" : "+v"(x));
  return (T)x;
}

// ONCE: what is not used again soon (the nt bit); 16-byte vectors only.
template <bool ONCE, class V> __device__ __forceinline__ V load_as(const void* p) {
  if constexpr (ONCE) return __builtin_bit_cast(V, __builtin_nontemporal_load((const u32x4*)p));
  else return *(const V*)p;
}
template <bool ONCE, class V> __device__ __forceinline__ void store_as(void* p, const V& v) {
  if constexpr (ONCE) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4*)p);
  else *(V*)p = v;
}

// How a head's row is cut into units.
struct Units {
  int nrot;   // rotated units
  int total;  // nrot + units of unrotated dims
  int half;   // rot / 2
};

// One unit of one head row on its way: get() reads it, put() rotates and writes it.  A
// kernel reads first and finds the position and the place meanwhile: both cost a
// memory latency or three.  cs/sn: the position's table rows (NULL: copy).
template <class T, bool VEC, bool INTER, bool ONCE = false> struct Unit {
  static constexpr int N = VEC ? 16 / (int)sizeof(T) : 1;  // elements of a vector
  static constexpr bool PAIR = !VEC || !INTER;             // firsts and seconds are two accesses
  std::conditional_t<VEC, Vec<T>, T> x, y;
  T* dst;
  const float *cs, *sn;
  int i;  // unit of its head

  __device__ __forceinline__ int first(const Units& u) const {
    return i >= u.nrot ? 2 * u.half + (i - u.nrot) * N : VEC || !INTER ? i * N : 2 * i;
  }
  __device__ __forceinline__ int second(const Units& u) const { return INTER ? 2 * i + 1 : i * N + u.half; }

  __device__ __forceinline__ void get(const T* src, const Units& u) {
    using V = decltype(x);
    x = load_as<ONCE, V>(src + first(u));
    if (PAIR && i < u.nrot) y = load_as<ONCE, V>(src + second(u));
  }
  __device__ __forceinline__ void put(const Units& u, float sgn) {
#pragma clang fp contract(off)
    using V = decltype(x);
    if (i < u.nrot && cs) {
      if constexpr (VEC && INTER) {
        typedef __attribute__((ext_vector_type(N / 2))) float pairs_t;
        const pairs_t c = *(const pairs_t*)(cs + i * N / 2), s = sgn * *(const pairs_t*)(sn + i * N / 2);
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
          const float a = to_f(x.v[2 * j]), b = to_f(x.v[2 * j + 1]);
          x.v[2 * j] = rounded<T>(__builtin_fmaf(b, s[j], a * c[j]));
          x.v[2 * j + 1] = rounded<T>(__builtin_fmaf(-a, s[j], b * c[j]));
        }
      } else if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
          const f32x4 c = *(const f32x4*)(cs + i * N + j), s = sgn * *(const f32x4*)(sn + i * N + j);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float a = to_f(x.v[j + k]), b = to_f(y.v[j + k]);
            x.v[j + k] = rounded<T>(__builtin_fmaf(b, s[k], a * c[k]));
            y.v[j + k] = rounded<T>(__builtin_fmaf(-a, s[k], b * c[k]));
          }
        }
      } else {
        const float a = to_f(x), b = to_f(y), c = cs[i], s = sgn * sn[i];
        x = rounded<T>(__builtin_fmaf(b, s, a * c));
        y = rounded<T>(__builtin_fmaf(-a, s, b * c));
      }
    }
    store_as<ONCE>(dst + first(u), x);
    if (PAIR && i < u.nrot) store_as<ONCE>(dst + second(u), y);
  }
};

struct RopeP {
  const void* x;
  void* out;
  const int32_t* pos;
  const float *cos, *sin;
  int32_t* err;
  int64_t T, rows, x_tok, x_head, out_tok, out_head;
  Units u;
  FastDiv by_units;  // units of a head
  FastDiv by_token;  // units of a token
  int tpb;           // tokens of a workgroup
  float sgn;
};

template <class T, bool VEC, bool INTER, bool ONCE>
__global__ __launch_bounds__(THREADS) void rope_kernel(RopeP p) {
  const int64_t t0 = (int64_t)blockIdx.x * p.tpb;
  const int nt = (int)(p.T - t0 < p.tpb ? p.T - t0 : p.tpb);
  const int n = nt * (int)p.by_token.d;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const uint32_t tl = div_by(i, p.by_token), j = i - tl * p.by_token.d;
    const uint32_t h = div_by(j, p.by_units);
    const int64_t t = t0 + tl;
    Unit<T, VEC, INTER, ONCE> m;
    m.i = j - h * p.by_units.d;
    m.get((const T*)p.x + t * p.x_tok + h * p.x_head, p.u);
    const int32_t pos = p.pos[t];
    const bool ok = pos >= 0 && pos < p.rows;
    if (!ok && pos >= 0 && j == 0) flag_err(p.err, ALTXS_EDEV_POS);
    m.cs = ok ? p.cos + (int64_t)pos * p.u.half : nullptr;
    m.sn = p.sin + (ok ? (int64_t)pos * p.u.half : 0);
    m.dst = (T*)p.out + t * p.out_tok + h * p.out_head;
    m.put(p.u, p.sgn);
  }
}

struct AppendP {
  const void *k, *v, *q;
  void *q_out, *k_cache, *v_cache;
  const int32_t *table, *pos, *cu;
  const float *cos, *sin;
  int32_t* err;
  int64_t T, n_pages, rope_rows;
  int64_t k_tok, k_head, v_tok, v_head, q_tok, q_head, qo_tok, qo_head;
  int64_t kv_page, kv_head, kv_slot;
  int B, Hq, Hkv, width, shift, W;  // Hq: query heads moved here (0: none); W: tokens of a segment (cu = NULL)
  Units u;
  FastDiv by_units, by_token;
  int tpb;
};

// A token's place: its rope row and its cache row's element offset (ok = 0: skipped).
struct Place {
  int64_t off;
  int32_t pos, ok;
};

constexpr int MAX_TPB = 64;

// The tokens' places are found by a wave each while the first units are read.
template <class T, bool VEC, bool INTER>
__global__ __launch_bounds__(THREADS) void append_kernel(AppendP p) {
  __shared__ Place place[MAX_TPB];
  const int64_t t0 = (int64_t)blockIdx.x * p.tpb;
  const int nt = (int)(p.T - t0 < p.tpb ? p.T - t0 : p.tpb);
  const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const int n = nt * (int)p.by_token.d;
  int tl = 0, h = 0;
  Unit<T, VEC, INTER> m;
  auto get = [&](int i) {
    tl = (int)div_by(i, p.by_token);
    const uint32_t j = i - tl * p.by_token.d;
    h = (int)div_by(j, p.by_units);
    m.i = (int)(j - h * p.by_units.d);
    const int64_t t = t0 + tl;
    const T* src = h < p.Hq           ? (const T*)p.q + t * p.q_tok + h * p.q_head
                   : h < p.Hq + p.Hkv ? (const T*)p.k + t * p.k_tok + (h - p.Hq) * p.k_head
                                      : (const T*)p.v + t * p.v_tok + (h - p.Hq - p.Hkv) * p.v_head;
    m.get(src, p.u);
  };
  auto put = [&]() {
    const Place pl = place[tl];
    if (!pl.ok) return;
    const bool is_v = h >= p.Hq + p.Hkv;
    m.dst = h < p.Hq ? (T*)p.q_out + (t0 + tl) * p.qo_tok + h * p.qo_head
            : is_v   ? (T*)p.v_cache + pl.off + (h - p.Hq - p.Hkv) * p.kv_head
                     : (T*)p.k_cache + pl.off + (h - p.Hq) * p.kv_head;
    m.cs = p.cos && !is_v ? p.cos + (int64_t)pl.pos * p.u.half : nullptr;
    m.sn = p.sin + (int64_t)pl.pos * p.u.half;
    m.put(p.u, 1.f);
  };
  if ((int)threadIdx.x < n) get(threadIdx.x);
  for (int i = wave; i < nt; i += THREADS / WAVE) {
    const int64_t t = t0 + i, cap = (int64_t)p.width << p.shift;
    Segment s;
    const int b = token_segment(p.cu, p.pos, p.B, p.W, t, p.T, (int)(cap < INT32_MAX ? cap : INT32_MAX), lane, s);
    if (lane == 0) {
      Place pl = {0, 0, 0};
      if (b >= 0) {  // rows behind the last segment belong to nobody
        const int32_t pos = s.pos + (int32_t)(t - s.t0);
        if (!s.ok || t < s.t0 || t >= s.t0 + s.n || (p.cos && pos >= p.rope_rows)) {
          flag_err(p.err, ALTXS_EDEV_POS);
        } else {
          const int32_t g = page_of(p.table + (int64_t)b * p.width, p.width, p.shift, p.n_pages, pos);
          if (g < 0) flag_err(p.err, ALTXS_EDEV_PAGE);
          else pl = Place{g * p.kv_page + (pos & ((1 << p.shift) - 1)) * p.kv_slot, pos, 1};
        }
      }
      place[i] = pl;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n;) {
    put();
    if ((i += THREADS) < n) get(i);
  }
}

int elem_size(int dtype) { return dtype == ALTXS_F32 ? 4 : 2; }

// Whether rows with these strides (in elements) at p can be moved in 16-byte vectors.
bool fits16(const void* p, int n, std::initializer_list<int64_t> strides) {
  bool ok = ((uintptr_t)p & 15) == 0;
  for (int64_t s : strides) ok = ok && s % n == 0;
  return ok;
}

// Vectors need whole ones in the head, the unrotated dims and each half (pairs).
bool dims_fit(int hd, int rot, bool inter, int n) { return hd % n == 0 && (inter ? rot % n == 0 : rot % (2 * n) == 0); }

Units units_of(int hd, int rot, bool vec, bool inter, int n) {
  Units u;
  u.half = rot / 2;
  if (!vec) n = 1;
  u.nrot = vec ? (inter ? rot / n : rot / 2 / n) : rot / 2;
  u.total = u.nrot + (hd - rot) / n;
  return u;
}

// f(T{}) for the type of dtype
template <class F> void by_type(int dtype, F f) {
  if (dtype == ALTXS_F32) f(float{});
  else if (dtype == ALTXS_BF16) f(__bf16{});
  else f(_Float16{});
}

}  // namespace

extern "C" int32_t altxs_rope(const AltxsRopeArgs* a, altxs_stream_t stream) {
  ALTXS_REQUIRE(a, "altxs_rope: null pointer");
  ALTXS_REQUIRE(a->dtype == ALTXS_F32 || a->dtype == ALTXS_BF16 || a->dtype == ALTXS_F16,
                "altxs_rope: dtype=%d", a->dtype);
  ALTXS_REQUIRE((a->flags & ~(ALTXS_ROPE_INTERLEAVED | ALTXS_ROPE_INVERSE)) == 0, "altxs_rope: unknown flags 0x%x",
                a->flags);
  ALTXS_REQUIRE(a->head_dim >= 2 && a->head_dim <= 1024, "altxs_rope: head_dim=%d", a->head_dim);
  ALTXS_REQUIRE(a->rot >= 2 && a->rot % 2 == 0 && a->rot <= a->head_dim,
                "altxs_rope: rot=%d must be even, 2 to head_dim=%d", a->rot, a->head_dim);
  ALTXS_REQUIRE(a->H >= 1 && a->H <= 4096, "altxs_rope: H=%d", a->H);
  ALTXS_REQUIRE(a->T >= 0 && a->rows >= 1, "altxs_rope: bad T or rows");
  if (a->T == 0) return ALTXS_OK;
  ALTXS_REQUIRE(a->x && a->out && a->pos && a->cos && a->sin, "altxs_rope: null pointer");
  const int n = 16 / elem_size(a->dtype);
  const bool inter = (a->flags & ALTXS_ROPE_INTERLEAVED) != 0;
  const bool vec = dims_fit(a->head_dim, a->rot, inter, n) && fits16(a->x, n, {a->x_tok, a->x_head}) &&
                   fits16(a->out, n, {a->out_tok, a->out_head}) && fits16(a->cos, 4, {(int64_t)a->rot / 2}) &&
                   fits16(a->sin, 4, {(int64_t)a->rot / 2});
  RopeP p;
  p.x = a->x; p.out = a->out; p.pos = a->pos; p.cos = a->cos; p.sin = a->sin; p.err = a->err;
  p.T = a->T; p.rows = a->rows;
  p.x_tok = a->x_tok; p.x_head = a->x_head; p.out_tok = a->out_tok; p.out_head = a->out_head;
  p.u = units_of(a->head_dim, a->rot, vec, inter, n);
  p.sgn = a->flags & ALTXS_ROPE_INVERSE ? -1.f : 1.f;
  if (a->x == a->out && a->x_tok == a->out_tok && a->x_head == a->out_head) p.u.total = p.u.nrot;  // the rest stays
  p.by_units = fast_div(p.u.total);
  p.by_token = fast_div(p.u.total * a->H);
  p.tpb = (int)p.by_token.d >= THREADS ? 1 : THREADS / (int)p.by_token.d;
  const int64_t wgs = (a->T + p.tpb - 1) / p.tpb;
  ALTXS_REQUIRE(wgs < (1ll << 24), "altxs_rope: T=%lld", (long long)a->T);  // 2^32 threads a launch
  const dim3 grid((unsigned)wgs);
  // Arrays that together pass the memory-side cache leave little in it for who reads the
  // result.  Marked as used once / not, two sets in turn: 536 MB 94.4 / 101 us, 268 MB 48.8 / 52.7, but 134 MB
  // 25.9 / 25.2, and one set over and over, which stays, 268 MB 48.3 / 45.0.
  const int es = elem_size(a->dtype);
  const bool once = vec && 2.0 * (double)a->T * a->H * a->head_dim * es > CACHE;
  by_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    auto* k = !vec    ? inter ? rope_kernel<T, false, true, false> : rope_kernel<T, false, false, false>
              : once  ? inter ? rope_kernel<T, true, true, true> : rope_kernel<T, true, false, true>
              : inter ? rope_kernel<T, true, true, false>
                      : rope_kernel<T, true, false, false>;
    hipLaunchKernelGGL(k, grid, dim3(THREADS), 0, (hipStream_t)stream, p);
  });
  ALTXS_CHECK_HIP(hipGetLastError());
  return ALTXS_OK;
}

extern "C" int32_t altxs_paged_append(const AltxsPagedAppendArgs* a, altxs_stream_t stream) {
  ALTXS_REQUIRE(a, "altxs_paged_append: null pointer");
  ALTXS_REQUIRE(a->dtype == ALTXS_F32 || a->dtype == ALTXS_BF16 || a->dtype == ALTXS_F16,
                "altxs_paged_append: dtype=%d", a->dtype);
  ALTXS_REQUIRE((a->flags & ~ALTXS_ROPE_INTERLEAVED) == 0, "altxs_paged_append: unknown flags 0x%x", a->flags);
  ALTXS_REQUIRE(a->head_dim >= 2 && a->head_dim <= 1024, "altxs_paged_append: head_dim=%d", a->head_dim);
  ALTXS_REQUIRE(a->rot >= 0 && a->rot % 2 == 0 && a->rot <= a->head_dim,
                "altxs_paged_append: rot=%d must be even, 0 to head_dim=%d", a->rot, a->head_dim);
  ALTXS_REQUIRE(a->Hkv >= 1 && a->Hkv <= 4096 && (!a->q || (a->H >= 1 && a->H <= 4096)), "altxs_paged_append: H=%d Hkv=%d",
                a->H, a->Hkv);
  ALTXS_REQUIRE(a->page_size >= 16 && a->page_size <= 1024 && (a->page_size & (a->page_size - 1)) == 0,
                "altxs_paged_append: page_size=%d must be a power of two from 16 to 1024", a->page_size);
  ALTXS_REQUIRE(a->T >= 0 && a->T < (1ll << 31) && a->B >= 0 && a->n_pages >= 0 && a->table_width >= 0,
                "altxs_paged_append: bad T, B, n_pages or table_width");
  ALTXS_REQUIRE(a->rot > 0 || !a->q, "altxs_paged_append: q without a rotation");
  for (int64_t st : {a->kv_page, a->kv_head, a->kv_slot})
    ALTXS_REQUIRE(st >= 0 && st < (1ll << 31), "altxs_paged_append: a cache stride of %lld elements", (long long)st);
  ALTXS_REQUIRE((a->kv_page > 0 || a->n_pages <= 1) && (a->kv_head > 0 || a->Hkv == 1) && a->kv_slot > 0,
                "altxs_paged_append: an expanded cache");
  if (a->T == 0 || a->B == 0) return ALTXS_OK;
  ALTXS_REQUIRE(a->cu || a->T % a->B == 0, "altxs_paged_append: T=%lld tokens are not B=%d equal segments",
                (long long)a->T, a->B);
  ALTXS_REQUIRE(a->k && a->v && a->k_cache && a->v_cache && a->table && a->pos && (!a->q || a->q_out) &&
                    (a->rot == 0 || (a->cos && a->sin)),
                "altxs_paged_append: null pointer");
  ALTXS_REQUIRE(a->rot == 0 || a->rope_rows >= 1, "altxs_paged_append: rope_rows=%lld", (long long)a->rope_rows);
  const int n = 16 / elem_size(a->dtype);
  const bool inter = (a->flags & ALTXS_ROPE_INTERLEAVED) != 0;
  bool vec = dims_fit(a->head_dim, a->rot, inter, n) && fits16(a->k, n, {a->k_tok, a->k_head}) &&
             fits16(a->v, n, {a->v_tok, a->v_head}) && fits16(a->k_cache, n, {a->kv_page, a->kv_head, a->kv_slot}) &&
             fits16(a->v_cache, n, {a->kv_page, a->kv_head, a->kv_slot});
  if (a->q) vec = vec && fits16(a->q, n, {a->q_tok, a->q_head}) && fits16(a->q_out, n, {a->q_out_tok, a->q_out_head});
  if (a->rot) vec = vec && fits16(a->cos, 4, {(int64_t)a->rot / 2}) && fits16(a->sin, 4, {(int64_t)a->rot / 2});
  AppendP p;
  p.k = a->k; p.v = a->v; p.q = a->q; p.q_out = a->q_out; p.k_cache = a->k_cache; p.v_cache = a->v_cache;
  p.table = a->table; p.pos = a->pos; p.cu = a->cu;
  p.cos = a->rot ? a->cos : nullptr; p.sin = a->sin; p.err = a->err;
  p.T = a->T; p.n_pages = a->n_pages; p.rope_rows = a->rope_rows;
  p.k_tok = a->k_tok; p.k_head = a->k_head; p.v_tok = a->v_tok; p.v_head = a->v_head;
  p.q_tok = a->q_tok; p.q_head = a->q_head; p.qo_tok = a->q_out_tok; p.qo_head = a->q_out_head;
  p.kv_page = a->kv_page; p.kv_head = a->kv_head; p.kv_slot = a->kv_slot;
  p.B = a->B; p.Hq = a->q ? a->H : 0; p.Hkv = a->Hkv; p.width = a->table_width;
  p.shift = __builtin_ctz((unsigned)a->page_size);
  p.W = a->cu ? 1 : (int)(a->T / a->B);
  p.u = units_of(a->head_dim, a->rot, vec, inter, n);
  p.by_units = fast_div(p.u.total);
  p.by_token = fast_div(p.u.total * (p.Hq + 2 * p.Hkv));
  p.tpb = (int)p.by_token.d >= THREADS ? 1 : THREADS / (int)p.by_token.d;
  if (p.tpb > MAX_TPB) p.tpb = MAX_TPB;
  const int64_t wgs = (a->T + p.tpb - 1) / p.tpb;
  ALTXS_REQUIRE(wgs < (1ll << 24), "altxs_paged_append: T=%lld", (long long)a->T);
  const dim3 grid((unsigned)wgs);
  by_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    auto* k = vec ? inter ? append_kernel<T, true, true> : append_kernel<T, true, false>
                  : inter ? append_kernel<T, false, true> : append_kernel<T, false, false>;
    hipLaunchKernelGGL(k, grid, dim3(THREADS), 0, (hipStream_t)stream, p);
  });
  ALTXS_CHECK_HIP(hipGetLastError());
  return ALTXS_OK;
}
