// Attention of the new tokens of every segment over its pages
// (altxs_paged_attn, include/altxs.h).
//
//   y = softmax(s) V,  s_key = bias(scale q . k_key),  key in [lo, hi)
//
// One wave per (token, head): 64 keys at a time, a key per lane for the scores
// and a dim per lane for the sum over V, with the running maximum and sum of the
// softmax in fp32.
#include "common.h"
#include "paged.h"

namespace {

using namespace altxs_paged;

constexpr int THREADS = 256, WAVES = THREADS / WAVE, TILE = 64;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_f(_Float16 x) { return (float)x; }

struct AttnP {
  const void *q, *k, *v;
  void* out;
  const int32_t *table, *pos, *cu, *starts, *prefix;
  const float* slopes;
  int32_t* err;
  int64_t T, n_pages, q_tok, q_head, o_tok, o_head;
  int64_t kc_page, kc_head, kc_slot, vc_page, vc_head, vc_slot;
  float scale, softcap;
  int B, W, H, Hkv, G, width, shift, cap, window;
};

// Scores in the base-2 domain of the softmax: log2(e) (cap tanh(scale x / cap) - slope |p - key|).
__device__ __forceinline__ float biased(const AttnP& a, float x, float slope, int p, int key) {
#pragma clang fp contract(off)
  x *= a.scale;
  if (a.softcap > 0.f) {
    const float e = __builtin_amdgcn_exp2f(x * (2.f * LOG2E / a.softcap));
    x = a.softcap * (1.f - 2.f / (1.f + e));
  }
  x *= LOG2E;
  return __builtin_fmaf(-slope * LOG2E, fabsf((float)(p - key)), x);
}

template <class T, int HD>
__global__ __launch_bounds__(THREADS) void attn_row_kernel(AttnP a) {
#pragma clang fp contract(off)
  constexpr int ND = HD / WAVE;
  __shared__ float qs[WAVES][HD];
  __shared__ float ps[WAVES][TILE];
  __shared__ int pg[WAVES][TILE];
  const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const int64_t row = (int64_t)blockIdx.x * WAVES + wave;
  if (row >= a.T * a.H) return;
  const int64_t t = row / a.H;
  const int h = (int)(row - t * a.H), hk = h / a.G;
  int b, c0, c1;
  if (a.cu) {
    b = 0;
    for (int i = 0; i < a.B; i += WAVE) b += __builtin_popcountll(__ballot(i + lane < a.B && a.cu[i + lane + 1] <= t));
    if (b >= a.B) return;  // behind the last segment
    c0 = a.cu[b];
    c1 = a.cu[b + 1];
  } else {
    b = (int)(t / a.W);
    c0 = b * a.W;
    c1 = c0 + a.W;
  }
  const Segment s = segment_of(c0, c1, a.pos[b], a.T, a.cap);
  Range r = {0, 0};
  const int p = s.pos + (int)(t - s.t0);
  if (s.ok && t >= s.t0)
    r = keys_seen(p, s.pos + s.n, a.window, a.starts ? a.starts[t] : 0, a.prefix ? a.prefix[b] : 0);
  else if (lane == 0) flag_err(a.err, ALTXS_EDEV_POS);
  const T* q = (const T*)a.q + t * a.q_tok + h * a.q_head;
#pragma unroll
  for (int i = 0; i < ND; ++i) qs[wave][lane + i * WAVE] = to_f(q[lane + i * WAVE]);
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  float m = -INFINITY, l = 0.f, o[ND] = {};
  for (int k0 = r.lo & ~(TILE - 1); k0 < r.hi; k0 += TILE) {
    const int key = k0 + lane;
    int g = -1;
    float x = -INFINITY;
    if (key >= r.lo && key < r.hi) {
      g = page_of(a.table + (int64_t)b * a.width, a.width, a.shift, a.n_pages, key);
      float acc = 0.f;
      if (g >= 0) {
        const T* k = (const T*)a.k + g * a.kc_page + hk * a.kc_head + (key & ((1 << a.shift) - 1)) * a.kc_slot;
#pragma unroll 8
        for (int d = 0; d < HD; ++d) acc = __builtin_fmaf(qs[wave][d], to_f(k[d]), acc);
      } else {
        flag_err(a.err, ALTXS_EDEV_PAGE);
      }
      x = biased(a, acc, slope, p, key);
    }
    const float mn = fmaxf(m, wave_max(x)), mu = mn == -INFINITY ? 0.f : mn;
    const float pr = __builtin_amdgcn_exp2f(x - mu), al = __builtin_amdgcn_exp2f(m - mu);
    ps[wave][lane] = pr;
    pg[wave][lane] = g;
    __builtin_amdgcn_wave_barrier();
    l = __builtin_fmaf(l, al, wave_sum(pr));
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] *= al;
    for (int j = 0; j < TILE; ++j) {
      const int gj = pg[wave][j];
      if (gj < 0) continue;
      const T* v = (const T*)a.v + gj * a.vc_page + hk * a.vc_head + ((k0 + j) & ((1 << a.shift) - 1)) * a.vc_slot;
#pragma unroll
      for (int i = 0; i < ND; ++i) o[i] = __builtin_fmaf(ps[wave][j], to_f(v[lane + i * WAVE]), o[i]);
    }
    __builtin_amdgcn_wave_barrier();
    m = mn;
  }
  T* out = (T*)a.out + t * a.o_tok + h * a.o_head;
#pragma unroll
  for (int i = 0; i < ND; ++i) out[lane + i * WAVE] = (T)(r.lo < r.hi ? o[i] / l : 0.f);
}

}  // namespace

static int32_t check(const AltxsPagedAttnArgs* a, const char* who) {
  ALTXS_REQUIRE(a, "%s: null pointer", who);
  ALTXS_REQUIRE(a->dtype == ALTXS_F32 || a->dtype == ALTXS_BF16 || a->dtype == ALTXS_F16, "%s: dtype=%d", who, a->dtype);
  ALTXS_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "%s: head_dim=%d (64 and 128 are built)", who, a->head_dim);
  ALTXS_REQUIRE(a->Hkv >= 1 && a->H >= a->Hkv && a->H <= 4096 && a->H % a->Hkv == 0, "%s: H=%d is not a multiple of Hkv=%d",
                who, a->H, a->Hkv);
  ALTXS_REQUIRE(a->page_size >= 16 && a->page_size <= 1024 && (a->page_size & (a->page_size - 1)) == 0,
                "%s: page_size=%d must be a power of two from 16 to 1024", who, a->page_size);
  ALTXS_REQUIRE(a->T >= 0 && a->T * a->H < (1ll << 31) && a->B >= 0 && a->n_pages >= 0 && a->table_width >= 0,
                "%s: bad T, B, n_pages or table_width", who);
  ALTXS_REQUIRE(a->max_len >= 0 && a->max_len <= (int64_t)a->table_width * a->page_size,
                "%s: max_len=%d is more than table_width * page_size", who, a->max_len);
  ALTXS_REQUIRE(a->scale > 0.f && a->scale < INFINITY, "%s: scale=%g must be positive", who, a->scale);
  ALTXS_REQUIRE(a->softcap >= 0.f && a->softcap < INFINITY, "%s: softcap=%g", who, a->softcap);
  ALTXS_REQUIRE(a->window >= 0, "%s: window=%d", who, a->window);
  ALTXS_REQUIRE(a->T == 0 || a->B == 0 || a->cu || a->T % a->B == 0, "%s: T=%lld tokens are not B=%d equal segments", who,
                (long long)a->T, a->B);
  return ALTXS_OK;
}

extern "C" int64_t altxs_paged_attn_workspace_bytes(const AltxsPagedAttnArgs* a) {
  const int32_t rc = check(a, "altxs_paged_attn_workspace_bytes");
  return rc ? rc : 0;
}

extern "C" int32_t altxs_paged_attn(const AltxsPagedAttnArgs* a, altxs_stream_t stream) {
  const int32_t rc = check(a, "altxs_paged_attn");
  if (rc) return rc;
  if (a->T == 0 || a->B == 0) return ALTXS_OK;
  ALTXS_REQUIRE(a->q && a->out && a->k_cache && a->v_cache && a->table && a->pos, "altxs_paged_attn: null pointer");
  AttnP p;
  p.q = a->q; p.k = a->k_cache; p.v = a->v_cache; p.out = a->out;
  p.table = a->table; p.pos = a->pos; p.cu = a->cu; p.starts = a->starts; p.prefix = a->prefix;
  p.slopes = a->slopes; p.err = a->err;
  p.T = a->T; p.n_pages = a->n_pages; p.q_tok = a->q_tok; p.q_head = a->q_head; p.o_tok = a->out_tok; p.o_head = a->out_head;
  p.kc_page = a->kc_page; p.kc_head = a->kc_head; p.kc_slot = a->kc_slot;
  p.vc_page = a->vc_page; p.vc_head = a->vc_head; p.vc_slot = a->vc_slot;
  p.scale = a->scale; p.softcap = a->softcap;
  p.B = a->B; p.W = a->cu ? 1 : (int)(a->T / a->B); p.H = a->H; p.Hkv = a->Hkv; p.G = a->H / a->Hkv;
  p.width = a->table_width; p.shift = __builtin_ctz((unsigned)a->page_size); p.cap = a->max_len; p.window = a->window;
  const dim3 grid((unsigned)((a->T * a->H + WAVES - 1) / WAVES));
  const hipStream_t s = (hipStream_t)stream;
#define GO(T)                                                                                                   \
  do {                                                                                                          \
    if (a->head_dim == 64) hipLaunchKernelGGL((attn_row_kernel<T, 64>), grid, dim3(THREADS), 0, s, p);          \
    else hipLaunchKernelGGL((attn_row_kernel<T, 128>), grid, dim3(THREADS), 0, s, p);                           \
  } while (0)
  if (a->dtype == ALTXS_F32) GO(float);
  else if (a->dtype == ALTXS_BF16) GO(__bf16);
  else GO(_Float16);
#undef GO
  ALTXS_CHECK_HIP(hipGetLastError());
  return ALTXS_OK;
}
