// Attention of the new tokens of every segment over its pages
// (altxs_paged_attn, include/altxs.h).
//
//   y = softmax(s) V,  s_key = bias(scale q . k_key),  key in [lo, hi)
//
// The softmax in one pass.  Keys come in tiles of 64 and chunks of 4 tiles.
// Inside a chunk a running maximum m, sum l and output O are kept over the tiles; a
// chunk starts afresh, and the chunks' (m, l, O) are folded in order:
//   M' = max(M, m), L' = L 2^(M - M') + l 2^(m - M'), O likewise.
// Tiles and chunks begin at multiples of their sizes from key 0, so a row's
// arithmetic is the same wherever its chunks are worked on -- one after the
// other by a workgroup that keeps the totals, or by workgroups of their own whose
// partial results a second launch folds.  That makes the bits of a row
// independent of batch, window width and launch, as in the dense attention, and
// lets long caches with few rows be split over the whole chip.
//
// Products (16-bit types): S^T = K Q^T and O^T = V^T P^T by v_mfma_f32_16x16x32.
// Lane 16 g + c of a score tile holds, for query row c, keys 16 kb + 4 g + i
// (kb, i < 4): a row's maximum and sum need two lane exchanges, and the lane's own
// eight values of blocks 2 s, 2 s + 1 are the P^T operand of step s when the
// contraction's keys are taken in the order 16 (j / 4) + 4 g + j % 4.  V's operand
// in that order comes out of row-major V tiles in LDS by ds_read_b64_tr_b16.
// Rows of a tile are (token, query head of the kv head's group) pairs, token-major:
// grouped heads and neighbouring tokens share every K and V read.
//
// Rounding.  In the 16-bit types the weights 2^(s - m) go into the P V products rounded to
// the type, and l sums the rounded ones.  The largest of a tile that moves m is one,
// exactly: m follows every tile's maximum for that (letting it trail by up to 8 powers of
// two, so that O is rescaled less often, saves 4% of chunk scoring and costs a third
// of the accuracy: error against 64 bits 1.25 to 1.4 times that of fp32 weights and a
// rounded output, against 1.07; a second product with the remainders would make it 1.0
// and chunk scoring 27% slower).  Everything else is fp32.
//
// Two kernels, one arithmetic:
//   few   up to 16 rows a segment and kv head on average (decode): 16-row tiles.  A
//         workgroup takes a chunk at a time, its four waves a tile each for the
//         scores (K straight into the operand registers) and a quarter of the
//         dims each for P V, so a chunk's loads are all in flight at once.
//   many  128-row tiles, 32 rows a wave (64 and 16 for rows of more than 128 bytes); K and
//         V tiles go through LDS, loaded ahead, and are read by all four waves.
// fp32 (the framework's exact mode) is the same with v_mfma_f32_16x16x4_f32, 4 keys or dims
// at a time, exact products and unrounded weights.
//
// Rows that a tile's rows do not all see.  Scores outside [lo, hi) become -inf.
// Keys outside the union of the tile's ranges, and keys of bad pages, are loaded
// from a row of zeros instead.  Only keys between can carry a neighbour's
// infinities or NaN into a row (0 * inf in P V): in tiles with such keys each wave looks
// through the V rows it loaded, before the workgroup meets, and zeroes what is not
// finite; if there was any, it is added to the rows that do see it when the chunk ends.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "paged.h"

namespace {

using namespace altxs_paged;

constexpr int THREADS = 256, WAVES = THREADS / WAVE, TILE = 64, CHUNK = 256, TPC = CHUNK / TILE;
static_assert(TPC == WAVES, "the few-row kernel gives each wave a tile of the chunk");
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_f(_Float16 x) { return (float)x; }

alignas(16) static __device__ const uint32_t kZeroRow[128] = {};  // a K or V row of zeros (128 fp32 values at most)

struct AttnP {
  const void *q, *k, *v;
  void* out;
  const int32_t *table, *pos, *cu, *starts, *prefix;
  const float* slopes;
  int32_t* err;
  int64_t T, n_pages, q_tok, q_head, o_tok, o_head;
  int64_t kv_head;
  uint32_t kv_page, kv_slot;
  float scale, softcap, scale2;  // scale2 = scale * log2(e)
  int B, W, H, Hkv, G, width, shift, cap, window;
  FastDiv by_g, by_hkv, by_b, by_pairs, by_tiles;  // by_tiles: row tiles of a segment (cu = NULL)
  // chunk partials: part[(row * nc + c) * HD + d] and ml[row * nc + c], row = t * H + h
  float* part;
  float2* ml;
  int nc;
  bool direct;  // a workgroup folds all its rows' chunks and writes out
};

// ---- rows ------------------------------------------------------------------

// A workgroup's row tile: rows r0 .. of segment b (rows of its tokens x group heads).
struct RowTile {
  int b, r0, rows;  // rows: of the whole segment; none left when r0 >= rows
  Segment s;
};

// Which tile slot `slot` is, of `br` rows; every wave finds it for itself, each lane with
// a segment's bounds and position.  One wave of each of the first slots also checks 64 of
// cu's entries (the search itself is safe with any).
__device__ __forceinline__ RowTile find_tile(const AttnP& a, int slot, int br, int lane, bool check) {
  RowTile t;
  t.b = a.B;
  t.r0 = t.rows = 0;
  if (!a.cu) {
    t.b = (int)div_by(slot, a.by_tiles);
    const int c0 = t.b * a.W;
    t.s = segment_of(c0, c0 + a.W, a.pos[t.b], a.T, a.cap);
    t.rows = a.W * a.G;
    t.r0 = (slot - t.b * (int)a.by_tiles.d) * br;
    return t;
  }
  if (check && slot < (a.B + WAVE - 1) / WAVE) {
    const int j = slot * WAVE + lane < a.B ? slot * WAVE + lane : a.B - 1;
    const int c0 = a.cu[j], c1 = a.cu[j + 1];
    if (__any(c1 < c0 || c1 > a.T || (j == 0 && c0 != 0)) && lane == 0) flag_err(a.err, ALTXS_EDEV_POS);
  }
  auto end_of = [&](int c1) { return c1 < 0 ? 0 : c1 > a.T ? (int)a.T : c1; };
  const int i = block_with_first(a.B, lane, [&](int j) { return first_slot(end_of(a.cu[j + 1]), a.G, br, j + 1) > slot; });
  const int j = i + lane < a.B ? i + lane : a.B - 1;
  const int c0 = a.cu[j], c1 = a.cu[j + 1], p = a.pos[j];
  const uint64_t later = __ballot(i + lane < a.B && first_slot(end_of(c1), a.G, br, j + 1) > slot);
  if (later) {
    const int n = __builtin_ctzll(later);
    t.b = i + n;
    t.s = segment_of(__builtin_amdgcn_readlane(c0, n), __builtin_amdgcn_readlane(c1, n), __builtin_amdgcn_readlane(p, n), a.T, a.cap);
    const int64_t k = slot - first_slot(t.s.t0, a.G, br, t.b);
    t.rows = t.s.n * a.G;
    t.r0 = k < 0 || k * br >= t.rows ? t.rows : (int)(k * br);
  }
  return t;
}

// One query row as a lane's column sees it.
struct Row {
  int lo, hi, p;      // rows past the segment's last, and rows that see nothing, let everything through
  float slope2;       // slope * log2(e)
  int64_t t;          // token
  int h;              // query head
  bool valid, empty;  // not valid: past the last, nothing is stored; empty: sees nothing, zeros are stored
};

__device__ __forceinline__ Row row_of(const AttnP& a, const RowTile& tile, int hk, int r) {
  Row o;
  o.valid = r < tile.rows;
  const int rr = o.valid ? r : 0;
  const int i = (int)div_by(rr, a.by_g);
  o.t = tile.s.t0 + i;
  o.h = hk * a.G + (rr - i * a.G);
  o.p = tile.s.pos + i;
  Range k = {0, 0};
  if (tile.s.ok)
    k = keys_seen(o.p, tile.s.pos + tile.s.n, a.window, a.starts ? a.starts[o.t] : 0, a.prefix ? a.prefix[tile.b] : 0);
  o.empty = o.valid && k.lo >= k.hi;
  o.lo = o.valid && !o.empty ? k.lo : 0;
  o.hi = o.valid && !o.empty ? k.hi : INT32_MAX;
  o.slope2 = a.slopes ? a.slopes[o.h] * LOG2E : 0.f;
  return o;
}

__device__ __forceinline__ int row16_imin(int v) {
  auto least = [](int a, int b) { return a < b ? a : b; };
  v = least(v, (int)dpp_u<DPP_XOR1>((uint32_t)v));
  v = least(v, (int)dpp_u<DPP_XOR2>((uint32_t)v));
  v = least(v, (int)dpp_u<DPP_HALF_MIRROR>((uint32_t)v));
  v = least(v, (int)dpp_u<DPP_MIRROR>((uint32_t)v));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int row16_imax(int v) { return -row16_imin(-v); }

// What a set of rows sees: the union [lo, hi) and what all of them see, [clo, chi); rows
// that see nothing do not count.
struct Seen {
  int lo, hi, clo, chi;
  __device__ bool full(int k0) const { return clo <= k0 && chi >= k0 + TILE; }
  // some key that is loaded (in [LO, HI)) is hidden from some row
  __device__ bool mixed(int k0, int LO, int HI) const {
    return clo > (k0 > LO ? k0 : LO) || chi < (k0 + TILE < HI ? k0 + TILE : HI);
  }
};
__device__ __forceinline__ Seen seen_by(const Row& r) {
  Seen s;
  const bool some = r.valid && !r.empty;
  s.lo = row16_imin(some ? r.lo : INT32_MAX);
  s.hi = row16_imax(some ? r.hi : 0);
  s.clo = row16_imax(r.lo);
  s.chi = row16_imin(r.hi);
  return s;
}
__device__ __forceinline__ Seen both(const Seen a, const Seen b) {
  return {a.lo < b.lo ? a.lo : b.lo, a.hi > b.hi ? a.hi : b.hi, a.clo > b.clo ? a.clo : b.clo, a.chi < b.chi ? a.chi : b.chi};
}

// ---- keys ----------------------------------------------------------------------

// The table entry of a key, read for the nearest key of the rows' union [LO, HI)
// (LO < HI <= what the table holds), and the page it names: -1 for a key outside the
// union or an entry that is no page (flagged).
__device__ __forceinline__ int key_entry(const AttnP& a, int b, int key, int LO, int HI) {
  const int k = key < LO ? LO : key >= HI ? HI - 1 : key;
  return a.table[(int64_t)b * a.width + (k >> a.shift)];
}
__device__ __forceinline__ int entry_page(const AttnP& a, int entry, int key, int LO, int HI) {
  const bool seen = key >= LO && key < HI, good = entry >= 0 && entry < a.n_pages;
  if (seen && !good) flag_err(a.err, ALTXS_EDEV_PAGE);
  return seen && good ? entry : -1;
}

// A key's row of kv head hk (head = its offset) in a cache, or the row of zeros.
template <class T>
__device__ __forceinline__ const T* key_row(const void* cache, int page, int key, int shift, uint32_t st_page, uint32_t st_slot,
                                            int64_t head) {
  const int64_t at = (int64_t)((uint64_t)(page < 0 ? 0 : page) * st_page + (uint64_t)(key & ((1 << shift) - 1)) * st_slot) + head;
  const T* p = (const T*)cache + at;
  return page < 0 ? (const T*)kZeroRow : p;
}

// ---- tile arithmetic ---------------------------------------------------------

// The same value, where rare paths start from it: what they compute stays in them
// instead of being kept in registers over the whole loop.
__device__ __forceinline__ int unhoisted(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Operands come in 16-byte pieces a lane: EL elements of each of the 4 lane groups, 4 EL
// along the contraction.  mfma(): the product of two pieces; fp32 has them as four
// v_mfma_f32_16x16x4_f32, whose k-th slice is element j of lane group k.
template <class T> struct Op;
template <> struct Op<__bf16> {
  static constexpr int EL = 8;
  static constexpr uint32_t EXP = 0x7f807f80u, ONE = 0x00800080u;  // exponent fields of a word, their lowest bits
  static constexpr uint32_t TOP = 0x80008000u, ONES = 0x3f803f80u; // the bits above them; a word of ones
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Op<_Float16> {
  static constexpr int EL = 8;
  static constexpr uint32_t EXP = 0x7c007c00u, ONE = 0x04000400u, TOP = 0x80008000u, ONES = 0x3c003c00u;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <> struct Op<float> {
  static constexpr int EL = 4;
  static constexpr uint32_t EXP = 0x7f800000u, ONE = 0x00800000u, TOP = 0x80000000u, ONES = 0x3f800000u;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
};
// Steps of P V over a tile: 32 keys (two score blocks) in the 16-bit types, 16 in fp32.
template <class T> constexpr int STEPS = TILE / (4 * Op<T>::EL);
template <class T, int HD> constexpr int PIECES = HD * (int)sizeof(T) / 16;  // of a K or V row

// The larger of two, NaN left out (fmaxf on values out of lane swaps would quiet them first).
__device__ __forceinline__ float max2(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_fmed3f(__uint_as_float(a), __uint_as_float(b), INFINITY);
}

// Products q.k of a tile -> scores (BIAS: finished, base 2; else still to be scaled by
// scale2) with -inf outside [lo, hi), and mx, their maximum over the row in the base-2 domain.
template <bool BIAS, int CB>
__device__ __forceinline__ void tile_scores(const AttnP& a, f32x4 (&S)[CB][4], float (&mx)[CB], const Row (&r)[CB], int k0, int g,
                                            bool full) {
#pragma clang fp contract(off)
  if constexpr (BIAS) {
    if (a.softcap > 0.f) {  // cap tanh(y) log2(e) = cap2 - 2 cap2 / (1 + 2^(2 log2(e) y)), y = scale x / cap
      const float e2 = 2.f * a.scale2 / a.softcap, cap2 = a.softcap * LOG2E;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const float e = __builtin_amdgcn_exp2f(S[cb][n / 4][n % 4] * e2);
          S[cb][n / 4][n % 4] = __builtin_fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(1.f + e), cap2);
        }
    } else {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int n = 0; n < 16; ++n) S[cb][n / 4][n % 4] *= a.scale2;
    }
    if (a.slopes) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        const int d0 = r[cb].p - (k0 + 4 * g);
#pragma unroll
        for (int n = 0; n < 16; ++n)
          S[cb][n / 4][n % 4] = __builtin_fmaf(-r[cb].slope2, fabsf((float)(d0 - (16 * (n / 4) + n % 4))), S[cb][n / 4][n % 4]);
      }
    }
  }
  if (!full) {
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      // keys lo .. hi - 1 of the lane's own: one comparison each, unsigned
      const uint32_t lo = r[cb].lo - (k0 + 4 * g), n_seen = r[cb].hi - r[cb].lo;
#pragma unroll
      for (int n = 0; n < 16; ++n)
        S[cb][n / 4][n % 4] = (uint32_t)(16 * (n / 4) + n % 4) - lo < n_seen ? S[cb][n / 4][n % 4] : -INFINITY;
    }
  }
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    float m = S[cb][0][0];
#pragma unroll
    for (int n = 1; n < 16; ++n) m = fmaxf(m, S[cb][n / 4][n % 4]);
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = max2(x[0], x[1]);
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = max2(y[0], y[1]);
    mx[cb] = BIAS ? m : m * a.scale2;
  }
}

// m after a tile of maximum mx, and the factor of what was summed before.
__device__ __forceinline__ float next_max(float& m, float mx) {
#pragma clang fp contract(off)
  const float old = m;
  m = fmaxf(old, mx);
  return m == old ? 1.f : __builtin_amdgcn_exp2f(old - m);
}

// Scores of step s -> weights 2^(s - m), as its P operand: rounded to the nearest value
// of a 16-bit type.
template <class T, bool BIAS>
__device__ __forceinline__ u32x4 step_weights(const AttnP& a, const f32x4 (&S)[4], int s, float m) {
#pragma clang fp contract(off)
  const float mu = m == -INFINITY ? 0.f : m, sc = BIAS ? 1.f : a.scale2;
  typedef __attribute__((ext_vector_type(Op<T>::EL))) T vec;
  vec w;
#pragma unroll
  for (int j = 0; j < Op<T>::EL; ++j)
    w[j] = (T)__builtin_amdgcn_exp2f(__builtin_fmaf(S[s * Op<T>::EL / 4 + j / 4][j % 4], sc, -mu));
  return __builtin_bit_cast(u32x4, w);
}

// V tiles in LDS: rows whose 16-byte pieces are permuted so that what a read takes of
// several rows falls into different banks -- 32 bytes of eight consecutive rows (16-bit
// types), 64 bytes of every fourth row (fp32).
template <class T, int HD> __device__ __forceinline__ int v_piece(int row, int piece) {
  return piece ^ (sizeof(T) == 4 ? 4 * ((row >> 2) & 3) : HD == 64 ? 2 * ((row >> 1) & 3) : 2 * (row & 7));
}
// K tiles: a lane reads whole pieces, 16 consecutive rows at the same one.
template <class T, int HD> __device__ __forceinline__ int k_piece(int row, int piece) {
  return piece ^ (PIECES<T, HD> == 8 ? (row >> 1) & 7 : row & 15);
}

typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short i16x4;
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef const __attribute__((address_space(1))) void glob_void;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(4))) int32_t const_i32;  // read by scalar loads

// 16 bytes a lane from global memory straight into LDS (lane l's at dst + 16 l).  ONCE: what
// nobody reads again soon (the nt bit).
template <bool ONCE = false> __device__ __forceinline__ void load_lds16(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds((glob_void*)src, (lds_void*)dst, 16, 0, ONCE ? 2 : 0);
}

// V operand of step s, dims 16 nb ..  16-bit types: ds_read_b64_tr_b16 gives lane i of each
// 16 lanes element i & 3 of the 8-byte pieces that lanes (i >> 2) + 4 j address, j < 4.
template <class T, int HD>
__device__ __forceinline__ u32x4 v_operand(const T* vt, int s, int nb, int lane) {
  const int g = lane >> 4, col = lane & 15;
  if constexpr (sizeof(T) == 4) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = 16 * s + 4 * g + j;
      v[j] = __float_as_uint(vt[row * HD + 4 * v_piece<T, HD>(row, 4 * nb + (col >> 2)) + (col & 3)]);
    }
    return v;
  } else {
    u32x2 h[2];
#pragma unroll
    for (int jb = 0; jb < 2; ++jb) {
      const int row = 32 * s + 16 * jb + 4 * g + (col >> 2);
      const T* at = vt + row * HD + 8 * v_piece<T, HD>(row, 2 * nb + ((col & 3) >> 1)) + 4 * (col & 1);
      h[jb] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at));
    }
    return u32x4{h[0][0], h[0][1], h[1][0], h[1][1]};
  }
}

// O += P V over one step's keys; O[cb][nb]: row block cb, 16 dims.  l += the sum of the
// weights, a product with ones: every register holds the row's sum (of the rounded
// weights, so that they add up to one after the division).
template <class T, int CB, int NB>
__device__ __forceinline__ void step_pv(f32x4 (&O)[CB][NB], f32x4 (&l)[CB], const u32x4 (&P)[CB], const u32x4 (&v)[NB]) {
  const u32x4 ones = {Op<T>::ONES, Op<T>::ONES, Op<T>::ONES, Op<T>::ONES};
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    l[cb] = Op<T>::mfma(ones, P[cb], l[cb]);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) O[cb][nb] = Op<T>::mfma(v[nb], P[cb], O[cb][nb]);
  }
}

// Zero what is not finite in a wave's N loads of V rows (LDS, 64 x 16 bytes each, `step` elements
// apart); whether any lane found some.  All is read before anything is written, and looked through
// by the largest magnitude, which is not finite from a full exponent field on.
template <class T, int N>
__device__ __forceinline__ bool take_odd(T* at, int step) {
  constexpr bool W = sizeof(T) == 4;
  u32x4 v[N];
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = *(const u32x4*)(at + n * step);
  uint32_t most = 0;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t mag = v[n][i] & ~Op<T>::TOP;
      if constexpr (W) most = mag > most ? mag : most;
      else most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, mag), __builtin_bit_cast(u16x2, most)));
    }
  const bool found = W ? most >= Op<T>::EXP : (most & 0xffff) >= (Op<T>::EXP & 0xffff) || most >= (Op<T>::EXP & 0xffff0000u);
  if (!__any(found)) return false;
#pragma unroll 1
  for (int n = 0; n < N; ++n) {
    u32x4 x = *(const u32x4*)(at + n * step);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a full exponent field carries into the bit above it
      const uint32_t f = ((x[i] & Op<T>::EXP) + Op<T>::ONE) & Op<T>::TOP;
      x[i] &= ~((f << 1) - (f >> (8 * sizeof(T) - 1)));
    }
    *(u32x4*)(at + n * step) = x;
  }
  return true;
}

// What take_odd() took out of tile k0's V, read again from the pages and added to the
// rows that see it (weight 1: infinities and NaN, whatever the weight); dims 16 (nb0 + nb)
// ..  Rare, and kept small so that it costs the loop around it no registers.
template <class T, int HD, int CB, int NB>
__device__ __forceinline__ void add_odd(const AttnP& a, int b, int hk, f32x4 (&O)[CB][NB], int nb0, const Row (&r)[CB], int k0,
                                        int LO, int HI, int lane) {
  const int first = k0 > LO ? k0 : LO, end = k0 + TILE < HI ? k0 + TILE : HI;
#pragma unroll 1
  for (int key = first; key < end; ++key) {
    const int entry = key_entry(a, b, key, LO, HI);
    if (entry < 0 || entry >= a.n_pages) continue;
    const T* v = key_row<T>(a.v, entry, key, a.shift, a.kv_page, a.kv_slot, hk * a.kv_head) + 16 * nb0 + 4 * (unhoisted(lane) >> 4);
    uint32_t in[CB];  // rows that see the key: all ones
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) in[cb] = key >= r[cb].lo && key < r[cb].hi ? ~0u : 0u;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // integers rather than comparisons, whose masks would spill the loop's scalar registers
        // (packed documents of 128 dims 57 us so, 49 without; the largest dense chunks 125 and 119)
        const uint32_t e = __float_as_uint(to_f(v[16 * nb + i]));
        const uint32_t is_odd = (uint32_t)((int32_t)(0x7f7fffffu - (e & 0x7fffffffu)) >> 31);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
          const uint32_t add = is_odd & in[cb];
          O[cb][nb][i] += __uint_as_float((e & add) | (0x80000000u & ~add));  // or -0, which changes nothing
        }
      }
  }
}

// Fold a chunk's (m, l) into the totals; its O goes by the factors: O fa + o fb.
struct Fold {
  float fa, fb;
};
__device__ __forceinline__ Fold fold(float& M, float& L, float m, float l) {
#pragma clang fp contract(off)
  Fold f;
  const float Mn = fmaxf(M, m);
  f.fa = M == Mn ? 1.f : __builtin_amdgcn_exp2f(M - Mn);
  f.fb = m == Mn ? 1.f : __builtin_amdgcn_exp2f(m - Mn);  // 0 where the row saw nothing of the chunk
  L = __builtin_fmaf(l, f.fb, L * f.fa);
  M = Mn;
  return f;
}
__device__ __forceinline__ float folded(const Fold f, float O, float o) {
#pragma clang fp contract(off)
  return __builtin_fmaf(o, f.fb, O * f.fa);
}

template <class T>
__device__ __forceinline__ void store_out(const AttnP& a, const Row& r, int d, const f32x4 o, float inv) {
#pragma clang fp contract(off)
  typedef __attribute__((ext_vector_type(4))) T T4;
  T4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (T)(r.empty ? 0.f : o[i] * inv);
  *(T4*)((T*)a.out + r.t * a.o_tok + r.h * a.o_head + d) = v;
}

template <int HD>
__device__ __forceinline__ void store_part(const AttnP& a, const Row& r, int c, int d, const f32x4 o) {
  *(f32x4*)(a.part + ((r.t * a.H + r.h) * a.nc + c) * HD + d) = o;
}

// (the largest instances would leave their lambdas as calls, their captures in scratch memory)
#define ALTXS_INLINE __attribute__((always_inline))

// ---- few rows ----------------------------------------------------------------
//
// Bound by the cache read.  64 segments decoding at 2048 keys of 8 x 64 bf16 (268 MB): 47 us,
// 5.7 TB/s; 256 at 4096 (2.1 GB): 332 us, 6.5 TB/s (a large copy moves 5.1, a large read
// 5.8).  A workgroup has its chunk's 64 KB in flight at once and a CU holds two of them, which
// is what covers the memory latency; one segment at 2048 is all latency: 5.6 us in 64 workgroups of
// a chunk each, and the fold's 3.8.  The loads are marked as read once: caches of several layers do
// not stay in the memory-side cache from step to step (357 us without, and 49.3 / 47.5 over ten
// caches of 64 segments, 34.6 / 31.6 of 32; caches that would stay, two of 32 segments, 29.2 / 31.1).

template <class T, int HD, bool BIAS>
__global__ __launch_bounds__(THREADS, HD * sizeof(T) > 256 ? 1 : 2) void attn_few_kernel(AttnP a) {
#pragma clang fp contract(off)
  constexpr int EL = Op<T>::EL, KS = HD / (4 * EL), ST = STEPS<T>;  // pieces of a score; steps of P V
  constexpr int NB = HD / 16 / WAVES;                              // 16-dim blocks of a wave's share of O
  constexpr int PR = PIECES<T, HD>, RPL = WAVE / PR;               // rows of one LDS load
  __shared__ alignas(16) T vt[TPC][TILE * HD];
  __shared__ u32x4 pt[TPC][ST][WAVE];
  __shared__ float tmax[TPC][16];
  __shared__ int odd[TPC];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
  const int g = lane >> 4, col = lane & 15;
  const int slot = (int)div_by(blockIdx.x, a.by_hkv), hk = blockIdx.x - slot * a.Hkv;
  const RowTile tile = find_tile(a, slot, 16, lane, hk == 0 && blockIdx.y == 0 && wave == 0);
  if (tile.r0 >= tile.rows) return;
  if (!tile.s.ok && lane == 0) flag_err(a.err, ALTXS_EDEV_POS);
  const Row row[1] = {row_of(a, tile, hk, tile.r0 + col)};
  const Row& r = row[0];
  const Seen seen = seen_by(r);
  u32x4 q[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    q[s] = r.valid ? *(const u32x4*)((const T*)a.q + r.t * a.q_tok + r.h * a.q_head + EL * (4 * s + g)) : u32x4{0, 0, 0, 0};
  float M = -INFINITY, L = 0.f;
  f32x4 O[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) O[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int c_end = (seen.hi + CHUNK - 1) / CHUNK;
  if (seen.lo < seen.hi) {
    // K of a chunk is loaded while the one before it goes through P V, and its page
    // entries another chunk ahead (read for the nearest key of the union, past the end too).
    u32x4 k[4][KS];
    auto entry_of = [&](int64_t c) {
      const int64_t key = c * CHUNK + wave * TILE + lane;
      return key_entry(a, tile.b, key < seen.hi ? (int)key : seen.hi, seen.lo, seen.hi);
    };
    auto load_k = [&](int c, int entry) ALTXS_INLINE {
      const int k0 = c * CHUNK + wave * TILE, pg = entry_page(a, entry, k0 + lane, seen.lo, seen.hi);
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        const int i = 16 * kb + col;
        const T* src = key_row<T>(a.k, __shfl(pg, i, WAVE), k0 + i, a.shift, a.kv_page, a.kv_slot, hk * a.kv_head);
#pragma unroll
        for (int s = 0; s < KS; ++s) k[kb][s] = __builtin_nontemporal_load((const u32x4*)(src + EL * (4 * s + g)));
      }
      return pg;
    };
    int c = seen.lo / CHUNK + blockIdx.y;
    if (c >= c_end) return;  // (a shared row tile: the workgroup has no chunk of it)
    int pg = load_k(c, entry_of(c)), entry = entry_of((int64_t)c + gridDim.y);
    for (; c < c_end; c += gridDim.y) {
      const int k0 = c * CHUNK + wave * TILE;
#pragma unroll
      for (int i = 0; i < TILE / RPL; ++i) {
        const int vr = i * RPL + lane / PR;
        const T* src = key_row<T>(a.v, __shfl(pg, vr, WAVE), k0 + vr, a.shift, a.kv_page, a.kv_slot, hk * a.kv_head);
        load_lds16<true>(src + EL * v_piece<T, HD>(vr, lane % PR), vt[wave] + i * RPL * HD);
      }
      f32x4 S[1][4];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        S[0][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) S[0][kb] = Op<T>::mfma(k[kb][s], q[s], S[0][kb]);
      }
      float mx[1];
      tile_scores<BIAS, 1>(a, S, mx, row, k0, g, seen.full(k0));
      if (g == 0) tmax[wave][col] = mx[0];
      __syncthreads();
      float m = -INFINITY, mw = 0.f, al[TPC];
#pragma unroll
      for (int t = 0; t < TPC; ++t) {
        al[t] = next_max(m, tmax[t][col]);
        if (t == wave) mw = m;
      }
#pragma unroll
      for (int s = 0; s < ST; ++s) pt[wave][s][lane] = step_weights<T, BIAS>(a, S[0], s, mw);
      __builtin_amdgcn_s_waitcnt(0);  // the wave's V tile
      if (seen.mixed(k0, seen.lo, seen.hi)) {
        const bool any = take_odd<T, TILE / RPL>(vt[wave] + EL * lane, RPL * HD);
        if (lane == 0) odd[wave] = any;
      }
      __syncthreads();
      if (c + (int)gridDim.y < c_end) {
        pg = load_k(c + gridDim.y, entry);
        entry = entry_of((int64_t)c + 2 * gridDim.y);
      }
      f32x4 l[1] = {f32x4{0.f, 0.f, 0.f, 0.f}}, o[1][NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) o[0][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < TPC; ++t) {
        l[0] *= al[t];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) o[0][nb] *= al[t];
#pragma unroll
        for (int s = 0; s < ST; ++s) {
          u32x4 v[NB];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) v[nb] = v_operand<T, HD>(vt[t], s, wave * NB + nb, lane);
          const u32x4 P[1] = {pt[t][s][lane]};
          step_pv<T, 1, NB>(o, l, P, v);
        }
      }
#pragma unroll 1
      for (int t = 0; t < TPC; ++t) {
        const int kt = c * CHUNK + t * TILE;
        if (seen.mixed(kt, seen.lo, seen.hi) && __builtin_amdgcn_readfirstlane(odd[t]))
          add_odd<T, HD, 1, NB>(a, tile.b, hk, o, wave * NB, row, kt, seen.lo, seen.hi, lane);
      }
      if (a.direct) {
        const Fold f = fold(M, L, m, l[0][0]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) O[nb][i] = folded(f, O[nb][i], o[0][nb][i]);
      } else if (r.valid) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) store_part<HD>(a, r, c, 16 * (wave * NB + nb) + 4 * g, o[0][nb]);
        if (wave == 0 && g == 0) a.ml[(r.t * a.H + r.h) * a.nc + c] = float2{m, l[0][0]};
      }
      __syncthreads();  // the chunk's LDS is free
    }
  }
  if (a.direct && r.valid) {
    const float inv = 1.f / L;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) store_out<T>(a, r, 16 * (wave * NB + nb) + 4 * g, O[nb], inv);
  }
}

// ---- many rows ---------------------------------------------------------------
//
// Bound by instruction issue: 16 x 2048 new tokens of 8 x 64 bf16 119 us, 577 TFLOP/s (of 1254 that
// a large product reaches), 128 dims 244 us, 563 TFLOP/s; the matrix cores are busy a
// quarter of the time and the vector units half of it (a score takes an fma, an exponential,
// half a conversion and its share of the maximum and the masks), at two waves a SIMD, which
// the accumulators of a chunk and of the total leave room for.  Eight waves of 16 rows
// (four a SIMD) spill them: 651 us for 244.  fp32, 4 x 2048: 188 us, 91 TFLOP/s.

constexpr int NW = 4;  // waves of a workgroup
// 16-row blocks of a wave, and rows of a workgroup
template <class T, int HD> constexpr int many_cb = HD * sizeof(T) == 128 ? 2 : 1;
template <class T, int HD> constexpr int many_rows = NW * 16 * many_cb<T, HD>;

// Workgroup i -> (slot, kv head).  The last row tiles of a segment see the most keys:
// they go first -- of equal segments all last tiles, then all second to last ones, each
// over (kv head, segment) with the segment running fastest: workgroups are dealt to the
// 8 XCDs in turn, so (for a multiple of 8 pairs) a pair's tiles share an L2, and an XCD's
// pairs spread over it (all of one kv head they would meet in an eighth of its sets:
// pages of 64 KB hold 8 KB a head).  Ragged segments: the slots backwards.
__device__ __forceinline__ int many_slot(const AttnP& a, int i, int& hk) {
  if (a.cu) {
    const int slot = (int)div_by(i, a.by_hkv);
    hk = i - slot * a.Hkv;
    return (int)(gridDim.x / a.Hkv) - 1 - slot;
  }
  const int back = (int)div_by(i, a.by_pairs), pair = i - back * (int)a.by_pairs.d;
  hk = (int)div_by(pair, a.by_b);
  return (pair - hk * a.B + 1) * (int)a.by_tiles.d - 1 - back;
}

template <class T, int HD, bool BIAS>
__global__ __launch_bounds__(NW* WAVE, HD * sizeof(T) > 256 ? 1 : 2) void attn_many_kernel(AttnP a) {
#pragma clang fp contract(off)
  constexpr int CB = many_cb<T, HD>, MANY = many_rows<T, HD>, EL = Op<T>::EL, KS = HD / (4 * EL), ST = STEPS<T>, NB = HD / 16;
  constexpr int PR = PIECES<T, HD>, RPW = WAVE / PR, RPL = NW * RPW, LOADS = TILE / RPL;  // rows of a wave's load, of the workgroup's; loads
  static_assert(16 % RPW == 0 && RPL % 8 == 0, "a load's rows lie in one page");
  constexpr int KINDS = RPL % 16 == 0 ? 1 : 2;  // pieces are permuted by the row modulo 16: alike in every load, or in every other
  // separate arrays: reads of one buffer do not wait for the loads into the other
  __shared__ alignas(16) T kt0[TILE * HD], kt1[TILE * HD], vt0[TILE * HD], vt1[TILE * HD];
  __shared__ int range[4][NW], odd[2][NW];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
  const int g = lane >> 4, col = lane & 15;
  int hk;
  const int slot = many_slot(a, blockIdx.x, hk);
  const RowTile tile = find_tile(a, slot, MANY, lane, hk == 0 && blockIdx.y == 0 && wave == 0);
  if (tile.r0 >= tile.rows) return;
  if (!tile.s.ok && threadIdx.x == 0) flag_err(a.err, ALTXS_EDEV_POS);
  Row r[CB];
  u32x4 q[CB][KS];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    r[cb] = row_of(a, tile, hk, tile.r0 + 16 * (wave * CB + cb) + col);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      q[cb][s] = r[cb].valid ? *(const u32x4*)((const T*)a.q + r[cb].t * a.q_tok + r[cb].h * a.q_head + EL * (4 * s + g))
                             : u32x4{0, 0, 0, 0};
  }
  Seen seen = seen_by(r[0]);
#pragma unroll
  for (int cb = 1; cb < CB; ++cb) seen = both(seen, seen_by(r[cb]));
  if (lane == 0) {
    range[0][wave] = seen.lo;
    range[1][wave] = seen.hi;
    range[2][wave] = seen.clo;
    range[3][wave] = seen.chi;
  }
  __syncthreads();
  Seen all = {INT32_MAX, 0, 0, INT32_MAX};
#pragma unroll
  for (int w = 0; w < NW; ++w) all = both(all, Seen{range[0][w], range[1][w], range[2][w], range[3][w]});
  const int LO = __builtin_amdgcn_readfirstlane(all.lo), HI = __builtin_amdgcn_readfirstlane(all.hi);
  // tiles [in0, in1) are seen whole by every row of the workgroup
  all.clo = __builtin_amdgcn_readfirstlane(all.clo);
  all.chi = __builtin_amdgcn_readfirstlane(all.chi);
  const int in0 = (all.clo + TILE - 1) / TILE, in1 = all.chi / TILE;

  float m[CB], M[CB], L[CB];
  f32x4 l[CB], O[CB][NB], Ot[CB][NB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    m[cb] = M[cb] = -INFINITY;
    L[cb] = 0.f;
    l[cb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) O[cb][nb] = Ot[cb][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int t_end = LO < HI ? (HI + TILE - 1) / TILE : 0, skip = TPC * ((int)gridDim.y - 1);
  auto after = [&](int t) { return (t & (TPC - 1)) == TPC - 1 ? t + 1 + skip : t + 1; };
  // Loads go by whole waves, 2 to 8 rows at a time, all in one page, whose entry is a
  // scalar; with pages of a tile or more one entry serves the whole tile.  Entries are
  // read for the nearest tile or key of the union (inside the table).
  const const_i32* entries = (const const_i32*)(a.table + (int64_t)tile.b * a.width);
  const bool large = a.shift >= 6;
  auto lookup = [&](int t, int (&e)[LOADS]) ALTXS_INLINE {
    if (large) {
      const int entry = entries[(t < t_end ? t : t_end - 1) >> (a.shift - 6)];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) e[i] = entry;
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        int key = t * TILE + i * RPL + wave * RPW;
        key = key < LO ? LO : key >= HI ? HI - 1 : key;
        e[i] = entries[key >> a.shift];
      }
    }
  };
  const uint32_t n_pages = a.n_pages < INT32_MAX ? (uint32_t)a.n_pages : INT32_MAX;
  const int whole0 = (LO + TILE - 1) / TILE;  // tiles all of whose keys are in the union
  const uint32_t wholes = HI / TILE > whole0 ? HI / TILE - whole0 : 0;
  const int krow = wave * RPW + lane / PR;
  const T *kl[KINDS], *vl[KINDS];
#pragma unroll
  for (int i = 0; i < KINDS; ++i) {
    kl[i] = (const T*)a.k + hk * a.kv_head + (uint64_t)krow * a.kv_slot + EL * k_piece<T, HD>(krow + i * RPL, lane % PR);
    vl[i] = (const T*)a.v + hk * a.kv_head + (uint64_t)krow * a.kv_slot + EL * v_piece<T, HD>(krow + i * RPL, lane % PR);
  }
  const uint64_t down = RPL * (uint64_t)a.kv_slot;  // a load's rows to the next one's
  auto load = [&](int t, const int (&e)[LOADS], T* kb, T* vb) ALTXS_INLINE {
    const bool whole = (uint32_t)(t - whole0) < wholes;
    if (large && whole && (uint32_t)e[0] < n_pages) {
      uint64_t at = (uint64_t)(uint32_t)e[0] * a.kv_page + (uint64_t)(uint32_t)((t << 6) & ((1 << a.shift) - 1)) * a.kv_slot;
#pragma unroll
      for (int i = 0; i < LOADS; ++i, at += down) {
        const int to = (i * RPL + wave * RPW) * HD;
        load_lds16(kl[i % KINDS] + at, kb + to);
        load_lds16(vl[i % KINDS] + at, vb + to);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int first = i * RPL, key = t * TILE + first + wave * RPW, entry = e[i];
      const bool good = (uint32_t)entry < n_pages;
      // kl and vl already stand krow rows into the page
      const uint64_t at = (uint64_t)(good ? (uint32_t)entry : 0) * a.kv_page +
                          (int64_t)((key & ((1 << a.shift) - 1)) - wave * RPW) * (int64_t)a.kv_slot;
      const T* ks = kl[i % KINDS] + at;
      const T* vs = vl[i % KINDS] + at;
      const int to = (first + wave * RPW) * HD;
      if (!(whole && good)) {
        const int ln = unhoisted(lane), row = first + wave * RPW + ln / PR;
        const bool in = key + ln / PR >= LO && key + ln / PR < HI;
        if (in && !good) flag_err(a.err, ALTXS_EDEV_PAGE);
        if (!in || !good) {
          ks = (const T*)kZeroRow + EL * k_piece<T, HD>(row, ln % PR);
          vs = (const T*)kZeroRow + EL * v_piece<T, HD>(row, ln % PR);
        }
      }
      load_lds16(ks, kb + to);
      load_lds16(vs, vb + to);
    }
  };

  int t = 0, tn = 0, odd_tiles = 0;  // odd_tiles: of the chunk, a bit each
  // One tile out of (kb, vb), buffer buf.  EDGE: some row does not see it whole.
  auto work = [&](auto edge, const T* kb, const T* vb, int buf) ALTXS_INLINE {
    constexpr bool EDGE = decltype(edge)::value;
    const int k0 = t * TILE;
    if (EDGE && !(seen.lo < k0 + TILE && seen.hi > k0)) return;  // no row of the wave sees any of it
    const int found = EDGE ? odd[buf][lane % NW] : 0;  // used at the end, if the tile is mixed
    f32x4 S[CB][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) S[cb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int row = 16 * j + col;
        const u32x4 k = *(const u32x4*)(kb + row * HD + EL * k_piece<T, HD>(row, 4 * s + g));
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) S[cb][j] = Op<T>::mfma(k, q[cb][s], S[cb][j]);
      }
    }
    float mx[CB], al[CB];
    tile_scores<BIAS, CB>(a, S, mx, r, k0, g, !EDGE || seen.full(k0));
    bool moved = false;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      al[cb] = next_max(m[cb], mx[cb]);
      moved = moved || al[cb] != 1.f;
    }
    if (__any(moved)) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        l[cb] *= al[cb];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) O[cb][nb] *= al[cb];
      }
    }
    u32x4 P[ST][CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int s = 0; s < ST; ++s) P[s][cb] = step_weights<T, BIAS>(a, S[cb], s, m[cb]);
#pragma unroll
    for (int s = 0; s < ST; ++s) {
      u32x4 v[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) v[nb] = v_operand<T, HD>(vb, s, nb, lane);
      step_pv<T, CB, NB>(O, l, P[s], v);
    }
    if (EDGE && all.mixed(k0, LO, HI)) {
      odd_tiles |= __any(found != 0) << (t & (TPC - 1));
    }
  };
  // Before the workgroup meets over tile t in buffer buf: the rows that this wave loaded.
  auto clean = [&](int t, T* vb, int buf) ALTXS_INLINE {
    if (!all.mixed(t * TILE, LO, HI)) return;
    const bool any = take_odd<T, LOADS>(vb + wave * RPW * HD + EL * lane, RPL * HD);
    if (lane == 0) odd[buf][wave] = any;
  };
  auto end_chunk = [&]() ALTXS_INLINE {
    for (; odd_tiles; odd_tiles &= odd_tiles - 1)
      add_odd<T, HD, CB, NB>(a, tile.b, hk, O, 0, r, (t / TPC * TPC + __builtin_ctz(odd_tiles)) * TILE, LO, HI, lane);
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      if (a.direct) {
        const Fold f = fold(M[cb], L[cb], m[cb], l[cb][0]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) Ot[cb][nb][i] = folded(f, Ot[cb][nb][i], O[cb][nb][i]);
      } else if (r[cb].valid) {
        const int c = (unsigned)t / TPC;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) store_part<HD>(a, r[cb], c, 16 * nb + 4 * g, O[cb][nb]);
        if (g == 0) a.ml[(r[cb].t * a.H + r[cb].h) * a.nc + c] = float2{m[cb], l[cb][0]};
      }
      m[cb] = -INFINITY;
      l[cb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) O[cb][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };
  // Tile t out of (kb, vb) while the next one, tn, whose entries are in en, is loaded into
  // (kn, vn), and the entries of the one after it are read; false after the last.
  int en[LOADS];
  const uint32_t n_in = in1 > in0 ? in1 - in0 : 0;
  auto step = [&](const T* kb, const T* vb, T* kn, T* vn, int buf) ALTXS_INLINE {
    if (tn < t_end) load(tn, en, kn, vn);
    const int tnn = after(tn);
    lookup(tnn, en);
    if ((uint32_t)(t - in0) < n_in) work(std::false_type{}, kb, vb, buf);
    else work(std::true_type{}, kb, vb, buf);
    if ((t & (TPC - 1)) == TPC - 1 || tn >= t_end) end_chunk();
    if (tn >= t_end) return false;
    __builtin_amdgcn_s_waitcnt(0);  // the wave's part of the next tile is there
    clean(tn, vn, buf ^ 1);
    __syncthreads();  // all of it is, and this one's buffer is free
    t = tn;
    tn = tnn;
    return true;
  };
  if (LO < HI) t = blockIdx.y == 0 ? LO / TILE : (LO / CHUNK + (int)blockIdx.y) * TPC;
  if (t < t_end) {
    lookup(t, en);
    load(t, en, kt0, vt0);
    tn = after(t);
    lookup(tn, en);
    __builtin_amdgcn_s_waitcnt(0);
    clean(t, vt0, 0);
    __syncthreads();
    while (step(kt0, vt0, kt1, vt1, 0) && step(kt1, vt1, kt0, vt0, 1)) {}
  }
  if (a.direct) {
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
      if (r[cb].valid) {
        const float inv = 1.f / L[cb];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) store_out<T>(a, r[cb], 16 * nb + 4 * g, Ot[cb][nb], inv);
      }
  }
}

// ---- folding the chunks' partial results ---------------------------------------

// One wave per (token, head): a dim (or two) per lane for O, and for each 64 chunks a
// chunk per lane for the factors -- the running maximum is a prefix maximum, so a
// scan over the lanes gives the values of fold() for all of them at once.  O is
// folded in order with the chunks' loads two groups ahead.  Bound by latency: 512 rows of
// 128 chunks (17.8 MB) 8.8 us, 1 row of 9 chunks 3.8 us, most of it the start of a launch; factors
// through LDS or 32 chunks ahead gain nothing (8.2 to 11.3 us).
template <class T, int HD>
__global__ __launch_bounds__(THREADS) void attn_fold_kernel(AttnP a) {
#pragma clang fp contract(off)
  constexpr int ND = HD / WAVE, AHEAD = 16;
  typedef __attribute__((ext_vector_type(ND))) float vec;
  const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const int64_t row = (int64_t)blockIdx.x * WAVES + wave;
  if (row >= a.T * a.H) return;
  const int64_t t = row / a.H;
  const int h = (int)(row - t * a.H);
  Segment s;
  const int b = token_segment(a.cu, a.pos, a.B, a.W, t, a.T, a.cap, lane, s);
  if (b < 0 || t < s.t0 || t >= s.t0 + s.n) return;
  Range r = {0, 0};
  if (s.ok) r = keys_seen(s.pos + (int)(t - s.t0), s.pos + s.n, a.window, a.starts ? a.starts[t] : 0, a.prefix ? a.prefix[b] : 0);
  const float* part = a.part + row * a.nc * HD + lane * ND;
  const float2* ml = a.ml + row * a.nc;
  const int c0 = __builtin_amdgcn_readfirstlane(r.lo / CHUNK), c1 = __builtin_amdgcn_readfirstlane((r.hi + CHUNK - 1) / CHUNK);
  float M = -INFINITY, L = 0.f;
  vec O = 0.f;
  vec o[2][AHEAD];
  auto get = [&](int c, vec (&o)[AHEAD]) {  // past the end: the last one again, unused
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) o[j] = *(const vec*)(part + (int64_t)(c + j < c1 ? c + j : c1 - 1) * HD);
  };
  for (int c = c0; c < c1; c += WAVE) {
    const float2 x = c + lane < c1 ? ml[c + lane] : float2{-INFINITY, 0.f};
    get(c, o[0]);
    float mx = fmaxf(x.x, M);  // maximum of the chunks up to the lane's
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) {
      const float up = __shfl_up(mx, d, WAVE);
      mx = fmaxf(mx, lane >= d ? up : -INFINITY);
    }
    const float up = __shfl_up(mx, 1, WAVE), before = lane ? up : M;
    const float fa = before == mx ? 1.f : __builtin_amdgcn_exp2f(before - mx);
    const float fb = x.x == mx ? 1.f : __builtin_amdgcn_exp2f(x.x - mx);
    auto add = [&](int j0, const vec (&o)[AHEAD]) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const float fj = lane_f(fa, j0 + j), gj = lane_f(fb, j0 + j), lj = lane_f(x.y, j0 + j);
        if (c + j0 + j < c1) {
          L = __builtin_fmaf(lj, gj, L * fj);
#pragma unroll
          for (int i = 0; i < ND; ++i) O[i] = __builtin_fmaf(o[j][i], gj, O[i] * fj);
        }
      }
    };
#pragma unroll
    for (int j0 = 0; j0 < WAVE; j0 += 2 * AHEAD) {
      if (c + j0 + AHEAD < c1) get(c + j0 + AHEAD, o[1]);
      add(j0, o[0]);
      if (c + j0 + 2 * AHEAD < c1 && j0 + 2 * AHEAD < WAVE) get(c + j0 + 2 * AHEAD, o[0]);
      if (c + j0 + AHEAD < c1) add(j0 + AHEAD, o[1]);
    }
    M = lane_f(mx, WAVE - 1);
  }
  const float inv = 1.f / L;
  T* out = (T*)a.out + t * a.o_tok + h * a.o_head + lane * ND;
#pragma unroll
  for (int i = 0; i < ND; ++i) out[i] = (T)(r.lo < r.hi ? O[i] * inv : 0.f);
}

// ---- host ------------------------------------------------------------------------

// How a call is launched (host decisions only; none of them changes a row's bits).
// Rows of a tile of the many-row kernel.
int many(const AltxsPagedAttnArgs* a) {
  if (a->dtype == ALTXS_F32) return a->head_dim == 64 ? many_rows<float, 64> : many_rows<float, 128>;
  return a->head_dim == 64 ? many_rows<__bf16, 64> : many_rows<__bf16, 128>;
}

struct Plan {
  bool few;
  int nc;       // chunks of max_len
  int64_t wgs;  // row-tile slots x kv heads
  int split;    // workgroups that share a row tile's chunks
  int64_t rows;
};

Plan plan_of(const AltxsPagedAttnArgs* a) {
  Plan p = {};
  p.rows = a->T * a->H;
  p.nc = (a->max_len + CHUNK - 1) / CHUNK;
  if (p.nc < 1) p.nc = 1;
  p.split = 1;
  if (a->T == 0 || a->B == 0) return p;
  const int G = a->H / a->Hkv;
  p.few = a->T * G <= 16 * (int64_t)a->B;
  const int br = p.few ? 16 : many(a);
  const int64_t slots = a->cu ? slot_count(a->T, G, br, a->B) : (int64_t)a->B * ((a->T / a->B * G + br - 1) / br);
  p.wgs = slots * a->Hkv;
  // Row tiles that there are, about: ragged segments' slots are up to B more.
  int64_t tiles = slots;
  if (a->cu) tiles = std::max(std::min((int64_t)a->B, a->T), (a->T * G + br - 1) / br);
  tiles *= a->Hkv;
  // Share a row tile's chunks among workgroups where the row tiles alone do not fill the
  // chip and that saves well more than the fold costs: a launch, and the partial results
  // written and read at ~3 TB/s.
  // Few: a workgroup takes a chunk in 3.6 us (rows of 128 bytes) to 9.3 (of 512), half as
  // long again where a CU holds two, and no call reads faster than ~6 TB/s.  Measured, one workgroup
  // against shared: 2 segments decoding at 2048 22.6 / 9.4 us, 40 (8 heads of 64) 42.8 / 36.0, 48 42.3 /
  // 43.6; 16 over 2 heads of 128 at 4096, 64 segments 85.7 / 58.1, 128 segments 97.3 / 114.6.
  // Many: ~4.8 us a chunk.  Windows of 512 tokens at 8000 163 / 37 us, but chunks of 1024 and 4096
  // tokens from position 0 24.2 / 23.5 and 81 / 87.
  // Shared no further than what is resident: few 64 segments of 16 over 2 heads of 128 at 4096 58.1
  // by 512 workgroups, 61.4 by 2048; many, those windows of 512 37.3 by 512, 40.4 by 1024; 48 drafts of up
  // to 9 tokens 33.7 us counted by their slots and 31.0 by their tiles.
  const int64_t fill = p.few ? 768 : 512;
  if (tiles < 384) {
    int64_t z = (fill + tiles - 1) / tiles;
    z = std::max<int64_t>(1, std::min<int64_t>({z, p.nc, 4 * fill / p.wgs}));  // idle segments' workgroups cost their start
    const int es = a->dtype == ALTXS_F32 ? 4 : 2;
    const double fold_us = 4.0 + (double)p.rows * p.nc * (a->head_dim + 2) * 8 / 3e6;
    const double chunk_us = p.few ? (1.7 + 1.9 * a->head_dim * es / 128) * (tiles > 256 ? 1.5 : 1.0) : 4.8;
    const double read_us = p.few ? (double)tiles * p.nc * CHUNK * a->head_dim * es * 2 / 6e6 : 0.0;
    const double one = std::max(p.nc * chunk_us, read_us), shared = std::max((p.nc + z - 1) / z * chunk_us, read_us) + fold_us;
    if (one > (p.few ? 1.15 : 1.5) * shared) p.split = (int)z;
  }
  return p;
}

int64_t ws_bytes(const Plan& p, int hd) { return p.split > 1 ? ((p.rows * p.nc + 1) / 2 * 4 + p.rows * p.nc * hd) * 4 : 0; }

}  // namespace

static int32_t check(const AltxsPagedAttnArgs* a, const char* who) {
  ALTXS_REQUIRE(a, "%s: null pointer", who);
  ALTXS_REQUIRE(a->dtype == ALTXS_F32 || a->dtype == ALTXS_BF16 || a->dtype == ALTXS_F16, "%s: dtype=%d", who, a->dtype);
  ALTXS_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "%s: head_dim=%d (64 and 128 are built)", who, a->head_dim);
  ALTXS_REQUIRE(a->Hkv >= 1 && a->H >= a->Hkv && a->H <= 4096 && a->H % a->Hkv == 0, "%s: H=%d is not a multiple of Hkv=%d",
                who, a->H, a->Hkv);
  ALTXS_REQUIRE(a->page_size >= 16 && a->page_size <= 1024 && (a->page_size & (a->page_size - 1)) == 0,
                "%s: page_size=%d must be a power of two from 16 to 1024", who, a->page_size);
  ALTXS_REQUIRE(a->T >= 0 && a->T < (1ll << 31) && a->T * a->H < (1ll << 31) && a->B >= 0 && a->n_pages >= 0 && a->table_width >= 0,
                "%s: bad T, B, n_pages or table_width", who);
  ALTXS_REQUIRE(a->max_len >= 0 && a->max_len <= (int64_t)a->table_width * a->page_size && a->max_len <= 1 << 30,
                "%s: max_len=%d is more than table_width * page_size or 2^30", who, a->max_len);
  for (int64_t st : {a->kv_page, a->kv_head, a->kv_slot})
    ALTXS_REQUIRE(st >= 0 && st < (1ll << 31), "%s: a cache stride of %lld elements", who, (long long)st);
  ALTXS_REQUIRE(a->scale > 0.f && a->scale * LOG2E < INFINITY, "%s: scale=%g must be positive", who, a->scale);
  ALTXS_REQUIRE(a->softcap == 0.f || (a->softcap > 0.f && a->softcap * LOG2E < INFINITY && 2.f * (a->scale * LOG2E) / a->softcap < INFINITY),
                "%s: softcap=%g", who, a->softcap);
  ALTXS_REQUIRE(a->window >= 0, "%s: window=%d", who, a->window);
  ALTXS_REQUIRE(a->T == 0 || a->B == 0 || a->cu || a->T % a->B == 0, "%s: T=%lld tokens are not B=%d equal segments", who,
                (long long)a->T, a->B);
  return ALTXS_OK;
}

extern "C" int64_t altxs_paged_attn_workspace_bytes(const AltxsPagedAttnArgs* a) {
  const int32_t rc = check(a, "altxs_paged_attn_workspace_bytes");
  return rc ? rc : ws_bytes(plan_of(a), a->head_dim);
}

extern "C" int32_t altxs_paged_attn(const AltxsPagedAttnArgs* a, altxs_stream_t stream) {
  const int32_t rc = check(a, "altxs_paged_attn");
  if (rc) return rc;
  if (a->T == 0 || a->B == 0) return ALTXS_OK;
  ALTXS_REQUIRE(a->q && a->out && a->k_cache && a->v_cache && a->table && a->pos, "altxs_paged_attn: null pointer");
  const Plan pl = plan_of(a);
  // 2^32 threads a launch; also B * Hkv < 2^24, as each segment has a tile
  ALTXS_REQUIRE(pl.wgs < (1ll << 24), "altxs_paged_attn: too many row tiles (T=%lld, B=%d)", (long long)a->T, a->B);
  uintptr_t bits = (uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->k_cache | (uintptr_t)a->v_cache;
  for (int64_t st : {a->q_tok, a->q_head, a->out_tok, a->out_head, a->kv_page, a->kv_head, a->kv_slot})
    bits |= (uintptr_t)(st * (a->dtype == ALTXS_F32 ? 4 : 2));
  ALTXS_REQUIRE((bits & 15) == 0, "altxs_paged_attn: rows of q, out and the caches must start at multiples of 16 bytes");
  const int64_t need = ws_bytes(pl, a->head_dim);
  ALTXS_REQUIRE(need == 0 || (a->ws && a->ws_bytes >= need && ((uintptr_t)a->ws & 15) == 0),
                "altxs_paged_attn: %lld workspace bytes needed, 16-byte aligned (%lld given)", (long long)need,
                (long long)a->ws_bytes);
  AttnP p;
  p.q = a->q; p.k = a->k_cache; p.v = a->v_cache; p.out = a->out;
  p.table = a->table; p.pos = a->pos; p.cu = a->cu; p.starts = a->starts; p.prefix = a->prefix;
  p.slopes = a->slopes; p.err = a->err;
  p.T = a->T; p.n_pages = a->n_pages; p.q_tok = a->q_tok; p.q_head = a->q_head; p.o_tok = a->out_tok; p.o_head = a->out_head;
  p.kv_page = (uint32_t)a->kv_page; p.kv_head = a->kv_head; p.kv_slot = (uint32_t)a->kv_slot;
  p.scale = a->scale; p.softcap = a->softcap; p.scale2 = a->scale * LOG2E;
  p.B = a->B; p.W = a->cu ? 1 : (int)(a->T / a->B); p.H = a->H; p.Hkv = a->Hkv; p.G = a->H / a->Hkv;
  p.width = a->table_width; p.shift = __builtin_ctz((unsigned)a->page_size); p.cap = a->max_len; p.window = a->window;
  p.by_g = fast_div(p.G); p.by_hkv = fast_div(p.Hkv); p.by_b = fast_div(p.B); p.by_pairs = fast_div((uint32_t)((int64_t)p.B * p.Hkv));
  const int br = pl.few ? 16 : many(a);
  p.by_tiles = fast_div((uint32_t)(((int64_t)p.W * p.G + br - 1) / br));
  p.nc = pl.nc; p.direct = pl.split == 1;
  p.ml = (float2*)a->ws;  // then O, from a multiple of 16 bytes on
  p.part = (float*)a->ws + (pl.rows * pl.nc + 1) / 2 * 4;
  const hipStream_t s = (hipStream_t)stream;
  const dim3 block(THREADS), by_row((unsigned)((pl.rows + WAVES - 1) / WAVES));
  const bool bias = a->softcap > 0.f || a->slopes;
#define ALTXS_HD_GO(K, ...)                                                          \
  do {                                                                               \
    if (a->head_dim == 64) hipLaunchKernelGGL((K<T, 64, ##__VA_ARGS__>), grid, block, 0, s, p);  \
    else hipLaunchKernelGGL((K<T, 128, ##__VA_ARGS__>), grid, block, 0, s, p);       \
  } while (0)
  auto go = [&](auto t) {
    using T = decltype(t);
    dim3 grid((unsigned)pl.wgs, (unsigned)pl.split);
    if (pl.few && bias) ALTXS_HD_GO(attn_few_kernel, true);
    else if (pl.few) ALTXS_HD_GO(attn_few_kernel, false);
    else {
      const dim3 block(NW * WAVE);
      if (bias) ALTXS_HD_GO(attn_many_kernel, true);
      else ALTXS_HD_GO(attn_many_kernel, false);
    }
    if (pl.split > 1) {
      grid = by_row;
      ALTXS_HD_GO(attn_fold_kernel);
    }
  };
  if (a->dtype == ALTXS_F32) go(float{});
  else if (a->dtype == ALTXS_BF16) go(__bf16{});
  else go(_Float16{});
#undef ALTXS_HD_GO
  ALTXS_CHECK_HIP(hipGetLastError());
  return ALTXS_OK;
}
