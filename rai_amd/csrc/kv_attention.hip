// Attention of packed rows of many requests over a paged cache of 8-bit codes (kv_cache.h), from one row a request to
// whole prompts.  No counterpart in the reference.
#include "kv_cache.h"

namespace rai {

typedef __attribute__((ext_vector_type(2))) __bf16 kv_bf16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 kv_bf16x8;
typedef __attribute__((ext_vector_type(4))) float kv_f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t kv_u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t kv_u32x2;
typedef __attribute__((ext_vector_type(2))) float kv_f32x2;

// One of the two kinds of work of a launch: tiles of few columns (16) or of many.
struct KvKind {
  int which;                     // requests served: 0 all, 1 those of up to 16 columns, 2 the others
  int blocks;                    // of the launch
  int workers;                   // of a key head, each with an even share of the steps; 0: a worker to a tile
  int each, extra;               // sixteenths of a key that a tile sees more than the one before it, and that its beginning and end are worth
  int least;                     // steps of a share at least
  double per_worker;             // 1 / workers
  float *part;                   // [Hkv * workers][2][columns of a tile][features] sums of a share's first and last tile
  float *part_m, *part_l;        // their maxima and sums of weights
  struct KvJoin *join;           // [Hkv * workers]
};
// The tile whose last part is a worker's first: workers first .. the worker itself have its parts.  (Whole 16 bytes: behind these of one kind lie the sums of the other,
// which are written 16 bytes at a time.)
struct alignas(16) KvJoin {
  int first;                     // -1: none
  int place;                     // which of the first worker's two parts
  int start, column, columns;    // the tile's request's first row, its first column and how many it has
};
struct KvAttnArgs {
  const void *q;
  void *out;
  int64_t q_row, q_head;
  const uint32_t *tables;
  int64_t table_ld, M, N;
  const int64_t *starts, *lens;
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  uint32_t pages;
  int dev, R, Hq, Hkv, G, D, features, page_shift;
  int64_t window;
  float scale_log2;              // |scale| * log2(e)
  uint32_t turn;                 // the signs of two bf16 where the scale is negative
  double per_group;              // 1 / G
  int reach;                     // keys that the oldest token of a tile sees, at most
  unsigned long long *errors;
  KvKind few, many;
};

// Eight codes as the eight bf16 of a fragment: every e4m3 value and every whole number up to 127 is a bf16.
template <int FMT> __device__ __forceinline__ kv_bf16x8 kv_unpack(uint32_t lo, uint32_t hi) {
  union { kv_bf16x2 p[4]; kv_bf16x8 v; } u;
  if constexpr (FMT == RAI_KV_E4M3) {
    u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = (int)(i < 2 ? lo : hi) >> (i & 1 ? 16 : 0);
      const kv_f32x2 f = {(float)(int8_t)x, (float)(int8_t)(x >> 8)};
      u.p[i] = __builtin_convertvector(f, kv_bf16x2);
    }
  }
  return u.v;
}

// Read by one tile alone, so not to be kept in the L2.
__device__ __forceinline__ kv_u32x4 fetch_once(const uint8_t *p) { return __builtin_nontemporal_load(reinterpret_cast<const kv_u32x4 *>(p)); }

// How many bf16 hold a value of type T: products with codes are then exact, so f16 and f32 rows lose nothing on the bf16 matrix instructions.  The softmax's
// weights are rounded to as many, to two at least: to 16 significant bits in every tile, so that neither the batch nor the width of its tables decides how far a
// result is off.  With one, results of bf16 rows are off by 0.0022 to 0.0024 of their size, with two by 0.0016 to 0.0017, which is the output's own rounding.  It
// costs nothing where a step waits for memory (64 requests 51 us either way), but an eighth where instructions bound it: prompts of 2300 rows 87 us for 77.
template <typename T> struct KvTerms;
template <> struct KvTerms<bf16_raw> { static constexpr int n = 1, weights = 2; };
template <> struct KvTerms<f16_raw> { static constexpr int n = 2, weights = 2; };
template <> struct KvTerms<float> { static constexpr int n = 3, weights = 3; };

__device__ __forceinline__ float bf16_part(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// Two values' terms: cut off (not rounded), so that what is left is exact, the last term rounded.
template <int TERMS> __device__ __forceinline__ void kv_split2(float x, float y, kv_bf16x2 *out) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    if (t == TERMS - 1) {
      const kv_f32x2 f = {x, y};
      out[t] = __builtin_convertvector(f, kv_bf16x2);
    } else {
      const float a = bf16_part(x), b = bf16_part(y);
      out[t] = __builtin_bit_cast(kv_bf16x2, (__float_as_uint(a) >> 16) | __float_as_uint(b));
      x -= a;
      y -= b;
    }
  }
}

// max and sum over the four lanes that hold a column (l, l ^ 16, l ^ 32, l ^ 48)
template <typename Op> __device__ __forceinline__ float column_fold(float v, Op op) {
  typedef __attribute__((ext_vector_type(2))) unsigned pair;
  pair p = __builtin_bit_cast(pair, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  v = op(__uint_as_float(p.x), __uint_as_float(p.y));
  p = __builtin_bit_cast(pair, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return op(__uint_as_float(p.x), __uint_as_float(p.y));
}
__device__ __forceinline__ float column_max(float v) { return column_fold(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float column_sum(float v) { return column_fold(v, [](float a, float b) { return a + b; }); }

constexpr float kNoScore = -3.402823466e38f;   // a running maximum before the first key
constexpr int kStep = 64;                      // keys of a step

// Blocks of a kernel that a CU holds.
constexpr int kv_blocks(int vt, int nc, int terms) { return vt > 8 || (nc > 1 && terms > 1 && vt > 4) ? 1 : nc > 1 || vt > 5 || terms > 1 ? 2 : 3; }
// Tiles of up to so many steps, which a table has room for, are not shared between workers; `full`: where tiles as they are keep half the card busy.  Measured, whole against
// shared: of few columns, 16 requests of up to 1200 keys over 8 heads (19 steps) 16 us against 18 and of up to 2048 over 32 heads (32, full) 24 against 27, but one
// of 2048 over 32 heads (not full) 18 against 13, and 16 of up to 4000 (63, full) 39 against 33; of many, 16 chunks of up to 256 behind up to 700 (11) 30 against 43, 8
// of up to 1024 with nothing before (16) 59 against 63, but a window of 1024 (18) 56 against 43 and one of 512 (10) 37 against 33, which goes through tiles of few.
constexpr int kv_alone(int nc, bool full) { return nc ? 16 : full ? 40 : 24; }
// Requests of many columns go through tiles of few as well where all tiles of 16 find room on the card at once and have up to so many steps for each place there: four
// waves then share a tile's steps, and no tile waits for another.  So against tiles of many: 9 chunks of up to 37 in a window of 512 keys (f32, 256 features, 4 steps a
// place) 25 us against 37, 640 rows behind nothing (10) 16 against 23, 4 chunks of up to 64 behind up to 4000 (15) 26 against 36, 16 of up to 64 behind
// up to 2000 (f32, 28) 36 against 39; beyond, 300 rows behind 5000 (35) 47 against 45, 16 chunks of up to 64 behind up to 4000 (56) 45 against 41.
constexpr int kv_small = 32;
// Steps of a share at least.  Of few columns with 8, with 4 and with 16: one request of 100000 keys 29, 43 and 23 us, of 8000 14, 13 and 17, four of 4000 over 8 heads 16, 19 and 20;
// of many with 2, 1 and 4: 700 rows behind 8000 keys 84 to 86.
constexpr int kv_least(int nc) { return nc ? 2 : 8; }
// Steps that a tile's beginning and end take as long as.  Prompts of 2300 rows 94 us with 3, 87 with 6, 93 with 9, 94 with 12; sixteen of them 275, 241, 246 and 257; one request of
// 8000 keys 13 to 14 with any.
constexpr int kv_extra = 6;

// How the work of a key head is dealt out.  A tile of a request is as long as the keys that its last row sees, which grows evenly from tile to
// tile, so that sums over tiles are known without a walk: in sixteenths of a key, tile t takes base + each * (t + 1), and `extra` for its beginning and end
// (queries, first loads, the merge), which a worker that goes on to another tile pays again.  These are prices, from which workers get their shares and tiles the seams between
// them; the steps themselves are a tile's own.  Behind a window the work no longer grows and the price still does, so that shares of prompts longer than a window
// of 1024 keys and more are uneven (8192 rows 275 us, without the window 368).
constexpr int kUnits = 16 * kStep;   // of a step
struct KvRequest {
  int start, n, tiles;           // first row, new tokens
  int len;                       // length, cut to its table's
  int64_t first;                 // position of the first row, by the whole length
};
__device__ __forceinline__ int64_t kv_base(const KvAttnArgs &a, const KvRequest &q) { return 16ll * min(max(q.len - q.n, 0), a.reach); }
__device__ __forceinline__ int64_t kv_units(const KvAttnArgs &a, const KvKind &d, const KvRequest &q, int64_t tile) { return kv_base(a, q) + d.extra + (int64_t)d.each * (tile + 1); }
// of the tiles before `tile`
__device__ __forceinline__ int64_t kv_units_before(const KvAttnArgs &a, const KvKind &d, const KvRequest &q, int64_t tile) { return tile * (kv_base(a, q) + d.extra) + d.each * (tile * (tile + 1) / 2); }

constexpr int64_t kKvFar = (int64_t)1 << 40;   // past every table and window
template <int QT> __device__ __forceinline__ KvRequest kv_request(const KvAttnArgs &a, const KvKind &d, int r) {
  KvRequest q;
  const int64_t start = min(max(a.starts[r], (int64_t)0), a.N), end = a.starts[r + 1], said = a.lens[r], most = a.M << a.page_shift;
  q.start = (int)start;
  q.n = (int)(min(max(end, start), a.N) - start);
  q.len = (int)min(max(said, (int64_t)0), most);
  int64_t first;                 // its rows end with the length, also where some are not there
  if (__builtin_sub_overflow(said, end, &first)) first = said < 0 ? -kKvFar : kKvFar;
  q.first = min(max(first, -kKvFar), kKvFar) + start;
  const int columns = q.n * a.G;
  q.tiles = d.which == 1 ? columns > 0 && columns <= 16 : d.which == 2 && columns <= 16 ? 0 : (columns + QT - 1) / QT;
  return q;
}
__device__ __forceinline__ int64_t wave_scan(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
}

// A worker's place in the work of a key head: its request and tile, and how far its share goes.
struct KvWork {
  KvRequest req;
  int r, tile;
  int64_t from, left;            // `from` units of the tile are others'
  int64_t share, tile_at;        // units before the tile
};
// Every wave sums over the requests by itself, 64 at a time, without LDS or barriers: tiles, if each is a worker's, or their units.  (The code
// around the steps is kept short all through: a wave runs it once, at the rate at which instructions arrive.)
template <int QT> __device__ __forceinline__ bool kv_deal(const KvAttnArgs &a, const KvKind &d, int kvh, int worker, KvWork *out) {
  const int lane = threadIdx.x & 63;
  KvRequest x;
  out->r = -1;
  out->tile = 0;
  out->from = 0;
  out->left = out->share = 1;
  int64_t own = 0, upto = 0, total = 0, u = worker;
  for (int pass = 0; pass < 2 && out->r < 0; ++pass) {
    int64_t at = 0;
#pragma unroll 1
    for (int i = 0; i < a.R; i += 64) {
      if (pass == 0 || a.R > 64) {
        x.tiles = 0;
        if (i + lane < a.R) x = kv_request<QT>(a, d, i + lane);
        own = d.workers == 0 ? x.tiles : x.tiles ? kv_units_before(a, d, x, x.tiles) : 0;
        upto = at + wave_scan(own, lane);
      }
      const uint64_t here = __ballot(pass == 1 && u < upto);
      if (here) {
        const int f = __builtin_ctzll(here);
        out->r = i + f;
        out->tile_at = lane_of(upto - own, f);
        out->req.start = __builtin_amdgcn_readlane(x.start, f);
        out->req.n = __builtin_amdgcn_readlane(x.n, f);
        out->req.len = __builtin_amdgcn_readlane(x.len, f);
        out->req.first = lane_of(x.first, f);
        out->req.tiles = __builtin_amdgcn_readlane(x.tiles, f);
        break;
      }
      at = lane_of(upto, 63);
    }
    if (pass == 0) {
      total = at;
      if (d.workers) {
        const int64_t even = (int64_t)((double)total * d.per_worker);
        out->share = max(even + 1 + (even >> 50), (int64_t)d.least * kUnits);   // times the workers: no less than the total
        u = worker * out->share;
        if (threadIdx.x == 0) d.join[(int64_t)kvh * d.workers + worker].first = -1;
      }
      if (u >= total) return false;
    }
  }
  if (out->r < 0) return false;
  if (d.workers) {
    int lo = 0, hi = out->req.tiles - 1;   // the tile that unit u lies in
#pragma unroll 1
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (kv_units_before(a, d, out->req, mid) <= u - out->tile_at) lo = mid;
      else hi = mid - 1;
    }
    out->tile = lo;
    out->tile_at += kv_units_before(a, d, out->req, lo);
    out->from = u - out->tile_at;
    out->left = min(out->share, total - u);
  } else {
    out->tile = (int)(u - out->tile_at);
    out->left = kv_units(a, d, out->req, out->tile);
  }
  return true;
}
// On to the next tile; false behind the worker's last.
template <int QT> __device__ __forceinline__ bool kv_next(const KvAttnArgs &a, const KvKind &d, int64_t size, int64_t to, KvWork *k) {
  k->left -= to - k->from;
  if (d.workers == 0 || k->left <= 0) return false;
  k->from = 0;
  k->tile_at += size;
  if (++k->tile >= k->req.tiles) {
    k->tile = 0;
    do {
      if (++k->r >= a.R) return false;
      k->req = kv_request<QT>(a, d, k->r);
    } while (k->req.tiles == 0);
  }
  return true;
}
// Which keys the tokens of a request see: of token i, oldest(i) .. newest(i), none where the oldest is the newer.
struct KvSeen {
  int64_t first, window;
  int len;
  double per_group;
  __device__ __forceinline__ int token(int x) const { return (int)(((double)x + 0.5) * per_group); }   // of column x
  __device__ __forceinline__ int64_t at(int i) const { return max(first + i, (int64_t)-1); }
  __device__ __forceinline__ int newest(int i) const { return (int)min(at(i), (int64_t)len - 1); }
  __device__ __forceinline__ int oldest(int i) const { return (int)min(max(at(i) - window + 1, (int64_t)0), (int64_t)len); }
};
// Columns of a tile, 16 to a lane group's place in NC: row of q and head, and what they see.
template <int NC> struct KvColumns {
  int rows[NC], heads[NC], hi[NC], lo[NC];
  bool live[NC];
};
template <int NC> __device__ __forceinline__ KvColumns<NC> kv_columns(const KvAttnArgs &a, const KvRequest &req, const KvSeen &see, int kvh, int x0, int columns) {
  KvColumns<NC> k;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int x = x0 + c * 16 + (threadIdx.x & 15);
    k.live[c] = x < columns;
    const int i = k.live[c] ? see.token(x) : 0;   // (a column behind the last repeats the first, and goes nowhere)
    k.rows[c] = req.start + i;
    k.heads[c] = kvh * a.G + (k.live[c] ? x - i * a.G : 0);
    k.hi[c] = k.live[c] ? see.newest(i) : -1;
    k.lo[c] = see.oldest(i);
  }
  return k;
}

// How a key's F features go into products of 32: in pieces of 64, 16 neighbouring ones to a lane group, so that a lane's 16 bytes of codes serve two
// products; what is left over by 8 bytes a lane where that is 32 or less.
template <int VT> struct KvFeatures {
  static constexpr int KR = VT % 4, KN = VT / 4 + (KR == 3), KS = 2 * KN + (KR == 1 || KR == 2);
  static constexpr bool TAIL = KR == 1 || KR == 2;
  static __device__ __forceinline__ int of_product(int s, int g) { return TAIL && s == KS - 1 ? KN * 64 + 8 * g : (s / 2) * 64 + 16 * g + 8 * (s & 1); }
};
template <typename T, int VT, int NC, bool TOGETHER>
__device__ __forceinline__ void kv_queries(const KvAttnArgs &a, const KvColumns<NC> &k, kv_bf16x8 (&qf)[NC][KvFeatures<VT>::KS][KvTerms<T>::n]) {
  constexpr int TERMS = KvTerms<T>::n, KS = KvFeatures<VT>::KS, WORDS = 2 * sizeof(T);
  struct alignas(16) Eight { uint32_t w[WORDS]; } all[NC][KS];
  // Lanes without these features take others and clear them by a mask.  No branch, and none for the compiler to make of a condition (it does not know
  // what the mask holds): in front of the end of one it has put copies of registers that belong behind it, so that they were made for some lanes only and
  // addresses were lost.
  uint32_t keep[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d0 = KvFeatures<VT>::of_product(s, (threadIdx.x & 63) >> 4);
    keep[s] = d0 < a.D ? 0xffffffffu : 0u;
    asm("" : "+v"(keep[s]));
#pragma unroll
    for (int c = 0; c < NC; ++c) all[c][s] = *reinterpret_cast<const Eight *>((const T *)a.q + (int64_t)k.rows[c] * a.q_row + (int64_t)k.heads[c] * a.q_head + (d0 & (int)keep[s]));
  }
  if (TOGETHER) __builtin_amdgcn_sched_barrier(0);   // all on their way before the first is waited for
  const uint32_t turn = sizeof(T) == 2 ? a.turn : a.turn & 0x80000000u;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Eight e = all[c][s];
#pragma unroll
      for (int j = 0; j < WORDS; ++j) e.w[j] = (e.w[j] ^ turn) & keep[s];
      if constexpr (TERMS == 1) {
        qf[c][s][0] = __builtin_bit_cast(kv_bf16x8, e);
      } else {
        struct Values { T v[8]; };
        const Values x = __builtin_bit_cast(Values, e);
        union { kv_bf16x2 p[4]; kv_bf16x8 v; } u[TERMS];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kv_bf16x2 t[TERMS];
          kv_split2<TERMS>((float)Scalar<T>::load(&x.v[2 * j]), (float)Scalar<T>::load(&x.v[2 * j + 1]), t);
#pragma unroll
          for (int i = 0; i < TERMS; ++i) u[i].p[j] = t[i];
        }
#pragma unroll
        for (int i = 0; i < TERMS; ++i) qf[c][s][i] = u[i].v;
      }
    }
  }
}

// Of sixteen keys: their page, and whether it is there.  Behind the context page 0 stands in.
struct KvPage { uint32_t id; bool there; };
struct KvScales { float k, v; bool there; };
__device__ __forceinline__ KvPage kv_page(const KvAttnArgs &a, uint32_t entry, int key, int len) {
  const bool there = key < len && entry < a.pages;
  return KvPage{there ? entry : 0u, there};
}
__device__ __forceinline__ KvScales kv_scales(const KvAttnArgs &a, KvPage p, int kvh) {
  const int64_t ph = (int64_t)p.id * a.Hkv + kvh;
  return KvScales{a.k_scale[ph], a.v_scale[ph], p.there};
}

// A running softmax over steps: per column its maximum and this lane's share of the sum, and the 16 features x 16 columns tiles of values.
template <int VT, int NC> struct KvState {
  kv_f32x4 o[NC][VT];
  float m[NC], l[NC];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      m[c] = kNoScore;
      l[c] = 0.f;
#pragma unroll
      for (int t = 0; t < VT; ++t) o[c][t] = kv_f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  // another's, over other keys of the same columns
  __device__ __forceinline__ void add(const KvState &y) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float up = fmaxf(m[c], y.m[c]), f1 = __builtin_amdgcn_exp2f(m[c] - up), f2 = __builtin_amdgcn_exp2f(y.m[c] - up);
      m[c] = up;
      l[c] = l[c] * f1 + y.l[c] * f2;
#pragma unroll
      for (int t = 0; t < VT; ++t) o[c][t] = o[c][t] * f1 + y.o[c][t] * f2;
    }
  }
};
// A step's scores s to weights pf, the state to their maximum.  Both scales go into the exponent: with x = s ks and y = x + log2(vs), exp2(y - m) is the
// weight times vs, and the sum of a lane's sixteen over vs is their share of the softmax's.  edge: some column does not see all of the step.
template <int VT, int NC, int TERMS>
__device__ __forceinline__ void kv_weights(kv_f32x4 (&s)[NC][4], KvState<VT, NC> &z, const KvColumns<NC> &k, const KvScales &sc, float scale_log2, int key0, bool edge,
                                           kv_bf16x8 (&pf)[NC][2][TERMS]) {
  const float ks = sc.k * scale_log2, vs = sc.there && sc.v > 0.f ? sc.v : 1.f;
  // log2(vs): its exponent, to which the logarithm of a power of two adds nothing
  const uint32_t bits = __float_as_uint(vs);
  const float up_v = (float)((int)(bits >> 23) - 127) + __builtin_amdgcn_logf(__uint_as_float((bits & 0x7fffffu) | 0x3f800000u)), over_v = __builtin_amdgcn_rcpf(vs);
  const float times = edge ? 1.f : ks;
  float top[NC];
  bool grows = false;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (edge)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + 4 * t + j;
          s[c][t][j] = key <= k.hi[c] && key >= k.lo[c] && sc.there ? s[c][t][j] * ks : -INFINITY;
        }
    float most = s[c][0][0];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) most = fmaxf(most, s[c][t][j]);
    top[c] = column_max(fmaxf(most * times, kNoScore));   // (times is not negative: a negative scale's sign is the queries')
    grows |= top[c] > z.m[c] + 8.f;
  }
  // a maximum that grew by less than 2^8 waits: weights stay below 2^8, and sums in f32 lose nothing by it
  if (__any(grows)) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float up = fmaxf(z.m[c], top[c]), f = __builtin_amdgcn_exp2f(z.m[c] - up);
      z.m[c] = up;
      z.l[c] *= f;
#pragma unroll
      for (int t = 0; t < VT; ++t) z.o[c][t] *= f;
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float down = up_v - z.m[c];
    float p[16], sum = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[4 * t + j] = __builtin_amdgcn_exp2f(fmaf(s[c][t][j], times, down));
        sum += p[4 * t + j];
      }
    z.l[c] = fmaf(sum, over_v, z.l[c]);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      union { kv_bf16x2 p[4]; kv_bf16x8 v; } f[TERMS];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        kv_bf16x2 t[TERMS];
        kv_split2<TERMS>(p[8 * u + 2 * j], p[8 * u + 2 * j + 1], t);
#pragma unroll
        for (int i = 0; i < TERMS; ++i) f[i].p[j] = t[i];
      }
#pragma unroll
      for (int i = 0; i < TERMS; ++i) pf[c][u][i] = f[i].v;
    }
  }
}
// The end of a tile, or of a worker's part of one.  The wave holds columns c0 .. of the tile and of their features the tiles t0, t0 + step, ..; held:
// whether it holds any.  A whole tile goes to the output, a part to the scratch, from where another launch joins them.  (Parts joined by the last
// block to leave a tile, without that launch, took as long or longer: 16 requests of up to 8000 keys over 16 heads 37 us for 34.)
template <typename T, int OT, int NC>
__device__ __forceinline__ void kv_finish(const KvAttnArgs &a, const KvKind &d, const KvWork &k, int kvh, int worker, bool first, int64_t size, int64_t to, int QT, int c0, int t0, int step,
                                          bool held, const KvColumns<NC> &cols, const KvState<OT, NC> &z) {
  const int col = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
  auto feature = [&](int i) { return 16 * (t0 + step * i) + 4 * g; };
  if (k.from != 0 || to != size) {
    const int64_t own = (int64_t)kvh * d.workers + worker;
    auto row_of = [&](int64_t place, int c) { return place * QT + c0 + c * 16 + col; };
    // the workers that have a part: from the one that the tile's first unit is in to the one that its last is in
    auto worker_of = [&](int64_t u) {
      int64_t w = (int64_t)((double)u / (double)k.share);
      return w + (w * k.share > u ? -1 : (w + 1) * k.share <= u ? 1 : 0);
    };
    const int64_t begin = worker_of(k.tile_at), place = k.tile_at != begin * k.share;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (!cols.live[c] || !held) continue;
      const int64_t e = row_of(2 * own + !first, c);
      if (g == 0 && t0 == 0) {
        d.part_m[e] = z.m[c];
        d.part_l[e] = z.l[c];
      }
#pragma unroll
      for (int i = 0; i < OT; ++i)
        if (feature(i) < a.features) *reinterpret_cast<kv_f32x4 *>(d.part + e * a.features + feature(i)) = z.o[c][i];
    }
    if (to == size && threadIdx.x == 0) d.join[own] = KvJoin{(int)begin, (int)place, k.req.start, k.tile * QT, min(QT, k.req.n * a.G - k.tile * QT)};
    return;
  }
  if (!held) return;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (!cols.live[c]) continue;
    const float f = z.l[c] == 0.f ? 0.f : 1.f / z.l[c];
    T *dst = (T *)a.out + ((int64_t)cols.rows[c] * a.Hq + cols.heads[c]) * a.D;
#pragma unroll
    for (int i = 0; i < OT; ++i) {
      struct alignas(sizeof(T) * 4) Four { T v[4]; } y;
#pragma unroll
      for (int j = 0; j < 4; ++j) Scalar<T>::store(&y.v[j], z.l[c] == 0.f ? 0.f : z.o[c][i][j] * f);
      if (feature(i) < a.D) *reinterpret_cast<Four *>(dst + feature(i)) = y;
    }
  }
}

// Blocks go to the XCDs in turn: each XCD gets neighbouring workers, whose keys are often the same; but not where workers are whole tiles, which
// are of different lengths from request to request.
__device__ __forceinline__ int kv_block(const KvKind &d, int block) { return d.workers && d.blocks % 8 == 0 ? block % 8 * (d.blocks / 8) + block / 8 : block; }

// What every wave has asked for or written is there, for all of them.
__device__ __forceinline__ void kv_meet() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Few columns: 16 to a tile, KW waves that share its steps in turn and merge through LDS.
// The columns of a request and key head are its new tokens times the query heads of the group, G to a token.  A step is 64 keys:
//     S^T = K . Q^T   (four tiles of 16 keys x 16 columns),      O^T = V^T . P^T   (VT tiles of 16 features x 16 columns)
// on v_mfma_f32_16x16x32_bf16.  Row 4 g + r of score tile t is key 16 g + 4 t + r of the step, so that the lane group g (lanes 16 g ..) holds
// the scores of sixteen neighbouring keys, which are the 16 bytes that it loads of a feature of V: the weights are the second product's
// fragments as they lie in registers, and every load of the cache is 16 bytes a lane, straight to registers.  Sixteen keys lie in one
// page, so a lane group has one page and one scale of keys and of values.
// Bound by memory and by what comes before the first step and behind the last: 64 requests of up to 16384 keys (236 MB) take 47 us and their join 4.7, 4.6 TB/s
// in all where a read alone reaches 7.1 and a copy 4.7; a lone row over 777 keys takes 11 us, a chain of trips (lengths, table, keys, merge) and of code that is
// run once.  A quarter of a wave reads sixteen keys' 16 bytes at a time: read as whole lines, at other results, the large case took 50 us.
template <typename T, int VT> constexpr int kv_few_lds() { return 4 * VT * 64 * 16 + 4 * 2 * 64 * 4; }
template <typename T, int FMT, int VT> __device__ __forceinline__ void kv_few(const KvAttnArgs &a, const KvKind &d, int block, uint8_t *lds) {
  typedef KvFeatures<VT> Fe;
  constexpr int TERMS = KvTerms<T>::n, WEIGHTS = KvTerms<T>::weights, QT = 16, KS = Fe::KS, KN = Fe::KN, KW = 4;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_head = d.blocks / a.Hkv, place = kv_block(d, block), kvh = place / per_head, worker = place % per_head;
  KvWork k;
  if (!kv_deal<QT>(a, d, kvh, worker, &k)) return;

  const int64_t head_bytes = ((int64_t)1 << a.page_shift) * a.features, page_bytes = a.Hkv * head_bytes;
  const uint8_t *const keys = a.k + kvh * head_bytes, *const values = a.v + kvh * head_bytes;
  const int slot_mask = (1 << a.page_shift) - 1, k_group = col >> 2;
  // Features behind the cache's last are read again from its beginning: q is zero there.
  int k_at[KN ? KN : 1];
#pragma unroll
  for (int i = 0; i < KN; ++i) k_at[i] = i * 64 + 16 * g < a.features ? i * 64 + 16 * g : 0;
  const int tail_at = KN * 64 + 8 * g < a.features ? KN * 64 + 8 * g : 0;
  int v_at[VT];
#pragma unroll
  for (int t = 0; t < VT; ++t) v_at[t] = (16 * t + col < a.features ? 16 * t + col : 0) << a.page_shift;

  for (bool first = true;; first = false) {
    const int64_t size = kv_units(a, d, k.req, k.tile), to = min(size, k.from + k.left);
    const int len = k.req.len, columns = k.req.n * a.G;
    const KvSeen see = {k.req.first, a.window, len, a.per_group};
    const KvColumns<1> cols = kv_columns<1>(a, k.req, see, kvh, k.tile * QT, columns);
    // of the tile's first and last token: every live column sees lo_last .. hi_first, none sees outside lo_first .. hi_last
    const int i_first = see.token(k.tile * QT), i_last = see.token(min((k.tile + 1) * QT, columns) - 1);
    const int hi_first = see.newest(i_first), hi_last = see.newest(i_last), lo_first = see.oldest(i_first), lo_last = see.oldest(i_last);
    const int step0 = lo_first / kStep, steps = hi_last >= lo_first ? hi_last / kStep + 1 - step0 : 0;
    const int s_begin = step0 + (int)min((int64_t)steps, max(k.from - d.extra, (int64_t)0) / kUnits), s_end = step0 + (to == size ? steps : (int)min((int64_t)steps, max(to - d.extra, (int64_t)0) / kUnits));

    // An entry of the table is asked for two steps ahead and looked at one step ahead: looked at sooner, it would wait for the loads that went
    // out with it.  So are scales: what a step hands to the next must not wait for keys.
    const uint32_t *const table = a.tables + (int64_t)k.r * a.table_ld;
    auto entry_of = [&](int key) __attribute__((always_inline)) { return table[key < len ? key >> a.page_shift : 0]; };
    struct { kv_u32x4 k[KN ? KN : 1][4]; kv_u32x2 tail[4]; kv_u32x4 v[VT]; } now;
    auto load_keys = [&](int st, KvPage p) __attribute__((always_inline)) {
      const int key = st * kStep + 16 * k_group + (col & 3);
      const uint8_t *base = keys + (int64_t)p.id * page_bytes + (key & slot_mask) * a.features;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < KN; ++i) now.k[i][t] = fetch_once(base + 4 * t * a.features + k_at[i]);
        if (Fe::TAIL) now.tail[t] = *reinterpret_cast<const kv_u32x2 *>(base + 4 * t * a.features + tail_at);
      }
    };
    auto load_values = [&](int st, KvPage p) __attribute__((always_inline)) {
      const uint8_t *base = values + (int64_t)p.id * page_bytes + ((st * kStep + 16 * g) & slot_mask);
#pragma unroll
      for (int t = 0; t < VT; ++t) now.v[t] = fetch_once(base + v_at[t]);
    };

    KvState<VT, 1> z;
    z.clear();
    int st = s_begin + w;
    bool missing = false;
    if (st < s_end) {
      const int last = s_end - 1;
      int next = min(st + KW, last);
      uint32_t nk = entry_of(st * kStep + 16 * k_group), nv = entry_of(st * kStep + 16 * g);
      KvScales scales;
      {
        const KvPage pk = kv_page(a, nk, st * kStep + 16 * k_group, len), pv = kv_page(a, nv, st * kStep + 16 * g, len);
        nk = entry_of(next * kStep + 16 * k_group);
        nv = entry_of(next * kStep + 16 * g);
        scales = kv_scales(a, pv, kvh);
        load_keys(st, pk);
        load_values(st, pv);
      }
      kv_bf16x8 qf[1][KS][TERMS];   // (behind the keys, which would wait for them)
      kv_queries<T, VT, 1, false>(a, cols, qf);
      for (; st < s_end; st += KW) {
        const int ahead = min(next + KW, last);
        const uint32_t ak = entry_of(ahead * kStep + 16 * k_group), av = entry_of(ahead * kStep + 16 * g);
        const KvPage of_k = kv_page(a, nk, next * kStep + 16 * k_group, len), of_v = kv_page(a, nv, next * kStep + 16 * g, len);
        const KvScales coming = kv_scales(a, of_v, kvh);
        const int key0 = st * kStep + 16 * g;   // this lane group's first
        const bool gone = key0 < len && !scales.there;
        missing |= gone && key0 + 15 >= lo_first && key0 <= hi_last;   // some row of the tile would see it
        if ((st + 1) * kStep > len || __any(gone)) {
          // codes behind the context may be anything; their weight is zero, and zero times a NaN would not be
          const int valid = scales.there ? min(len - key0, 16) : 0;
          uint32_t keep[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int b = min(max(valid - 4 * j, 0), 4);
            keep[j] = b == 4 ? 0xffffffffu : (1u << 8 * b) - 1;
          }
#pragma unroll
          for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) now.v[t][j] &= keep[j];
        }
        kv_f32x4 s[1][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          s[0][t] = kv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < KS; ++e) {
            kv_bf16x8 f;
            if (Fe::TAIL && e == KS - 1) f = kv_unpack<FMT>(now.tail[t].x, now.tail[t].y);
            else f = kv_unpack<FMT>(now.k[e / 2][t][2 * (e & 1)], now.k[e / 2][t][2 * (e & 1) + 1]);
#pragma unroll
            for (int i = 0; i < TERMS; ++i) s[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, qf[0][e][i], s[0][t], 0, 0, 0);
          }
        }
        load_keys(next, of_k);
        kv_bf16x8 pf[1][2][WEIGHTS];
        kv_weights<VT, 1, WEIGHTS>(s, z, cols, scales, a.scale_log2, key0, (st + 1) * kStep - 1 > hi_first || st * kStep < lo_last || __any(gone), pf);
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const kv_bf16x8 f = kv_unpack<FMT>(now.v[t][2 * u], now.v[t][2 * u + 1]);
#pragma unroll
            for (int i = 0; i < WEIGHTS; ++i) z.o[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, pf[0][u][i], z.o[0][t], 0, 0, 0);
          }
        load_values(next, of_v);
        next = ahead;
        nk = ak;
        nv = av;
        scales = coming;
      }
    }
    if (kvh == 0) {
      const bool past = k.from == 0 && k.tile == 0 && w == 0 && a.lens[k.r] > a.M << a.page_shift;
      if ((__any(missing) || past) && lane == 0) atomicAdd(a.errors, 1ull);
    }
    z.l[0] = column_sum(z.l[0]);

    // every wave's sums to LDS as they lie in registers, and every fourth tile of features to a wave
    constexpr int OT = (VT + 3) / 4;
    kv_f32x4 (*const sums)[VT][64] = reinterpret_cast<kv_f32x4 (*)[VT][64]>(lds);
    float (*const stats)[2][64] = reinterpret_cast<float (*)[2][64]>(lds + 4 * VT * 64 * 16);
    __syncthreads();   // (nobody reads the tile before any more)
#pragma unroll
    for (int t = 0; t < VT; ++t) sums[w][t][lane] = z.o[0][t];
    stats[w][0][lane] = z.m[0];
    stats[w][1][lane] = z.l[0];
    __syncthreads();
    KvState<OT, 1> y;
    y.clear();
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y.m[0] = fmaxf(y.m[0], stats[i][0][lane]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = __builtin_amdgcn_exp2f(stats[i][0][lane] - y.m[0]);
      y.l[0] = fmaf(stats[i][1][lane], f[i], y.l[0]);
#pragma unroll
      for (int t = 0; t < OT; ++t) y.o[0][t] += sums[i][min(4 * t + w, VT - 1)][lane] * f[i];
    }
    kv_finish<T, OT, 1>(a, d, k, kvh, worker, first, size, to, QT, 0, w, 4, true, cols, y);
    if (!kv_next<QT>(a, d, size, to, &k)) return;
  }
}

// 16 bytes a lane straight to LDS, at `to` (the wave's) + 16 * lane.  Not by the builtin, behind which the compiler puts a wait for all that is on its way before the
// next read of LDS, of the other buffer too: kv_meet waits, before a barrier.  The instruction writes no register.
__device__ __forceinline__ void kv_to_lds(const uint8_t *from, uint32_t to) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(to), "v"(from) : "memory");
}

// Many columns: two waves of 16 NC columns each for the even steps of a tile and two for the odd ones, merged through LDS at its end.  Keys and values come
// through LDS as codes, two buffers of two steps, one barrier for both: each byte of the cache reaches a CU once for 32 NC columns, and no
// register holds what is on its way.  Keys lie in LDS in the order of the score tiles'
// rows, their 16-byte pieces exchanged so that sixteen rows' reads spread over the banks; values as sixteen keys of a feature.
// Bound by the instructions around the products: a step of 32 columns takes 96 matrix instructions (1536 clocks of a SIMD) and about 370 vector ones
// (1900: codes to bf16 128, the softmax 160, weights in two terms 80) and as many scalar ones in between, two waves to a SIMD.  Prompts of 2300 rows over up to 5000 keys,
// 34.6 GFLOP, take 87 us with their join; sixteen of them 241 us, 495 TFLOP/s of the 1370 that a large product reaches.
template <int VT> constexpr int kv_wide_lds() { return 8 * 64 * 16 * VT; }
template <typename T, int FMT, int VT, int NC> __device__ __forceinline__ void kv_wide(const KvAttnArgs &a, const KvKind &d, int block, uint8_t *lds) {
  typedef KvFeatures<VT> Fe;
  constexpr int TERMS = KvTerms<T>::n, WEIGHTS = KvTerms<T>::weights, QT = 32 * NC, KS = Fe::KS, BYTES = 64 * 16 * VT, LOADS = (2 * VT + 3) / 4;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = w >> 1;
  const int per_head = d.blocks / a.Hkv, place = kv_block(d, block), kvh = place / per_head, worker = place % per_head;
  KvWork k;
  if (!kv_deal<QT>(a, d, kvh, worker, &k)) return;

  const int64_t head_bytes = ((int64_t)1 << a.page_shift) * a.features, page_bytes = a.Hkv * head_bytes;
  const uint8_t *const keys = a.k + kvh * head_bytes, *const values = a.v + kvh * head_bytes;
  const int slot_mask = (1 << a.page_shift) - 1;
  // A step's pieces of 16 bytes are asked for in runs of 64, VT runs of keys and VT of values, every fourth a wave's.  Where VT is a multiple of 4 a run
  // lies in sixteen keys (KEYED: keys in their order in LDS), a wave's i-th run of values in the same as its i-th of keys, so that their page and first byte are
  // found by scalar instructions, once for both, and a lane adds an offset that does not change; else each lane finds its own, and keys lie in the order
  // of the score tiles' rows.  Found by lane all through, addresses took as many instructions as everything between the products.
  constexpr bool KEYED = VT % 4 == 0;
  constexpr int ASKS = KEYED ? VT / 4 : LOADS;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
  auto exchange = [](int column) { return VT == 4 ? column >> 2 : VT == 8 ? column >> 1 : VT == 16 ? column : 0; };
  int key_of[ASKS], at_of[LOADS];   // first key of the piece (KEYED: of its run), bytes from there on
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int run = i * 4 + w, piece = (run < VT ? run : run - VT) * 64 + lane;
    if (run < VT) {
      const int row = piece / VT, j = KEYED ? (row & 3) | (row >> 4) << 2 : row & 15, part = (piece % VT) ^ exchange(j);
      if (!KEYED) key_of[i % ASKS] = 16 * (j >> 2) + 4 * (row >> 4) + (j & 3);
      at_of[i] = (KEYED ? row % 16 * a.features : 0) + (16 * part < a.features ? 16 * part : 0);
    } else {
      const int d = piece % (16 * VT);
      if (!KEYED) key_of[i % ASKS] = 16 * (piece / (16 * VT));
      at_of[i] = (d < a.features ? d : 0) << a.page_shift;
    }
  }
  if (KEYED)
#pragma unroll
    for (int i = 0; i < ASKS; ++i) key_of[i] = (i * 4 + w) * 4 / VT * 16;
  int k_at[4];   // this lane's row of score tile t in LDS
#pragma unroll
  for (int t = 0; t < 4; ++t) k_at[t] = (KEYED ? 16 * (col >> 2) + 4 * t + (col & 3) : 16 * t + col) * 16 * VT;

  for (bool first = true;; first = false) {
    const int64_t size = kv_units(a, d, k.req, k.tile), to = min(size, k.from + k.left);
    const int len = k.req.len, columns = k.req.n * a.G;
    const KvSeen see = {k.req.first, a.window, len, a.per_group};
    const int x0 = k.tile * QT, xw = x0 + (w & 1) * 16 * NC;
    const KvColumns<NC> cols = kv_columns<NC>(a, k.req, see, kvh, xw, columns);
    // what the tile's first and last token see, for the steps; and this wave's, for what it may skip or need not mask
    const int i_first = see.token(x0), i_last = see.token(min(x0 + QT, columns) - 1);
    const int lo_first = see.oldest(i_first), hi_last = see.newest(i_last);
    const int step0 = lo_first / kStep, steps = hi_last >= lo_first ? hi_last / kStep + 1 - step0 : 0;
    const int s_begin = step0 + (int)min((int64_t)steps, max(k.from - d.extra, (int64_t)0) / kUnits), s_end = step0 + (to == size ? steps : (int)min((int64_t)steps, max(to - d.extra, (int64_t)0) / kUnits));
    const int iw_first = see.token(min(xw, columns - 1)), iw_last = see.token(min(xw + 16 * NC, columns) - 1);
    const int hi_near = see.newest(iw_first), hi_far = xw < columns ? see.newest(iw_last) : -1, lo_near = see.oldest(iw_last), lo_far = see.oldest(iw_first);

    const uint32_t *const table = a.tables + (int64_t)k.r * a.table_ld;
    auto entry_of = [&](int key) __attribute__((always_inline)) { return table[key < len ? key >> a.page_shift : 0]; };
    // the two steps from `st` on; a step behind the last is asked for as the last
    const int last = s_end - 1;
    auto ask = [&](int st, uint32_t (&e)[2][ASKS], uint32_t &of_scales) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < ASKS; ++i) {
          const int key = min(st + h, last) * kStep + key_of[i];
          if constexpr (KEYED) e[h][i] = ((const __attribute__((address_space(4))) uint32_t *)table)[key < len ? key >> a.page_shift : 0];
          else e[h][i] = entry_of(key);
        }
      of_scales = entry_of(min(st + half, last) * kStep + 16 * g);
    };
    auto load = [&](int st, const uint32_t (&e)[2][ASKS], uint32_t to_lds) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < ASKS; ++i) {
          const int run = i * 4 + w, key = min(st + h, last) * kStep + key_of[i], slot = key & slot_mask;
          const int64_t page = (int64_t)kv_page(a, e[h][i], key, len).id * page_bytes;
          if constexpr (KEYED) {
            kv_to_lds(keys + (page + slot * a.features) + at_of[i], to_lds + h * 2 * BYTES + run * 1024);
            kv_to_lds(values + (page + slot) + at_of[i + ASKS], to_lds + h * 2 * BYTES + (VT + run) * 1024);
          } else {
            if (run >= 2 * VT) break;
            kv_to_lds((run < VT ? keys : values) + page + slot * (run < VT ? a.features : 1) + at_of[i], to_lds + h * 2 * BYTES + run * 1024);
          }
        }
      }
    };

    KvState<VT, NC> z;
    z.clear();
    bool missing = false;
    if (s_begin < s_end) {
      uint32_t entries[2][ASKS], e_scales;
      ask(s_begin, entries, e_scales);
      KvScales scales = kv_scales(a, kv_page(a, e_scales, min(s_begin + half, last) * kStep + 16 * g, len), kvh);
      kv_meet();   // (nobody reads the tile before any more)
      load(s_begin, entries, lds_at);
      ask(min(s_begin + 2, last), entries, e_scales);
      kv_bf16x8 qf[NC][KS][TERMS];
      kv_queries<T, VT, NC, true>(a, cols, qf);
      for (int st0 = s_begin, b = 0; st0 < s_end; st0 += 2, b ^= 1) {
        kv_meet();   // these steps' pieces, of every wave
        const int st = st0 + half, next = min(st0 + 2, last), key0 = st * kStep + 16 * g;
        const KvScales coming = kv_scales(a, kv_page(a, e_scales, min(next + half, last) * kStep + 16 * g, len), kvh);
        load(next, entries, lds_at + (b ^ 1) * 4 * BYTES);
        ask(min(st0 + 4, last), entries, e_scales);
        const bool gone = st < s_end && key0 < len && !scales.there;
        missing |= gone && key0 + 15 >= lo_first && key0 <= hi_last;   // some row of the tile would see it
        uint8_t *const kt = lds + (b * 4 + half * 2) * BYTES, *const vt = kt + BYTES;
        if (st < s_end && ((st + 1) * kStep > len || __any(gone))) {
          // codes behind the context may be anything; their weight is zero, and zero times a NaN would not be.  (Each wave does it for itself: the
          // step's other one writes the same.)
          const int valid = scales.there ? min(len - key0, 16) : 0;
          for (int t = 0; t < VT; ++t) {
            kv_u32x4 *const p = reinterpret_cast<kv_u32x4 *>(vt + (g * 16 * VT + 16 * t + col) * 16);
            kv_u32x4 x = *p;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int n = min(max(valid - 4 * j, 0), 4);
              x[j] &= n == 4 ? 0xffffffffu : (1u << 8 * n) - 1;
            }
            *p = x;
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        if (st < s_end && st * kStep <= hi_far && (st + 1) * kStep > lo_far) {
          kv_f32x4 s[NC][4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int c = 0; c < NC; ++c) s[c][t] = kv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < KS; ++e) {
              kv_bf16x8 f;
              if (Fe::TAIL && e == KS - 1) {
                const int part = min(4 * Fe::KN + (g >> 1), VT - 1) ^ exchange(col);
                const kv_u32x2 x = *reinterpret_cast<const kv_u32x2 *>(kt + k_at[t] + 16 * part + 8 * (g & 1));
                f = kv_unpack<FMT>(x.x, x.y);
              } else {
                const int part = (4 * (e / 2) + g) ^ exchange(col);
                const kv_u32x2 x = *reinterpret_cast<const kv_u32x2 *>(kt + k_at[t] + 16 * part + 8 * (e & 1));
                f = kv_unpack<FMT>(x.x, x.y);
              }
#pragma unroll
              for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < TERMS; ++i) s[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, qf[c][e][i], s[c][t], 0, 0, 0);
            }
          }
          kv_bf16x8 pf[NC][2][WEIGHTS];
          kv_weights<VT, NC, WEIGHTS>(s, z, cols, scales, a.scale_log2, key0, (st + 1) * kStep - 1 > hi_near || st * kStep < lo_near || __any(gone), pf);
#pragma unroll
          for (int t = 0; t < VT; ++t) {
            const kv_u32x4 v = *reinterpret_cast<const kv_u32x4 *>(vt + (g * 16 * VT + 16 * t + col) * 16);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const kv_bf16x8 f = kv_unpack<FMT>(v[2 * u], v[2 * u + 1]);
#pragma unroll
              for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < WEIGHTS; ++i) z.o[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, pf[c][u][i], z.o[c][t], 0, 0, 0);
            }
          }
        }
        scales = coming;
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last step asked once more: nothing may land in LDS behind the block's end
    }
    if (kvh == 0 && (w & 1) == 0) {
      const bool past = w == 0 && k.from == 0 && k.tile == 0 && a.lens[k.r] > a.M << a.page_shift;
      if ((__any(missing) || past) && lane == 0) atomicAdd(a.errors, 1ull);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) z.l[c] = column_sum(z.l[c]);
    // the odd steps' sums to the waves of the even ones, as they lie in registers
    kv_f32x4 (*const sums)[NC][VT][64] = reinterpret_cast<kv_f32x4 (*)[NC][VT][64]>(lds);
    float (*const stats)[NC][2][64] = reinterpret_cast<float (*)[NC][2][64]>(lds + 2 * NC * VT * 1024);
    static_assert(2 * NC * VT * 1024 + 2 * NC * 2 * 256 <= kv_wide_lds<VT>(), "the merge's room");
    kv_meet();
    if (half == 1) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int t = 0; t < VT; ++t) sums[w & 1][c][t][lane] = z.o[c][t];
        stats[w & 1][c][0][lane] = z.m[c];
        stats[w & 1][c][1][lane] = z.l[c];
      }
    }
    kv_meet();
    if (half == 0) {
      KvState<VT, NC> y;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int t = 0; t < VT; ++t) y.o[c][t] = sums[w][c][t][lane];
        y.m[c] = stats[w][c][0][lane];
        y.l[c] = stats[w][c][1][lane];
      }
      z.add(y);
    }
    kv_finish<T, VT, NC>(a, d, k, kvh, worker, first, size, to, QT, (w & 1) * 16 * NC, 0, 1, half == 0, cols, z);
    if (!kv_next<QT>(a, d, size, to, &k)) return;
  }
}

// Requests of few columns and those of many in one launch, the larger work first.  NC = 0: no request has many.
template <typename T, int FMT, int VT, int NC>
__global__ void __launch_bounds__(256, kv_blocks(VT, NC ? NC : 1, KvTerms<T>::n)) k_kv_attention(KvAttnArgs a) {
  constexpr int FEW = kv_few_lds<T, VT>(), WIDE = NC ? kv_wide_lds<VT>() : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[FEW > WIDE ? FEW : WIDE];
  if constexpr (NC > 0) {
    if ((int)blockIdx.x < a.many.blocks) {
      kv_wide<T, FMT, VT, NC>(a, a.many, blockIdx.x, lds);
      return;
    }
  }
  kv_few<T, FMT, VT>(a, a.few, blockIdx.x - (NC ? a.many.blocks : 0), lds);
}

// The parts of tiles that workers share, to the output.  Blocks for each worker that had a tile's last part, over the tile's columns: a wave reads whole rows of
// as many columns as fit it.  4.7 us behind 64 requests, 9 behind prompts of 2300 rows as a trace has it, most of it the launch and one trip.  PARTS: the block's waves take every fourth part each and meet in LDS (a context over many workers); else each its own columns.
template <typename T, bool PARTS> __device__ __forceinline__ void kv_join(const KvAttnArgs &a, const KvKind &d, int QT, int worker, int kvh, int z, kv_f32x4 (*sums)[64], float (*stats)[2][64]) {
  const int64_t base = (int64_t)kvh * d.workers;
  const KvJoin j = d.join[base + worker];
  const int F4 = a.features / 4, per_wave = 64 / F4, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = (PARTS ? z : z * 4 + w) * per_wave + lane / F4, f = lane % F4 * 4;
  const bool live = j.first >= 0 && lane / F4 < per_wave && c < j.columns;
  if (j.first < 0 || (PARTS && z * per_wave >= j.columns)) return;
  const int cc = live ? c : 0;
  float m = kNoScore, l = 0.f;
  kv_f32x4 o = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float pm, float pl, kv_f32x4 y) __attribute__((always_inline)) {
    const float up = fmaxf(m, pm), f1 = __builtin_amdgcn_exp2f(m - up), f2 = __builtin_amdgcn_exp2f(pm - up);
    m = up;
    l = l * f1 + pl * f2;
    o = o * f1 + y * f2;
  };
  constexpr int AT_ONCE = 4, STEP = PARTS ? 4 : 1;
  for (int k = j.first + (PARTS ? w : 0); k <= worker; k += AT_ONCE * STEP) {
    float pm[AT_ONCE], pl[AT_ONCE];
    kv_f32x4 y[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int p = min(k + u * STEP, worker);
      const int64_t row = (2 * (base + p) + (p == j.first ? j.place : 0)) * QT + cc;
      pm[u] = k + u * STEP <= worker ? d.part_m[row] : kNoScore;
      pl[u] = k + u * STEP <= worker ? d.part_l[row] : 0.f;
      y[u] = *reinterpret_cast<const kv_f32x4 *>(d.part + row * a.features + f);
      if (k + u * STEP > worker) y[u] = kv_f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) add(pm[u], pl[u], y[u]);
  }
  if constexpr (PARTS) {
    sums[w][lane] = o;
    stats[w][0][lane] = m;
    stats[w][1][lane] = l;
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int u = 1; u < 4; ++u) add(stats[u][0][lane], stats[u][1][lane], sums[u][lane]);
  }
  if (!live || f >= a.D) return;
  const int x = j.column + c, i = x / a.G;
  const float over = l == 0.f ? 0.f : 1.f / l;
  struct alignas(sizeof(T) * 4) Four { T v[4]; } y;
#pragma unroll
  for (int u = 0; u < 4; ++u) Scalar<T>::store(&y.v[u], l == 0.f ? 0.f : o[u] * over);
  *reinterpret_cast<Four *>((T *)a.out + (((int64_t)j.start + i) * a.Hq + (int64_t)kvh * a.G + x - i * a.G) * a.D + f) = y;
}

// Of few columns alone, a grid of workers, heads and columns; or of both kinds, `few` blocks, zf to a worker, then those of many columns, zm to a worker.  (One launch for
// both: a chunk of 64 rows behind 30000 keys 51 us, with two 61; but found from one number, a block's place costs the few alone 1.7 us.)
template <typename T, bool BOTH> __global__ void __launch_bounds__(256) k_kv_attention_join(KvAttnArgs a, int few, int zf, int zm, int QT) {
  __shared__ kv_f32x4 sums[4][64];
  __shared__ float stats[4][2][64];
  if constexpr (!BOTH) kv_join<T, true>(a, a.few, 16, blockIdx.x, blockIdx.y, blockIdx.z, sums, stats);
  else {
    int b = blockIdx.x;
    if (b < few) {
      const int z = b % zf, own = b / zf;
      kv_join<T, true>(a, a.few, 16, own % a.few.workers, own / a.few.workers, z, sums, stats);
    } else {
      b -= few;
      const int z = b % zm, own = b / zm;
      kv_join<T, false>(a, a.many, QT, own % a.many.workers, own / a.many.workers, z, sums, stats);
    }
  }
}

// Tiles of 16 columns to a wave of a wide block: as many as registers hold.
template <typename T> constexpr int wide_tiles(int features) { return KvTerms<T>::n == 1 || (KvTerms<T>::n == 2 && features <= 128) ? 2 : 1; }

// Rows of D features off 16-byte boundaries to ones of F, zeros behind the D; and the other way, of the rows that are a request's.
struct KvRowsArgs {
  const void *src;
  void *dst;
  int64_t row, head, N;          // strides of the rows that are not contiguous
  int H, D, F, R;
  const int64_t *starts;
};
template <typename T> __global__ void __launch_bounds__(256) k_kv_rows_widen(KvRowsArgs a) {
  const int64_t total = a.N * a.H * a.F;
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < total; e += gridDim.x * 256ll) {
    const int64_t rh = e / a.F, n = rh / a.H;
    const int d = (int)(e - rh * a.F), h = (int)(rh - n * a.H);
    T v;
    memset(&v, 0, sizeof(T));
    if (d < a.D) v = ((const T *)a.src)[n * a.row + h * a.head + d];
    ((T *)a.dst)[e] = v;
  }
}
template <typename T> __global__ void __launch_bounds__(256) k_kv_rows_narrow(KvRowsArgs a) {
  const int64_t total = a.N * a.H * a.D, first = a.starts[0], last = a.starts[a.R];
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < total; e += gridDim.x * 256ll) {
    const int64_t rh = e / a.D, n = rh / a.H;
    if (n >= first && n < last) ((T *)a.dst)[e] = ((const T *)a.src)[rh * a.F + e - rh * a.D];
  }
}

// A kind's workers and what it takes of the scratch.
template <typename T, int VT, int NC> struct KvShares {
  static constexpr int QT = NC ? 32 * NC : 16;
  int workers;
  int64_t parts;
  // tiles: as many as there may be.  No more workers than the least share allows: blocks that find nothing to do take their time too.
  KvShares(const KvAttnArgs &a, int64_t steps, int64_t tiles) {
    const int64_t slots = (int64_t)device_cu_count(a.dev) * kv_blocks(VT, NC ? NC : 1, KvTerms<T>::n) / a.Hkv, useful = (tiles * (steps + kv_extra) + kv_least(NC) - 1) / kv_least(NC);
    const int64_t n = slots < useful ? slots : useful;
    workers = steps <= kv_alone(NC, 2 * tiles >= slots) ? 0 : n < 1 ? 1 : (int)n;
    parts = 2ll * QT * a.Hkv * workers;
  }
  static_assert(QT * sizeof(float) % 16 == 0 && sizeof(KvJoin) % 16 == 0, "whole 16 bytes of scratch");
  size_t bytes(const KvAttnArgs &a) const { return (size_t)(parts * (a.features + 2) * 4) + (size_t)a.Hkv * workers * sizeof(KvJoin); }
  KvKind kind(const KvAttnArgs &a, int which, void *ws) const {
    KvKind d;
    memset(&d, 0, sizeof(d));
    d.which = which;
    d.workers = workers;
    d.blocks = (workers ? workers : (int)(which == 1 ? a.R : a.N * a.G / QT + a.R)) * a.Hkv;
    d.each = (16 * QT + a.G - 1) / a.G;
    d.extra = kv_extra * kUnits;
    d.least = kv_least(NC);
    d.per_worker = workers ? 1.0 / workers : 0;
    d.part = (float *)ws;
    d.part_m = d.part + parts * a.features;
    d.part_l = d.part_m + parts;
    d.join = (KvJoin *)(d.part_l + parts);
    return d;
  }
};

template <typename T, int FMT, int VT> static int launch_kv_attention(hipStream_t st, KvAttnArgs a, const KvRowsArgs &odd, bool wide, int64_t steps) {
  constexpr int NC = wide_tiles<T>(16 * VT);
  const int64_t tiles = (a.N * a.G / 16 + a.R) * a.Hkv, slots = (int64_t)device_cu_count(a.dev) * kv_blocks(VT, 1, KvTerms<T>::n);
  if (tiles <= slots && tiles * steps <= kv_small * slots) wide = false;
  const KvShares<T, VT, 0> few(a, steps, wide ? a.R : a.N * a.G / 16 + a.R);
  const KvShares<T, VT, NC> many(a, steps, a.N * a.G / (32 * NC) + a.R);
  const size_t of_few = few.bytes(a), of_many = wide ? many.bytes(a) : 0;
  const size_t rows = odd.src ? ((size_t)a.N * a.Hq * a.features * sizeof(T) + 15) / 16 * 16 : 0;
  WorkspaceHold hold;
  void *ws = nullptr;
  if (of_few + of_many + rows) RAI_TRY(workspace(a.dev, of_few + of_many + 2 * rows, &ws, &hold));
  char *const base = (char *)ws;
  const int64_t most = kNumCU * 32;
  KvRowsArgs in = odd, back = odd;
  if (odd.src) {
    a.q = in.dst = base;
    a.out = base + rows;
    back.src = a.out;
    a.q_row = (int64_t)a.Hq * a.features;
    a.q_head = a.D = a.features;
    const int64_t blocks = (a.N * a.Hq * a.features + 255) / 256;
    hipLaunchKernelGGL((k_kv_rows_widen<T>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, in);
    RAI_TRY(launch_check("kv_rows_widen"));
  }
  a.few = few.kind(a, wide ? 1 : 0, base + 2 * rows);
  if (wide) a.many = many.kind(a, 2, base + 2 * rows + of_few);
  RAI_REQUIRE(((uintptr_t)a.few.part | (uintptr_t)a.many.part) % 16 == 0, RAI_ERR_UNSUPPORTED, "kv_attention: scratch of %zu and %zu bytes off 16", of_few, of_many);
  dim3 grid;
  RAI_TRY(grid_of_blocks((int64_t)a.few.blocks + a.many.blocks, 256, &grid));
  RAI_REQUIRE(grid.y == 1, RAI_ERR_UNSUPPORTED, "kv_attention: %d blocks", a.few.blocks + a.many.blocks);
  if (wide) {
    hipLaunchKernelGGL((k_kv_attention<T, FMT, VT, NC>), grid, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((k_kv_attention<T, FMT, VT, 0>), grid, dim3(256), 0, st, a);
  }
  RAI_TRY(launch_check("kv_attention"));
  const int per_wave = 256 / a.features, zf = (few.QT + per_wave - 1) / per_wave, zm = (many.QT + 4 * per_wave - 1) / (4 * per_wave);
  const int64_t of_few_tiles = (int64_t)a.few.workers * a.Hkv * zf, joins = of_few_tiles + (int64_t)a.many.workers * a.Hkv * zm;
  if (a.many.workers) hipLaunchKernelGGL((k_kv_attention_join<T, true>), dim3((unsigned)joins), dim3(256), 0, st, a, (int)of_few_tiles, zf, zm, many.QT);
  else if (a.few.workers) hipLaunchKernelGGL((k_kv_attention_join<T, false>), dim3((unsigned)a.few.workers, (unsigned)a.Hkv, (unsigned)zf), dim3(256), 0, st, a, 0, 0, 0, 0);
  RAI_TRY(launch_check("kv_attention_join"));
  if (odd.src) {
    const int64_t blocks = (a.N * a.Hq * odd.D + 255) / 256;
    hipLaunchKernelGGL((k_kv_rows_narrow<T>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, back);
    RAI_TRY(launch_check("kv_rows_narrow"));
  }
  return RAI_OK;
}

template <typename T, int FMT> static int launch_by_features(hipStream_t st, const KvAttnArgs &a, const KvRowsArgs &odd, bool wide, int64_t steps) {
  if (a.features <= 64) return launch_kv_attention<T, FMT, 4>(st, a, odd, wide, steps);
  if (a.features <= 80) return launch_kv_attention<T, FMT, 5>(st, a, odd, wide, steps);
  if (a.features <= 128) return launch_kv_attention<T, FMT, 8>(st, a, odd, wide, steps);
  return launch_kv_attention<T, FMT, 16>(st, a, odd, wide, steps);
}

}  // namespace rai

using namespace rai;

extern "C" int rai_hip_kv_attention(int dev, const rai_hip_tensor *q, const rai_hip_tensor *tables, const rai_hip_tensor *starts, const rai_hip_tensor *lens, int32_t format,
                                    const rai_hip_tensor *k, const rai_hip_tensor *v, const rai_hip_tensor *k_scale, const rai_hip_tensor *v_scale, double scale, int32_t window,
                                    const rai_hip_tensor *out) {
  KvCacheView c;
  RAI_TRY(kv_cache_view("kv_attention", format, k, v, k_scale, v_scale, &c));
  RAI_TRY(validate(q, "q"));
  RAI_TRY(validate(tables, "tables"));
  RAI_TRY(validate(starts, "starts"));
  RAI_TRY(validate(lens, "lens"));
  RAI_TRY(validate(out, "out"));
  RAI_REQUIRE(q->dtype == RAI_BF16 || q->dtype == RAI_F16 || q->dtype == RAI_F32, RAI_ERR_BAD_DTYPE, "kv_attention: q is bf16, f16 or f32");
  RAI_REQUIRE(out->dtype == q->dtype && tables->dtype == RAI_U32 && starts->dtype == RAI_I64 && lens->dtype == RAI_I64, RAI_ERR_BAD_DTYPE,
              "kv_attention: out has q's dtype, tables are u32, starts and lens i64");
  RAI_REQUIRE(q->rank == 3 && same_shape(q, out) && is_contiguous(out), RAI_ERR_BAD_SHAPE, "kv_attention: q is [rows, heads, features], out contiguous of its shape");
  RAI_REQUIRE(tables->rank == 2 && starts->rank == 1 && lens->rank == 1 && lens->shape[0] == tables->shape[0] && starts->shape[0] == tables->shape[0] + 1, RAI_ERR_BAD_SHAPE,
              "kv_attention: tables [R, M], starts [R + 1], lens [R]");
  const int64_t N = q->shape[0], Hq = q->shape[1], D = q->shape[2], R = tables->shape[0], M = tables->shape[1];
  RAI_REQUIRE(Hq > 0 && Hq % c.heads == 0 && Hq <= 65535, RAI_ERR_BAD_SHAPE, "kv_attention: %lld query heads over %d of the cache", (long long)Hq, c.heads);
  RAI_REQUIRE(D > 0 && (D + 15) / 16 * 16 == c.features, RAI_ERR_BAD_SHAPE, "kv_attention: heads of %lld features want a cache of %lld, not %d", (long long)D,
              (long long)((D + 15) / 16 * 16), c.features);
  RAI_REQUIRE(M * c.page < (int64_t)1 << 31 && N < (int64_t)1 << 31 && R < (int64_t)1 << 24, RAI_ERR_UNSUPPORTED, "kv_attention: rows and tokens of a table are below 2^31, requests below 2^24");
  RAI_REQUIRE((D == 1 || q->stride[2] == 1) && (M <= 1 || tables->stride[1] == 1) && is_contiguous(starts) && is_contiguous(lens), RAI_ERR_BAD_STRIDE,
              "kv_attention: features and pages of a table have unit stride, starts and lens are contiguous");
  RAI_REQUIRE(window >= 0, RAI_ERR_BAD_ARG, "kv_attention: window %d", window);
  const rai_hip_tensor *ins[] = {q, tables, starts, lens, k, v, k_scale, v_scale};
  for (const rai_hip_tensor *i : ins) RAI_REQUIRE(!overlap(i, out), RAI_ERR_BAD_ARG, "kv_attention: out lies over an input");
  RAI_REQUIRE((N * (Hq / c.heads) / 16 + R) * c.heads < (int64_t)1 << 23, RAI_ERR_UNSUPPORTED, "kv_attention: %lld rows of %lld heads over %d and %lld requests are more than 2^23 tiles", (long long)N,
              (long long)Hq, c.heads, (long long)R);
  hipStream_t st = stream_of(dev);
  if (!st) return RAI_ERR_HIP;
  if (N == 0 || R == 0) return RAI_OK;
  KvAttnArgs a;
  memset(&a, 0, sizeof(a));
  const int64_t es = (int64_t)dtype_size(q->dtype);
  a.q = base_ptr(q);
  a.out = base_ptr(out);
  a.q_row = q->stride[0];
  a.q_head = q->stride[1];
  a.tables = (const uint32_t *)base_ptr(tables);
  a.table_ld = tables->stride[0];
  a.M = M; a.N = N;
  a.starts = (const int64_t *)base_ptr(starts);
  a.lens = (const int64_t *)base_ptr(lens);
  a.k = c.k; a.v = c.v; a.k_scale = c.k_scale; a.v_scale = c.v_scale;
  a.pages = (uint32_t)(M == 0 ? 0 : c.pages < (int64_t)UINT32_MAX ? c.pages : (int64_t)UINT32_MAX);
  a.R = (int)R; a.Hq = (int)Hq; a.Hkv = c.heads; a.G = (int)(Hq / c.heads); a.D = (int)D;
  a.features = c.features; a.page_shift = c.page_shift;
  a.window = window > 0 ? window : 2 * kKvFar;
  a.reach = window > 0 && window < INT32_MAX - kStep ? window + kStep : INT32_MAX;
  a.per_group = 1.0 / a.G;
  // rows off 16-byte boundaries, and heads of features in no whole eights, go through rows of the cache's features
  const bool even = D % 8 == 0 && (uintptr_t)a.q % 16 == 0 && (uintptr_t)a.out % 16 == 0 && (N == 1 || a.q_row * es % 16 == 0) && (Hq == 1 || a.q_head * es % 16 == 0);
  KvRowsArgs odd;
  memset(&odd, 0, sizeof(odd));
  if (!even) {
    odd.src = a.q;
    odd.dst = a.out;
    odd.row = a.q_row;
    odd.head = a.q_head;
    odd.N = N; odd.H = a.Hq; odd.D = a.D; odd.F = a.features; odd.R = a.R;
    odd.starts = a.starts;
  }
  a.scale_log2 = (float)(fabs(scale) * 1.4426950408889634);
  a.turn = scale < 0 ? 0x80008000u : 0;
  a.errors = index_error_counter(dev);

  a.dev = dev;
  const bool wide = N * a.G > 16 * R;   // some request has more than one tile of 16 columns
  // steps of a tile, at most
  const int64_t all = (M * c.page + kStep - 1) / kStep, seen = ((int64_t)a.reach + kStep - 1) / kStep + 1, steps = all < seen ? all : seen;
#define KV_ATTENTION(T) return format == RAI_KV_E4M3 ? launch_by_features<T, RAI_KV_E4M3>(st, a, odd, wide, steps) : launch_by_features<T, RAI_KV_INT8>(st, a, odd, wide, steps)
  if (q->dtype == RAI_BF16) KV_ATTENTION(bf16_raw);
  if (q->dtype == RAI_F16) KV_ATTENTION(f16_raw);
  KV_ATTENTION(float);
#undef KV_ATTENTION
}
