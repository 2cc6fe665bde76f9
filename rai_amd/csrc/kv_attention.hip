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

struct KvAttnArgs {
  const void *q;
  void *out;
  int64_t q_row, q_head;
  const uint32_t *tables;
  int64_t table_ld, M, N;
  const int64_t *starts, *lens;
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  int64_t pages;
  int dev, R, Hq, Hkv, G, D, features, page_shift, window;
  float scale_log2;              // scale * log2(e)
  double per_group;              // 1 / G
  int reach;                     // keys that the oldest token of a tile sees, at most
  int which;                     // requests served: 0 all, 1 those of up to 16 columns, 2 the others
  int each;                      // sixteenths of a key that a tile sees more than the one before it
  double per_worker;             // 1 / workers
  int workers;                   // of a key head, each with an even share of the steps; 0: a worker to a tile
  int least;                     // steps of a share at least
  float *part;                   // [Hkv * workers][2][columns of a tile][features] sums of a share's first and last tile
  float *part_m, *part_l;        // their maxima and sums of weights
  struct KvJoin *join;           // [Hkv * workers]
  unsigned long long *errors;
};

// The tile whose last part is a worker's first: workers first .. the worker itself have its parts.
struct KvJoin {
  int first;                     // -1: none
  int place;                     // which of the first worker's two parts
  int start, column, columns;    // the tile's request's first row, its first column and how many it has
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

// ONCE: read by one tile alone, so not to be kept in the L2.
template <bool ONCE> __device__ __forceinline__ kv_u32x4 fetch(const uint8_t *p) {
  const kv_u32x4 *q = reinterpret_cast<const kv_u32x4 *>(p);
  return ONCE ? __builtin_nontemporal_load(q) : *q;
}

// How many bf16 hold a value of type T: products with codes are then exact, so f16 and f32 rows lose nothing on the bf16 matrix instructions.
template <typename T> struct KvTerms;
template <> struct KvTerms<bf16_raw> { static constexpr int n = 1; };
template <> struct KvTerms<f16_raw> { static constexpr int n = 2; };
template <> struct KvTerms<float> { static constexpr int n = 3; };

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
constexpr int kv_blocks(int vt, int nc) { return nc > 1 || vt > 8 ? 1 : vt > 5 ? 2 : 3; }
// Contexts of up to so many steps are not shared between workers.
constexpr int kv_alone(int kw) { return kw == 1 ? 8 : 16; }
constexpr int kv_least(int kw) { return kw == 1 ? 2 : 8; }

// How the work of a key head is dealt out.  A tile of a request is as long as the keys that its last row sees, which grows evenly from tile to
// tile, so that sums over tiles are known without a walk: in sixteenths of a key, tile t takes base + each * (t + 1).
constexpr int kUnits = 16 * kStep;   // of a step
struct KvRequest {
  int start, n, tiles;           // first row, new tokens
  int len, first;                // length, cut to its table's; position of the first new token
};
__device__ __forceinline__ int64_t kv_base(const KvAttnArgs &a, const KvRequest &q) { return 16ll * min(max(q.len - q.n, 0), a.reach); }
__device__ __forceinline__ int64_t kv_units(const KvAttnArgs &a, const KvRequest &q, int64_t tile) { return kv_base(a, q) + (int64_t)a.each * (tile + 1); }
// of the tiles before `tile`
__device__ __forceinline__ int64_t kv_units_before(const KvAttnArgs &a, const KvRequest &q, int64_t tile) { return tile * kv_base(a, q) + a.each * (tile * (tile + 1) / 2); }

template <int QT> __device__ __forceinline__ KvRequest kv_request(const KvAttnArgs &a, int r) {
  KvRequest q;
  const int64_t start = min(max(a.starts[r], (int64_t)0), a.N), said = a.lens[r], most = a.M << a.page_shift;
  q.start = (int)start;
  q.n = (int)(min(max(a.starts[r + 1], start), a.N) - start);
  q.len = (int)min(max(said, (int64_t)0), most);
  q.first = (int)min(max(said, -(1ll << 30)), most) - q.n;
  const int columns = q.n * a.G;
  q.tiles = a.which == 1 ? columns > 0 && columns <= 16 : a.which == 2 && columns <= 16 ? 0 : (columns + QT - 1) / QT;
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

// The columns of a request and key head are its new tokens times the query heads of the group, G to a token; a tile is 16 NC of them.  A
// step is 64 keys:
//     S^T = K . Q^T   (four tiles of 16 keys x 16 columns),      O^T = V^T . P^T   (VT tiles of 16 features x 16 columns)
// on v_mfma_f32_16x16x32_bf16.  Row 4 g + r of score tile t is key 16 g + 4 t + r of the step, so that the lane group g (lanes 16 g ..) holds
// the scores of sixteen neighbouring keys, which are the 16 bytes that it loads of a feature of V: the weights are the second product's
// fragments as they lie in registers, and every load of the cache is 16 bytes a lane, straight to registers.  Sixteen keys lie in one
// page, so a lane group has one page and one scale of keys and of values; both go into the exponent: with x = s ks and y = x + log2(vs),
// exp2(y - m) is the weight times vs, and the sum of sixteen of them over vs is their share of the softmax's.
// KW waves share a tile's steps in turn and merge through LDS; with KW = 1 a wave is a worker by itself and blocks are four of them.
template <typename T, int FMT, int VT, int NC, int KW>
__global__ void __launch_bounds__(256, NC * VT <= 8 ? 2 : 1) k_kv_attention(KvAttnArgs a) {
  constexpr int TERMS = KvTerms<T>::n, QT = 16 * NC, KL = VT / 4, KR = VT % 4;   // 16-byte loads of a key's features; features left
  constexpr int KS = 2 * KL + (KR == 0 ? 0 : KR == 3 ? 2 : 1);                     // products along the features
  constexpr int KN = KL + (KR == 3);                                               // whole 16-byte loads
  constexpr bool TAIL = KR == 1 || KR == 2;                                        // and one of 8 bytes
  constexpr int WPB = 4 / KW;                                                      // workers of a block
  constexpr bool HOIST = NC > 1 && VT <= 8 && TERMS == 1;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Blocks go to the XCDs in turn: each gets neighbouring workers, whose keys are often the same.
  const int blocks = gridDim.x * gridDim.y, linear = blockIdx.y * gridDim.x + blockIdx.x;
  const int place = blocks % 8 == 0 ? linear % 8 * (blocks / 8) + linear / 8 : linear;
  const int kvh = place / gridDim.x, worker = place % gridDim.x * WPB + (KW == 1 ? w : 0);

  // ------------------------------------------------ this worker's first request and tile, and how far its share goes
  // Every wave sums over the requests by itself, 64 at a time, without LDS or barriers: tiles, if each is a worker's, or their units.  (The code
  // is kept short all through: a wave runs most of it once, at the rate at which instructions arrive.)
  KvRequest req;
  int r = -1, tile = 0;
  int64_t from = 0, left = 1, share = 1, tile_at = 0;   // `from` units of the tile are others'; tile_at: units before the tile
  {
    KvRequest x;
    int64_t own = 0, upto = 0, total = 0, u = worker;
    for (int pass = 0; pass < 2 && r < 0; ++pass) {
      int64_t at = 0;
#pragma unroll 1
      for (int i = 0; i < a.R; i += 64) {
        if (pass == 0 || a.R > 64) {
          x.tiles = 0;
          if (i + lane < a.R) x = kv_request<QT>(a, i + lane);
          own = a.workers == 0 ? x.tiles : x.tiles ? kv_units_before(a, x, x.tiles) : 0;
          upto = at + wave_scan(own, lane);
        }
        const uint64_t here = __ballot(pass == 1 && u < upto);
        if (here) {
          const int f = __builtin_ctzll(here);
          r = i + f;
          tile_at = lane_of(upto - own, f);
          req.start = __builtin_amdgcn_readlane(x.start, f);
          req.n = __builtin_amdgcn_readlane(x.n, f);
          req.len = __builtin_amdgcn_readlane(x.len, f);
          req.first = __builtin_amdgcn_readlane(x.first, f);
          req.tiles = __builtin_amdgcn_readlane(x.tiles, f);
          break;
        }
        at = lane_of(upto, 63);
      }
      if (pass == 0) {
        total = at;
        if (a.workers) {
          share = max((int64_t)((double)total * a.per_worker) + 1, (int64_t)a.least * kUnits);   // times the workers: no less than the total
          u = worker * share;
          if ((KW == 1 ? lane : threadIdx.x) == 0) a.join[(int64_t)kvh * a.workers + worker].first = -1;
        }
        if (u >= total) return;
      }
    }
    if (r < 0) return;
    if (a.workers) {
      int lo = 0, hi = req.tiles - 1;   // the tile that unit u lies in
#pragma unroll 1
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (kv_units_before(a, req, mid) <= u - tile_at) lo = mid;
        else hi = mid - 1;
      }
      tile = lo;
      tile_at += kv_units_before(a, req, tile);
      from = u - tile_at;
      left = min(share, total - u);
    } else {
      tile = (int)(u - tile_at);
      left = kv_units(a, req, tile);
    }
  }

  const int64_t head_bytes = ((int64_t)1 << a.page_shift) * a.features;
  const int slot_mask = (1 << a.page_shift) - 1, k_group = col >> 2;
  // Features behind the cache's last are read again from its beginning: q is zero there.
  int k_at[KN ? KN : 1];
#pragma unroll
  for (int i = 0; i < KN; ++i) k_at[i] = i * 64 + 16 * g < a.features ? i * 64 + 16 * g : 0;
  const int tail_at = KN * 64 + 8 * g < a.features ? KN * 64 + 8 * g : 0;
  int v_at[VT];
#pragma unroll
  for (int t = 0; t < VT; ++t) v_at[t] = (16 * t + col < a.features ? 16 * t + col : 0) << a.page_shift;

  bool first = true;   // of the worker's tiles
  for (;; first = false) {
    // ---------------------------------------------- the tile: its columns, the steps of it that are this worker's
    const int64_t size = kv_units(a, req, tile), to = min(size, from + left);
    const int len = req.len, columns = req.n * a.G;
    int rows[NC], heads[NC], hi[NC], lo[NC];
    bool live[NC];
    // how far token i sees: keys lo .. hi
    auto token = [&](int x) { return (int)(((double)x + 0.5) * a.per_group); };
    auto newest = [&](int i) { return min(max(req.first + i, -1), len - 1); };
    auto oldest = [&](int i) { return max(max(req.first + i, -1) - a.window + 1, 0); };
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int x = tile * QT + c * 16 + col;
      live[c] = x < columns;
      const int i = live[c] ? token(x) : 0;   // (a column behind the last repeats the first, and goes nowhere)
      rows[c] = req.start + i;
      heads[c] = kvh * a.G + (live[c] ? x - i * a.G : 0);
      hi[c] = live[c] ? newest(i) : -1;
      lo[c] = oldest(i);
    }
    // of the tile's first and last token: every live column sees lo_last .. hi_first, none sees outside lo_first .. hi_last
    const int i_first = token(tile * QT), i_last = token(min((tile + 1) * QT, columns) - 1);
    const int hi_first = newest(i_first), hi_last = newest(i_last), lo_first = oldest(i_first), lo_last = oldest(i_last);
    const int step0 = lo_first / kStep, steps = hi_last >= lo_first ? hi_last / kStep + 1 - step0 : 0;
    const int s_begin = step0 + (int)min((int64_t)steps, from / kUnits), s_end = step0 + (to == size ? steps : (int)min((int64_t)steps, to / kUnits));

    kv_bf16x8 qf[NC][KS][TERMS];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const T *src = (const T *)a.q + (int64_t)rows[c] * a.q_row + (int64_t)heads[c] * a.q_head;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d0 = TAIL && s == KS - 1 ? KN * 64 + 8 * g : (s / 2) * 64 + 16 * g + 8 * (s & 1);
        struct alignas(16) Eight { T v[8]; } e = *reinterpret_cast<const Eight *>(src + (d0 < a.D ? d0 : 0));
        if (d0 >= a.D) memset(&e, 0, sizeof(e));
        if constexpr (TERMS == 1) {
          qf[c][s][0] = __builtin_bit_cast(kv_bf16x8, e);
        } else {
          union { kv_bf16x2 p[4]; kv_bf16x8 v; } u[TERMS];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            kv_bf16x2 t[TERMS];
            kv_split2<TERMS>((float)Scalar<T>::load(&e.v[2 * j]), (float)Scalar<T>::load(&e.v[2 * j + 1]), t);
#pragma unroll
            for (int i = 0; i < TERMS; ++i) u[i].p[j] = t[i];
          }
#pragma unroll
          for (int i = 0; i < TERMS; ++i) qf[c][s][i] = u[i].v;
        }
      }
    }

    // ---------------------------------------------- the cache
    const uint32_t *const table = a.tables + (int64_t)r * a.table_ld;
    // Of sixteen keys from `key` on: their page, and whether it is there.  Behind the context page 0 stands in.  An entry is asked for two
    // steps ahead and looked at one step ahead: looked at sooner, it would wait for the loads that went out with it.
    struct Page { uint32_t id; bool there; };
    auto entry_of = [&](int key) __attribute__((always_inline)) { return table[key < len ? key >> a.page_shift : 0]; };
    auto page_of = [&](uint32_t id, int key) __attribute__((always_inline)) {
      const bool there = key < len && id < a.pages;
      return Page{there ? id : 0u, there};
    };
    struct Step { kv_u32x4 k[KN ? KN : 1][4]; kv_u32x2 tail[4]; kv_u32x4 v[VT]; };
    struct Scales { float k, v; bool there; };
    Step now;
    auto scales_of = [&](Page pv) __attribute__((always_inline)) {
      const int64_t ph = (int64_t)pv.id * a.Hkv + kvh;
      return Scales{a.k_scale[ph], a.v_scale[ph], pv.there};
    };
    auto load_keys = [&](int st, Page pk) __attribute__((always_inline)) {
      Step &s = now;
      const int key = st * kStep + 16 * k_group + (col & 3);
      const uint8_t *base = a.k + ((int64_t)pk.id * a.Hkv + kvh) * head_bytes + (key & slot_mask) * a.features;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < KN; ++i) s.k[i][t] = fetch<KW != 1>(base + 4 * t * a.features + k_at[i]);
        if (TAIL) s.tail[t] = *reinterpret_cast<const kv_u32x2 *>(base + 4 * t * a.features + tail_at);
      }
    };
    auto load_values = [&](int st, Page pv) __attribute__((always_inline)) {
      const uint8_t *values = a.v + ((int64_t)pv.id * a.Hkv + kvh) * head_bytes + ((st * kStep + 16 * g) & slot_mask);
#pragma unroll
      for (int t = 0; t < VT; ++t) now.v[t] = fetch<KW != 1>(values + v_at[t]);
    };

    kv_f32x4 o[NC][VT];
    float m[NC], l[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      m[c] = kNoScore;
      l[c] = 0.f;
#pragma unroll
      for (int t = 0; t < VT; ++t) o[c][t] = kv_f32x4{0.f, 0.f, 0.f, 0.f};
    }

    int st = s_begin + (KW == 1 ? 0 : w);
    bool missing = false;
    if (st < s_end) {
      const int last = s_end - 1;
      int next = min(st + KW, last);
      uint32_t nk = entry_of(st * kStep + 16 * k_group), nv = entry_of(st * kStep + 16 * g);
      Scales scales;
      {
        const Page pk = page_of(nk, st * kStep + 16 * k_group), pv = page_of(nv, st * kStep + 16 * g);
        nk = entry_of(next * kStep + 16 * k_group);
        nv = entry_of(next * kStep + 16 * g);
        scales = scales_of(pv);
        load_keys(st, pk);
        load_values(st, pv);
      }
      for (; st < s_end; st += KW) {
        const int ahead = min(next + KW, last);
        const uint32_t ak = entry_of(ahead * kStep + 16 * k_group), av = entry_of(ahead * kStep + 16 * g);
        const Page of_k = page_of(nk, next * kStep + 16 * k_group), of_v = page_of(nv, next * kStep + 16 * g);
        const Scales coming = scales_of(of_v);   // (ahead of the keys: what a step hands to the next must not wait for those)
        const int key0 = st * kStep + 16 * g;   // this lane group's first
        const bool there = scales.there, gone = key0 < len && !there;
        missing |= gone;
        if ((st + 1) * kStep > len || __any(gone)) {
          // codes behind the context may be anything; their weight is zero, and zero times a NaN would not be
          const int valid = there ? (int)min(len - key0, (int64_t)16) : 0;
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
        kv_f32x4 s[NC][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int c = 0; c < NC; ++c) s[c][t] = kv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < KS; ++e) {
            kv_bf16x8 f;
            if (TAIL && e == KS - 1) f = kv_unpack<FMT>(now.tail[t].x, now.tail[t].y);
            else f = kv_unpack<FMT>(now.k[e / 2][t][2 * (e & 1)], now.k[e / 2][t][2 * (e & 1) + 1]);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
              for (int i = 0; i < TERMS; ++i) s[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, qf[c][e][i], s[c][t], 0, 0, 0);
          }
        }
        // With several tiles to share them V's fragments are made here, beside the scores' products, and its registers are free for the next step's
        kv_bf16x8 vf[HOIST ? VT : 1][2];
        if constexpr (HOIST) {
#pragma unroll
          for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) vf[t][u] = kv_unpack<FMT>(now.v[t][2 * u], now.v[t][2 * u + 1]);
        }
        const float ks = scales.k * a.scale_log2, vs = there && scales.v > 0.f ? scales.v : 1.f;
        load_keys(next, of_k);
        if constexpr (HOIST) load_values(next, of_v);

        // log2(vs): its exponent, to which the logarithm of a power of two adds nothing
        const uint32_t bits = __float_as_uint(vs);
        const float up_v = (float)((int)(bits >> 23) - 127) + __builtin_amdgcn_logf(__uint_as_float((bits & 0x7fffffu) | 0x3f800000u)), over_v = __builtin_amdgcn_rcpf(vs);
        const bool edge = (st + 1) * kStep - 1 > hi_first || st * kStep < lo_last || __any(gone);
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
                s[c][t][j] = key <= hi[c] && key >= lo[c] && there ? s[c][t][j] * ks : -INFINITY;
              }
          float most = s[c][0][0], least = s[c][0][0];
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) most = fmaxf(most, s[c][t][j]), least = fminf(least, s[c][t][j]);
          top[c] = column_max(fmaxf(times < 0.f ? least * times : most * times, kNoScore));
          grows |= top[c] > m[c] + 8.f;
        }
        // a maximum that grew by less than 2^8 waits: weights stay below 2^8, and sums in f32 lose nothing by it
        if (__any(grows)) {
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const float up = fmaxf(m[c], top[c]), f = __builtin_amdgcn_exp2f(m[c] - up);
            m[c] = up;
            l[c] *= f;
#pragma unroll
            for (int t = 0; t < VT; ++t) o[c][t] *= f;
          }
        }
        kv_bf16x8 pf[NC][2][TERMS];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float down = up_v - m[c];
          float p[16], sum = 0.f;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              p[4 * t + j] = __builtin_amdgcn_exp2f(fmaf(s[c][t][j], times, down));
              sum += p[4 * t + j];
            }
          l[c] = fmaf(sum, over_v, l[c]);
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
          if constexpr (HOIST)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int t = 0; t < VT; ++t)
#pragma unroll
                for (int i = 0; i < TERMS; ++i) o[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[t][u], pf[c][u][i], o[c][t], 0, 0, 0);
        }
        if constexpr (!HOIST) {
#pragma unroll
          for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const kv_bf16x8 f = kv_unpack<FMT>(now.v[t][2 * u], now.v[t][2 * u + 1]);
#pragma unroll
              for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < TERMS; ++i) o[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, pf[c][u][i], o[c][t], 0, 0, 0);
            }
          load_values(next, of_v);
        }
        next = ahead;
        nk = ak;
        nv = av;
        scales = coming;
      }
    }
    if (kvh == 0) {
      const bool past = from == 0 && tile == 0 && (KW == 1 || w == 0) && a.lens[r] > a.M << a.page_shift;
      if ((__any(missing) || past) && lane == 0) atomicAdd(a.errors, 1ull);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) l[c] = column_sum(l[c]);

    if constexpr (KW > 1) {
      // the upper half of the waves hands its sums to the lower, until one is left; values lie in LDS as in registers
      static_assert(NC == 1, "waves that share steps have one tile of 16 columns");
      __shared__ kv_f32x4 sums[KW / 2][VT][64];
      __shared__ float stats[KW / 2][2][64];
#pragma unroll
      for (int half = KW / 2; half > 0; half /= 2) {
        __syncthreads();
        if (w >= half && w < 2 * half) {
#pragma unroll
          for (int t = 0; t < VT; ++t) sums[w - half][t][lane] = o[0][t];
          stats[w - half][0][lane] = m[0];
          stats[w - half][1][lane] = l[0];
        }
        __syncthreads();
        if (w < half) {
          const float m2 = stats[w][0][lane], l2 = stats[w][1][lane], up = fmaxf(m[0], m2);
          const float f1 = __builtin_amdgcn_exp2f(m[0] - up), f2 = __builtin_amdgcn_exp2f(m2 - up);
          m[0] = up;
          l[0] = l[0] * f1 + l2 * f2;
#pragma unroll
          for (int t = 0; t < VT; ++t) o[0][t] = o[0][t] * f1 + sums[w][t][lane] * f2;
        }
      }
    }

    // ---------------------------------------------- out, or to the tile's other parts
    const bool whole = from == 0 && to == size;
    if (KW == 1 || w == 0) {
      const int64_t own = (int64_t)kvh * a.workers + worker, part = (2 * own + !first) * QT;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (!live[c]) continue;
        if (!whole) {
          const int64_t e = part + c * 16 + col;
          if (g == 0) {
            a.part_m[e] = m[c];
            a.part_l[e] = l[c];
          }
#pragma unroll
          for (int t = 0; t < VT; ++t)
            if (16 * t < a.features) *reinterpret_cast<kv_f32x4 *>(a.part + e * a.features + 16 * t + 4 * g) = o[c][t];
          continue;
        }
        const float f = l[c] == 0.f ? 0.f : 1.f / l[c];
        T *dst = (T *)a.out + ((int64_t)rows[c] * a.Hq + heads[c]) * a.D + 4 * g;
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          struct alignas(sizeof(T) * 4) Four { T v[4]; } y;
#pragma unroll
          for (int j = 0; j < 4; ++j) Scalar<T>::store(&y.v[j], l[c] == 0.f ? 0.f : o[c][t][j] * f);
          if (16 * t + 4 * g < a.D) *reinterpret_cast<Four *>(dst + 16 * t) = y;
        }
      }
      if (!whole && to == size && lane == 0) {
        int64_t begin = (int64_t)((double)tile_at / (double)share);
        begin += begin * share > tile_at ? -1 : (begin + 1) * share <= tile_at ? 1 : 0;
        a.join[own] = KvJoin{(int)begin, tile_at != begin * share, req.start, tile * QT, min(QT, columns - tile * QT)};
      }
    }
    left -= to - from;
    if (a.workers == 0 || left <= 0) return;
    from = 0;
    tile_at += size;
    if (++tile >= req.tiles) {
      tile = 0;
      do {
        if (++r >= a.R) return;
        req = kv_request<QT>(a, r);
      } while (req.tiles == 0);
    }
  }
}

// The parts of tiles that workers share, to the output: a block for each worker that had a tile's last part.
template <typename T> __global__ void __launch_bounds__(256) k_kv_attention_join(KvAttnArgs a, int QT) {
  const int64_t worker = blockIdx.x, own = (int64_t)blockIdx.y * a.workers + worker;
  const KvJoin j = a.join[own];
  if (j.first < 0) return;
  const int F4 = a.features / 4;
  for (int e = threadIdx.x; e < j.columns * F4; e += 256) {
    const int c = e / F4, d = (e - c * F4) * 4, x = j.column + c, i = x / a.G;
    auto part_of = [&](int64_t k) { return (2 * ((int64_t)blockIdx.y * a.workers + k) + (k == j.first ? j.place : 0)) * QT + c; };
    float m = kNoScore, l = 0.f;
    kv_f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int64_t k = j.first; k <= worker; k += 4) {   // four parts asked for at a time
      float pm[4], pl[4], up = m;
      kv_f32x4 y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t p = part_of(min(k + u, worker));
        pm[u] = a.part_m[p];
        pl[u] = a.part_l[p];
        y[u] = *reinterpret_cast<const kv_f32x4 *>(a.part + p * a.features + d);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (k + u > worker) pm[u] = kNoScore, pl[u] = 0.f, y[u] = kv_f32x4{0.f, 0.f, 0.f, 0.f};
        up = fmaxf(up, pm[u]);
      }
      const float f = __builtin_amdgcn_exp2f(m - up);
      l *= f;
      o *= f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float g = __builtin_amdgcn_exp2f(pm[u] - up);
        l = fmaf(pl[u], g, l);
#pragma unroll
        for (int v = 0; v < 4; ++v) o[v] = fmaf(y[u][v], g, o[v]);
      }
      m = up;
    }
    const float f = l == 0.f ? 0.f : 1.f / l;
    T *dst = (T *)a.out + (((int64_t)j.start + i) * a.Hq + (int64_t)blockIdx.y * a.G + x - i * a.G) * a.D + d;
    struct alignas(sizeof(T) * 4) Four { T v[4]; } y;
#pragma unroll
    for (int u = 0; u < 4; ++u) Scalar<T>::store(&y.v[u], l == 0.f ? 0.f : o[u] * f);
    if (d < a.D) *reinterpret_cast<Four *>(dst) = y;
  }
}

// Tiles of 16 columns to a wave that is a worker by itself: as many as registers hold.
template <typename T> constexpr int wide_tiles(int features) { return (features <= 128 ? 2 : 1) * (KvTerms<T>::n == 1 ? 2 : 1); }

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

// What a launch takes of the scratch: parts of tiles, and the words about them.
struct KvPlanOfWork {
  int workers, columns;          // of a key head; of a tile
  size_t bytes(const KvAttnArgs &a) const { return workers ? (size_t)a.Hkv * workers * (2ll * columns * (a.features + 2) * 4 + sizeof(KvJoin)) : 0; }
};
template <typename T, int VT, int NC, int KW> static KvPlanOfWork plan_of_work(const KvAttnArgs &a, int64_t steps) {
  constexpr int WPB = 4 / KW;
  if (steps <= kv_alone(KW)) return {0, 16 * NC};
  const int64_t workers = (int64_t)device_cu_count(a.dev) * kv_blocks(VT, NC) * WPB / a.Hkv;
  return {(int)(workers < WPB ? WPB : workers / WPB * WPB), 16 * NC};
}

template <typename T, int FMT, int VT, int NC, int KW> static int launch_tiles(hipStream_t st, KvAttnArgs a, int64_t steps, void *ws) {
  constexpr int QT = 16 * NC, WPB = 4 / KW;
  const KvPlanOfWork p = plan_of_work<T, VT, NC, KW>(a, steps);
  a.each = (16 * QT + a.G - 1) / a.G;
  a.workers = p.workers;
  if (a.workers) {
    const int64_t parts = 2 * QT * (int64_t)a.Hkv * a.workers;
    a.least = kv_least(KW);
    a.per_worker = 1.0 / a.workers;
    a.part = (float *)ws;
    a.part_m = a.part + parts * a.features;
    a.part_l = a.part_m + parts;
    a.join = (KvJoin *)(a.part_l + parts);
  }
  const int64_t slots = a.which == 1 ? a.R : a.N * a.G / QT + a.R, x = a.workers ? a.workers / WPB : (slots + WPB - 1) / WPB;
  hipLaunchKernelGGL((k_kv_attention<T, FMT, VT, NC, KW>), dim3((unsigned)x, (unsigned)a.Hkv), dim3(256), 0, st, a);
  RAI_TRY(launch_check("kv_attention"));
  if (a.workers) {
    hipLaunchKernelGGL((k_kv_attention_join<T>), dim3((unsigned)a.workers, (unsigned)a.Hkv), dim3(256), 0, st, a, QT);
    RAI_TRY(launch_check("kv_attention_join"));
  }
  return RAI_OK;
}

template <typename T, int FMT, int VT> static int launch_kv_attention(hipStream_t st, KvAttnArgs a, const KvRowsArgs &odd, bool wide, int64_t steps) {
  constexpr int NC = wide_tiles<T>(16 * VT);
  // the two launches run one after the other and may use the same scratch
  size_t parts = plan_of_work<T, VT, 1, 4>(a, steps).bytes(a);
  if (wide) {
    const size_t others = plan_of_work<T, VT, NC, 1>(a, steps).bytes(a);
    if (others > parts) parts = others;
  }
  const size_t rows = odd.src ? ((size_t)a.N * a.Hq * a.features * sizeof(T) + 15) / 16 * 16 : 0;
  WorkspaceHold hold;
  void *ws = nullptr;
  if (parts + rows) RAI_TRY(workspace(a.dev, parts + 2 * rows, &ws, &hold));
  const int64_t most = kNumCU * 32;
  KvRowsArgs in = odd, back = odd;
  if (odd.src) {
    a.q = in.dst = (char *)ws + parts;
    a.out = (char *)ws + parts + rows;
    back.src = a.out;
    a.q_row = (int64_t)a.Hq * a.features;
    a.q_head = a.D = a.features;
    const int64_t blocks = (a.N * a.Hq * a.features + 255) / 256;
    hipLaunchKernelGGL((k_kv_rows_widen<T>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, in);
    RAI_TRY(launch_check("kv_rows_widen"));
  }
  if (wide) {
    a.which = 2;
    RAI_TRY((launch_tiles<T, FMT, VT, NC, 1>(st, a, steps, ws)));
    a.which = 1;
  }
  RAI_TRY((launch_tiles<T, FMT, VT, 1, 4>(st, a, steps, ws)));
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
  RAI_REQUIRE(N * (Hq / c.heads) / 16 + R < (int64_t)1 << 23, RAI_ERR_UNSUPPORTED, "kv_attention: %lld rows of %lld heads to a key head and %lld requests", (long long)N, (long long)(Hq / c.heads), (long long)R);
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
  a.pages = M == 0 ? 0 : c.pages;
  a.R = (int)R; a.Hq = (int)Hq; a.Hkv = c.heads; a.G = (int)(Hq / c.heads); a.D = (int)D;
  a.features = c.features; a.page_shift = c.page_shift;
  a.window = window > 0 ? window : INT32_MAX;
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
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.errors = index_error_counter(dev);

  a.dev = dev;
  const bool wide = N * a.G > 16 * R;   // some request has more than one tile of 16 columns
  const int64_t steps = (M * c.page + kStep - 1) / kStep;
#define KV_ATTENTION(T) return format == RAI_KV_E4M3 ? launch_by_features<T, RAI_KV_E4M3>(st, a, odd, wide, steps) : launch_by_features<T, RAI_KV_INT8>(st, a, odd, wide, steps)
  if (q->dtype == RAI_BF16) KV_ATTENTION(bf16_raw);
  if (q->dtype == RAI_F16) KV_ATTENTION(f16_raw);
  KV_ATTENTION(float);
#undef KV_ATTENTION
}
