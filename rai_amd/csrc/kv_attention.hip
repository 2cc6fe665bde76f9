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
  int R, Hq, Hkv, G, D, features, page_shift, window;
  int q_aligned, out_aligned;
  float scale_log2;              // scale * log2(e)
  int splits, least;             // parts of a context, and steps of a part at least
  int which;                     // requests served: 0 all, 1 those of up to 16 columns, 2 the others
  float *part;                   // [N * Hq][splits][features] sums, then their maxima and sums of weights
  float *part_m, *part_l;
  int *parts;                    // [N * Hq]: how many of `splits` there are
  unsigned long long *errors;
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

// The columns of a request and key head are its new tokens times the query heads of the group, G to a token; a tile is 16 NC of them.  A
// step is 64 keys:
//     S^T = K . Q^T   (four tiles of 16 keys x 16 columns),      O^T = V^T . P^T   (VT tiles of 16 features x 16 columns)
// on v_mfma_f32_16x16x32_bf16.  Row 4 g + r of score tile t is key 16 g + 4 t + r of the step, so that the lane group g (lanes 16 g ..) holds
// the scores of sixteen neighbouring keys, which are the 16 bytes that it loads of a feature of V: the weights are the second product's
// fragments as they lie in registers, and every load of the cache is 16 bytes a lane, straight to registers.  Sixteen keys lie in one
// page, so a lane group has one page and one scale of keys and of values: scores and weights are multiplied by them.
// KW waves share a tile's steps in turn and merge through LDS; with KW = 1 a wave has a tile to itself and blocks are four of them.
template <typename T, int FMT, int VT, int NC, int KW>
__global__ void __launch_bounds__(256, NC * VT <= 8 ? 2 : 1) k_kv_attention(KvAttnArgs a) {
  constexpr int TERMS = KvTerms<T>::n, QT = 16 * NC, KL = VT / 4, KR = VT % 4;   // 16-byte loads of a key's features; features left
  constexpr int KS = 2 * KL + (KR == 0 ? 0 : KR == 3 ? 2 : 1);                     // products along the features
  constexpr int KN = KL + (KR == 3);                                               // whole 16-byte loads
  constexpr bool TAIL = KR == 1 || KR == 2;                                        // and one of 8 bytes
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t slot = KW == 1 ? (int64_t)blockIdx.x * 4 + w : blockIdx.x;
  const int kvh = blockIdx.y;

  // request r has the tiles that begin at starts[r] * G / QT + r: intervals of slots that are always wide enough
  int r = -1;
  for (int i = 0; i < a.R; i += 64) {
    bool before = false;
    if (i + lane < a.R) before = (int64_t)((uint64_t)min(max(a.starts[i + lane], (int64_t)0), a.N) * a.G / QT) + i + lane <= slot;
    r += __popcll(__ballot(before));
  }
  if (r < 0) return;
  r = __builtin_amdgcn_readfirstlane(r);
  const int64_t start = min(max(a.starts[r], (int64_t)0), a.N), stop = min(max(a.starts[r + 1], start), a.N);
  const int64_t tile = slot - (start * a.G / QT + r), columns = (stop - start) * a.G;
  if (tile * QT >= columns) return;
  if (a.which == 1 ? columns > 16 : a.which == 2 && columns <= 16) return;
  const int64_t most = a.M << a.page_shift, said = a.lens[r], len = min(max(said, (int64_t)0), most), n = stop - start;
  if (said > most && tile == 0 && blockIdx.z == 0 && kvh == 0 && threadIdx.x % (KW * 64) == 0) atomicAdd(a.errors, 1ull);

  // this lane's columns: row of q and head, newest and oldest key they see
  int64_t rows[NC];
  int heads[NC];
  int hi[NC], lo[NC];
  bool live[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int64_t x = tile * QT + c * 16 + col;
    live[c] = x < columns;
    const int64_t i = live[c] ? x / a.G : 0;
    rows[c] = start + i;
    heads[c] = kvh * a.G + (live[c] ? (int)(x - i * a.G) : 0);
    const int64_t p = said - n + i;
    hi[c] = live[c] ? (int)min(max(p, (int64_t)-1), len - 1) : -1;
    lo[c] = a.window > 0 ? (int)min(max(p - a.window + 1, (int64_t)0), len) : 0;
  }
  // of the tile's first and last token: every live column sees [lo_last, hi_first], none sees outside [lo_first, hi_last]
  const int64_t p_first = said - n + tile * QT / a.G, p_last = said - n + (min((tile + 1) * QT, columns) - 1) / a.G;
  const int hi_first = (int)min(max(p_first, (int64_t)-1), len - 1), hi_last = (int)min(max(p_last, (int64_t)-1), len - 1);
  const int lo_first = a.window > 0 ? (int)min(max(p_first - a.window + 1, (int64_t)0), len) : 0, lo_last = a.window > 0 ? (int)min(max(p_last - a.window + 1, (int64_t)0), len) : 0;
  const int step0 = lo_first / kStep, steps = max(hi_last / kStep + 1 - step0, 0) * (hi_last >= 0);
  const int share = max((steps + a.splits - 1) / a.splits, a.least), parts = max((steps + share - 1) / share, 1);
  const int z = blockIdx.z;
  if (z >= parts) return;
  const int s_begin = step0 + z * share, s_end = step0 + min(steps, (z + 1) * share);

  kv_bf16x8 qf[NC][KS][TERMS];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const T *src = (const T *)a.q + rows[c] * a.q_row + (int64_t)heads[c] * a.q_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d0 = TAIL && s == KS - 1 ? KN * 64 + 8 * g : (s / 2) * 64 + 16 * g + 8 * (s & 1);
      float x[8];
      if (a.q_aligned && d0 + 8 <= a.D) {
        struct alignas(16) Eight { T v[8]; };
        const Eight e = *reinterpret_cast<const Eight *>(src + d0);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = live[c] ? (float)Scalar<T>::load(&e.v[j]) : 0.f;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = live[c] && d0 + j < a.D ? (float)Scalar<T>::load(src + d0 + j) : 0.f;
      }
      union { kv_bf16x2 p[4]; kv_bf16x8 v; } u[TERMS];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        kv_bf16x2 t[TERMS];
        kv_split2<TERMS>(x[2 * j], x[2 * j + 1], t);
#pragma unroll
        for (int i = 0; i < TERMS; ++i) u[i].p[j] = t[i];
      }
#pragma unroll
      for (int i = 0; i < TERMS; ++i) qf[c][s][i] = u[i].v;
    }
  }

  const uint32_t *const table = a.tables + (int64_t)r * a.table_ld;
  const int64_t head_bytes = ((int64_t)1 << a.page_shift) * a.features;
  const int slot_mask = (1 << a.page_shift) - 1, k_group = col >> 2;
  // Of sixteen keys from `key` on: their page, and whether it is there.  Behind the context page 0 stands in.
  struct Page { uint32_t id; bool there; };
  auto page_of = [&](int key) __attribute__((always_inline)) {
    const bool inside = key < len;
    const uint32_t id = table[inside ? key >> a.page_shift : 0];
    return Page{inside && id < a.pages ? id : 0u, inside && id < a.pages};
  };
  auto lost = [&](const Page &p, int key) __attribute__((always_inline)) { return key < len && !p.there; };

  struct Keys { kv_u32x4 x[KN ? KN : 1][4]; kv_u32x2 tail[4]; };
  struct Step { Keys k; float ks, vs; Page of_v; };
  // Features behind the cache's last are read again from its beginning: q is zero there.
  int k_at[KN ? KN : 1];
#pragma unroll
  for (int i = 0; i < KN; ++i) k_at[i] = i * 64 + 16 * g < a.features ? i * 64 + 16 * g : 0;
  const int tail_at = KN * 64 + 8 * g < a.features ? KN * 64 + 8 * g : 0;
  auto load_keys = [&](int st, Page pk, Page pv) __attribute__((always_inline)) {
    Step s;
    s.of_v = pv;
    const int64_t ph = (int64_t)pv.id * a.Hkv + kvh;
    s.ks = a.k_scale[ph];
    s.vs = a.v_scale[ph];
    const int key = st * kStep + 16 * k_group + (col & 3);
    const uint8_t *base = a.k + ((int64_t)pk.id * a.Hkv + kvh) * head_bytes + (key & slot_mask) * a.features;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < KN; ++i) s.k.x[i][t] = *reinterpret_cast<const kv_u32x4 *>(base + 4 * t * a.features + k_at[i]);
      if (TAIL) s.k.tail[t] = *reinterpret_cast<const kv_u32x2 *>(base + 4 * t * a.features + tail_at);
    }
    return s;
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

  constexpr int STRIDE = KW;
  int st = s_begin + (KW == 1 ? 0 : w);
  bool missing = false;
  if (st < s_end) {
    const int last = s_end - 1;
    Page pk = page_of(st * kStep + 16 * k_group), pv = page_of(st * kStep + 16 * g);
    Step now = load_keys(st, pk, pv);
    int ahead = min(st + STRIDE, last);
    Page nk = page_of(ahead * kStep + 16 * k_group), nv = page_of(ahead * kStep + 16 * g);
    for (; st < s_end; st += STRIDE) {
      const int key0 = st * kStep + 16 * g;   // this lane group's first
      kv_u32x4 v[VT];
      {
        const uint8_t *base = a.v + ((int64_t)now.of_v.id * a.Hkv + kvh) * head_bytes + (key0 & slot_mask);
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          const int d = 16 * t + col;
          v[t] = *reinterpret_cast<const kv_u32x4 *>(base + ((int64_t)(d < a.features ? d : 0) << a.page_shift));
        }
      }
      kv_f32x4 s[NC][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int c = 0; c < NC; ++c) s[c][t] = kv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < KS; ++e) {
          kv_bf16x8 f;
          if (TAIL && e == KS - 1) f = kv_unpack<FMT>(now.k.tail[t].x, now.k.tail[t].y);
          else f = kv_unpack<FMT>(now.k.x[e / 2][t][2 * (e & 1)], now.k.x[e / 2][t][2 * (e & 1) + 1]);
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < TERMS; ++i) s[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, qf[c][e][i], s[c][t], 0, 0, 0);
        }
      }
      const Page of_v = now.of_v;
      const float ks = of_v.there ? now.ks * a.scale_log2 : 0.f, vs = of_v.there ? now.vs : 0.f;
      const int next = min(st + STRIDE, last);
      now = load_keys(next, nk, nv);
      ahead = min(next + STRIDE, last);
      nk = page_of(ahead * kStep + 16 * k_group);
      nv = page_of(ahead * kStep + 16 * g);

      const bool gone = lost(of_v, key0);
      missing |= gone;
      const bool edge = (st + 1) * kStep - 1 > hi_first || st * kStep < lo_last || __any(gone);
      if ((st + 1) * kStep > len || __any(gone)) {
        // codes behind the context may be anything; their weight is zero, and zero times a NaN would not be
        const int valid = of_v.there ? (int)min(len - key0, (int64_t)16) : 0;
        uint32_t keep[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int b = min(max(valid - 4 * j, 0), 4);
          keep[j] = b == 4 ? 0xffffffffu : (1u << 8 * b) - 1;
        }
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[t][j] &= keep[j];
      }
      kv_bf16x8 pf[NC][2][TERMS];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float top = kNoScore;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float x = s[c][t][j] * ks;
            if (edge) {
              const int key = key0 + 4 * t + j;
              x = key <= hi[c] && key >= lo[c] && of_v.there ? x : -INFINITY;
            }
            s[c][t][j] = x;
            top = fmaxf(top, x);
          }
        top = column_max(top);
        // a maximum that grew by less than 2^8 waits: weights stay below 2^8, and sums in f32 lose nothing by it
        if (__any(top > m[c] + 8.f)) {
          const float up = fmaxf(m[c], top), f = __builtin_amdgcn_exp2f(m[c] - up);
          m[c] = up;
          l[c] *= f;
#pragma unroll
          for (int t = 0; t < VT; ++t) o[c][t] *= f;
        }
        float p[16];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = __builtin_amdgcn_exp2f(s[c][t][j] - m[c]);
            l[c] += x;
            p[4 * t + j] = x * vs;
          }
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
#pragma unroll
      for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const kv_bf16x8 f = kv_unpack<FMT>(v[t][2 * u], v[t][2 * u + 1]);
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < TERMS; ++i) o[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, pf[c][u][i], o[c][t], 0, 0, 0);
        }
    }
  }
  if (__any(missing) && kvh == 0 && lane == 0) atomicAdd(a.errors, 1ull);
#pragma unroll
  for (int c = 0; c < NC; ++c) l[c] = column_sum(l[c]);

  if constexpr (KW > 1) {
    // the upper half of the waves hands its sums to the lower, until one is left; values lie in LDS as in registers
    static_assert(NC == 1, "waves that share steps have one tile of 16 columns");
    __shared__ kv_f32x4 sums[KW / 2][VT][64];
    __shared__ float stats[KW / 2][2][64];
#pragma unroll
    for (int half = KW / 2; half > 0; half /= 2) {
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
      __syncthreads();
    }
    if (w > 0) return;
  }

#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (!live[c]) continue;
    const int64_t at = rows[c] * a.Hq + heads[c];
    if (parts > 1) {
      const int64_t e = at * a.splits + z;
      if (g == 0) {
        a.part_m[e] = m[c];
        a.part_l[e] = l[c];
        if (z == 0) a.parts[at] = parts;
      }
#pragma unroll
      for (int t = 0; t < VT; ++t)
        if (16 * t < a.features) *reinterpret_cast<kv_f32x4 *>(a.part + e * a.features + 16 * t + 4 * g) = o[c][t];
      continue;
    }
    if (a.splits > 1 && g == 0) a.parts[at] = 1;
    const float f = l[c] == 0.f ? 0.f : 1.f / l[c];
    T *dst = (T *)a.out + at * a.D;
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      const int d = 16 * t + 4 * g;
      struct alignas(sizeof(T) * 4) Four { T v[4]; } y;
#pragma unroll
      for (int j = 0; j < 4; ++j) Scalar<T>::store(&y.v[j], l[c] == 0.f ? 0.f : o[c][t][j] * f);
      if (a.out_aligned && d + 4 <= a.D) *reinterpret_cast<Four *>(dst + d) = y;
      else
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d + j < a.D) dst[d + j] = y.v[j];
    }
  }
}

// The parts of a row and head to its output: a wave each.
template <typename T> __global__ void __launch_bounds__(256) k_kv_attention_merge(KvAttnArgs a, int64_t begin, int64_t end) {
  const int64_t at = begin + (int64_t)(blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (at >= end) return;
  // rows that belong to no request have no parts
  const int64_t row = at / a.Hq;
  if (row < min(max(a.starts[0], (int64_t)0), a.N) || row >= min(max(a.starts[a.R], (int64_t)0), a.N)) return;
  const int parts = min(a.parts[at], a.splits);
  if (parts <= 1) return;
  float m = kNoScore;
  for (int z = 0; z < parts; ++z) m = fmaxf(m, a.part_m[at * a.splits + z]);
  float l = 0.f, o[kKvMaxFeatures / 64] = {};
  for (int z = 0; z < parts; ++z) {
    const int64_t e = at * a.splits + z;
    const float f = __builtin_amdgcn_exp2f(a.part_m[e] - m);
    l = fmaf(a.part_l[e], f, l);
#pragma unroll
    for (int i = 0; i < kKvMaxFeatures / 64; ++i)
      if (i * 64 + lane < a.features) o[i] = fmaf(a.part[e * a.features + i * 64 + lane], f, o[i]);
  }
  const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < kKvMaxFeatures / 64; ++i)
    if (i * 64 + lane < a.D) Scalar<T>::store((T *)a.out + at * a.D + i * 64 + lane, l == 0.f ? 0.f : o[i] * f);
}

template <typename T, int FMT, int VT, int NC, int KW> static void launch_tiles(hipStream_t st, const KvAttnArgs &a) {
  const int64_t slots = a.N * a.G / (16 * NC) + a.R;
  hipLaunchKernelGGL((k_kv_attention<T, FMT, VT, NC, KW>), dim3((unsigned)(KW == 1 ? (slots + 3) / 4 : slots), (unsigned)a.Hkv, (unsigned)a.splits), dim3(256), 0, st, a);
}

// Tiles of 16 columns to a wave that has a tile to itself: as many as registers hold.
template <typename T> constexpr int wide_tiles(int features) { return (features <= 128 ? 2 : 1) * (KvTerms<T>::n == 1 ? 2 : 1); }

template <typename T, int FMT, int VT> static int launch_kv_attention(hipStream_t st, KvAttnArgs a, bool wide) {
  constexpr int NC = wide_tiles<T>(16 * VT);
  if (wide) {
    a.which = 2;
    launch_tiles<T, FMT, VT, NC, 1>(st, a);
    RAI_TRY(launch_check("kv_attention"));
    a.which = 1;
  }
  launch_tiles<T, FMT, VT, 1, 4>(st, a);
  RAI_TRY(launch_check("kv_attention"));
  if (a.splits > 1) {
    const int64_t waves = a.N * a.Hq;
    dim3 grid;
    RAI_TRY(grid_of_blocks((waves + 3) / 4, 256, &grid));
    hipLaunchKernelGGL((k_kv_attention_merge<T>), grid, dim3(256), 0, st, a, (int64_t)0, waves);
    RAI_TRY(launch_check("kv_attention_merge"));
  }
  return RAI_OK;
}

template <typename T, int FMT> static int launch_by_features(hipStream_t st, const KvAttnArgs &a, bool wide) {
  if (a.features <= 64) return launch_kv_attention<T, FMT, 4>(st, a, wide);
  if (a.features <= 80) return launch_kv_attention<T, FMT, 5>(st, a, wide);
  if (a.features <= 128) return launch_kv_attention<T, FMT, 8>(st, a, wide);
  return launch_kv_attention<T, FMT, 16>(st, a, wide);
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
  a.features = c.features; a.page_shift = c.page_shift; a.window = window;
  a.q_aligned = (uintptr_t)a.q % 16 == 0 && (N == 1 || a.q_row * es % 16 == 0) && (Hq == 1 || a.q_head * es % 16 == 0);
  a.out_aligned = (uintptr_t)a.out % (4 * es) == 0 && D % 4 == 0;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.errors = index_error_counter(dev);

  const bool wide = N * a.G > 16 * R;   // some request has more than one tile of 16 columns
  const int nc = q->dtype == RAI_BF16 ? wide_tiles<bf16_raw>(a.features) : wide_tiles<float>(a.features);
  const int64_t tiles = (N * a.G / (wide ? 16 * nc : 16) + R) * a.Hkv, steps = (M * c.page + kStep - 1) / kStep;
  int64_t splits = 2048 / tiles;
  a.least = 8;
  if (splits > (steps + a.least - 1) / a.least) splits = (steps + a.least - 1) / a.least;
  if (splits > 64) splits = 64;
  if (splits < 1) splits = 1;
  a.splits = (int)splits;
  WorkspaceHold hold;
  if (splits > 1) {
    const int64_t cells = N * Hq * splits;
    void *ws = nullptr;
    RAI_TRY(workspace(dev, (size_t)(cells * (a.features + 2) + N * Hq) * 4, &ws, &hold));
    a.part = (float *)ws;
    a.part_m = a.part + cells * a.features;
    a.part_l = a.part_m + cells;
    a.parts = (int *)(a.part_l + cells);
  }
#define KV_ATTENTION(T) return format == RAI_KV_E4M3 ? launch_by_features<T, RAI_KV_E4M3>(st, a, wide) : launch_by_features<T, RAI_KV_INT8>(st, a, wide)
  if (q->dtype == RAI_BF16) KV_ATTENTION(bf16_raw);
  if (q->dtype == RAI_F16) KV_ATTENTION(f16_raw);
  KV_ATTENTION(float);
#undef KV_ATTENTION
}
