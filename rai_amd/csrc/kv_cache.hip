// Pages of an 8-bit key/value cache: which tokens of a step go where (k_kv_plan), and the step's keys and values into
// their pages (k_kv_append).  No counterpart in the reference, whose models concatenate their caches (phi2.rs:233-243).
#include "kv_cache.h"

namespace rai {

static void span(const rai_hip_tensor *t, uintptr_t *lo, uintptr_t *hi) {
  const size_t es = dtype_size(t->dtype);
  *lo = (uintptr_t)t->data + t->offset * es;
  int64_t last = 0;
  for (int i = 0; i < t->rank; ++i) last += (t->shape[i] - 1) * t->stride[i];
  *hi = *lo + (last + 1) * es;
}

bool overlap(const rai_hip_tensor *a, const rai_hip_tensor *b) {
  if (numel(a) == 0 || numel(b) == 0) return false;
  uintptr_t a0, a1, b0, b1;
  span(a, &a0, &a1);
  span(b, &b0, &b1);
  return a0 < b1 && b0 < a1;
}

int kv_cache_view(const char *what, int32_t format, const rai_hip_tensor *k, const rai_hip_tensor *v, const rai_hip_tensor *k_scale,
                  const rai_hip_tensor *v_scale, KvCacheView *out) {
  RAI_TRY(validate(k, "k"));
  RAI_TRY(validate(v, "v"));
  RAI_TRY(validate(k_scale, "k_scale"));
  RAI_TRY(validate(v_scale, "v_scale"));
  RAI_REQUIRE(format == RAI_KV_E4M3 || format == RAI_KV_INT8, RAI_ERR_BAD_ARG, "%s: format %d", what, format);
  RAI_REQUIRE(k->dtype == RAI_U8 && v->dtype == RAI_U8 && k_scale->dtype == RAI_F32 && v_scale->dtype == RAI_F32, RAI_ERR_BAD_DTYPE,
              "%s: the cache is u8 codes and f32 scales", what);
  RAI_REQUIRE(k->rank == 4 && v->rank == 4 && k_scale->rank == 2 && v_scale->rank == 2, RAI_ERR_BAD_SHAPE,
              "%s: the cache is k [pages, heads, page, features], v [pages, heads, features, page], scales [pages, heads]", what);
  const int64_t P = k->shape[0], H = k->shape[1], B = k->shape[2], D = k->shape[3];
  RAI_REQUIRE(v->shape[0] == P && v->shape[1] == H && v->shape[2] == D && v->shape[3] == B, RAI_ERR_BAD_SHAPE,
              "%s: v must be [pages, heads, features, page] of k's sizes", what);
  RAI_REQUIRE(k_scale->shape[0] == P && k_scale->shape[1] == H && same_shape(k_scale, v_scale), RAI_ERR_BAD_SHAPE,
              "%s: scales must be [pages, heads]", what);
  RAI_REQUIRE(P > 0 && P < (int64_t)1 << 31 && H > 0 && H <= 65535, RAI_ERR_BAD_SHAPE, "%s: %lld pages of %lld heads", what, (long long)P, (long long)H);
  RAI_REQUIRE(B >= 16 && B <= 256 && (B & (B - 1)) == 0, RAI_ERR_BAD_SHAPE, "%s: a page is 16, 32, 64, 128 or 256 tokens, not %lld", what, (long long)B);
  RAI_REQUIRE(D > 0 && D % 16 == 0 && D <= kKvMaxFeatures, RAI_ERR_BAD_SHAPE,
              "%s: the cache's features are a multiple of 16 up to %d, not %lld", what, kKvMaxFeatures, (long long)D);
  RAI_REQUIRE(is_contiguous(k) && is_contiguous(v) && is_contiguous(k_scale) && is_contiguous(v_scale), RAI_ERR_BAD_STRIDE,
              "%s: the cache must be contiguous", what);
  RAI_REQUIRE((uintptr_t)base_ptr(k) % 16 == 0 && (uintptr_t)base_ptr(v) % 16 == 0, RAI_ERR_BAD_STRIDE, "%s: the cache must begin on 16 bytes", what);
  out->k = (uint8_t *)base_ptr(k);
  out->v = (uint8_t *)base_ptr(v);
  out->k_scale = (float *)base_ptr(k_scale);
  out->v_scale = (float *)base_ptr(v_scale);
  out->pages = P;
  out->heads = (int)H;
  out->page = (int)B;
  out->page_shift = __builtin_ctz((unsigned)B);
  out->features = (int)D;
  out->format = format;
  return RAI_OK;
}

// ---------------------------------------------------------------- plan
constexpr int kPlanThreads = 256;
constexpr int kPlanRequests = 4096;   // what a block's scan holds in LDS

struct KvPlanArgs {
  const int64_t *lens, *add, *taken;
  const uint32_t *free_pages, *tables;
  int64_t free_stride, table_ld;
  uint32_t *out_tables;
  int64_t out_ld;
  int64_t *out_lens, *out_taken, *starts, *positions;
  uint32_t *runs;
  int64_t F, M, N, W;
  int R, shift;
  unsigned long long *errors;
};

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int64_t wave_scan(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
// The sum of what the threads before this one hold; `total`: of all.  Two barriers.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *total, int64_t *sums) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t upto = wave_scan(v, lane);
  if (lane == 63) sums[w] = upto;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    if (i < w) before += sums[i];
    all += sums[i];
  }
  __syncthreads();
  *total = all;
  return before + upto - v;
}
// The first of n rising numbers that is greater than x (n where none is).
__device__ __forceinline__ int first_above(const uint32_t *a, int n, uint32_t x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Lengths to pages, in one launch.  With c = ceil(len / page) and need = ceil((len + add) / page) - c, request r takes the free
// pages taken + E_r .. + need_r - 1, E the sum of the needs before it; its new tokens are rows starts[r] .. of the batch, and each
// page they touch gives a run (page, first slot, first row, rows).  Every block sums over all requests by itself (4096 at most: 64 KB
// out of L2) rather than wait for another, keeps the three running sums in LDS, and then does its share of the runs, rows and table
// entries, each of which finds its request by bisection there.  Bound by its chain of trips: lengths read in each of three passes (a thread's requests
// lie next to each other, so a wave's reads are spread), sums, bisection, table entry, store; 64 requests take 5.3 us, 512 with
// 160 new rows each and tables of 1024 entries 9.2, a launch alone 4.2.
__global__ void __launch_bounds__(kPlanThreads) k_kv_plan(KvPlanArgs a) {
  extern __shared__ uint32_t plan_lds[];
  __shared__ int64_t sums[kPlanThreads / 64];
  uint32_t *const row_end = plan_lds, *const piece_end = plan_lds + a.R, *const page_at = plan_lds + 2 * a.R;
  const int R = a.R, per = (R + kPlanThreads - 1) / kPlanThreads, r0 = threadIdx.x * per, r1 = min(r0 + per, R);
  const int64_t room_for = a.M << a.shift, whole = (1 << a.shift) - 1;
  const bool first = blockIdx.x == 0;
  // a length no table could hold counts as one row too many, so that sums of 4096 stay in range
  auto rows_of = [&](int64_t add) { return add < 0 ? 0 : add < ((int64_t)1 << 40) ? add : (int64_t)1 << 40; };
  auto pages_of = [&](int64_t tokens) { return (tokens + whole) >> a.shift; };

  int64_t total, rows = 0;
  for (int r = r0; r < r1; ++r) rows += rows_of(a.add[r]);
  rows = block_scan(rows, &total, sums);
  const int64_t all_rows = total;
  int64_t need = 0, end = rows;
  auto fits = [&](int64_t len, int64_t add, int64_t end_row) { return len >= 0 && add >= 0 && len <= room_for && add <= room_for && len + add <= room_for && end_row <= a.N; };
  for (int r = r0; r < r1; ++r) {
    const int64_t len = a.lens[r], add = a.add[r];
    end += rows_of(add);
    if (fits(len, add, end)) need += pages_of(len + add) - pages_of(len);
  }
  need = block_scan(need, &total, sums);
  const int64_t taken = a.taken[0], room = taken < 0 || taken > a.F ? 0 : a.F - taken;
  int64_t pieces = 0, most = 0;
  end = rows;
  int64_t upto = need;
  int bad = 0;
  for (int r = r0; r < r1; ++r) {
    const int64_t len = a.lens[r], add = a.add[r], start = end;
    end += rows_of(add);
    const bool fit = fits(len, add, end);
    const int64_t want = fit ? pages_of(len + add) - pages_of(len) : 0;
    upto += want;
    const bool served = fit && (want == 0 || upto <= room);
    if (served && want) most = upto;
    if (!served) ++bad;
    const int64_t touched = served && add > 0 ? ((len + add - 1) >> a.shift) - (len >> a.shift) + 1 : 0;
    pieces += touched;
    row_end[r] = (uint32_t)(end < 0xffffffffll ? end : 0xffffffffll);
    piece_end[r] = (uint32_t)touched;
    page_at[r] = served ? (uint32_t)(upto - want) : 0xffffffffu;
    if (first) {
      a.starts[r] = start;
      a.out_lens[r] = served ? len + add : len;
    }
  }
  pieces = block_scan(pieces, &total, sums);
  const int64_t all_pieces = total;
  for (int r = r0; r < r1; ++r) piece_end[r] = (uint32_t)(pieces += piece_end[r]);
  if (first) {
    if (threadIdx.x == 0) a.starts[R] = all_rows;
    if (bad) atomicAdd(a.errors, (unsigned long long)bad);
  }
  // the largest sum that was served: the needs are not negative, so it is the last thread's that served any
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) most = max(most, (int64_t)__shfl_xor(most, o, 64));
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = most;
  __syncthreads();
  if (first && threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < kPlanThreads / 64; ++i) most = max(most, sums[i]);
    a.out_taken[0] = taken + most;
  }

  const int64_t step = (int64_t)gridDim.x * kPlanThreads, at = (int64_t)blockIdx.x * kPlanThreads + threadIdx.x;
  for (int64_t w = at; w < a.W; w += step) {
    uint32_t page = 0, slot = 0, row = 0, count = 0;
    if (w < all_pieces) {
      const int r = first_above(piece_end, R, (uint32_t)w);
      const int64_t len = a.lens[r], stop = len + a.add[r], held = pages_of(len);
      const int64_t start = r ? row_end[r - 1] : 0, i = (len >> a.shift) + w - (r ? piece_end[r - 1] : 0);
      const int64_t from = max(len, i << a.shift), to = min(stop, (i + 1) << a.shift);
      if (i >= held) {
        page = a.free_pages[(taken + page_at[r] + i - held) * a.free_stride];
        a.out_tables[r * a.out_ld + i] = page;
      } else {
        page = a.tables[r * a.table_ld + i];
      }
      slot = (uint32_t)(from & whole);
      row = (uint32_t)(start + from - len);
      count = (uint32_t)(to - from);
    }
    a.runs[w] = page;
    a.runs[a.W + w] = slot;
    a.runs[2 * a.W + w] = row;
    a.runs[3 * a.W + w] = count;
  }
  for (int64_t n = at; n < a.N; n += step) {
    int64_t p = -1;
    if (n < all_rows) {
      const int r = first_above(row_end, R, (uint32_t)n);
      if (page_at[r] != 0xffffffffu) p = a.lens[r] + n - (r ? row_end[r - 1] : 0);
    }
    a.positions[n] = p;
  }
  if (a.out_tables != a.tables)
    for (int64_t e = at; e < R * a.M; e += step) {
      const int64_t r = e / a.M, i = e - r * a.M;
      if (page_at[r] != 0xffffffffu) {
        const int64_t len = a.lens[r];
        if (i >= pages_of(len) && i < pages_of(len + a.add[r])) continue;   // a run's
      }
      a.out_tables[r * a.out_ld + i] = a.tables[r * a.table_ld + i];
    }
}

// ---------------------------------------------------------------- append
struct KvAppendArgs {
  KvCacheView c;
  const void *src[2];            // new keys, new values
  int64_t row[2], head[2];       // strides
  const uint32_t *runs;
  int64_t N, W;
  int D;                         // the rows' features; those up to c.features are zero in the cache
  int rounds;                    // units a wave (or block) does in turn
  unsigned long long *errors;
};

template <int FMT> struct KvFormat;
template <> struct KvFormat<RAI_KV_E4M3> {
  static constexpr float kLargest = 448.f;
  static constexpr int kMostExp = 119;
  // e so that `largest` <= kLargest 2^e, for largest = m 2^x, m in [1/2, 1)
  static __device__ __forceinline__ int exponent(float m, int x) { return x - 9 + (m > 0.875f); }
  static __device__ __forceinline__ uint32_t code2(float a, float b) { return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu; }
  static __device__ __forceinline__ float value(uint32_t byte) { return __builtin_amdgcn_cvt_f32_fp8(byte, 0); }
};
template <> struct KvFormat<RAI_KV_INT8> {
  static constexpr float kLargest = 127.f;
  static constexpr int kMostExp = 121;
  static __device__ __forceinline__ int exponent(float m, int x) { return x - 7 + (m > 127.f / 128.f); }
  static __device__ __forceinline__ uint32_t code2(float a, float b) {
    return ((uint32_t)(int)rintf(a) & 0xffu) | ((uint32_t)(int)rintf(b) & 0xffu) << 8;
  }
  static __device__ __forceinline__ float value(uint32_t byte) { return (float)(int8_t)byte; }
};
constexpr int kKvLeastExp = -100;   // of a scale; a page of zeros has it

// A value over its scale: a NaN is zero and what lies outside is the largest, as in the library's casts to whole numbers.
template <int FMT> __device__ __forceinline__ float kv_clamp(float x) {
  return x != x ? 0.f : fminf(fmaxf(x, -KvFormat<FMT>::kLargest), KvFormat<FMT>::kLargest);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// V features of a row as they are read; those from D on are zero.
template <typename T, bool VEC, int V> struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) KvPack { T v[V]; };
template <typename T, bool VEC, int V> __device__ __forceinline__ KvPack<T, VEC, V> kv_load(const T *src, uint32_t d, uint32_t D) {
  KvPack<T, VEC, V> p;
  if constexpr (VEC) {
    memset(&p, 0, sizeof(p));
    if (d < D) p = *reinterpret_cast<const KvPack<T, VEC, V> *>(src + d);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      memset(&p.v[j], 0, sizeof(T));
      if (d + j < D) p.v[j] = src[d + j];
    }
  }
  return p;
}
// Keeps what was read in the registers as it is: widened copies of it would take twice as many.
template <typename P> __device__ __forceinline__ void kv_keep(P &p) {
  struct Words { uint32_t w[sizeof(P) / 4]; } x = __builtin_bit_cast(Words, p);
#pragma unroll
  for (size_t i = 0; i < sizeof(P) / 4; ++i) asm volatile("" : "+v"(x.w[i]));
  p = __builtin_bit_cast(P, x);
}
template <typename T> __device__ __forceinline__ float finite_size(const T &v) {
  const float x = fabsf((float)Scalar<T>::load(&v));
  return x < INFINITY ? x : 0.f;
}
template <int FMT> __device__ __forceinline__ uint32_t kv_codes4(float a, float b, float c, float d) {
  typedef KvFormat<FMT> Fm;
  return Fm::code2(kv_clamp<FMT>(a), kv_clamp<FMT>(b)) | Fm::code2(kv_clamp<FMT>(c), kv_clamp<FMT>(d)) << 16;
}
// Four codes to another scale.
template <int FMT> __device__ __forceinline__ uint32_t kv_rescale4(uint32_t x, float ratio) {
  typedef KvFormat<FMT> Fm;
  return kv_codes4<FMT>(Fm::value(x & 0xff) * ratio, Fm::value(x >> 8 & 0xff) * ratio, Fm::value(x >> 16 & 0xff) * ratio, Fm::value(x >> 24) * ratio);
}

// A unit is a run's keys or values of one head: their largest finite magnitude, the scale 2^e that holds it (and what the page holds already, whose
// codes are taken to the new scale where it is another), the codes.  Scales are powers of two, so a code's value over the old
// scale is exact and one in e4m3 is not rounded again unless it falls below the normal numbers.
// WAVES waves share a unit: one for pages of up to 4096 values, four beyond.  Keys go eight features of a token to a thread; of the
// values, which lie transposed, a wave takes sixteen tokens and a thread two features of them, so that it reads four (f32: eight) bytes of each token and
// writes whole 16-byte pieces of both features, without a trip through LDS.  What the first pass read stays in registers where a thread has
// no more than four packs of keys or one piece of values, and is read again from the caches otherwise.
// A unit owns its page and head alone: a run whose page an earlier run of the call names is refused.
// Bound by vector instructions and by trips: 16 prompts of up to 1300 rows of 8 heads of 128 features (61 MB) take 23 us, 2.6 TB/s, a copy of as many bytes 13.  All of
// a unit stays in registers there; 9.0 million vector instructions are 15 us of every SIMD's time, and the way from the run over its rows and their largest to the first
// code, which the four waves of a SIMD hide in part, takes the rest.  64 single tokens 5.8 us, a launch and the same way once.
template <typename T, int FMT, bool VEC, int WAVES>
__global__ void __launch_bounds__(256) k_kv_append(KvAppendArgs a) {
  typedef KvFormat<FMT> Fm;
  typedef KvPack<T, VEC, 8> Eight;
  typedef KvPack<T, VEC, 2> Two;
  constexpr int HELD = 4, LANES = 64 * WAVES;
  __shared__ float tops[4];
  const int w = blockIdx.x;
  const uint32_t page = a.runs[w], at = a.runs[a.W + w], row = a.runs[2 * a.W + w], count = a.runs[3 * a.W + w];
  if (count == 0) return;
  if (page >= a.c.pages || at >= (uint32_t)a.c.page || count > a.c.page - at || row >= a.N || count > a.N - row) {
    if (blockIdx.y == 0 && threadIdx.x == 0) atomicAdd(a.errors, 1ull);
    return;
  }
  bool again = false;   // an earlier run has the page; asked for ahead of the values, answered behind them
  for (int64_t i = threadIdx.x; i < w; i += 256)
    if (a.runs[i] == page && a.runs[3 * a.W + i] != 0) again = true;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, t = threadIdx.x % LANES, B = a.c.page;
  const uint32_t F = a.c.features, D = a.D, packs = F / 8, items = count * packs;        // of keys
  const int piece0 = at / 16 + wave % WAVES, pieces = (at + count - 1) / 16 + 1;         // of values: pieces of 16 slots, this wave's first
  for (int g = 0; g < a.rounds; ++g) {
    const int unit = (blockIdx.y * a.rounds + g) * (4 / WAVES) + wave / WAVES, h = unit >> 1, side = unit & 1;
    if (g > 0 && h >= a.c.heads) break;   // (in the first round every wave comes to the barrier)
    const bool live = h < a.c.heads;
    const int64_t stride = a.row[side], ph = (int64_t)page * a.c.heads + h;
    const T *const src = (const T *)a.src[side] + (int64_t)row * stride + (int64_t)h * a.head[side];
    float *const scale = (side ? a.c.v_scale : a.c.k_scale) + ph;
    uint8_t *const codes = (side ? a.c.v : a.c.k) + ph * B * F;
    const float s_old = at > 0 && live ? *scale : 0.f;

    Eight keys[HELD];
    Two values[16];
    float top = 0.f;
    auto key_pack = [&](uint32_t e) __attribute__((always_inline)) {
      const uint32_t s = e / packs;
      return kv_load<T, VEC, 8>(src + s * stride, (e - s * packs) * 8, D);
    };
    // Sixteen tokens of features d and d + 1; slots of the piece without a new token repeat the nearest one, which changes no maximum.
    auto value_piece = [&](int p, uint32_t d, Two *out) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 16; ++j) out[j] = kv_load<T, VEC, 2>(src + min(max(16 * p + j - (int)at, 0), (int)count - 1) * stride, d, D);
    };
    if (!live) {
    } else if (side == 0) {
#pragma unroll
      for (int i = 0; i < HELD; ++i) keys[i] = key_pack(min((uint32_t)(t + i * LANES), items - 1));
#pragma unroll
      for (int i = 0; i < HELD; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, finite_size(keys[i].v[j]));
      for (uint32_t e = t + HELD * LANES; e < items; e += LANES) {
        const Eight x = key_pack(e);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, finite_size(x.v[j]));
      }
    } else {
      if (piece0 < pieces) value_piece(piece0, 2 * lane, values);
      if (piece0 < pieces)
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(fmaxf(top, finite_size(values[j].v[0])), finite_size(values[j].v[1]));
      for (int p = piece0; p < pieces; p += WAVES)
        for (uint32_t d0 = p == piece0 ? 128 : 0; d0 < F; d0 += 128) {
          Two x[16];
          value_piece(p, d0 + 2 * lane, x);
#pragma unroll
          for (int j = 0; j < 16; ++j) top = fmaxf(fmaxf(top, finite_size(x[j].v[0])), finite_size(x[j].v[1]));
        }
    }
    top = wave_max(top);
    if (WAVES == 4 && lane == 0) tops[wave] = top;
    if (g == 0) {
      if (__syncthreads_or(again)) {
        if (blockIdx.y == 0 && threadIdx.x == 0) atomicAdd(a.errors, 1ull);
        return;
      }
      if (!live) return;
    } else if (WAVES == 4) {
      __syncthreads();
    }
    if constexpr (WAVES == 4) {
      top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      __syncthreads();   // (tops serves the next unit; and every thread has read the old scale)
    }
    int ex = kKvLeastExp;
    if (top > 0.f) {
      int x;
      const float m = frexpf(top, &x);
      ex = min(max(Fm::exponent(m, x), kKvLeastExp), Fm::kMostExp);
    }
    if (side == 0) {
#pragma unroll
      for (int i = 0; i < HELD; ++i) kv_keep(keys[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) kv_keep(values[j]);
    }
    const float s_own = power_of_two(ex), s_new = s_old >= s_own ? s_old : s_own, inverse = 1.f / s_new, ratio = s_old / s_new;
    const bool rescale = at > 0 && s_old != s_new;
    if (t == 0) *scale = s_new;
    auto number = [&](const T &v) __attribute__((always_inline)) { return (float)Scalar<T>::load(&v) * inverse; };
    if (side == 0) {
      auto store = [&](uint32_t e, const Eight &x) __attribute__((always_inline)) {
        *reinterpret_cast<uint2 *>(codes + at * F + 8 * e) = make_uint2(kv_codes4<FMT>(number(x.v[0]), number(x.v[1]), number(x.v[2]), number(x.v[3])),
                                                                        kv_codes4<FMT>(number(x.v[4]), number(x.v[5]), number(x.v[6]), number(x.v[7])));
      };
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (t + i * LANES < items) store(t + i * LANES, keys[i]);
      for (uint32_t e = t + HELD * LANES; e < items; e += LANES) store(e, key_pack(e));
      if (rescale)
        for (uint32_t e = t; e < at * F / 16; e += LANES) {
          uint4 *const p = reinterpret_cast<uint4 *>(codes) + e, x = *p;
          *p = make_uint4(kv_rescale4<FMT>(x.x, ratio), kv_rescale4<FMT>(x.y, ratio), kv_rescale4<FMT>(x.z, ratio), kv_rescale4<FMT>(x.w, ratio));
        }
    } else {
      auto store = [&](int p, uint32_t d, const Two *x) __attribute__((always_inline)) {
        if (d >= F) return;
        const int first = (int)at - 16 * p, behind = first + (int)count;   // new tokens are slots first .. behind - 1 of the piece
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t c[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) c[j] = kv_codes4<FMT>(number(x[4 * j].v[i]), number(x[4 * j + 1].v[i]), number(x[4 * j + 2].v[i]), number(x[4 * j + 3].v[i]));
          uint4 *const dst = reinterpret_cast<uint4 *>(codes + (d + i) * B + 16 * p);
          if (first > 0 || behind < 16) {
            const uint4 was = *dst;
            const uint32_t old[4] = {was.x, was.y, was.z, was.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int lo = min(max(first - 4 * j, 0), 4), hi = min(max(behind - 4 * j, 0), 4);
              const uint32_t before = lo == 4 ? 0xffffffffu : (1u << 8 * lo) - 1, upto = hi == 4 ? 0xffffffffu : (1u << 8 * hi) - 1;
              const uint32_t kept = rescale ? kv_rescale4<FMT>(old[j], ratio) : old[j];
              c[j] = (kept & before) | (c[j] & upto & ~before) | (old[j] & ~upto & ~before);
            }
          }
          *dst = make_uint4(c[0], c[1], c[2], c[3]);
        }
      };
      if (piece0 < pieces) store(piece0, 2 * lane, values);
      for (int p = piece0; p < pieces; p += WAVES)
        for (uint32_t d0 = p == piece0 ? 128 : 0; d0 < F; d0 += 128) {
          Two x[16];
          value_piece(p, d0 + 2 * lane, x);
          store(p, d0 + 2 * lane, x);
        }
      if (rescale)   // whole pieces before the run's first
        for (uint32_t e = t; e < at / 16 * F; e += LANES) {
          const uint32_t p = e / F, d = e - p * F;
          uint4 *const dst = reinterpret_cast<uint4 *>(codes + d * B + 16 * p), x = *dst;
          *dst = make_uint4(kv_rescale4<FMT>(x.x, ratio), kv_rescale4<FMT>(x.y, ratio), kv_rescale4<FMT>(x.z, ratio), kv_rescale4<FMT>(x.w, ratio));
        }
    }
  }
}

template <typename T, int FMT> static void launch_kv_append(hipStream_t st, KvAppendArgs a, bool vec) {
  const bool wide = a.c.page * a.c.features > 4096;
  const int per_block = wide ? 1 : 4, groups = (2 * a.c.heads + per_block - 1) / per_block;
  // A block looks once for its page among the runs before its own; where runs are many it then does several units' work.
  int64_t rounds = a.W * groups / 4096;
  a.rounds = (int)(rounds < 1 ? 1 : rounds < groups ? rounds : groups);
  const dim3 grid((unsigned)a.W, (unsigned)((groups + a.rounds - 1) / a.rounds));
  if (wide && vec) hipLaunchKernelGGL((k_kv_append<T, FMT, true, 4>), grid, dim3(256), 0, st, a);
  else if (wide) hipLaunchKernelGGL((k_kv_append<T, FMT, false, 4>), grid, dim3(256), 0, st, a);
  else if (vec) hipLaunchKernelGGL((k_kv_append<T, FMT, true, 1>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_kv_append<T, FMT, false, 1>), grid, dim3(256), 0, st, a);
}

}  // namespace rai

using namespace rai;

extern "C" int rai_hip_kv_plan(int dev, const rai_hip_tensor *lens, const rai_hip_tensor *add, const rai_hip_tensor *free_pages, const rai_hip_tensor *taken,
                               const rai_hip_tensor *tables, int32_t page, const rai_hip_tensor *out_tables, const rai_hip_tensor *out_lens,
                               const rai_hip_tensor *out_taken, const rai_hip_tensor *starts, const rai_hip_tensor *positions, const rai_hip_tensor *runs) {
  RAI_TRY(validate(lens, "lens"));
  RAI_TRY(validate(add, "add"));
  RAI_TRY(validate(free_pages, "free_pages"));
  RAI_TRY(validate(taken, "taken"));
  RAI_TRY(validate(tables, "tables"));
  RAI_TRY(validate(out_tables, "out_tables"));
  RAI_TRY(validate(out_lens, "out_lens"));
  RAI_TRY(validate(out_taken, "out_taken"));
  RAI_TRY(validate(starts, "starts"));
  RAI_TRY(validate(positions, "positions"));
  RAI_TRY(validate(runs, "runs"));
  for (const rai_hip_tensor *t : {lens, add, taken, out_lens, out_taken, starts, positions})
    RAI_REQUIRE(t->dtype == RAI_I64 && t->rank == 1 && is_contiguous(t), RAI_ERR_BAD_DTYPE, "kv_plan: lengths, starts and positions are contiguous rank-1 i64");
  for (const rai_hip_tensor *t : {free_pages, tables, out_tables, runs})
    RAI_REQUIRE(t->dtype == RAI_U32, RAI_ERR_BAD_DTYPE, "kv_plan: pages, tables and runs are u32");
  RAI_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0, RAI_ERR_BAD_ARG, "kv_plan: a page is 16, 32, 64, 128 or 256 tokens, not %d", page);
  RAI_REQUIRE(free_pages->rank == 1 && tables->rank == 2 && same_shape(tables, out_tables) && runs->rank == 2 && runs->shape[0] == 4, RAI_ERR_BAD_SHAPE,
              "kv_plan: free_pages [F], tables and out_tables [R, M], runs [4, W]");
  const int64_t R = tables->shape[0], M = tables->shape[1], N = positions->shape[0], W = runs->shape[1];
  RAI_REQUIRE(lens->shape[0] == R && add->shape[0] == R && out_lens->shape[0] == R && starts->shape[0] == R + 1 && taken->shape[0] == 1 &&
                  out_taken->shape[0] == 1,
              RAI_ERR_BAD_SHAPE, "kv_plan: lens, add and out_lens [R], starts [R + 1], taken and out_taken [1], for R = %lld", (long long)R);
  RAI_REQUIRE(R <= kPlanRequests, RAI_ERR_UNSUPPORTED, "kv_plan: %lld requests, %d at most", (long long)R, kPlanRequests);
  RAI_REQUIRE(N < (int64_t)1 << 31 && M < (int64_t)1 << 31 && free_pages->shape[0] < (int64_t)1 << 31, RAI_ERR_UNSUPPORTED, "kv_plan: rows, pages of a table and free pages are below 2^31");
  RAI_REQUIRE(W >= (N < N / page + 2 * R ? N : N / page + 2 * R), RAI_ERR_BAD_SHAPE, "kv_plan: %lld runs; %lld rows of %lld requests may need min(rows, rows / page + 2 requests)",
              (long long)W, (long long)N, (long long)R);
  RAI_REQUIRE((M <= 1 || (tables->stride[1] == 1 && out_tables->stride[1] == 1)) && is_contiguous(runs), RAI_ERR_BAD_STRIDE, "kv_plan: rows of tables have unit stride, runs are contiguous");
  RAI_REQUIRE(R <= 1 || out_tables->stride[0] >= M, RAI_ERR_BAD_STRIDE, "kv_plan: rows of out_tables overlap");
  const bool same = R == 0 || M == 0 || (base_ptr(tables) == base_ptr(out_tables) && (R == 1 || tables->stride[0] == out_tables->stride[0]));
  const rai_hip_tensor *outs[] = {out_tables, out_lens, out_taken, starts, positions, runs}, *ins[] = {lens, add, free_pages, taken, tables};
  for (const rai_hip_tensor *o : outs) {
    for (const rai_hip_tensor *i : ins)
      RAI_REQUIRE((o == out_tables && i == tables && same) || !overlap(o, i), RAI_ERR_BAD_ARG, "kv_plan: an output lies over an input (out_tables may be tables itself)");
    for (const rai_hip_tensor *p : outs) RAI_REQUIRE(o == p || !overlap(o, p), RAI_ERR_BAD_ARG, "kv_plan: two outputs overlap");
  }
  hipStream_t st = stream_of(dev);
  if (!st) return RAI_ERR_HIP;
  KvPlanArgs a;
  a.lens = (const int64_t *)base_ptr(lens);
  a.add = (const int64_t *)base_ptr(add);
  a.taken = (const int64_t *)base_ptr(taken);
  a.free_pages = (const uint32_t *)base_ptr(free_pages);
  a.free_stride = free_pages->stride[0];
  a.tables = (const uint32_t *)base_ptr(tables);
  a.table_ld = tables->stride[0];
  a.out_tables = (uint32_t *)base_ptr(out_tables);
  a.out_ld = out_tables->stride[0];
  if (same) a.out_tables = (uint32_t *)a.tables, a.out_ld = a.table_ld;
  a.out_lens = (int64_t *)base_ptr(out_lens);
  a.out_taken = (int64_t *)base_ptr(out_taken);
  a.starts = (int64_t *)base_ptr(starts);
  a.positions = (int64_t *)base_ptr(positions);
  a.runs = (uint32_t *)base_ptr(runs);
  a.F = free_pages->shape[0]; a.M = M; a.N = N; a.W = W;
  a.R = (int)R;
  a.shift = __builtin_ctz((unsigned)page);
  a.errors = index_error_counter(dev);
  // A block for every 1024 runs, rows or (where they are copied) 4096 table entries: what a block repeats, the sums, is worth that much.
  const int64_t share = (N > W ? N : W) / 1024, copied = same ? 0 : R * M / 4096, blocks = 1 + (share > copied ? share : copied);
  hipLaunchKernelGGL(k_kv_plan, dim3((unsigned)(blocks < 512 ? blocks : 512)), dim3(kPlanThreads), 3 * R * sizeof(uint32_t), st, a);
  return launch_check("kv_plan");
}

extern "C" int rai_hip_kv_append(int dev, const rai_hip_tensor *new_k, const rai_hip_tensor *new_v, const rai_hip_tensor *runs, int32_t format, const rai_hip_tensor *k,
                                 const rai_hip_tensor *v, const rai_hip_tensor *k_scale, const rai_hip_tensor *v_scale) {
  KvAppendArgs a;
  RAI_TRY(kv_cache_view("kv_append", format, k, v, k_scale, v_scale, &a.c));
  RAI_TRY(validate(new_k, "new_k"));
  RAI_TRY(validate(new_v, "new_v"));
  RAI_TRY(validate(runs, "runs"));
  RAI_REQUIRE(new_k->dtype == new_v->dtype && (new_k->dtype == RAI_BF16 || new_k->dtype == RAI_F16 || new_k->dtype == RAI_F32), RAI_ERR_BAD_DTYPE,
              "kv_append: new_k and new_v are both bf16, f16 or f32");
  RAI_REQUIRE(runs->dtype == RAI_U32, RAI_ERR_BAD_DTYPE, "kv_append: runs are u32");
  RAI_REQUIRE(new_k->rank == 3 && same_shape(new_k, new_v) && new_k->shape[1] == a.c.heads, RAI_ERR_BAD_SHAPE, "kv_append: new_k and new_v are [rows, %d, features]", a.c.heads);
  const int64_t N = new_k->shape[0], D = new_k->shape[2];
  RAI_REQUIRE(D > 0 && (D + 15) / 16 * 16 == a.c.features, RAI_ERR_BAD_SHAPE, "kv_append: heads of %lld features want a cache of %lld, not %d", (long long)D,
              (long long)((D + 15) / 16 * 16), a.c.features);
  RAI_REQUIRE(runs->rank == 2 && runs->shape[0] == 4 && is_contiguous(runs), RAI_ERR_BAD_SHAPE, "kv_append: runs are contiguous [4, W]");
  RAI_REQUIRE(N < (int64_t)1 << 31 && runs->shape[1] < (int64_t)1 << 31, RAI_ERR_UNSUPPORTED, "kv_append: rows and runs are below 2^31");
  RAI_REQUIRE(D == 1 || (new_k->stride[2] == 1 && new_v->stride[2] == 1), RAI_ERR_BAD_STRIDE, "kv_append: features must have unit stride");
  const rai_hip_tensor *held[] = {k, v, k_scale, v_scale}, *ins[] = {new_k, new_v, runs};
  for (const rai_hip_tensor *o : held) {
    for (const rai_hip_tensor *i : ins) RAI_REQUIRE(!overlap(o, i), RAI_ERR_BAD_ARG, "kv_append: the cache lies over an input");
    for (const rai_hip_tensor *p : held) RAI_REQUIRE(o == p || !overlap(o, p), RAI_ERR_BAD_ARG, "kv_append: parts of the cache overlap");
  }
  hipStream_t st = stream_of(dev);
  if (!st) return RAI_ERR_HIP;
  a.N = N;
  a.W = runs->shape[1];
  if (N == 0 || a.W == 0) return RAI_OK;
  a.D = (int)D;
  a.src[0] = base_ptr(new_k);
  a.src[1] = base_ptr(new_v);
  a.row[0] = new_k->stride[0]; a.head[0] = new_k->stride[1];
  a.row[1] = new_v->stride[0]; a.head[1] = new_v->stride[1];
  a.runs = (const uint32_t *)base_ptr(runs);
  a.errors = index_error_counter(dev);
  const int64_t es = (int64_t)dtype_size(new_k->dtype);
  auto aligned = [&](const rai_hip_tensor *t) {
    return (uintptr_t)base_ptr(t) % 16 == 0 && (N == 1 || t->stride[0] * es % 16 == 0) && (a.c.heads == 1 || t->stride[1] * es % 16 == 0);
  };
  const bool vec = D % 8 == 0 && aligned(new_k) && aligned(new_v);
#define KV_APPEND(T)                                                                                              \
  do {                                                                                                            \
    if (format == RAI_KV_E4M3) launch_kv_append<T, RAI_KV_E4M3>(st, a, vec);                                      \
    else launch_kv_append<T, RAI_KV_INT8>(st, a, vec);                                                            \
  } while (0)
  if (new_k->dtype == RAI_BF16) KV_APPEND(bf16_raw);
  else if (new_k->dtype == RAI_F16) KV_APPEND(f16_raw);
  else KV_APPEND(float);
#undef KV_APPEND
  return launch_check("kv_append");
}
