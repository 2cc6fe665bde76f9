// Rotary embedding of rows that each have a position of their own, in both layouts of a pair, and its gradient.
// Reference for the half layout at one offset: rai-models/src/llm/phi2.rs:44-78, qwen2.rs:33-72 (rai_hip_rope).
#include "kv_cache.h"
#include "rotary.h"

namespace rai {

struct RopeRowsArgs {
  const void *x;
  void *out;
  int64_t row, head;             // strides of x; features have stride 1
  const int64_t *positions;
  const double *frequencies;
  int64_t N;
  int H, D, rot, inverse;
  int tokens;                    // rows to a block
  double magnitude;
};

// Cosine and sine of a turn, times the magnitude, and a pair by them: of 16-bit rows in f32 (off by 2^-21, their own rounding is 2^-11 or more), of f32 rows in
// f64, so that either is rounded once that shows.  (8192 f32 rows of 64 heads of 80 features 67 us, in f32
// 69; 4099 of 16 heads of 128, all turned, 13.0 for 11.5.)
template <typename T> struct Turn {
  typedef float2 type;
  static __device__ __forceinline__ float2 of(double turns, double magnitude) {
    float s, c;
    sincospif(2.f * (float)turns, &s, &c);
    return make_float2(c * (float)magnitude, s * (float)magnitude);
  }
};
template <> struct Turn<float> {
  typedef double2 type;
  static __device__ __forceinline__ double2 of(double turns, double magnitude) {
    double s, c;
    sincospi(2.0 * turns, &s, &c);
    return make_double2(c * magnitude, s * magnitude);
  }
};
template <typename T> __device__ __forceinline__ void rotate(T *u, T *v, float2 c) {
  const float x = (float)Scalar<T>::load(u), y = (float)Scalar<T>::load(v);
  Scalar<T>::store(u, fmaf(x, c.x, -y * c.y));
  Scalar<T>::store(v, fmaf(y, c.x, x * c.y));
}
__device__ __forceinline__ void rotate(float *u, float *v, double2 c) {
  const double x = *u, y = *v;
  *u = (float)fma(x, c.x, -y * c.y);
  *v = (float)fma(y, c.x, x * c.y);
}

// A block turns `tokens` rows.  Every thread takes V features of a head and, in the half layout, their partners; it asks for kAtOnce such items before anything
// else.  Meanwhile the cosines and sines of the block's rows go to LDS, each angle once for all heads: position x frequency in 64 bits, whole turns taken off,
// so that far positions lose nothing (a product in 32 bits is off by 0.03 radians at position 10^6).  Bound by memory: x read once, out written once; 8192 rows
// of 64 heads of 80 bf16 features take 35 us, as a copy of those 84 MB does (items one after another behind the angles 49 us, four at once 37, eight 39).
constexpr int kAtOnce = 2;
template <typename T, bool INTERLEAVED, int V>
__global__ void __launch_bounds__(256) k_rope_rows(RopeRowsArgs a) {
  typedef typename Turn<T>::type Angle;
  extern __shared__ __attribute__((aligned(16))) uint8_t turns_lds[];
  Angle *const turn = reinterpret_cast<Angle *>(turns_lds);   // [tokens][rot / 2]
  struct alignas(sizeof(T) * V) Pack { T v[V]; };
  const int half = a.rot / 2;
  const int64_t n0 = (int64_t)blockIdx.x * a.tokens;
  const int rows = (int)min((int64_t)a.tokens, a.N - n0);
  // Items of a head: interleaved packs are pairs by themselves; otherwise packs that are turned with their partners (V == 1: pairs of
  // either layout), then packs that are not.
  constexpr bool SELF = INTERLEAVED && V > 1;
  const int turned = SELF ? (a.rot + V - 1) / V : half / V, items = SELF ? a.D / V : turned + (a.D - a.rot) / V;
  const uint32_t total = (uint32_t)rows * a.H * items;
  for (uint32_t e0 = threadIdx.x; e0 < total || e0 == threadIdx.x; e0 += 256 * kAtOnce) {
    Pack p[kAtOnce], q[kAtOnce];
    int t[kAtOnce], it[kAtOnce], d[kAtOnce];
    T *dst[kAtOnce];
    const int apart = INTERLEAVED ? 1 : half;   // partners
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const uint32_t e = e0 + 256 * u, r = e / items;
      if (e >= total) break;
      it[u] = e - r * items;
      t[u] = r / a.H;
      const uint32_t h = r - t[u] * a.H;
      d[u] = SELF ? it[u] * V : it[u] >= turned ? a.rot + (it[u] - turned) * V : INTERLEAVED ? 2 * it[u] : it[u] * V;
      const T *const src = (const T *)a.x + (n0 + t[u]) * a.row + (int64_t)h * a.head + d[u];
      dst[u] = (T *)a.out + ((n0 + t[u]) * a.H + h) * a.D + d[u];
      p[u] = *reinterpret_cast<const Pack *>(src);
      if (!SELF && it[u] < turned) q[u] = *reinterpret_cast<const Pack *>(src + apart);
    }
    if (e0 == threadIdx.x) {
      for (int e = threadIdx.x; e < rows * half; e += 256) {
        const int n = e / half, i = e - n * half;
        const double turns = (double)a.positions[n0 + n] * a.frequencies[i] * 0.15915494309189533577;   // of 2 pi
        Angle c = Turn<T>::of(turns - rint(turns), a.magnitude);
        if (a.inverse) c.y = -c.y;
        turn[e] = c;
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (e0 + 256 * u >= total) break;
      if (it[u] < turned) {
        const Angle *const c = turn + t[u] * half;
        if constexpr (SELF) {
#pragma unroll
          for (int j = 0; j < V; j += 2)
            if (d[u] + j < a.rot) rotate(&p[u].v[j], &p[u].v[j + 1], c[(d[u] + j) / 2]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) rotate(&p[u].v[j], &q[u].v[j], c[it[u] * V + j]);
          *reinterpret_cast<Pack *>(dst[u] + apart) = q[u];
        }
      }
      *reinterpret_cast<Pack *>(dst[u]) = p[u];
    }
  }
}

template <typename T> static void launch_rope_rows(hipStream_t st, const RopeRowsArgs &a, bool interleaved, bool vec) {
  constexpr int V = 16 / sizeof(T);
  const dim3 grid((unsigned)((a.N + a.tokens - 1) / a.tokens));
  const size_t lds = (size_t)a.tokens * (a.rot / 2) * sizeof(typename Turn<T>::type);
  if (interleaved && vec) hipLaunchKernelGGL((k_rope_rows<T, true, V>), grid, dim3(256), lds, st, a);
  else if (interleaved) hipLaunchKernelGGL((k_rope_rows<T, true, 1>), grid, dim3(256), lds, st, a);
  else if (vec) hipLaunchKernelGGL((k_rope_rows<T, false, V>), grid, dim3(256), lds, st, a);
  else hipLaunchKernelGGL((k_rope_rows<T, false, 1>), grid, dim3(256), lds, st, a);
}

__global__ void __launch_bounds__(256) k_rope_frequencies(double *out, int n, double base, double factor, double low, double high, double original) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  double f = pow(base, -2.0 * i / (2 * n));
  if (factor > 0) {
    const double wave = 6.283185307179586476925 / f;
    if (wave > original / low) f /= factor;
    else if (wave >= original / high) {
      const double s = (original / wave - low) / (high - low);
      f = (1.0 - s) * f / factor + s * f;
    }
  }
  out[i] = f;
}

}  // namespace rai

using namespace rai;

extern "C" int rai_hip_rope_frequencies(int dev, double base, double factor, double low, double high, double original, const rai_hip_tensor *out) {
  RAI_TRY(validate(out, "out"));
  RAI_REQUIRE(out->dtype == RAI_F64, RAI_ERR_BAD_DTYPE, "rope_frequencies: out is f64");
  RAI_REQUIRE(out->rank == 1 && is_contiguous(out) && out->shape[0] < 1 << 20, RAI_ERR_BAD_SHAPE, "rope_frequencies: out is contiguous [rotated features / 2]");
  RAI_REQUIRE(base > 0 && base < INFINITY, RAI_ERR_BAD_ARG, "rope_frequencies: base %g", base);
  RAI_REQUIRE(factor == 0 || (factor > 0 && factor < INFINITY && low > 0 && high > low && high < INFINITY && original > 0 && original < INFINITY), RAI_ERR_BAD_ARG,
              "rope_frequencies: factor %g, low %g, high %g, original %g", factor, low, high, original);
  hipStream_t st = stream_of(dev);
  if (!st) return RAI_ERR_HIP;
  const int n = (int)out->shape[0];
  if (n == 0) return RAI_OK;
  hipLaunchKernelGGL(k_rope_frequencies, dim3((n + 255) / 256), dim3(256), 0, st, (double *)base_ptr(out), n, base, factor, low, high, original);
  return launch_check("rope_frequencies");
}

extern "C" int rai_hip_rope_positions(int dev, const rai_hip_tensor *x, const rai_hip_tensor *positions, const rai_hip_tensor *frequencies, int32_t interleaved,
                                      int32_t inverse, double magnitude, const rai_hip_tensor *out) {
  RAI_TRY(validate(x, "x"));
  RAI_TRY(validate(positions, "positions"));
  RAI_TRY(validate(frequencies, "frequencies"));
  RAI_TRY(validate(out, "out"));
  RAI_REQUIRE(x->dtype == RAI_F32 || x->dtype == RAI_BF16 || x->dtype == RAI_F16, RAI_ERR_BAD_DTYPE, "rope_positions: f32, bf16 or f16 required");
  RAI_REQUIRE(x->dtype == out->dtype && positions->dtype == RAI_I64 && frequencies->dtype == RAI_F64, RAI_ERR_BAD_DTYPE,
              "rope_positions: out has x's dtype, positions are i64, frequencies f64");
  RAI_REQUIRE(x->rank == 3 && same_shape(x, out) && is_contiguous(out), RAI_ERR_BAD_SHAPE, "rope_positions: x is [rows, heads, features], out contiguous of its shape");
  const int64_t N = x->shape[0], H = x->shape[1], D = x->shape[2];
  RAI_REQUIRE(positions->rank == 1 && positions->shape[0] == N && is_contiguous(positions), RAI_ERR_BAD_SHAPE, "rope_positions: positions are contiguous [%lld]", (long long)N);
  RAI_REQUIRE(frequencies->rank == 1 && is_contiguous(frequencies) && 2 * frequencies->shape[0] <= D, RAI_ERR_BAD_SHAPE,
              "rope_positions: frequencies are contiguous, one for each pair of at most %lld features", (long long)D);
  RAI_REQUIRE(D <= 1024 && H < (int64_t)1 << 20 && N < (int64_t)1 << 31, RAI_ERR_UNSUPPORTED, "rope_positions: %lld rows of %lld heads of %lld features", (long long)N, (long long)H, (long long)D);
  RAI_REQUIRE(D == 1 || x->stride[2] == 1, RAI_ERR_BAD_STRIDE, "rope_positions: features must have unit stride");
  RAI_REQUIRE(!overlap(x, out) && !overlap(positions, out) && !overlap(frequencies, out), RAI_ERR_BAD_ARG, "rope_positions: out lies over an input");
  hipStream_t st = stream_of(dev);
  if (!st) return RAI_ERR_HIP;
  if (numel(out) == 0) return RAI_OK;
  RopeRowsArgs a;
  a.x = base_ptr(x);
  a.out = base_ptr(out);
  a.row = x->stride[0];
  a.head = x->stride[1];
  a.positions = (const int64_t *)base_ptr(positions);
  a.frequencies = (const double *)base_ptr(frequencies);
  a.N = N; a.H = (int)H; a.D = (int)D;
  a.rot = 2 * (int)frequencies->shape[0];
  a.inverse = inverse != 0;
  a.magnitude = magnitude;
  const int V = (int)(16 / dtype_size(x->dtype));
  const bool vec = (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.out % 16 == 0 && (N == 1 || a.row % V == 0) && (H == 1 || a.head % V == 0) && D % V == 0 &&
                   (interleaved || (a.rot / 2 % V == 0));
  // Rows enough for what a thread asks for at once, but 2048 blocks first
  int64_t tokens = (kAtOnce * 256 * (vec ? V : 2) + H * D - 1) / (H * D);
  if (tokens > (N + 2047) / 2048) tokens = (N + 2047) / 2048;
  a.tokens = (int)tokens;
  if (x->dtype == RAI_F32) launch_rope_rows<float>(st, a, interleaved != 0, vec);
  else if (x->dtype == RAI_BF16) launch_rope_rows<bf16_raw>(st, a, interleaved != 0, vec);
  else launch_rope_rows<f16_raw>(st, a, interleaved != 0, vec);
  return launch_check("rope_positions");
}
