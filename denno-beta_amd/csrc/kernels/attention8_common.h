// Shared by the matrix-core kernels of attention over the cache in 8 bits (attention8_single.hip, attention8_portions.hip).
#pragma once
#include "cache8.h"

namespace attend8 {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t u32x4;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4;
typedef __attribute__((__vector_size__(2 * sizeof(float)))) float floatx2;

constexpr float LOG2E = 1.44269504088896340736f;
// what a running maximum starts from: below any score, and finite, so that differences of it are numbers
constexpr float LOWEST = -3.0e38f;

// eight e4m3 numbers, as they lie in two words, in bfloat16: exact
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi) {
  u32x4 w;
  w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
  w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
  w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  return __builtin_bit_cast(bf16x8, w);
}

// eight numbers in bfloat16, two per conversion, to nearest
__device__ __forceinline__ bf16x8 to_bf16x8(const float* v) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{v[2 * i], v[2 * i + 1]}, bf16x2));
  return __builtin_bit_cast(bf16x8, w);
}

// Eight 32-bit numbers as PARTS numbers of bfloat16 whose sum they are: each part is what the parts before leave, rounded.  Three
// parts hold all 24 digits of a number, so a product of 32-bit rows with the cache (whose numbers are exact in bfloat16) is three
// products on the matrix cores with nothing lost but the 32-bit sums' own roundings; one part is a rounding to bfloat16.
template <int PARTS>
__device__ __forceinline__ void split(const float* v, bf16x8* parts) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = v[i];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    parts[p] = to_bf16x8(rest);
    if (p + 1 < PARTS) {
      const u32x4 w = __builtin_bit_cast(u32x4, parts[p]);
#pragma unroll
      for (int i = 0; i < 8; ++i) rest[i] -= __uint_as_float((i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
  }
}

// cap * tanh(s / cap) of a score in units of log2(e): s2 = s log2(e).  With x = s / cap, up to 0.625: tanh(x) = x (1 + x^2 P(x^2)), P of degree four through
// Chebyshev's nodes in 64 bits, off by 2^-25 of tanh at most; a score that is small beside the cap so comes out as itself, however
// large the cap.  Elsewhere 1 - 2 / (e^2x + 1), whose error of some 1e-7 is that of tanh itself there (near 0 it would be 1e-7 of the cap,
// not of the score).  The whole is off by 14 half units of the result's last place at most, hardware's power and reciprocal taken a unit off each.
struct Cap {      // (made on the host, so that its numbers take no vector registers)
  float cap2, per_cap, to_tanh;      // cap log2(e) (0: no cap), its inverse, 2 / cap (finite, so that a score of 0 stays 0 under the smallest caps)
  explicit Cap(float cap) : cap2(cap * LOG2E), per_cap(1.0f / cap2), to_tanh(fminf(2.0f / cap, 3.0e38f)) {}
  static constexpr float NEAR = 0.625f;
  __device__ __forceinline__ float near(float s2) const {
    const float x = s2 * per_cap, z = x * x;
    float p = -6.104945778808797e-3f;
    p = fmaf(p, z, 2.100363925867268e-2f);
    p = fmaf(p, z, -5.3852496893706345e-2f);
    p = fmaf(p, z, 0.13332782257758075f);
    p = fmaf(p, z, -0.3333332909943444f);
    return fmaf(s2 * z, p, s2);
  }
  __device__ __forceinline__ float any(float s2) const {
    const float e = __builtin_amdgcn_exp2f(s2 * to_tanh);
    const float far = cap2 * fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
    return fabsf(s2 * per_cap) < NEAR ? near(s2) : far;
  }
  // A lane's N scores, get(i) * by, to put(i, .).  Power and reciprocal take as long as eight other operations, and most tiles of most models' scores
  // have nothing beyond NEAR: those go without (the same bits; 0.62: whatever the two products are rounded to, none is beyond it).  2,048
  // rows of two prompts, 25 heads of 64: 31.3 us with a cap of 30 and 37.5 with one of 3, 24.5 without a cap.
  template <int N, class Get, class Put>
  __device__ __forceinline__ void of(float by, Get get, Put put) const {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(get(i)));
    if (__builtin_amdgcn_ballot_w64(!(most * fabsf(by * per_cap) < 0.62f)) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        put(i, near(get(i) * by));
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);      // (four at a time: registers)
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        put(i, any(get(i) * by));
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

// Results of a row's keys that n_splits workgroups shared out, for every row and head: [rows][heads][n_splits][dh + 2], the running maximum
// (in units of log2(e)), the sum, the weighted values.  A tile's rows are row0 .. row0 + nrows (no nrows: one).
struct Parts {
  const float* part;
  int n_splits;
  const int32_t *tile_seq, *tile_row0, *tile_nrows;
  const float* sink_at;
  int sink, H, dh, ldo;
};

// the splits' results of a tile's rows and a head, in their order
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const Parts a, T* __restrict__ out) {
  const int tile = blockIdx.y, head = blockIdx.x;
  if (a.tile_seq[tile] < 0) return;
  const int row0 = a.tile_row0[tile], nrows = a.tile_nrows ? a.tile_nrows[tile] : 1;
  for (int x = blockIdx.z * 256 + threadIdx.x; x < nrows * a.dh; x += 256 * gridDim.z) {
    const int row = row0 + x / a.dh, d = x % a.dh;
    const float* part = a.part + (static_cast<size_t>(row) * a.H + head) * a.n_splits * (a.dh + 2);
    float m = LOWEST, l = 0.f, v = 0.f;
    for (int s0 = 0; s0 < a.n_splits; s0 += 8) {      // (eight asked for at a time)
      float ms[8], ls[8], vs[8], top = m;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float* p = part + static_cast<size_t>(min(s0 + j, a.n_splits - 1)) * (a.dh + 2);
        ms[j] = p[0], ls[j] = p[1], vs[j] = p[2 + d];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, ms[j]);
      const float f0 = __builtin_amdgcn_exp2f(m - top);
      m = top, l *= f0, v *= f0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = s0 + j < a.n_splits ? __builtin_amdgcn_exp2f(ms[j] - m) : 0.f;
        l = fmaf(ls[j], f, l);
        v = fmaf(vs[j], f, v);
      }
    }
    if (a.sink) l += __builtin_amdgcn_exp2f((a.sink_at ? a.sink_at[head] : 0.f) * LOG2E - m);
    out[static_cast<size_t>(row) * a.ldo + head * a.dh + d] = from_float<T>(l == 0.f ? 0.f : v / l);      // (a row that reads nothing: zeros)
  }
}

static inline void join(const Parts& a, void* out, int n_tiles, int dtype, hipStream_t stream) {
  const dim3 grid(a.H, n_tiles, a.tile_nrows ? 16 : 1);      // (a tile of 128 rows: 8 of them a workgroup)
  if (dtype == DN_BF16) join_kernel<bf16_t><<<grid, 256, 0, stream>>>(a, static_cast<bf16_t*>(out));
  else join_kernel<float><<<grid, 256, 0, stream>>>(a, static_cast<float*>(out));
}

}  // namespace attend8
