// A step's rows into the paged cache in 8 bits, and attention over it for every size (cache8.h has the layout).
#include "cache8.h"

#include <math.h>

// =======================================================================================
// append: a step's queries and keys turned by their positions, keys and values to the pages
// =======================================================================================
namespace append {
constexpr int THREADS = 256;
constexpr int CHUNK = 16;        // rows whose cos and sin lie in LDS at a time
constexpr int SCALE_MIN = -117;  // the least exponent of a scale: its smallest number, 2^-9, is then 2^-126, a normal 32-bit one

// sin and cos of a 64-bit angle.  The angle less the nearest multiple k of pi/2, taken off in three parts (each product k * part
// is exact inside its fma, so what is lost is some k * 2^-161), leaves |r| <= pi/4; there Taylor's series up to r^15 and r^16 are off by
// less than (pi/4)^17 / 17! = 5e-17.
__device__ __forceinline__ void sin_cos(double a, double& s, double& c) {
  const double k = rint(a * 0.63661977236758134308);
  double r = fma(-k, 1.57079632679489655800, a);
  r = fma(-k, 6.12323399573676603587e-17, r);
  r = fma(-k, -1.49738490485916983e-33, r);
  const double z = r * r;
  double p = -1.0 / 1307674368000.0;
  p = fma(p, z, 1.0 / 6227020800.0);
  p = fma(p, z, -1.0 / 39916800.0);
  p = fma(p, z, 1.0 / 362880.0);
  p = fma(p, z, -1.0 / 5040.0);
  p = fma(p, z, 1.0 / 120.0);
  p = fma(p, z, -1.0 / 6.0);
  const double sr = fma(p * z, r, r);
  p = 1.0 / 20922789888000.0;
  p = fma(p, z, -1.0 / 87178291200.0);
  p = fma(p, z, 1.0 / 479001600.0);
  p = fma(p, z, -1.0 / 3628800.0);
  p = fma(p, z, 1.0 / 40320.0);
  p = fma(p, z, -1.0 / 720.0);
  p = fma(p, z, 1.0 / 24.0);
  p = fma(p, z, -0.5);
  const double cr = fma(p, z, 1.0);
  const long long q = static_cast<long long>(k);
  s = (q & 1) ? cr : sr;
  c = (q & 1) ? sr : cr;
  if (q & 2) s = -s;
  if ((q + 1) & 2) c = -c;
}

// a 64-bit number as the 32-bit one towards zero, its last bit set if anything was cut off: rounding that to fewer digits (a scale of
// two's powers does not touch them) gives what rounding the 64-bit number would
__device__ __forceinline__ float to_odd(double y) {
  float f = static_cast<float>(y);
  const double b = static_cast<double>(f);
  if (b != y && fabs(y) < INFINITY) {
    uint32_t u = __float_as_uint(f);
    if (fabs(b) > fabs(y)) u -= 1;
    f = __uint_as_float(u | 1u);
  }
  return f;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }      // (no for NaN)

// the least e with top <= 448 * 2^e (448 = 1.75 * 2^8), at least SCALE_MIN
__device__ __forceinline__ int scale_exponent(float top) {
  const uint32_t u = __float_as_uint(top);
  const int e = static_cast<int>(u >> 23) - 127;
  return max((u & 0x7fffffu) <= 0x600000u ? e - 8 : e - 7, SCALE_MIN);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// the nearest e4m3 number to y * unit (ties to even); y * unit is at most 448, or not finite: then NaN
__device__ __forceinline__ uint8_t number_of(float y, float unit) {
  const float f = y * unit;
  if (!finite(f)) return 0x7f;
  return static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f, f, 0, false) & 0xff);
}
__device__ __forceinline__ float value_of(uint8_t b) { return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(b), 0); }

// A workgroup takes the rows of one page (a row in whose page the row before does not stand begins such a run) and four
// tasks of these rows, one a wave: a key head, a value head, a query head.
template <typename T>
__global__ __launch_bounds__(THREADS) void kernel(const T* __restrict__ src, int ld, int k_col, int v_col,
                                                  const int32_t* __restrict__ slot_map, uint8_t* __restrict__ k_pool,
                                                  uint8_t* __restrict__ v_pool, float* __restrict__ k_scale, float* __restrict__ v_scale,
                                                  int n_pages, const int32_t* __restrict__ positions, const float* __restrict__ freq,
                                                  int dims, int halves, float mag, int q_col, int n_heads, T* q_out, int ldq, int rows,
                                                  int Hkv, int dh, int page_size) {
  extern __shared__ double turn[];      // [CHUNK][dims / 2] pairs (cos, sin)
  const int t0 = blockIdx.x;
  auto page_of = [&](int t) {
    const int s = slot_map[t];
    const int p = s < 0 ? -1 : s / page_size;
    return p < n_pages ? p : -1;
  };
  const int page = page_of(t0);
  if (page >= 0 && t0 > 0 && page_of(t0 - 1) == page) return;      // the whole workgroup: this row is another run's
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  // the run's rows t0 .. t0 + n (a row without a page is a run of its own)
  int n = 1;
  if (page >= 0) {
    for (;;) {
      const int t = t0 + n + lane;
      const bool same = t < rows && page_of(min(t, rows - 1)) == page;
      const uint64_t other = ~__builtin_amdgcn_ballot_w64(same);
      const int more = other ? __builtin_ctzll(other) : 64;
      n += more;
      if (more < 64) break;
    }
  }
  const int half = dims / 2;
  const int task = blockIdx.y * (THREADS / 64) + wave;
  const int kind = task < Hkv ? 0 : task < 2 * Hkv ? 1 : task < 2 * Hkv + n_heads ? 2 : 3;
  const bool idle = kind == 3 || (kind < 2 && page < 0);
  const int head = kind == 0 ? task : kind == 1 ? task - Hkv : task - 2 * Hkv;
  const int col = (kind == 0 ? k_col : kind == 1 ? v_col : q_col) + head * dh;
  const int turned = kind == 1 ? 0 : half;      // pairs that this task's heads turn
  const int units = turned + dh - 2 * turned;   // a row's units: a pair each, then a number each
  const size_t block = (static_cast<size_t>(max(page, 0)) * Hkv + head) * page_size * dh;

  // unit u of row r (of the chunk that begins with row c): its numbers, at entries i and j (j < 0: one number)
  auto unit = [&](int c, int r, int u, int& i, int& j, double& a, double& b) {
    const T* x = src + static_cast<size_t>(t0 + c + r) * ld + col;
    if (u < turned) {
      i = halves ? u : 2 * u;
      j = halves ? u + half : 2 * u + 1;
      const double* cs = turn + (static_cast<size_t>(r) * half + u) * 2;
      const double p = to_float(x[i]), q = to_float(x[j]);
      a = (p * cs[0] - q * cs[1]) * mag;
      b = (q * cs[0] + p * cs[1]) * mag;
    } else {
      i = u + turned;
      j = -1;
      a = to_float(x[i]);
      b = 0.0;
    }
  };
  auto angles = [&](int c) {      // cos and sin of the chunk's rows, by the whole workgroup
    __syncthreads();
    for (int x = threadIdx.x; x < min(CHUNK, n - c) * half; x += THREADS) {
      double s, k;
      sin_cos(static_cast<double>(positions[t0 + c + x / half]) * static_cast<double>(freq[x % half]), s, k);
      turn[2 * x] = k;
      turn[2 * x + 1] = s;
    }
    __syncthreads();
  };

  // first the largest finite magnitude of what is new, and whether a row begins the page; queries are done with here
  float top = 0.f;
  bool anew = false;
  for (int c = 0; c < n; c += CHUNK) {
    if (half > 0) angles(c);
    if (idle) continue;
    const int m = min(CHUNK, n - c) * units;
    for (int x = lane; x < m; x += 64) {
      int i, j;
      double a, b;
      unit(c, x / units, x % units, i, j, a, b);
      if (kind == 2) {
        T* o = q_out + static_cast<size_t>(t0 + c + x / units) * ldq + head * dh;
        o[i] = from_float<T>(static_cast<float>(a));
        if (j >= 0) o[j] = from_float<T>(static_cast<float>(b));
      } else {
        const float fa = fabsf(to_odd(a)), fb = fabsf(to_odd(b));
        top = fmaxf(top, finite(fa) ? fa : 0.f);
        top = fmaxf(top, finite(fb) ? fb : 0.f);
      }
    }
    if (kind < 2)
      for (int r = 0; r < min(CHUNK, n - c); ++r) anew = anew || slot_map[t0 + c + r] % page_size == 0;
  }
  // (every wave of the workgroup has to pass every barrier below, tasks or none)
  const bool writes = !idle && kind < 2;
  float now = 1.f;
  if (writes) {
    uint8_t* pool = (kind == 0 ? k_pool : v_pool) + block;
    float* scale = (kind == 0 ? k_scale : v_scale) + static_cast<size_t>(page) * Hkv + head;
    top = wave_max(top);
    const float was = anew ? 0.f : *scale;
    now = fmaxf(power_of_two(scale_exponent(top)), was);
    if (now != was) {
      const float ratio = was / now;
      for (int x = lane; x < page_size * dh; x += 64) pool[x] = anew ? 0 : number_of(value_of(pool[x]), ratio);
      if (lane == 0) *scale = now;
      // the run's own numbers are stored over these below, by other lanes
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
      __builtin_amdgcn_wave_barrier();
    }
  }
  // then the numbers themselves
  const float per = 1.0f / now;
  for (int c = 0; c < n; c += CHUNK) {
    if (half > 0 && n > CHUNK) angles(c);
    if (!writes) continue;
    uint8_t* pool = (kind == 0 ? k_pool : v_pool) + block;
    const int m = min(CHUNK, n - c) * units;
    for (int x = lane; x < m; x += 64) {
      const int r = x / units, place = slot_map[t0 + c + r] % page_size;
      int i, j;
      double a, b;
      unit(c, r, x % units, i, j, a, b);
      pool[kind == 0 ? place * dh + i : i * page_size + place] = number_of(to_odd(a), per);
      if (j >= 0) pool[kind == 0 ? place * dh + j : j * page_size + place] = number_of(to_odd(b), per);
    }
  }
}
}  // namespace append

extern "C" int dn_kv_append8(const void* src, int ld, int k_col, int v_col, const int32_t* slot_map, void* k_pool, void* v_pool,
                             float* k_scale, float* v_scale, int n_pages, const int32_t* positions, const float* freq, int dims,
                             int halves, float mag, int q_col, int n_heads, void* q_out, int ldq, int T, int Hkv, int dh, int page_size,
                             int dtype, hipStream_t stream) {
  if (dims < 0 || dims % 2 != 0 || dims > dh || dh < 1 || dh > 256 || page_size < 1 || Hkv < 1 || n_heads < 0 || n_pages < 1) return DN_ERR_SHAPE;
  if (dtype != DN_F32 && dtype != DN_BF16) return DN_ERR_DTYPE;
  if (T == 0) return 0;
  const dim3 grid(T, (2 * Hkv + n_heads + 3) / 4);
  const size_t lds = static_cast<size_t>(append::CHUNK) * dims * sizeof(double);
#define DN_APPEND(TYPE)                                                                                                          \
  append::kernel<TYPE><<<grid, append::THREADS, lds, stream>>>(                                                                  \
      static_cast<const TYPE*>(src), ld, k_col, v_col, slot_map, static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool),   \
      k_scale, v_scale, n_pages, positions, freq, dims, halves, mag, q_col, n_heads, static_cast<TYPE*>(q_out), ldq, T, Hkv, dh, \
      page_size)
  if (dtype == DN_F32) DN_APPEND(float);
  else DN_APPEND(bf16_t);
#undef DN_APPEND
  return dn_launch_status();
}

// =======================================================================================
// attention, for every size: a wave for a row and a head
// =======================================================================================
namespace plain8 {
constexpr int KEYS = 64;

// One pass over the keys that the row reads, 64 at a time (a lane a key, then a lane up to four dims), with the softmax's running
// maximum and sum, all in 32 bits.  Only keys that the row reads are touched, so what stands in the others does not matter.
template <typename T>
__global__ __launch_bounds__(64) void kernel(const T* __restrict__ q, int ldq, T* __restrict__ out, int ldo,
                                             const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool,
                                             const float* __restrict__ k_scale, const float* __restrict__ v_scale, int n_pages,
                                             const int32_t* __restrict__ block_tables, int max_blocks,
                                             const int32_t* __restrict__ tile_seq, const int32_t* __restrict__ tile_row0,
                                             const int32_t* __restrict__ tile_nrows, const int32_t* __restrict__ tile_pos0, int H,
                                             int Hkv, int dh, int page_size, float scale, int window, int keep, int sink,
                                             const float* __restrict__ sink_at, float cap) {
  __shared__ float qs[256], ps[KEYS];
  __shared__ long long at[KEYS];      // where a key's head begins in the values' pool, plus its place there; -1: the row does not read it
  __shared__ float vs[KEYS];
  const int tile = blockIdx.x / 16, r = blockIdx.x % 16, h = blockIdx.y, lane = threadIdx.x;
  const int seq = tile_seq[tile];
  if (seq < 0 || r >= tile_nrows[tile]) return;
  const int row = tile_row0[tile] + r, pos = tile_pos0[tile] + r, hk = h / (H / Hkv);
  const int lo = window > 0 ? max(0, pos - window + 1) : 0;
  const int32_t* bt = block_tables + static_cast<size_t>(seq) * max_blocks;
  for (int d = lane; d < dh; d += 64) qs[d] = to_float(q[static_cast<size_t>(row) * ldq + h * dh + d]);
  __syncthreads();
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  float m = -3.0e38f, l = 0.f;
  const int keep_end = (min(keep, pos + 1) + KEYS - 1) / KEYS * KEYS, rest = max(lo / KEYS * KEYS, keep_end);
  for (int kt = keep_end > 0 ? 0 : rest; kt <= pos; kt = kt + KEYS == keep_end ? rest : kt + KEYS) {
    const int key = kt + lane, b = key / page_size;
    bool ok = key <= pos && (key >= lo || key < keep) && b < max_blocks;
    const int page = ok ? bt[b] : -1;
    ok = ok && page >= 0 && page < n_pages;
    float s = -INFINITY;
    long long v_at = -1;
    if (ok) {
      const size_t ph = static_cast<size_t>(page) * Hkv + hk;
      const uint8_t* kr = k_pool + (ph * page_size + key % page_size) * dh;
      float dot = 0.f;
      for (int d = 0; d < dh; ++d) dot = fmaf(qs[d], __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(kr[d]), 0), dot);
      s = dot * k_scale[ph] * scale;
      if (cap > 0.f) s = cap * tanhf(s / cap);
      v_at = static_cast<long long>(ph * dh) * page_size + key % page_size;
      vs[lane] = v_scale[ph];
    }
    if (__builtin_amdgcn_ballot_w64(ok) == 0) continue;      // (one wave: no barrier is passed by)
    const float m_new = fmaxf(m, wave_max(s));
    const float alpha = expf(m - m_new);
    const float p = ok ? expf(s - m_new) : 0.f;
    l = l * alpha + wave_sum(p);
    m = m_new;
    ps[lane] = p;
    at[lane] = v_at;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      o[i] *= alpha;
      if (d < dh)
        for (int j = 0; j < KEYS; ++j)
          if (at[j] >= 0)
            o[i] = fmaf(ps[j] * vs[j], __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(v_pool[at[j] + static_cast<long long>(d) * page_size]), 0), o[i]);
    }
    __syncthreads();
  }
  if (sink) l += expf((sink_at ? sink_at[h] : 0.f) - m);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < dh) out[static_cast<size_t>(row) * ldo + h * dh + d] = from_float<T>(l == 0.f ? 0.f : o[i] / l);      // (a row that reads nothing: zeros)
  }
}
}  // namespace plain8

extern "C" int dn_attention8(const void* q, int ldq, void* out, int ldo, const void* k_pool, const void* v_pool, const float* k_scale,
                             const float* v_scale, int n_pages, const int32_t* block_tables, int max_blocks, const int32_t* tile_seq,
                             const int32_t* tile_row0, const int32_t* tile_nrows, const int32_t* tile_pos0, int n_tiles, int H, int Hkv,
                             int dh, int page_size, float scale, int window, int keep, int sink, const float* sink_at, float cap,
                             int dtype, hipStream_t stream) {
  if (dh < 1 || dh > 256 || Hkv < 1 || H % Hkv != 0 || page_size < 1 || window < 0 || keep < 0 || (keep > 0 && window == 0) || !(cap >= 0.f))
    return DN_ERR_SHAPE;
  if (dtype != DN_F32 && dtype != DN_BF16) return DN_ERR_DTYPE;
  if (n_tiles == 0) return 0;
  const dim3 grid(n_tiles * 16, H);
#define DN_PLAIN8(TYPE)                                                                                                              \
  plain8::kernel<TYPE><<<grid, 64, 0, stream>>>(                                                                                     \
      static_cast<const TYPE*>(q), ldq, static_cast<TYPE*>(out), ldo, static_cast<const uint8_t*>(k_pool),                           \
      static_cast<const uint8_t*>(v_pool), k_scale, v_scale, n_pages, block_tables, max_blocks, tile_seq, tile_row0, tile_nrows,     \
      tile_pos0, H, Hkv, dh, page_size, scale, window, keep, sink, sink_at, cap)
  if (dtype == DN_F32) DN_PLAIN8(float);
  else DN_PLAIN8(bf16_t);
#undef DN_PLAIN8
  return dn_launch_status();
}
