// A step's rows into the paged cache in 8 bits, and attention over it for every size (cache8.h has the layout).
#include "cache8.h"

#include <math.h>

// =======================================================================================
// append: a step's queries and keys turned by their positions, keys and values to the pages
// =======================================================================================
namespace append {
constexpr int ANY_TASKS = 4;     // tasks of a workgroup of the kernel for any size, one a wave
constexpr int HEADS = 4;         // heads of a workgroup of the other, one a wave
constexpr int ALL_SIDE_BY_SIDE = 4;      // up to so many rows of a workgroup its runs are all of rows side by side
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
  const int q = static_cast<int>(k - 4.0 * floor(k * 0.25));
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

struct Args {
  const void* src;
  const int32_t* slot_map;
  uint8_t *k_pool, *v_pool;
  float *k_scale, *v_scale;
  const int32_t* positions;
  const float* freq;
  void* q_out;
  int ld, k_col, v_col, n_pages, dims, halves, q_col, n_heads, ldq, rows, Hkv, dh, page_size, page_shift;      // page_shift: -1 if page_size is no power of two
  float mag;
  // (a division by a number known only at run time is some twenty-five instructions)
  __device__ __forceinline__ int over_page(int slot) const { return page_shift >= 0 ? slot >> page_shift : slot / page_size; }
};

// the page of row t, -1: none
__device__ __forceinline__ int page_of(const Args& a, int t) {
  const int s = a.slot_map[t];
  const int p = s < 0 ? -1 : a.over_page(s);
  return p < a.n_pages ? p : -1;
}

// how many rows from t0 on stand in `page`
__device__ __forceinline__ int rows_in_page(const Args& a, int t0, int page, int lane) {
  int n = 1;
  for (;;) {
    const int t = t0 + n + lane;
    const bool same = t < a.rows && page_of(a, min(t, a.rows - 1)) == page;
    const uint64_t other = ~__builtin_amdgcn_ballot_w64(same);
    const int more = other ? __builtin_ctzll(other) : 64;
    n += more;
    if (more < 64) return n;
  }
}

// Every size and any order of a page's rows.  A workgroup takes the rows t0 .. t0 + n of one page and four tasks of these rows, one a
// wave: a key head, a value head, a query head; a number, or a pair of them, at a time.
template <typename T>
__device__ __forceinline__ void any_size(const Args& a, double* turn, int t0, int n, int page, int first_task, int wave, int lane) {
  const int half = a.dims / 2, dh = a.dh, page_size = a.page_size, Hkv = a.Hkv;
  const T* src = static_cast<const T*>(a.src);
  const int task = first_task + wave;
  const int kind = task < Hkv ? 0 : task < 2 * Hkv ? 1 : task < 2 * Hkv + a.n_heads ? 2 : 3;
  const bool idle = kind == 3 || (kind < 2 && page < 0);
  const int head = kind == 0 ? task : kind == 1 ? task - Hkv : task - 2 * Hkv;
  const int col = (kind == 0 ? a.k_col : kind == 1 ? a.v_col : a.q_col) + head * dh;
  const int turned = kind == 1 ? 0 : half;      // pairs that this task's heads turn
  const int units = turned + dh - 2 * turned;   // a row's units: a pair each, then a number each
  const size_t block = (static_cast<size_t>(max(page, 0)) * Hkv + head) * page_size * dh;

  // unit u of row r (of the chunk that begins with row c): its numbers, at entries i and j (j < 0: one number)
  auto unit = [&](int c, int r, int u, int& i, int& j, double& p, double& q) {
    const T* x = src + static_cast<size_t>(t0 + c + r) * a.ld + col;
    if (u < turned) {
      i = a.halves ? u : 2 * u;
      j = a.halves ? u + half : 2 * u + 1;
      const double* cs = turn + (static_cast<size_t>(r) * half + u) * 2;
      const double v = to_float(x[i]), w = to_float(x[j]);
      p = (v * cs[0] - w * cs[1]) * a.mag;
      q = (w * cs[0] + v * cs[1]) * a.mag;
    } else {
      i = u + turned;
      j = -1;
      p = to_float(x[i]);
      q = 0.0;
    }
  };
  auto angles = [&](int c) {      // cos and sin of the chunk's rows, by the whole workgroup
    __syncthreads();
    for (int x = threadIdx.x; x < min(CHUNK, n - c) * half; x += blockDim.x) {
      double s, k;
      sin_cos(static_cast<double>(a.positions[t0 + c + x / half]) * static_cast<double>(a.freq[x % half]), s, k);
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
      double p, q;
      unit(c, x / units, x % units, i, j, p, q);
      if (kind == 2) {
        T* o = static_cast<T*>(a.q_out) + static_cast<size_t>(t0 + c + x / units) * a.ldq + head * dh;
        o[i] = from_float<T>(static_cast<float>(p));
        if (j >= 0) o[j] = from_float<T>(static_cast<float>(q));
      } else {
        const float fp = fabsf(to_odd(p)), fq = fabsf(to_odd(q));
        top = fmaxf(top, finite(fp) ? fp : 0.f);
        top = fmaxf(top, finite(fq) ? fq : 0.f);
      }
    }
    if (kind < 2)
      for (int r = 0; r < min(CHUNK, n - c); ++r) anew = anew || a.slot_map[t0 + c + r] % page_size == 0;
  }
  // (every wave of the workgroup has to pass every barrier below, tasks or none)
  const bool writes = !idle && kind < 2;
  float now = 1.f;
  uint8_t* pool = (kind == 0 ? a.k_pool : a.v_pool) + block;
  if (writes) {
    float* scale = (kind == 0 ? a.k_scale : a.v_scale) + static_cast<size_t>(page) * Hkv + head;
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
    const int m = min(CHUNK, n - c) * units;
    for (int x = lane; x < m; x += 64) {
      const int r = x / units, place = a.slot_map[t0 + c + r] % page_size;
      int i, j;
      double p, q;
      unit(c, r, x % units, i, j, p, q);
      pool[kind == 0 ? place * dh + i : i * page_size + place] = number_of(to_odd(p), per);
      if (j >= 0) pool[kind == 0 ? place * dh + j : j * page_size + place] = number_of(to_odd(q), per);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(64 * ANY_TASKS) void any_size_kernel(const Args a) {
  extern __shared__ double turn[];      // [CHUNK][dims / 2] pairs (cos, sin)
  const int t0 = blockIdx.x, page = page_of(a, t0);
  if (page >= 0 && t0 > 0 && page_of(a, t0 - 1) == page) return;      // the whole workgroup: this row is another run's
  const int lane = threadIdx.x % 64;
  const int n = page >= 0 ? rows_in_page(a, t0, page, lane) : 1;      // (a row without a page is a run of its own)
  any_size<T>(a, turn, t0, n, page, blockIdx.y * ANY_TASKS, threadIdx.x / 64, lane);
}

// The sizes of models: heads of a multiple of 8, turned entries likewise, pages of a multiple of 16, rows 16-byte aligned.  What bounds
// these calls is bytes (portions) or a chain of a few trips to memory (single rows), so numbers move eight at a time, and the
// angles' sines, some 60 instructions of 64 bits each, are made once per workgroup for the HEADS heads that it turns at a time.
//   keys and queries: a lane takes a unit of 8 entries of a row: two runs of four, side by side, or with halves half a turn apart;
//   values: a lane takes two dims and a block of 16 places, so that a dim's 16 numbers, which lie side by side in the page, leave
//   in one store; what the page holds in that block already is read beside the rows.
typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t u32x4;
typedef __attribute__((__vector_size__(2 * sizeof(uint32_t)))) uint32_t u32x2;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4;

__device__ __forceinline__ void load4(const bf16_t* p, float* v) {
  const u32x2 w = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float((i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
}
__device__ __forceinline__ void load4(const float* p, float* v) {
  const floatx4 w = *reinterpret_cast<const floatx4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = w[i];
}
__device__ __forceinline__ void load2(const bf16_t* p, float* v) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
  v[0] = __uint_as_float(w << 16), v[1] = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void load2(const float* p, float* v) { v[0] = p[0], v[1] = p[1]; }
__device__ __forceinline__ void store4(bf16_t* p, const float* v) {
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = static_cast<uint32_t>(from_float<bf16_t>(v[2 * i]).bits) | static_cast<uint32_t>(from_float<bf16_t>(v[2 * i + 1]).bits) << 16;
  *reinterpret_cast<u32x2*>(p) = w;
}
__device__ __forceinline__ void store4(float* p, const float* v) { *reinterpret_cast<floatx4*>(p) = floatx4{v[0], v[1], v[2], v[3]}; }

// four numbers of a page (number_of), in one word
__device__ __forceinline__ uint32_t numbers_of(const float* y, float unit) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = y[i] * unit;
    f[i] = finite(f[i]) ? f[i] : NAN;
  }
  return __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false), true);
}
// a word of numbers in a page whose scale grew
__device__ __forceinline__ uint32_t renumbered(uint32_t w, float ratio) {
  const float y[4] = {__builtin_amdgcn_cvt_f32_fp8(w, 0), __builtin_amdgcn_cvt_f32_fp8(w, 1), __builtin_amdgcn_cvt_f32_fp8(w, 2), __builtin_amdgcn_cvt_f32_fp8(w, 3)};
  return numbers_of(y, ratio);
}

// The angles' sines of rows t0 .. t0 + n, by the whole workgroup.  turn: [rows][4][dims / 8] pairs (cos, sin): pair 4 u + k at [k][u], so
// that lanes side by side read side by side.
__device__ __forceinline__ void angles(const Args& a, double* turn, int t0, int n, int wave, int lane) {
  // (half up to 128: a power of two of threads, the least that holds a row's pairs, takes a row)
  const int half = a.dims / 2, bits = half > 1 ? 32 - __builtin_clz(half - 1) : 0;
  const int x = wave * 64 + lane, p = x & ((1 << bits) - 1);
  if (p < half) {
    const double f = a.freq[p];
    for (int r = x >> bits; r < n; r += 64 * HEADS >> bits) {
      double s, c;
      sin_cos(static_cast<double>(a.positions[t0 + r]) * f, s, c);
      double* to = turn + 2 * (r * half + p % 4 * (half / 4) + p / 4);
      to[0] = c * a.mag;
      to[1] = s * a.mag;
    }
  }
  __syncthreads();
}

// A lane's unit u of a row: its two runs of four entries begin at ea and eb.
// how the first dims of a head are turned
enum Turn { NOT, PAIRS, HALF };

template <typename T, Turn TURN>
struct Unit {
  int u, ea, eb, half;
  bool turned;
  __device__ __forceinline__ Unit(const Args& a, int u_) : u(u_), half(a.dims / 2), turned(TURN != NOT && u_ < a.dims / 8) {
    ea = TURN == HALF && turned ? 4 * u : 8 * u;
    eb = TURN == HALF && turned ? half + 4 * u : 8 * u + 4;
  }
  __device__ __forceinline__ void load(const T* row, float* v) const { load4(row + ea, v), load4(row + eb, v + 4); }
  // turned as row r's angles say, rounded to 32 bits.  KEYS: so that a second rounding to e4m3 is what rounding the 64-bit number would be,
  // and so that the largest magnitude compares with 1.75 * 2^k as the 64-bit one does.  Either can go wrong only where the 32-bit number
  // stands on a border itself, and those have zeros in their last 19 bits: there (once in half a million) the last bit is set odd.
  template <bool KEYS>
  __device__ __forceinline__ void turn(const double* angles, int r, float* v) const {
    if (!turned) return;
    float w[8];
    bool border = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const double* cs = angles + 2 * (r * half + k * (half / 4) + u);
      const int i = TURN == HALF ? k : 2 * k, j = TURN == HALF ? 4 + k : 2 * k + 1;
      const double c = cs[0], s = cs[1], p = v[i], q = v[j];
      w[i] = static_cast<float>(p * c - q * s);
      w[j] = static_cast<float>(q * c + p * s);
      if (KEYS) border = border | ((__float_as_uint(w[i]) & 0x7ffffu) == 0) | ((__float_as_uint(w[j]) & 0x7ffffu) == 0);
    }
    if (KEYS && __builtin_amdgcn_ballot_w64(border) != 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const double* cs = angles + 2 * (r * half + k * (half / 4) + u);
        const int i = TURN == HALF ? k : 2 * k, j = TURN == HALF ? 4 + k : 2 * k + 1;
        const double c = cs[0], s = cs[1], p = v[i], q = v[j];
        w[i] = to_odd(p * c - q * s);
        w[j] = to_odd(q * c + p * s);
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = w[k];
  }
};
constexpr int UNITS = 4, KEY_UNITS = 4;      // units of a lane in flight (keys take more registers)

// rows t0 .. t0 + n (n <= UNITS) of the queries
template <typename T, Turn TURN>
__device__ __forceinline__ void turn_queries(const Args& a, double* turn, int t0, int n, int wave, int lane) {
  const int per_row = a.dh / 8, span = 64 / per_row, of = lane / per_row;
  const Unit<T, TURN> unit(a, lane % per_row);
  const T* x = static_cast<const T*>(a.src) + static_cast<size_t>(t0) * a.ld + a.q_col;
  T* o = static_cast<T*>(a.q_out) + static_cast<size_t>(t0) * a.ldq;
  float v[UNITS][8];
  auto load = [&](int head) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i)
      unit.load(x + static_cast<size_t>(min(i, n - 1)) * a.ld + head * a.dh, v[i]);
  };
  const int first = of < span ? wave * span + of : a.n_heads;
  load(min(first, a.n_heads - 1));
  angles(a, turn, t0, n, wave, lane);
  for (int head = first; head < a.n_heads; head += HEADS * span) {
    if (head != first) load(head);
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      if (i < n) {
        unit.template turn<false>(turn, i, v[i]);
        T* to = o + static_cast<size_t>(i) * a.ldq + head * a.dh;
        store4(to + unit.ea, v[i]);
        store4(to + unit.eb, v[i] + 4);
      }
      __builtin_amdgcn_sched_barrier(0);      // (one unit's 64-bit numbers at a time)
    }
  }
}

// The rows t0 .. t0 + n, which stand in one page, of HEADS key heads (group < ceil(Hkv / HEADS)) or value heads (the groups behind).
template <typename T, Turn TURN>
__device__ __forceinline__ void run_of_rows(const Args& a, double* turn, int* row_in, int group, int t0, int n, int page, int place0, bool odd, int wave,
                                            int lane) {
  const int ps = a.page_size, dh = a.dh, kv_groups = (a.Hkv + HEADS - 1) / HEADS;
  const bool values = group >= kv_groups;
  const int head = (values ? group - kv_groups : group) * HEADS + wave;
  if (odd) {      // (the same for every wave of the workgroup) rows in another order than their places': the row of every place, -1: none
    for (int i = threadIdx.x; i < ps; i += 64 * HEADS) row_in[i] = -1;
    __syncthreads();
    for (int r = threadIdx.x; r < n; r += 64 * HEADS) row_in[a.slot_map[t0 + r] - page * ps] = r;
    __syncthreads();
  }
  auto row_at = [&](int place) {
    if (odd) return row_in[place];
    return place >= place0 && place < place0 + n ? place - place0 : -1;
  };
  const T* src = static_cast<const T*>(a.src) + static_cast<size_t>(t0) * a.ld;
  const bool anew = odd ? row_in[0] >= 0 : place0 == 0;

  if (values) {
    if (head >= a.Hkv) return;      // (no barrier in this part)
    const T* x = src + a.v_col + head * dh;
    uint8_t* pool = a.v_pool + (static_cast<size_t>(page) * a.Hkv + head) * ps * dh;
    float* scale = a.v_scale + static_cast<size_t>(page) * a.Hkv + head;
    const float was = anew ? 0.f : *scale;
    if (n == 1 && !anew) {
      // one row, as a decode step brings it: unless the scale grows, its bytes are all that is stored
      float y[4][2], top = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int d = 2 * lane + 128 * i;
        y[i][0] = y[i][1] = 0.f;
        if (d < dh) load2(x + d, y[i]);
#pragma unroll
        for (int j = 0; j < 2; ++j) top = fmaxf(top, finite(y[i][j]) ? fabsf(y[i][j]) : 0.f);
      }
      top = wave_max(top);
      const float now = fmaxf(power_of_two(scale_exponent(top)), was);
      if (now == was) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int d = 2 * lane + 128 * i;
          if (d < dh) {
            pool[static_cast<size_t>(d) * ps + place0] = number_of(y[i][0], 1.0f / now);
            pool[static_cast<size_t>(d + 1) * ps + place0] = number_of(y[i][1], 1.0f / now);
          }
        }
        return;
      }
    }
    // a lane's unit x: a pair of dims and a block of 16 places
    const int pairs = dh / 2, units = pairs * (ps / 16);
    const int b0 = odd ? 0 : place0 / 16, b1 = odd ? ps / 16 - 1 : (place0 + n - 1) / 16;      // the blocks that rows bring something to
    const bool once = units <= 64;      // (rows and page stay in registers)
    float y[16][2];
    uint32_t mask[4];      // the bytes of the block that rows bring
    u32x4 held[2];
    auto load = [&](int d, int b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // (never a conditional load, here and below: sixteen branches cost more than sixteen loads of a row already asked for; 10.1 -> 7.1 us)
        const int r = row_at(16 * b + i);
        load2(x + static_cast<size_t>(max(r, 0)) * a.ld + d, y[i]);
        if (r < 0) y[i][0] = y[i][1] = 0.f;
        const uint32_t byte = r >= 0 ? 0xffu << (8 * (i % 4)) : 0u;
        mask[i / 4] = i % 4 == 0 ? byte : mask[i / 4] | byte;
      }
    };
    auto load_held = [&](int d, int b) {
#pragma unroll
      for (int j = 0; j < 2; ++j) held[j] = anew ? u32x4{0u, 0u, 0u, 0u} : *reinterpret_cast<const u32x4*>(pool + static_cast<size_t>(d + j) * ps + 16 * b);
    };
    float top = 0.f;
    for (int i = lane; i < units; i += 64) {
      const int b = i / pairs, d = 2 * (i - b * pairs);
      if (once) load_held(d, b);
      if (once || (b >= b0 && b <= b1)) load(d, b);
      if (b >= b0 && b <= b1) {
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) top = fmaxf(top, finite(y[k][j]) ? fabsf(y[k][j]) : 0.f);
      }
    }
    top = wave_max(top);
    const float now = fmaxf(power_of_two(scale_exponent(top)), was), per = 1.0f / now, ratio = was / now;
    const bool grown = now != was;
    if (grown && lane == 0) *scale = now;
    for (int i = lane; i < units; i += 64) {
      const int b = i / pairs, d = 2 * (i - b * pairs);
      if (!grown && (b < b0 || b > b1)) continue;
      if (!once) {
        load_held(d, b);
        if (b >= b0 && b <= b1) {
          load(d, b);
        } else {      // a block that no row brings anything to
#pragma unroll
          for (int k = 0; k < 16; ++k) y[k][0] = y[k][1] = 0.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) mask[q] = 0u;
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        u32x4 w;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float z[4] = {y[4 * q][j], y[4 * q + 1][j], y[4 * q + 2][j], y[4 * q + 3][j]};
          const uint32_t old = grown && !anew ? renumbered(held[j][q], ratio) : held[j][q];
          w[q] = (numbers_of(z, per) & mask[q]) | (old & ~mask[q]);
        }
        *reinterpret_cast<u32x4*>(pool + static_cast<size_t>(d + j) * ps + 16 * b) = w;
      }
    }
    return;
  }

  // keys: `span` rows at a time
  const int per_row = dh / 8, span = 64 / per_row, of = lane / per_row;
  const Unit<T, TURN> unit(a, lane % per_row);
  const int end = of < span && head < a.Hkv ? n : 0;      // (a lane without work has no rows)
  const T* x = src + a.k_col + min(head, a.Hkv - 1) * dh;
  float v[KEY_UNITS][8];
  auto load = [&](int r0) {
#pragma unroll
    for (int i = 0; i < KEY_UNITS; ++i) unit.load(x + static_cast<size_t>(min(r0 + of + i * span, n - 1)) * a.ld, v[i]);
  };
  auto turn_all = [&](int r0) {
#pragma unroll
    for (int i = 0; i < KEY_UNITS; ++i) {
      if (r0 + of + i * span < end) unit.template turn<true>(turn, r0 + of + i * span, v[i]);
      __builtin_amdgcn_sched_barrier(0);      // (one unit's 64-bit numbers at a time)
    }
  };
  load(0);
  float* scale = a.k_scale + static_cast<size_t>(page) * a.Hkv + head;
  const float was = anew || head >= a.Hkv ? 0.f : *scale;
  if (TURN != NOT) angles(a, turn, t0, n, wave, lane);
  if (head >= a.Hkv) return;      // (no barrier below)
  uint8_t* pool = a.k_pool + (static_cast<size_t>(page) * a.Hkv + head) * ps * dh;
  const bool once = n <= KEY_UNITS * span;
  float top = 0.f;
  for (int r0 = 0; r0 < n; r0 += KEY_UNITS * span) {
    if (r0 > 0) load(r0);
    turn_all(r0);
#pragma unroll
    for (int i = 0; i < KEY_UNITS; ++i)
      if (r0 + of + i * span < end) {
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, finite(v[i][k]) ? fabsf(v[i][k]) : 0.f);
      }
  }
  top = wave_max(top);
  const float now = fmaxf(power_of_two(scale_exponent(top)), was), per = 1.0f / now;
  if (now != was) {      // what the page holds in other places
    if (lane == 0) *scale = now;
    const float ratio = was / now;
    for (int place = of; place < ps && of < span; place += span) {
      if (row_at(place) >= 0) continue;
      u32x2* at = reinterpret_cast<u32x2*>(pool + static_cast<size_t>(place) * dh + unit.u * 8);
      u32x2 w = {0u, 0u};
      if (!anew) w = *at, w = u32x2{renumbered(w[0], ratio), renumbered(w[1], ratio)};
      *at = w;
    }
  }
  for (int r0 = 0; r0 < n; r0 += KEY_UNITS * span) {
    if (!once) load(r0), turn_all(r0);      // (read a second time, out of the caches)
#pragma unroll
    for (int i = 0; i < KEY_UNITS; ++i) {
      const int r = r0 + of + i * span;
      if (r < end) {
        uint8_t* to = pool + static_cast<size_t>(odd ? a.slot_map[t0 + r] - page * ps : place0 + r) * dh;
        *reinterpret_cast<uint32_t*>(to + unit.ea) = numbers_of(v[i], per);
        *reinterpret_cast<uint32_t*>(to + unit.eb) = numbers_of(v[i] + 4, per);
      }
    }
  }
}

// The first workgroups take Q rows of queries each.  Of the others, each takes the runs of rows in one page that begin among its R rows side by
// side.  With more than four of them runs of one row, as decoded tokens are, go to the workgroups in turn instead (block, block + blocks,
// ...), so that no workgroup has many one after the other: 64 of them in front of 1,984 rows of prompts, 25 heads of 64, 14.6 us, all side by
// side 26.0 (prompts alone 13.2 and 12.0; 256 single rows, four a workgroup, 14.6 and 13.4).  Runs of pages in turn as well would leave some
// workgroups two or three of the long ones: 2,799 rows of 32 + 8 + 8 heads of 128 30.4 us for 20.5.
// (A workgroup that finds none costs 2.7 ns of the launch all the same: with one for every row, 2,136 rows of 32 + 8 + 8 heads of 128 took
// 68 us.)
// Four waves per SIMD where nothing is turned (4,096 rows of 25 heads of 64 21.0 us, with three 26.5, before single rows went in turn; five keep registers in memory), three where
// the 64-bit numbers want the registers.
template <typename T, Turn TURN>
__global__ __launch_bounds__(64 * HEADS) __attribute__((amdgpu_waves_per_eu(TURN == NOT ? 4 : 3))) void kernel(const Args a, int q_blocks, int Q, int R, int blocks) {
  extern __shared__ double turn[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  if (TURN != NOT && static_cast<int>(blockIdx.x) < q_blocks) {
    const int t0 = blockIdx.x * Q;
    turn_queries<T, TURN>(a, turn, t0, min(Q, a.rows - t0), wave, lane);
    return;
  }
  int* const row_in = reinterpret_cast<int*>(turn + static_cast<size_t>(min(a.page_size, a.rows)) * a.dims);
  const int groups = 2 * ((a.Hkv + HEADS - 1) / HEADS), group = (blockIdx.x - q_blocks) % groups, block = (blockIdx.x - q_blocks) / groups;
  const int ps = a.page_size;
  auto page_at = [&](int slot) {
    const int its = a.over_page(slot);
    return slot < 0 || its >= a.n_pages ? -1 : its;
  };
  // slots of the rows from the one before this workgroup's first on, and of the rows that are its own in turn (R <= 32; every wave writes the same)
  __shared__ int side_by_side[64], in_turn[32];
  const int first = block * R - 1;
  uint64_t runs, singles = 0;
  auto slot_at = [&](int t) { return a.slot_map[min(max(t, 0), a.rows - 1)]; };      // (never a conditional load; what is none is left out behind it)
  auto is_row = [&](int t) { return t >= 0 && t < a.rows; };
  int window = slot_at(first + lane);
  if (R <= ALL_SIDE_BY_SIDE) {
    window = is_row(first + lane) ? window : -1;
    const int its = page_at(window), before = __shfl(its, lane - 1);
    runs = __builtin_amdgcn_ballot_w64(lane >= 1 && lane <= R && its >= 0 && before != its);
  } else {
    const int t = block + lane * blocks;
    int lone = slot_at(t), lone_before = slot_at(t - 1), lone_behind = slot_at(t + 1);
    window = is_row(first + lane) ? window : -1;
    lone = lane < R && is_row(t) ? lone : -1;
    lone_before = t > 0 ? lone_before : -1;
    lone_behind = t + 1 < a.rows ? lone_behind : -1;
    if (lane < 32) in_turn[lane] = lone;
    const int its = page_at(window), before = __shfl(its, lane - 1), behind = __shfl(its, lane + 1), page = page_at(lone);
    runs = __builtin_amdgcn_ballot_w64(lane >= 1 && lane <= R && its >= 0 && before != its && behind == its);
    singles = __builtin_amdgcn_ballot_w64(page >= 0 && page_at(lone_before) != page && page_at(lone_behind) != page);
  }
  side_by_side[lane] = window;
  while ((runs | singles) != 0) {
    int t0, n = 1, slot0;
    bool odd = false;
    if (runs != 0) {
      const int i = __builtin_ctzll(runs);
      runs &= runs - 1;
      t0 = first + i;
      slot0 = __builtin_amdgcn_readlane(window, i);
      n = __builtin_ctzll(~(__builtin_amdgcn_ballot_w64(page_at(window) == page_at(slot0)) >> i));      // (the bits shifted in are zeros: i >= 1)
      if (n == 64 - i) n = rows_in_page(a, t0, page_at(slot0), lane);
      // rows in another order than their places'
      odd = n > ps - (slot0 - page_at(slot0) * ps) || (lane >= i && lane < i + n && window != slot0 + lane - i);
      for (int r = 64 - i + lane; r < n; r += 64) odd = odd || a.slot_map[t0 + r] != slot0 + r;
      odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    } else {
      const int i = __builtin_ctzll(singles);
      singles &= singles - 1;
      t0 = block + i * blocks;
      slot0 = __builtin_amdgcn_readfirstlane(in_turn[i]);
    }
    const int page = page_at(slot0);
    // (more rows than places have a slot twice, which is not allowed: those behind are left out, so that what LDS holds suffices)
    run_of_rows<T, TURN>(a, turn, row_in, group, t0, min(n, ps), page, slot0 - page * ps, odd, wave, lane);
    if ((runs | singles) == 0) break;
    __syncthreads();      // (the next run's angles and places take these ones' room)
    window = side_by_side[lane];      // (so that it takes no register meanwhile)
  }
}
}  // namespace append

extern "C" int dn_kv_append8(const void* src, int ld, int k_col, int v_col, const int32_t* slot_map, void* k_pool, void* v_pool,
                             float* k_scale, float* v_scale, int n_pages, const int32_t* positions, const float* freq, int dims,
                             int halves, float mag, int q_col, int n_heads, void* q_out, int ldq, int T, int Hkv, int dh, int page_size,
                             int dtype, hipStream_t stream) {
  if (dims < 0 || dims % 2 != 0 || dims > dh || dh < 1 || dh > 256 || page_size < 1 || Hkv < 1 || n_heads < 0 || (n_heads > 0 && dims == 0) || n_pages < 1) return DN_ERR_SHAPE;
  if (dtype != DN_F32 && dtype != DN_BF16) return DN_ERR_DTYPE;
  if (T == 0) return 0;
  int page_shift = 0;
  while ((1 << page_shift) < page_size) ++page_shift;
  if ((1 << page_shift) != page_size) page_shift = -1;
  const append::Args a = {src, slot_map, static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool), k_scale, v_scale, positions, freq, q_out,
                          ld, k_col, v_col, n_pages, dims, halves, q_col, n_heads, ldq, T, Hkv, dh, page_size, page_shift, mag};
  // a run's rows in LDS at a time, and a page's places; the kernel for other sizes takes rows 16 at a time, whatever the page
  const size_t lds = static_cast<size_t>(append::CHUNK) * dims * sizeof(double),
               lds_page = static_cast<size_t>(min(page_size, T)) * dims * sizeof(double) + page_size * sizeof(int);
  const int size = dtype == DN_F32 ? 4 : 2;
  auto whole = [&](const void* p, int stride, int col) {
    return (reinterpret_cast<uintptr_t>(p) + static_cast<size_t>(col) * size) % 16 == 0 && static_cast<size_t>(stride) * size % 16 == 0;
  };
  const bool fast = dh % 8 == 0 && dims % 8 == 0 && page_size % 16 == 0 && lds_page <= 128 * 1024 + 4096 && whole(src, ld, k_col) && whole(src, ld, v_col) &&
                    (n_heads == 0 || (whole(src, ld, q_col) && whole(q_out, ldq, 0))) && reinterpret_cast<uintptr_t>(k_pool) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(v_pool) % 16 == 0;
  if (fast) {
    // A workgroup for every row as long as that makes no more than 1,024, else for 2, 4, 8, ... rows, up to a page's: more would be runs
    // one after the other (4,096 rows of 25 heads of 64 with 64 rows a workgroup: 126 us, with 16 23.4).
    const int groups = 2 * ((Hkv + append::HEADS - 1) / append::HEADS), Q = T <= 512 ? 1 : append::UNITS, q_blocks = n_heads > 0 ? (T + Q - 1) / Q : 0;
    int R = 1;
    while (static_cast<long>((T + R - 1) / R) * groups > 1024 && 2 * R <= min(page_size, 32)) R *= 2;
    const int blocks = (T + R - 1) / R;
    const dim3 grid(q_blocks + blocks * groups);
#define DN_APPEND(TYPE, TURN)                                                                                                          \
  do {                                                                                                                                 \
    auto* fn = &append::kernel<TYPE, append::TURN>;                                                                                    \
    if (lds_page > 60 * 1024) {                                                                                                        \
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, lds_page); \
      if (e != hipSuccess) return static_cast<int>(e);                                                                                 \
    }                                                                                                                                  \
    fn<<<grid, 64 * append::HEADS, lds_page, stream>>>(a, q_blocks, Q, R, blocks);                                                     \
  } while (0)
    if (dtype == DN_F32) {
      if (dims == 0) DN_APPEND(float, NOT);
      else if (halves) DN_APPEND(float, HALF);
      else DN_APPEND(float, PAIRS);
    } else {
      if (dims == 0) DN_APPEND(bf16_t, NOT);
      else if (halves) DN_APPEND(bf16_t, HALF);
      else DN_APPEND(bf16_t, PAIRS);
    }
#undef DN_APPEND
  } else {
    const dim3 grid(T, (2 * Hkv + n_heads + append::ANY_TASKS - 1) / append::ANY_TASKS);
    if (dtype == DN_F32) append::any_size_kernel<float><<<grid, 64 * append::ANY_TASKS, lds, stream>>>(a);
    else append::any_size_kernel<bf16_t><<<grid, 64 * append::ANY_TASKS, lds, stream>>>(a);
  }
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
  if (dh < 1 || dh > 256 || Hkv < 1 || H % Hkv != 0 || page_size < 1 || window < 0 || keep < 0 || (keep > 0 && window == 0) || !(cap >= 0.f && cap < INFINITY))
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
