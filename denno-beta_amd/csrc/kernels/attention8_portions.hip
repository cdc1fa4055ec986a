// Attention over the cache in 8 bits for portions of prompts: two products of the rows with the keys and the values, so the matrix
// instructions are what it takes, and what stands between them (widening the cache's numbers, the softmax) has to be little.
//
// A workgroup takes up to RG x 32 rows of one request and one head: wave w owns 32 of them (row group w % RG), and its KG
// key groups (w / RG) share out the keys, 64 by 64, and join at the end.  A group's tile of 64 keys comes from the pages 16 bytes a thread,
// is widened to bfloat16 times its page's scale on the way into LDS (v_cvt_scalef32_pk_bf16_fp8: the scale, a power of two,
// costs nothing there and nothing behind), and serves all row groups; two tiles deep, the one after the next on its way to registers.
//   S^T = K Q^T by v_mfma_f32_32x32x16_bf16: lane (column: a row of q; half g) gets 16 keys of every 32, so the running softmax is
//   inside a lane but for one exchange between the halves, and its weights are, eight by eight, B operands of
//   O^T += V^T P^T, whose k-th slots are the keys 16 a + 4 g + {0..3, 8..11}: the values lie in LDS in that order, 16 bytes a read.
// 32-bit rows: three bfloat16 parts of the queries and of the weights (attend8::split), three products for one.  bfloat16 rows: one part of the
// weights, that is, a weight (at most 1, the largest so exact) rounded to 8 digits in front of the second product, whose operands have no more; the sum under the
// softmax is of the 32-bit weights.  Beside the rounding of the result itself (0.0016 of its size) it is hardly seen: 0.0017 off 64 bits.
//
// Measured: 1,986 rows of 32 heads of 128 behind 2,001 to 8,192 tokens 262 us, 822 TFLOP/s, a third of what the matrix units could do and two thirds of
// what a large product reaches.  They are busy a third of the time (33 %), the vector units 46 %, LDS 39 % (a third of that for banks asked for twice), and what keeps
// the sum of the three from becoming the largest is a wave's own chain from product to softmax to product, with two waves per SIMD, which is what 228
// registers of 512 leave room for.  Two prompts of 1,024 rows of 25 heads of 64 23.1 us (matrix units 9 %, vector 29 %, LDS 15 %), a 32-bit prompt of 1,001 22.8.
// Sums of weights by the matrix units, as a product with ones, were slower (16 more registers: 408 -> 658 us undivided).
#include "attention8_common.h"

namespace portions8 {
using namespace attend8;
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float floatx16;

struct Args {
  const void* q;
  void* out;
  const uint8_t *k_pool, *v_pool;
  const float *k_scale, *v_scale;
  const int32_t *block_tables, *tile_seq, *tile_row0, *tile_nrows, *tile_pos0;
  const float* sink_at;
  float* part;      // attend8::Parts' results, with more than one split
  int ldq, ldo, n_pages, max_blocks, n_splits, H, Hkv, page_shift, window, keep, sink;      // pages of 1 << page_shift keys
  float scale;
  Cap cap;
};

__device__ __forceinline__ u32x4 widen_scaled(uint32_t lo, uint32_t hi, float scale) {
  u32x4 w;
  w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
  w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
  w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
  return w;
}

// A wait for products that are read behind a branch, which the compiler does not always leave room for: 16 cycles, as a product of 32 x 32 wants at least
__device__ __forceinline__ void settle(floatx16& a, floatx16& b) { asm volatile("s_nop 15" : "+v"(a), "+v"(b)); }

// the largest scale whose products with all numbers are finite (448 2^119 = 1.75 2^127)
constexpr float LARGEST = 0x1p119f;

// the upper bit of those of a word's four e4m3 numbers that are NaN (0x7f or 0xff)
__device__ __forceinline__ uint32_t nan_in(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

template <int DH16, int PARTS, int RG, int KG>
constexpr int waves_per_simd() {      // (with room for one wave only, the compiler moves results to and fro between two sets of registers)
  return DH16 * (4 * PARTS + 8) > 128 ? 1 : 2;
}

// CAPPED: scores have a soft cap (a kernel of its own: what the cap takes of registers cost heads of 96, 160 and 256 without one 6 % of their time)
template <int DH16, int PARTS, int RG, int KG, bool CAPPED>
__global__ __launch_bounds__(64 * RG * KG) __attribute__((amdgpu_waves_per_eu(waves_per_simd<DH16, PARTS, RG, KG>()))) void kernel(const Args a) {
  constexpr int DH = DH16 * 16, DB = (DH + 31) / 32;
  // elements of a key's row, of a dim's row of 64 keys, 16 bytes of padding each; and 64 bytes more behind every 16 keys, so that the four
  // blocks of keys that lanes side by side write do not ask for the same banks
  constexpr int KROW = DH + 8, VROW = 72, BLOCK_PAD = 32;
  constexpr int KSZ = 64 * KROW + 4 * BLOCK_PAD, TSZ = KSZ + DH * VROW;  // of a tile's keys, of a tile
  constexpr int THREADS = 64 * RG;                       // of a key group
  constexpr int CHUNKS = 64 * DH16;                      // 16-byte chunks of a tile's keys, and of its values
  constexpr int U = (CHUNKS + THREADS - 1) / THREADS;
  constexpr int JOIN = 2 + 16 * DB;
  constexpr int BYTES_TILES = 2 * KG * TSZ * 2, BYTES_JOIN = (KG - 1) * THREADS * JOIN * 4;
  constexpr int SUBS = 4 / RG;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  bf16_t* const tiles = reinterpret_cast<bf16_t*>(smem);                        // [2][KG][keys | values]
  constexpr int FLAGS_AT = BYTES_TILES > BYTES_JOIN ? BYTES_TILES : BYTES_JOIN;
  int* const flags = reinterpret_cast<int*>(smem + FLAGS_AT);                   // [2][KG][4 blocks: whether there is a page]
  int* const seen = flags + 2 * KG * 4;                                         // whether there was a value that is NaN

  // consecutive workgroups go to different XCDs: the heads of one key head are Hkv workgroups apart, so that with 8 key heads (or a
  // multiple) an XCD's L2 holds the keys of its own heads only
  const int G = a.H / a.Hkv;
  // Tiles come with the longest first.  The first 256 workgroups go to a CU each, and the next 256 to the same CUs in the same order: those
  // are taken the other way round (in eights, which go to the eight XCDs), so that the longest have the shortest beside them (two prompts
  // of 1,024 with 25 heads of 64: 28.3 -> 26.8 us; workgroups of 8 waves, of which a CU holds one, wait for a free CU and stay in order).
  int bx = blockIdx.x, by = blockIdx.y;
  if constexpr (RG == 2) {
    const int b = by * gridDim.x + bx, eights = gridDim.x * gridDim.y / 8, end = min(eights, 64);
    if (b >= 256 && b / 8 < end) {
      const int other = (32 + end - 1 - b / 8) * 8 + b % 8;
      by = other / gridDim.x, bx = other % gridDim.x;
    }
  }
  const int hk = bx % a.Hkv, h = hk * G + bx / a.Hkv;
  const int tile = by / SUBS, sub = SUBS - 1 - by % SUBS;
  const int seq = a.tile_seq[tile];
  const int r0 = sub * 32 * RG;
  const int nrows = min(a.tile_nrows[tile] - r0, 32 * RG);
  if (seq < 0 || nrows <= 0) return;      // the whole workgroup
  const int row0 = a.tile_row0[tile] + r0, pos0 = a.tile_pos0[tile] + r0;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int kg = wave / RG, rg = wave % RG, t = threadIdx.x % THREADS;
  const int col = lane % 32, g = lane / 32;
  const int32_t* bt = a.block_tables + static_cast<size_t>(seq) * a.max_blocks;
  const int wrow0 = rg * 32;
  const bool has_rows = wrow0 < nrows;      // (a wave without rows carries tiles all the same)
  const bool row_ok = wrow0 + col < nrows;
  const int my_row = min(wrow0 + col, nrows - 1), my_pos = pos0 + my_row;
  auto first_key = [&](int pos) { return a.window > 0 ? max(0, pos - a.window + 1) : 0; };
  const int my_lo = first_key(my_pos), lo_w = first_key(pos0 + wrow0), hi_w = pos0 + min(wrow0 + 31, nrows - 1), lo_last = first_key(hi_w);
  const int lo_g = first_key(pos0), hi_g = pos0 + nrows - 1, lo_g_last = first_key(hi_g);

  bf16x8 qf[DH16][PARTS];
#pragma unroll
  for (int c = 0; c < DH16; ++c) {
    const size_t at = static_cast<size_t>(row0 + my_row) * a.ldq + h * DH + c * 16 + g * 8;
    if constexpr (PARTS == 1) {
      qf[c][0] = *reinterpret_cast<const bf16x8*>(static_cast<const bf16_t*>(a.q) + at);
    } else {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = static_cast<const float*>(a.q)[at + j];
      split<PARTS>(v, qf[c]);
    }
  }
  floatx16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m_run = LOWEST, l_run = 0.f;
  const float scale2 = a.scale * LOG2E;
  const float per_score = CAPPED ? 1.0f : scale2;      // what is left to multiply a score with

  // Steps of 64 KG keys: `kept` ones from the start, then those from the window's first key on.  Step i begins with key_of(i).
  constexpr int STEP = 64 * KG;
  const int kept = a.keep > 0 ? (min(a.keep, hi_g + 1) + STEP - 1) / STEP : 0;
  const int rest = max(lo_g / STEP, kept);
  const int steps = kept + max(0, hi_g / STEP - rest + 1);
  auto key_of = [&](int i) { return STEP * (i < kept ? i : rest + i - kept); };
  const int share = blockIdx.z, per = (steps + a.n_splits - 1) / a.n_splits, i0 = share * per, i1 = min(steps, i0 + per);      // this workgroup's

  // This thread's chunks of its group's tile are all of block t % 4, its 16 keys, so that a thread has one page a tile: chunk x = t / 4 +
  // THREADS / 4 u is, of the keys, 16 dims (x % DH16) of key x / DH16, and of the values dim x.  A tile begins at a multiple of 64, so in
  // pages of up to 64 keys a block's place in its page is always the same, and in longer ones what is added to it is the same for all threads.
  constexpr int BLOCK_CHUNKS = CHUNKS / 4;
  const int in_page = (1 << a.page_shift) - 1;
  const uint32_t page_bytes = static_cast<uint32_t>(a.Hkv) * DH << a.page_shift;
  const int off = 16 * (t % 4);
  // (the chunks of one thread lie evenly apart if a group's threads take whole keys at a time: one place to keep then)
  constexpr bool EVEN = CHUNKS % THREADS == 0 && THREADS / 4 % DH16 == 0;
  constexpr int PLACES = EVEN ? 1 : U;
  uint32_t k_at[PLACES], v_at[PLACES];
  struct Raw {                   // a tile on its way
    u32x4 k[U], v[U];
    float k_by, v_by;
    bool there;                  // whether it has a page
  };
#pragma unroll
  for (int u = 0; u < PLACES; ++u) {
    // (a thread without a chunk takes another's)
    const uint32_t x = CHUNKS % THREADS == 0 ? t / 4 + THREADS / 4 * u : min(t / 4 + THREADS / 4 * u, BLOCK_CHUNKS - 1);
    k_at[u] = ((hk << a.page_shift) + (off & in_page) + x / DH16) * DH + x % DH16 * 16;
    v_at[u] = ((hk * DH + x) << a.page_shift) + (off & in_page);
  }
  // The page of the block of 16 keys that key kt + off stands in (off < 64): what the table says is asked for a step before it is
  // needed (page_entry), and looked at when it is (page_of; -1: none, or behind the last row): looked at at once, it would be waited for at
  // once, and with it the keys and values on their way.
  auto page_entry = [&](int kt, int off) { return bt[min((kt >> a.page_shift) + (off >> a.page_shift), a.max_blocks - 1)]; };
  auto page_of = [&](int kt, int off, int entry) {
    return (kt >> a.page_shift) + (off >> a.page_shift) < a.max_blocks && kt + (off & ~15) <= hi_g && entry < a.n_pages ? entry : -1;
  };
  auto entry_of = [&](int i) { return page_entry(key_of(i) + 64 * kg, off); };      // (a step behind the last one begins behind the last row)
  auto fetch = [&](int i, int entry, Raw& raw) {      // (what has no page reads the pools' first: no row reads what comes of it)
    const int kt = key_of(i) + 64 * kg, far = kt & in_page, found = page_of(kt, off, entry);
    const uint32_t page = max(found, 0);
    raw.there = found >= 0;
    const size_t begin = static_cast<size_t>(page) * page_bytes;
    raw.k_by = a.k_scale[page * a.Hkv + hk];
    raw.v_by = a.v_scale[page * a.Hkv + hk];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw.k[u] = *reinterpret_cast<const u32x4*>(a.k_pool + begin + (k_at[EVEN ? 0 : u] + (EVEN ? THREADS / 4 / DH16 * DH * u : 0) + far * DH));
      raw.v[u] = *reinterpret_cast<const u32x4*>(a.v_pool + begin + (v_at[EVEN ? 0 : u] + ((EVEN ? THREADS / 4 * u : 0) << a.page_shift) + far));
    }
  };
  auto stash = [&](Raw& raw, int buf) {
    bf16_t* dst = tiles + (buf * KG + kg) * TSZ;
    // Values that are NaN go in as zeros (a weight of zero, of a row that does not read the value, would make NaN of its result), and the
    // rows that do read them are seen to at the end.
    uint32_t nan = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int w = 0; w < 4; ++w) nan |= (raw.v[u][w] & 0x7f7f7f7fu) + 0x01010101u;
    nan &= 0x80808080u;
    // So would a value beyond the largest number (256 2^120, which a value above 0.97 of it is rounded to): of a page with a scale so large
    // numbers go in as at most 240, within the rounding that they have had.  What has no page has no scale either.  A page whose scale is no
    // finite number (none that was written into a cache is) goes in as one of values that are NaN.
    float v_by = raw.there ? raw.v_by : 1.0f;
    if (__builtin_amdgcn_ballot_w64(nan != 0 || !(fabsf(v_by) <= LARGEST)) != 0) {
      const bool scaled = fabsf(v_by) < INFINITY;
      v_by = scaled ? v_by : 1.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          raw.v[u][w] &= scaled ? ~((nan_in(raw.v[u][w]) >> 7) * 0xffu) : 0u;
          const uint32_t high = fabsf(v_by) > LARGEST ? (((raw.v[u][w] & 0x7f7f7f7fu) + 0x08080808u) & 0x80808080u) >> 7 : 0u;      // from 256 on
          raw.v[u][w] = (raw.v[u][w] & ~(high * 0x7fu)) | high * 0x77u;
        }
      if (raw.there && (nan != 0 || !scaled)) *seen = 1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = t / 4 + THREADS / 4 * u;
      if (CHUNKS % THREADS == 0 || x < BLOCK_CHUNKS) {
        u32x4* to = reinterpret_cast<u32x4*>(dst + (off + x / DH16) * KROW + t % 4 * BLOCK_PAD + x % DH16 * 16);
        to[0] = widen_scaled(raw.k[u][0], raw.k[u][1], raw.k_by);
        to[1] = widen_scaled(raw.k[u][2], raw.k[u][3], raw.k_by);
        to = reinterpret_cast<u32x4*>(dst + KSZ + x * VROW + off);
        to[0] = widen_scaled(raw.v[u][0], raw.v[u][2], v_by);
        to[1] = widen_scaled(raw.v[u][1], raw.v[u][3], v_by);
      }
    }
    if (t < 4) flags[(buf * KG + kg) * 4 + t] = raw.there;
  };

  if (threadIdx.x == 0) *seen = 0;
  __syncthreads();
  Raw raw;
  int entry;
  {      // the first two tiles are asked for at once
    Raw first;
    const int entry0 = entry_of(i0), entry1 = entry_of(i0 + 1);
    entry = entry_of(i0 + 2);
    fetch(i0, entry0, first);
    fetch(i0 + 1, entry1, raw);
    stash(first, 0);
  }
  __syncthreads();
  int buf = 0;
  for (int i = i0; i < i1; ++i, buf ^= 1) {
    // The next tile on its way to LDS, the one after it to registers: the first key group does this in front of its products, the others behind
    // theirs, and products go in front of what the other waves of a SIMD do beside them, so that one wave's products run beside another's
    // other work: 2,048 rows of 32 heads of 128 behind 4,000 tokens 204.4 -> 196.1 us (groups alone 214.9, priorities alone 205.5), 1,280 rows 33.0 -> 31.8,
    // 512 15.0 -> 13.7, two prompts of 1,024 of 25 heads of 64 25.1 -> 24.9.  With one key group there is nobody beside a wave to
    // take turns with, and priorities cost 2 %.
    auto next = [&]() {
      if (i + 1 < i1) stash(raw, buf ^ 1);
      if (i + 2 < i1) fetch(i + 2, entry, raw);
      entry = entry_of(i + 3);
    };
    if (KG == 1 || kg == 0) next();

    const int kw = key_of(i) + 64 * kg;
    // a tile that no row of the wave reads is stepped over
    if (has_rows && kw <= hi_w && (kw + 63 >= lo_w || kw < a.keep)) {
      const bf16_t* Kb = tiles + (buf * KG + kg) * TSZ;
      const bf16_t* Vb = Kb + KSZ;
      const int* flag = flags + (buf * KG + kg) * 4;
      const floatx16 zero16 = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      const u32x4 there4 = *reinterpret_cast<const u32x4*>(flag);      // blocks with a page
      // The operands that LDS gives come four at a time, one such group ahead of the products (a read takes as long as three or four
      // products), the values' first group while the softmax is made.
      auto key_part = [&](int f) { return *reinterpret_cast<const bf16x8*>(Kb + f / DH16 * (32 * KROW + 2 * BLOCK_PAD) + col * KROW + col / 16 * BLOCK_PAD + f % DH16 * 16 + g * 8); };
      auto value_part = [&](int f) {      // f: block of 16 keys, then of 32 dims
        return *reinterpret_cast<const bf16x8*>(Vb + min(32 * (f % DB) + col, DH - 1) * VROW + 16 * (f / DB) + 8 * g);
      };
      constexpr int KF = 2 * DH16, VF = 4 * DB;
      bf16x8 part[2][4];
      floatx16 s[2];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < KF) part[0][j] = key_part(j);
      if (KG > 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int f = 0; f < KF; f += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (f + 4 + j < KF) part[(f / 4 + 1) % 2][j] = key_part(f + 4 + j);
          else if (f + 4 >= KF && j < VF) part[(f / 4 + 1) % 2][j] = value_part(j);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (f + j < KF) {
            const int c = (f + j) / DH16, d = (f + j) % DH16;
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
              s[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(part[f / 4 % 2][j], qf[d][p], d == 0 && p == 0 ? zero16 : s[c], 0, 0, 0);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (KG > 1) __builtin_amdgcn_s_setprio(0);
      settle(s[0], s[1]);
      const int there = __builtin_amdgcn_readfirstlane(there4[0] | there4[1] << 1 | there4[2] << 2 | there4[3] << 3);
      // an edge: a key that one of the wave's rows does not read.  The same for the whole wave.
      const bool edge = kw + 63 > pos0 + wrow0 || (kw < lo_last && kw + 63 >= a.keep) || there != 15;
      // whether this lane's row reads its i-th key of the half tile c (no branches: all of it is one comparison after the other)
      auto reads = [&](int c, int i) {
        const int key = kw + 32 * c + 8 * (i / 4) + 4 * g + i % 4;
        return ((there >> (2 * c + i / 8) & 1) != 0) & (key <= my_pos) & ((key >= my_lo) | (key < a.keep));
      };
      if constexpr (CAPPED) {
#pragma unroll
        for (int c = 0; c < 2; ++c) a.cap.of<16>(scale2, [&](int i) { return s[c][i]; }, [&](int i, float v) { s[c][i] = v; });
      }
      if (edge) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[c][i] = reads(c, i) ? s[c][i] : -INFINITY;
      }
      float top = LOWEST, tops[4] = {LOWEST, LOWEST, LOWEST, LOWEST};
#pragma unroll
      for (int i = 0; i < 16; ++i) tops[i % 4] = fmaxf(fmaxf(tops[i % 4], s[0][i]), s[1][i]);
      top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      top = fmaxf(top, other_half(top));
      // (moving the maximum only once it has grown by 2^6, so that the results so far are rarely multiplied, is no faster here, 268.0 us and 268.1,
      // and the largest weights, which are ones so, would be rounded as the others are: 0.0019 off 64 bits for 0.0017)
      const float m_new = fmaxf(m_run, top * per_score), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
      if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
      }
      constexpr int V0 = (KF + 3) / 4;      // the group of `part` that the values begin in
      float sums[4] = {0.f, 0.f, 0.f, 0.f};
      bf16x8 pf[4][PARTS];
      auto weigh = [&](int c) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[c][i] = __builtin_amdgcn_exp2f(fmaf(s[c][i], per_score, -m_new));
          sums[i % 4] += s[c][i];
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float p[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) p[j] = s[c][8 * x + j];
          split<PARTS>(p, pf[2 * c + x]);
        }
      };
      // (the second half's weights are made beside the first half's products: the 32-bit prompt of 1,001 26.5 -> 24.9 us; heads of up to 32 have
      // both halves among their first four products)
      weigh(0);
      if (DB == 1) weigh(1);
      __builtin_amdgcn_sched_barrier(0);
      if (KG > 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int f = 0; f < VF; f += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (f + 4 + j < VF) part[(V0 + f / 4 + 1) % 2][j] = value_part(f + 4 + j);
        if (f == VF / 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (f + j < VF) {
            const int x = (f + j) / DB, d = (f + j) % DB;
#pragma unroll
            for (int pt = 0; pt < PARTS; ++pt) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(part[(V0 + f / 4) % 2][j], pf[x][pt], o[d], 0, 0, 0);
          }
        if (f == 0 && DB > 1) weigh(1);
      }
      if (KG > 1) __builtin_amdgcn_s_setprio(0);
      l_run += (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }
    if (KG > 1 && kg > 0) next();
    __syncthreads();
  }
  l_run += other_half(l_run);

  if constexpr (KG > 1) {
    // the other key groups hand maxima, sums and weighted values to the first, lane to lane; the tiles in LDS are done with
    if (kg > 0) {
      float* join = reinterpret_cast<float*>(smem) + ((kg - 1) * THREADS + t) * JOIN;
      join[0] = m_run;
      join[1] = l_run;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) join[2 + 16 * d + i] = o[d][i];
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int k = 0; k < KG - 1; ++k) {
      const float* join = reinterpret_cast<const float*>(smem) + (k * THREADS + t) * JOIN;
      const float m_new = fmaxf(m_run, join[0]);
      const float f0 = __builtin_amdgcn_exp2f(m_run - m_new), f1 = __builtin_amdgcn_exp2f(join[0] - m_new);
      l_run = l_run * f0 + join[1] * f1;
      m_run = m_new;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * f0 + join[2 + 16 * d + i] * f1;
    }
  }
  float* const part = a.part + ((static_cast<size_t>(row0 + my_row) * a.H + h) * a.n_splits + share) * (DH + 2);      // (of this lane's row)
  if (row_ok && a.n_splits > 1) {
    if (g == 0) part[0] = m_run, part[1] = l_run;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int dim = 32 * d + 8 * (i / 4) + 4 * g + i % 4;
        if (dim < DH) part[2 + dim] = o[d][i];
      }
  } else if (row_ok) {
    if (a.sink) l_run += __builtin_amdgcn_exp2f((a.sink_at ? a.sink_at[h] : 0.f) * LOG2E - m_run);
    const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;      // (a row that reads nothing: zeros)
    const size_t at = static_cast<size_t>(row0 + my_row) * a.ldo + h * DH;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int dim = 32 * d + 8 * x + 4 * g;
        if (dim < DH) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float r = o[d][4 * x + j] * inv;
            if (PARTS == 1) static_cast<bf16_t*>(a.out)[at + dim + j] = from_float<bf16_t>(r);
            else static_cast<float*>(a.out)[at + dim + j] = r;
          }
        }
      }
  }
  if (*seen != 0 && has_rows) {
    // a value that is NaN reaches the rows that read it and no other: once more over the values, whose rows' results become NaN in the
    // value's dim (behind this wave's own stores above)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_wave_barrier();
    for (int i = i0 * KG; i < i1 * KG; ++i) {
      const int kt = key_of(i / KG) + 64 * (i % KG);
      for (int x = lane; x < DH * 4; x += 64) {
        const int dim = x / 4, first = kt + 16 * (x % 4), page = page_of(kt, 16 * (x % 4), page_entry(kt, 16 * (x % 4)));
        if (page < 0) continue;
        const uint8_t* v = a.v_pool + static_cast<size_t>(page) * page_bytes + (((hk * DH + dim) << a.page_shift) + (first & in_page));
        const bool scaled = fabsf(a.v_scale[static_cast<size_t>(page) * a.Hkv + hk]) < INFINITY;
        for (int j = 0; j < 16; ++j) {
          if (scaled && (v[j] & 0x7f) != 0x7f) continue;
          const int key = first + j;
          for (int r = wrow0; r < min(wrow0 + 32, nrows); ++r) {
            const int pos = pos0 + r;
            if (key > pos || (key < first_key(pos) && key >= a.keep)) continue;
            const size_t at = static_cast<size_t>(row0 + r) * a.ldo + h * DH + dim;
            if (a.n_splits > 1) a.part[((static_cast<size_t>(row0 + r) * a.H + h) * a.n_splits + share) * (DH + 2) + 2 + dim] = NAN;
            else if (PARTS == 1) static_cast<bf16_t*>(a.out)[at] = bf16_t{0x7fc0};
            else static_cast<float*>(a.out)[at] = NAN;
          }
        }
      }
    }
  }
}

template <int DH16, int PARTS, int RG, int KG, bool CAPPED>
static int launch_as(const Args& a, int n_tiles, hipStream_t stream) {
  constexpr int DH = DH16 * 16, DB = (DH + 31) / 32;
  constexpr int TILES = 2 * KG * (64 * (DH + 8) + 128 + DH * 72) * 2, JOIN = (KG - 1) * 64 * RG * (2 + 16 * DB) * 4;
  constexpr int BYTES = (TILES > JOIN ? TILES : JOIN) + 2 * KG * 4 * 4 + 16;
  static_assert(BYTES <= 160 * 1024, "LDS");
  auto* fn = &kernel<DH16, PARTS, RG, KG, CAPPED>;
  if (BYTES > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    if (e != hipSuccess) return static_cast<int>(e);
  }
  fn<<<dim3(a.H, n_tiles * (4 / RG), a.n_splits), 64 * RG * KG, BYTES, stream>>>(a);
  return 0;
}

template <int DH16, int PARTS, int RG, int KG>
static int launch(const Args& a, int n_tiles, hipStream_t stream) {
  return a.cap.cap2 > 0.f ? launch_as<DH16, PARTS, RG, KG, true>(a, n_tiles, stream) : launch_as<DH16, PARTS, RG, KG, false>(a, n_tiles, stream);
}

template <int DH16, int PARTS>
static int by_shape(const Args& a, int n_tiles, int rows, int groups, hipStream_t stream) {
  if (rows == 4 && groups == 1) return launch<DH16, PARTS, 4, 1>(a, n_tiles, stream);
  if constexpr (DH16 <= (PARTS == 1 ? 8 : 6)) {
    if (rows == 4 && groups == 2) return launch<DH16, PARTS, 4, 2>(a, n_tiles, stream);
    if (rows == 2 && groups == 2) return launch<DH16, PARTS, 2, 2>(a, n_tiles, stream);
  }
  return DN_ERR_SHAPE;
}

template <int PARTS>
static int by_dim(const Args& a, int n_tiles, int dh, int rows, int groups, hipStream_t stream) {
  switch (dh / 16) {
#define DN_DIM(N) case N: return by_shape<N, PARTS>(a, n_tiles, rows, groups, stream);
    DN_DIM(1) DN_DIM(2) DN_DIM(3) DN_DIM(4) DN_DIM(5) DN_DIM(6) DN_DIM(7) DN_DIM(8)
    DN_DIM(9) DN_DIM(10) DN_DIM(11) DN_DIM(12) DN_DIM(13) DN_DIM(14) DN_DIM(15) DN_DIM(16)
#undef DN_DIM
  }
  return DN_ERR_SHAPE;
}
}  // namespace portions8

extern "C" int dn_attention8_portions(const void* q, int ldq, void* out, int ldo, const void* k_pool, const void* v_pool,
                                      const float* k_scale, const float* v_scale, int n_pages, const int32_t* block_tables, int max_blocks,
                                      const int32_t* tile_seq, const int32_t* tile_row0, const int32_t* tile_nrows,
                                      const int32_t* tile_pos0, int n_tiles, float* part, int n_splits, int rows, int groups, int H,
                                      int Hkv, int dh, int page_size, float scale, int window, int keep, int sink, const float* sink_at, float cap, int dtype,
                                      hipStream_t stream) {
  if (dh < 16 || dh > 256 || dh % 16 != 0 || Hkv < 1 || H % Hkv != 0 || page_size < 16 || (page_size & (page_size - 1)) != 0 || !(scale > 0.f) ||
      n_pages < 1 || max_blocks < 1 || static_cast<size_t>(n_pages) * Hkv >= (1ull << 31) || static_cast<size_t>(Hkv) * dh * page_size >= (1ull << 31) ||
      window < 0 || keep < 0 || (keep > 0 && window == 0) || !(cap >= 0.f && cap < INFINITY) || ldq % 8 != 0 || n_splits < 1 || (n_splits > 1 && !part))
    return DN_ERR_SHAPE;
  if (dtype != DN_F32 && dtype != DN_BF16) return DN_ERR_DTYPE;
  if (n_tiles == 0) return 0;
  const portions8::Args a = {q, out, static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool), k_scale, v_scale,
                             block_tables, tile_seq, tile_row0, tile_nrows, tile_pos0, sink_at, part, ldq, ldo, n_pages, max_blocks, n_splits, H, Hkv,
                             __builtin_ctz(page_size), window, keep, sink, scale, attend8::Cap(cap)};
  const int rc = dtype == DN_BF16 ? portions8::by_dim<1>(a, n_tiles, dh, rows, groups, stream)
                                  : portions8::by_dim<3>(a, n_tiles, dh, rows, groups, stream);
  if (rc != 0) return rc;
  if (n_splits > 1)
    attend8::join(attend8::Parts{part, n_splits, tile_seq, tile_row0, tile_nrows, sink_at, sink, H, dh, ldo}, out, n_tiles, dtype, stream);
  return dn_launch_status();
}
