// Attention over the cache in 8 bits for steps of single rows: the bytes of the keys and values are what it takes, so every one is read
// once, 16 at a time, straight into the registers from which the matrix instructions are fed.
//
// A workgroup takes one row, up to 16 query heads that share a key head, and a run of the row's tiles of 64 keys; its waves take
// the run's tiles in turn, each with a softmax of its own (running maximum and sum, 32-bit), and join at the end.
//   A tile is four blocks of 16 keys, each inside one page.  S = K Q^T by v_mfma_f32_16x16x32_bf16: rows are keys, columns heads.  Which
//   key stands in which row is free: row r of the t-th product is key 4 t + r % 4 of block r / 4, so that lane (column c, group g) gets, over
//   the four products, the 16 keys of block g for head c: one scale of keys and one of values per lane, and its 16 weights are, eight
//   by eight, what the second product wants as its B operand if the k-th slots of group g are block g's keys.
//   O^T = V^T P^T: lane (dim r, group g) reads its dim's 16 values of block g, 16 bytes side by side.
// No LDS, no exchange between lanes but the maximum's over the four groups, and no number is touched on the way but by the conversion
// (v_cvt_scalef32_pk_bf16_fp8, two numbers each).  Dims go the same way: 16 bytes of a key are dims 16 g .. 16 g + 15 of a run of 64.
// 32-bit rows: three bfloat16 parts of the query and of the weights (attend8::split), three products for one.  bfloat16 rows: one part, the weight
// rounded to 8 digits, as the second product takes it (the sum under the softmax is of the 32-bit weights): 0.0016 to 0.0018 off 64 bits, of
// which the result's own rounding is 0.0016.
//
// Measured: 64 rows behind 100 to 1,020 tokens, 25 heads of 64, 24.2 us, 4.7 TB/s; one row over 131,072 keys, 32 heads over 8 of 128, 46 us, 5.8 TB/s where the
// memory-side cache has a part of it, 4.9 where it has none; 518 keys of 25 heads 5.1 us, of which 3 are the launch and a trip to memory for the tables.
#include "attention8_common.h"

namespace single8 {
using namespace attend8;

struct Args {
  const void* q;
  void* out;
  const uint8_t *k_pool, *v_pool;
  const float *k_scale, *v_scale;
  const int32_t *block_tables, *tile_seq, *tile_row0, *tile_pos0;
  const float* sink_at;
  float* part;      // attend8::Parts' results
  int ldq, ldo, n_pages, max_blocks, n_splits, H, Hkv, page_shift, window, keep, sink;      // pages of 1 << page_shift keys
  float scale;
  Cap cap;
};

// a value from the lane 16 away, and the one 32 away
__device__ __forceinline__ float across16(float v) { return __shfl_xor(v, 16); }

// CAPPED: scores have a soft cap (a kernel of its own, as for portions: 64 rows of 25 heads of 64 without one 24.7 -> 24.2 us)
template <int DH16, int PARTS, int WAVES, bool CAPPED>
__global__ __launch_bounds__(WAVES * 64) void kernel(const Args a) {
  constexpr int DH = DH16 * 16, NC = (DH16 + 3) / 4;
  extern __shared__ float lds[];      // [WAVES][16] maxima, [WAVES][16] sums, [WAVES][heads here][64 dims, or the head's fewer]
  const int G = a.H / a.Hkv, blocks = (G + 15) / 16;
  const int tile = blockIdx.z, sp = blockIdx.x, hk = blockIdx.y / blocks, h0 = blockIdx.y % blocks * 16;
  const int seq = a.tile_seq[tile];
  if (seq < 0) return;
  const int row = a.tile_row0[tile], pos = a.tile_pos0[tile];
  const int heads = min(G - h0, 16);      // of this workgroup
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int c16 = lane % 16, g = lane / 16, kg = c16 / 4;      // column or row; group; the block of this lane's row of keys
  const int in_page = (1 << a.page_shift) - 1;
  const int32_t* bt = a.block_tables + static_cast<size_t>(seq) * a.max_blocks;

  // the tiles that the row reads: `kept` ones from the start, then those from the window's first key on; this split's are i0 .. i1
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int kept = a.keep > 0 ? (min(a.keep, pos + 1) + 63) / 64 : 0;
  const int rest = max(lo / 64, kept);
  const int n_tiles = kept + max(0, pos / 64 - rest + 1);
  const int per = (n_tiles + a.n_splits - 1) / a.n_splits;
  const int i0 = sp * per, i1 = min(n_tiles, i0 + per);

  bf16x8 qf[NC][2][PARTS];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float v[8];
      const bool ok = c16 < heads && 4 * c + g < DH16;
      const size_t at = static_cast<size_t>(row) * a.ldq + (hk * G + h0 + (ok ? c16 : 0)) * DH + (ok ? c * 64 + g * 16 + m * 8 : 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = PARTS == 1 ? to_float(static_cast<const bf16_t*>(a.q)[at + j]) : static_cast<const float*>(a.q)[at + j];
        v[j] = ok ? x : 0.f;
      }
      split<PARTS>(v, qf[c][m]);
    }

  floatx4 o[DH16];
#pragma unroll
  for (int d = 0; d < DH16; ++d) o[d] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m_run = LOWEST, l_run = 0.f;
  const float scale2 = a.scale * LOG2E;

  // the page of the block that begins with `key` and the key's place in it; -1 where the row reads none of it
  auto page_of = [&](int key) {
    const int b = key >> a.page_shift;
    const int page = key <= pos && b < a.max_blocks ? bt[b] : -1;
    return page < a.n_pages ? page : -1;
  };
  for (int i = i0 + wave; i < i1; i += WAVES) {
    const int kt = 64 * (i < kept ? i : rest + i - kept);
    const int kb = kt + 16 * kg, vb = kt + 16 * g;
    const int k_page = page_of(kb), v_page = page_of(vb);
    const size_t kph = static_cast<size_t>(max(k_page, 0)) * a.Hkv + hk, vph = static_cast<size_t>(max(v_page, 0)) * a.Hkv + hk;
    const uint8_t* kp = a.k_pool + ((kph << a.page_shift) + (kb & in_page) + c16 % 4) * DH + g * 16;
    const uint8_t* vp = a.v_pool + ((vph * DH + c16) << a.page_shift) + (vb & in_page);
    u32x4 kr[4][NC], vr[DH16];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < NC; ++c) kr[t][c] = *reinterpret_cast<const u32x4*>(kp + t * 4 * DH + (4 * c + g < DH16 ? c * 64 : -g * 16));
#pragma unroll
    for (int d = 0; d < DH16; ++d) vr[d] = *reinterpret_cast<const u32x4*>(vp + (static_cast<size_t>(d) * 16 << a.page_shift));
    const float ks = a.k_scale[vph] * scale2;
    float vs = a.v_scale[vph];

    floatx4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (4 * c + 3 >= DH16 && 4 * c + g >= DH16) kr[t][c] = u32x4{0u, 0u, 0u, 0u};      // (dims past the head's end)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const bf16x8 kf = widen(kr[t][c][2 * m], kr[t][c][2 * m + 1]);
#pragma unroll
          for (int p = 0; p < PARTS; ++p) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[c][m][p], s[t], 0, 0, 0);
        }
      }
    }
    // s[t][j]: key vb + 4 t + j, head of this lane's column
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[t][j] *= ks;
    // (every product is read before the first branch behind it: the compiler left out the wait for one that is read behind a branch)
    if constexpr (CAPPED) a.cap.of<16>(1.0f, [&](int i) { return s[i / 4][i % 4]; }, [&](int i, float v) { s[i / 4][i % 4] = v; });
    // a tile at an edge, or with a page that is given back: what the row does not read is -inf, and its values are zeros, whatever
    // stands there (a weight of zero times NaN would be NaN), and so is the scale of a block of which it reads nothing.  The same for
    // the whole wave.
    const bool edge = kt + 63 > pos || kt < lo || __builtin_amdgcn_ballot_w64(v_page < 0) != 0;
    if (edge) {
      uint32_t mask[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = vb + 4 * t + j;
          const bool ok = v_page >= 0 && key <= pos && (key >= lo || key < a.keep);
          s[t][j] = ok ? s[t][j] : -INFINITY;
          mask[t] |= ok ? 0xffu << (8 * j) : 0u;
        }
#pragma unroll
      for (int d = 0; d < DH16; ++d)
#pragma unroll
        for (int t = 0; t < 4; ++t) vr[d][t] &= mask[t];
      vs = (mask[0] | mask[1] | mask[2] | mask[3]) != 0 ? vs : 0.f;
    }
    float top = LOWEST;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, s[t][j]);
    top = fmaxf(top, across16(top));
    top = fmaxf(top, other_half(top));
    const float m_new = fmaxf(m_run, top), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
    m_run = m_new;
    float p[16], sum = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = __builtin_amdgcn_exp2f(s[t][j] - m_new);
        sum += e;
        p[4 * t + j] = e * vs;      // (a power of two: the rounding below is the weight's)
      }
    l_run = l_run * alpha + sum;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
      for (int d = 0; d < DH16; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d][j] *= alpha;
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      bf16x8 pf[PARTS];
      split<PARTS>(p + 8 * m, pf);
#pragma unroll
      for (int d = 0; d < DH16; ++d) {
        const bf16x8 vf = widen(vr[d][2 * m], vr[d][2 * m + 1]);
#pragma unroll
        for (int pt = 0; pt < PARTS; ++pt) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[pt], o[d], 0, 0, 0);
      }
    }
  }
  l_run += across16(l_run);
  l_run += other_half(l_run);

  // the waves' results meet in LDS, 64 dims at a time: o[d][j] is dim 16 d + 4 g + j of head c16
  float* const ms = lds;
  float* const ls = lds + WAVES * 16;
  float* const os = lds + 2 * WAVES * 16;
  if (g == 0) ms[wave * 16 + c16] = m_run, ls[wave * 16 + c16] = l_run;
#pragma unroll
  for (int d0 = 0; d0 < DH16; d0 += 4) {
    constexpr int WIDE = DH16 < 4 ? DH : 64;
    const int wide = min(64, DH - d0 * 16);
    if (d0 > 0) __syncthreads();
    if (c16 < heads) {
#pragma unroll
      for (int d = d0; d < min(d0 + 4, DH16); ++d)
        *reinterpret_cast<floatx4*>(os + (wave * heads + c16) * WIDE + 16 * (d - d0) + 4 * g) = o[d];
    }
    __syncthreads();
    for (int x = threadIdx.x; x < heads * wide; x += WAVES * 64) {
      const int h = x / wide, d = x % wide;
      float m = LOWEST, l = 0.f, v = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) m = fmaxf(m, ms[w * 16 + h]);
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(ms[w * 16 + h] - m);
        l = fmaf(ls[w * 16 + h], f, l);
        v = fmaf(os[(w * heads + h) * WIDE + d], f, v);
      }
      const int head = hk * G + h0 + h;
      if (a.n_splits > 1) {
        float* part = a.part + ((static_cast<size_t>(row) * a.H + head) * a.n_splits + sp) * (DH + 2);
        part[2 + d0 * 16 + d] = v;
        if (d0 + d == 0) part[0] = m, part[1] = l;
      } else {
        if (a.sink) l += __builtin_amdgcn_exp2f((a.sink_at ? a.sink_at[head] : 0.f) * LOG2E - m);
        const float r = l == 0.f ? 0.f : v / l;      // (a row that reads nothing: zeros)
        const size_t at = static_cast<size_t>(row) * a.ldo + head * DH + d0 * 16 + d;
        if (PARTS == 1) static_cast<bf16_t*>(a.out)[at] = from_float<bf16_t>(r);
        else static_cast<float*>(a.out)[at] = r;
      }
    }
  }
}

template <int DH16, int PARTS>
static int launch(const Args& a, int n_tiles, hipStream_t stream) {
  // (heads beyond 128 leave the registers for four waves; up to there eight are faster than four: 16 rows in a window of 4,096 26.8 us and
  // 29.5, 64 rows over some 700 keys 24.6 and 25.3)
  constexpr int WAVES = DH16 <= 8 ? 8 : 4;
  const int G = a.H / a.Hkv, blocks = (G + 15) / 16;
  const size_t lds = (2 * WAVES * 16 + static_cast<size_t>(WAVES) * min(G, 16) * (DH16 < 4 ? DH16 * 16 : 64)) * sizeof(float);
  const dim3 grid(a.n_splits, a.Hkv * blocks, n_tiles);
  if (a.cap.cap2 > 0.f) kernel<DH16, PARTS, WAVES, true><<<grid, WAVES * 64, lds, stream>>>(a);
  else kernel<DH16, PARTS, WAVES, false><<<grid, WAVES * 64, lds, stream>>>(a);
  return 0;
}

template <int PARTS>
static int by_dim(const Args& a, int n_tiles, int dh, hipStream_t stream) {
  switch (dh / 16) {
#define DN_DIM(N) case N: return launch<N, PARTS>(a, n_tiles, stream);
    DN_DIM(1) DN_DIM(2) DN_DIM(3) DN_DIM(4) DN_DIM(5) DN_DIM(6) DN_DIM(7) DN_DIM(8)
    DN_DIM(9) DN_DIM(10) DN_DIM(11) DN_DIM(12) DN_DIM(13) DN_DIM(14) DN_DIM(15) DN_DIM(16)
#undef DN_DIM
  }
  return DN_ERR_SHAPE;
}
}  // namespace single8

extern "C" int dn_attention8_single(const void* q, int ldq, void* out, int ldo, const void* k_pool, const void* v_pool,
                                    const float* k_scale, const float* v_scale, int n_pages, const int32_t* block_tables, int max_blocks,
                                    const int32_t* tile_seq, const int32_t* tile_row0, const int32_t* tile_pos0, int n_tiles, float* part,
                                    int n_splits, int H, int Hkv, int dh, int page_size, float scale, int window, int keep,
                                    int sink, const float* sink_at, float cap, int dtype, hipStream_t stream) {
  if (dh < 16 || dh > 256 || dh % 16 != 0 || Hkv < 1 || H % Hkv != 0 || page_size < 16 || (page_size & (page_size - 1)) != 0 || window < 0 || keep < 0 ||
      (keep > 0 && window == 0) || !(cap >= 0.f && cap < INFINITY) || n_splits < 1 || (n_splits > 1 && !part))
    return DN_ERR_SHAPE;
  if (dtype != DN_F32 && dtype != DN_BF16) return DN_ERR_DTYPE;
  if (n_tiles == 0) return 0;
  const single8::Args a = {q, out, static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool), k_scale, v_scale,
                           block_tables, tile_seq, tile_row0, tile_pos0, sink_at, part, ldq, ldo, n_pages, max_blocks, n_splits, H, Hkv,
                           __builtin_ctz(page_size), window, keep, sink, scale, attend8::Cap(cap)};
  const int rc = dtype == DN_BF16 ? single8::by_dim<1>(a, n_tiles, dh, stream) : single8::by_dim<3>(a, n_tiles, dh, stream);
  if (rc != 0) return rc;
  if (n_splits > 1)
    attend8::join(attend8::Parts{part, n_splits, tile_seq, tile_row0, nullptr, sink_at, sink, H, dh, ldo}, out, n_tiles, dtype, stream);
  return dn_launch_status();
}
