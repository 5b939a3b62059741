// Attention of new tokens' queries over a paged cache of keys and values in the OCP MX block formats
// (the layout of mx_cache.hip), for single tokens, drafted tokens and prefill chunks.
//
// Math, for query row i of a sequence with n new tokens of L held ones, head h of group g = h / G:
//   s_j = scale * (q . k_j),  j < limit = L - n + i + 1 (causal) or L,  clamped to [0, L]
//   m = max s_j,  p_j = exp(s_j - m),  o = sum p_j v_j / sum p_j,  lse = m + log sum p_j
// A row without a visible key (or whose scores are all -inf: sum p = 0) gives o = 0 and lse = -inf.
//
// One pass over the keys with a running maximum and sum.  Scores and products run on the matrix cores
// (v_mfma_f32_16x16x32_bf16): an e2m1 or e4m3 element times its power-of-two scale is exact in bf16, so
// K and V enter the products exactly, decoded by v_cvt_scalef32_pk_bf16_{fp4,fp8} in registers.  What is
// not exact in bf16 is split into bf16 parts, each product summed in fp32: queries of bf16 are 1 part,
// of fp16 2 (11 bits), of fp32 3 (24 bits), all exact; probabilities are rounded to 2 parts (off by at
// most 2^-16, where the output's own half step is 2^-8 or 2^-11) and to 3 for fp32 outputs (2^-24).  Maxima,
// sums and outputs are held in fp32.
//
// The products are laid out so that nothing crosses lanes.  A lane is (n = lane % 16, g = lane / 16).
//   S^T = K Q^T: A = K, row n of 16-token tile u holds token 8 (n / 4) + n % 4 + 4 u of the 32; the
//     contraction's order is free, so lane g takes dims g D/4 .. (g + 1) D/4 - 1: whole MX blocks, one
//     contiguous load.  B = Q^T, column n = query row.  The result's lane holds query row n and tokens
//     8 g + (0..3) of tile 0 and 8 g + (4..7) of tile 1:
//   O^T = V^T P^T: which is B's layout, P^T: column n, tokens 8 g .. 8 g + 7.  A = V^T: tile j's row n is
//     dim n D/16 + j, so a lane decodes D/16 consecutive dims of 8 consecutive tokens, and pairs tokens
//     by one byte permutation for each two elements.
//   A query row's maximum, sum and rescaling are its lane's own (the four g's share the maximum).
#include "mx_device.h"

namespace {

using namespace vg;

constexpr int kTile = 32;   // keys of one step
constexpr int kWaves = 4;   // waves of a workgroup
constexpr int kRows = 16;   // query rows of a wave
#ifndef VG_STEP_GROUPS
#define VG_STEP_GROUPS 8
#endif
constexpr int kStepGroups = VG_STEP_GROUPS;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
  const void* q;
  const uint8_t *kc, *ks, *vc, *vs;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;   // NULL: one new token for each sequence
  void* out;
  float* lse;              // may be NULL
  float* part_o;           // [q_tokens * q_heads, splits, dim] when splits > 1
  float* part_ml;          // [q_tokens * q_heads, splits, 2]
  int64_t q_t, q_h;        // strides of q in elements
  int64_t table_stride;
  int32_t q_tokens, batch, q_heads, kv_heads, group;
  int32_t width;           // pages of a row of the table
  int32_t pages, page_shift;
  int32_t causal;
  int32_t row_tiles, tile_rows;
  int32_t chunk, splits;   // keys of a split (a multiple of kTile), splits of the longest sequence
  float scale_log2;        // scale * log2(e)
};

// The rows that one workgroup takes: rows row0 .. of the `rows` = new * group (token, head) pairs of
// sequence seq (-1: rows that belong to none, `length` 0).
struct RowTile {
  int32_t seq, tok0, fresh, length;  // fresh: new tokens of the sequence
  int32_t row0, rows;
};

// bounds(0) = 0, bounds(i) = starts[i - 1], bounds(batch + 2) = q_tokens: rows of no sequence come first
// and last, so that every row of the output is written.
__device__ inline int32_t row_bound(const AttnArgs& a, int32_t i) {
  if (i <= 0) return 0;
  if (i > a.batch + 1) return a.q_tokens;
  const int32_t x = a.starts[i - 1];
  return x < 0 ? 0 : (x > a.q_tokens ? a.q_tokens : x);
}

// The last i of 0 .. batch + 1 with floor(bounds(i) * scale / tile) + (count ? i : 0) <= at, 64 bounds a
// step.
__device__ inline int32_t find_bound(const AttnArgs& a, int32_t scale, int32_t tile, bool count, int32_t at) {
  const int32_t lane = threadIdx.x & 63;
  int32_t n = 0;
  for (int32_t i0 = 0; i0 < a.batch + 2; i0 += 64) {
    const int32_t i = i0 + lane;
    const bool below = i < a.batch + 2 && row_bound(a, i) * scale / tile + (count ? i : 0) <= at;
    n += __popcll(__ballot(below));
  }
  return n - 1;
}

__device__ inline int32_t held_tokens(const AttnArgs& a, int32_t seq) {
  if (seq < 0 || seq >= a.batch) return 0;
  const int64_t most = (int64_t)a.width << a.page_shift;
  const int64_t x = a.lengths[seq];
  return (int32_t)(x < 0 ? 0 : (x > most ? most : x));
}

__device__ inline RowTile find_tile(const AttnArgs& a, int32_t tile, int32_t tile_rows) {
  RowTile r;
  if (a.starts == nullptr) {
    const int32_t per = (a.group + tile_rows - 1) / tile_rows;
    r.seq = tile / per;
    r.row0 = (tile - r.seq * per) * tile_rows;
    r.tok0 = r.seq;
    r.fresh = 1;
  } else {
    const int32_t i = find_bound(a, a.group, tile_rows, true, tile);
    r.tok0 = row_bound(a, i);
    r.fresh = row_bound(a, i + 1) - r.tok0;
    r.row0 = (tile - (r.tok0 * a.group / tile_rows + i)) * tile_rows;
    r.seq = i - 1 < a.batch ? i - 1 : -1;
  }
  r.rows = r.fresh * a.group;
  r.length = held_tokens(a, r.seq);
  return r;
}

// Keys that new token i of the tile's sequence sees.
__device__ inline int32_t row_limit(const AttnArgs& a, const RowTile& r, int32_t i) {
  int32_t x = a.causal ? r.length - r.fresh + i + 1 : r.length;
  if (x > r.length) x = r.length;
  return x < 0 ? 0 : x;
}

// Splits that a tile whose rows see up to `limit` keys has.
__device__ inline int32_t splits_of(const AttnArgs& a, int32_t limit) {
  return limit <= a.chunk ? 1 : (limit + a.chunk - 1) / a.chunk;
}

// Elements 2 SEL and 2 SEL + 1 of a word of codes, times 2^(scale's exponent), as a bf16 pair.
template <int FMT>
__device__ __forceinline__ uint32_t decode_pair(uint32_t w, float scale, int sel) {
  bf16x2 r;
  if constexpr (FMT == VELOGRAD_MX_E2M1) {
    switch (sel) {
      case 0: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0); break;
      case 1: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1); break;
      case 2: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2); break;
      default: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3); break;
    }
  } else {
    r = sel == 0 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)
                 : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
  }
  return __builtin_bit_cast(uint32_t, r);
}

__device__ __forceinline__ float scale_arg(uint32_t code) {
  return __builtin_bit_cast(float, (code & 0xffu) << 23);
}

__device__ __forceinline__ f32x4 mfma(const u32x4 x, const u32x4 y, const f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y),
                                                 c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  const bf16x2 p = {(__bf16)x, (__bf16)y};
  return __builtin_bit_cast(uint32_t, p);
}

// f[8] as PARTS bf16 fragments whose sum is f (to 8 PARTS bits); the rest goes back into f.  A value that
// is not finite stays in the first part alone.
template <int PARTS>
__device__ __forceinline__ void split_parts(float* f, u32x4* out) {
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = pack_bf16(f[2 * i], f[2 * i + 1]);
      out[p][i] = w;
      if (p + 1 < PARTS) {
        const float a = __builtin_bit_cast(float, w << 16), b = __builtin_bit_cast(float, w & 0xffff0000u);
        f[2 * i] = __builtin_isfinite(a) ? f[2 * i] - a : 0.0f;
        f[2 * i + 1] = __builtin_isfinite(b) ? f[2 * i + 1] - b : 0.0f;
      }
    }
  }
}

// The same for probabilities (in [0, 2^8], or NaN): no infinities to look for.
template <int PARTS>
__device__ __forceinline__ void split_probs(float* f, u32x4* out) {
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = pack_bf16(f[2 * i], f[2 * i + 1]);
      out[p][i] = w;
      if (p + 1 < PARTS) {
        f[2 * i] -= __builtin_bit_cast(float, w << 16);
        f[2 * i + 1] -= __builtin_bit_cast(float, w & 0xffff0000u);
      }
    }
  }
}

__device__ __forceinline__ float across_g(float v, bool sum) {
  const float x = __shfl_xor(v, 16);
  v = sum ? v + x : __builtin_fmaxf(v, x);
  const float y = __shfl_xor(v, 32);
  return sum ? v + y : __builtin_fmaxf(v, y);
}

template <int D, int FMT, int DT>
struct Shape {
  static constexpr int kSteps = D / 32;                              // products of S^T
  static constexpr int kOut = D / 16;                                // 16-dim tiles of O^T
  static constexpr int kRowBytes = FMT == VELOGRAD_MX_E2M1 ? D / 2 : D;
  static constexpr int kKBytes = kRowBytes / 4;                      // a lane's bytes of a key
  static constexpr int kVBytes = kRowBytes / 16;                     // a lane's bytes of a value
  static constexpr int kPerWord = FMT == VELOGRAD_MX_E2M1 ? 4 : 2;   // pairs in a word of codes
  static constexpr int kKScales = D / 4 >= 32 ? D / 128 : 1;         // blocks of a lane's part of a key
  static constexpr int kQParts = DT == VELOGRAD_DTYPE_BF16 ? 1 : DT == VELOGRAD_DTYPE_F16 ? 2 : 3;
  static constexpr int kPParts = DT == VELOGRAD_DTYPE_F32 ? 3 : 2;
};

template <int BYTES>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (BYTES == 2) {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (BYTES == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (BYTES == 8) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    w[0] = v[0];
    w[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const u32x4 v = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
    }
  }
}

template <int D, int FMT, int DT>
__global__ __launch_bounds__(kWaves * 64) void mx_attention_kernel(const AttnArgs a) {
  using S = Shape<D, FMT, DT>;
  constexpr int kWordsK = S::kKBytes / 4;
  constexpr int kWordsV = S::kVBytes < 4 ? 1 : S::kVBytes / 4;
  // Heads fastest, then row tiles, then splits.
  const uint32_t tile_split = blockIdx.x / (uint32_t)a.kv_heads;
  const int32_t h = (int32_t)(blockIdx.x - tile_split * (uint32_t)a.kv_heads);
  const int32_t split = (int32_t)(tile_split / (uint32_t)a.row_tiles);
  const RowTile r = find_tile(a, (int32_t)(tile_split - (uint32_t)split * (uint32_t)a.row_tiles), kWaves * kRows);
  if (r.row0 < 0 || r.row0 >= r.rows) return;
  const int32_t here = r.rows - r.row0 < kWaves * kRows ? r.rows - r.row0 : kWaves * kRows;
  // Few rows: all waves take the same ones and share the keys out; else every wave takes its own.
  const bool share = here <= kRows;
  const int32_t wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int32_t wrow = share ? r.row0 : r.row0 + wave * kRows;
  const int32_t tile_limit = row_limit(a, r, (r.row0 + here - 1) / a.group);
  const int32_t active = splits_of(a, tile_limit);
  if (split >= active) return;

  const int32_t row = wrow + n;
  const bool row_ok = row < r.rows;
  const int32_t fresh = row_ok ? row / a.group : 0;
  const int32_t head = h * a.group + (row_ok ? row - fresh * a.group : 0);
  const int32_t limit = row_ok ? row_limit(a, r, fresh) : 0;
  const int64_t tok = r.tok0 + fresh;

  // The query row's fragments: dims g D/4 + 8 s .. + 7 for product s.
  u32x4 qf[S::kSteps][S::kQParts];
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) {
    float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row_ok) {
      const int64_t e = tok * a.q_t + head * a.q_h + g * (D / 4) + 8 * s;
      Codec<DT>::unpack(load16_any<DT>(a.q, e), f);
      if constexpr (DT == VELOGRAD_DTYPE_F32) Codec<DT>::unpack(load16_any<DT>(a.q, e + 4), f + 4);
    }
    split_parts<S::kQParts>(f, qf[s]);
  }

  f32x4 acc[S::kOut];
#pragma unroll
  for (int j = 0; j < S::kOut; ++j) acc[j] = f32x4{0, 0, 0, 0};
  float m = -3.0e38f, l = 0.0f;

  // The wave's keys: [begin, end) in steps; all its rows see every key below `clear`.
  int32_t end = (split + 1) * a.chunk;
  const int32_t last_row = (wrow + kRows < r.rows ? wrow + kRows : r.rows) - 1;
  const int32_t wave_limit = wrow < r.rows ? row_limit(a, r, last_row / a.group) : 0;
  if (end > wave_limit) end = wave_limit;
  const int32_t clear = wrow < r.rows ? row_limit(a, r, wrow / a.group) : 0;
  const int32_t begin = split * a.chunk + (share ? wave * kTile : 0);
  const int32_t stride = share ? kWaves * kTile : kTile;
  const int32_t* table = a.table + (int64_t)(r.seq < 0 ? 0 : r.seq) * a.table_stride;
  const int32_t page_mask = (1 << a.page_shift) - 1;

  for (int32_t t0 = begin; t0 < end; t0 += stride) {
    const int32_t tk = t0 + 8 * (n >> 2) + (n & 3), tv = t0 + 8 * g;
    int32_t ik = tk >> a.page_shift, iv = tv >> a.page_shift;
    if (ik >= a.width) ik = a.width - 1;
    if (iv >= a.width) iv = a.width - 1;
    int32_t pk = table[ik], pv = table[iv];
    const bool bad = (uint32_t)pv >= (uint32_t)a.pages;
    if ((uint32_t)pk >= (uint32_t)a.pages) pk = 0;
    if (bad) pv = 0;
    const int64_t hk = (int64_t)pk * a.kv_heads + h, hv = (int64_t)pv * a.kv_heads + h;
    const int32_t ok = tk & page_mask, ov = tv & page_mask;

    const uint8_t* kp = a.kc + ((hk << a.page_shift) + ok) * S::kRowBytes + g * S::kKBytes;
    const uint8_t* vp = a.vc + ((hv << a.page_shift) + ov) * S::kRowBytes + n * S::kVBytes;
    uint32_t kw[2][kWordsK], vw[8][kWordsV], kscale[2][S::kKScales];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      load_words<S::kKBytes>(kp + 4 * u * S::kRowBytes, kw[u]);
#pragma unroll
      for (int b = 0; b < S::kKScales; ++b)
        kscale[u][b] = a.ks[((hk * (D / 32) + (g * (D / 4)) / 32 + b) << a.page_shift) + ok + 4 * u];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) load_words<S::kVBytes>(vp + i * S::kRowBytes, vw[i]);
    u32x2 vscale = *reinterpret_cast<const u32x2*>(
        a.vs + ((hv * (D / 32) + (n * (D / 16)) / 32) << a.page_shift) + ov);

    // Scores.
    f32x4 sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) {
        u32x4 kf;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int pair = 4 * s + i;  // of the lane's D/8 pairs
          kf[i] = decode_pair<FMT>(kw[u][pair / S::kPerWord], scale_arg(kscale[u][pair / 16 % S::kKScales]),
                                   pair % S::kPerWord);
        }
#pragma unroll
        for (int p = S::kQParts - 1; p >= 0; --p) sc[u] = mfma(kf, qf[s][p], sc[u]);
      }
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = sc[i >> 2][i & 3] * a.scale_log2;

    const bool masked = t0 + kTile > clear || __ballot(bad) != 0;
    if (masked) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (bad || tv + i >= limit) x[i] = -__builtin_inff();
        // Nothing is read of what lies behind the sequence's end: its codes may be anything.
        if (bad || tv + i >= r.length) {
#pragma unroll
          for (int w = 0; w < kWordsV; ++w) vw[i][w] = 0;
          vscale[i >> 2] = (vscale[i >> 2] & ~(0xffu << (8 * (i & 3)))) | (127u << (8 * (i & 3)));
        }
      }
    }

    // The running maximum moves only when a row's new maximum passes it by 8 (p stays below 2^8, which
    // costs fp32 nothing): most steps rescale nothing.
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, x[i]);
    if (__ballot(top > m + 8.0f) != 0) {
      top = across_g(top, false);
      const float next = top > m + 8.0f ? top : m;  // for each row by itself
      const float f = __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= f;
#pragma unroll
      for (int j = 0; j < S::kOut; ++j) acc[j] *= f;
    }
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(x[i] - m);
      l += p[i];
    }
    u32x4 pf[S::kPParts];
    split_parts<S::kPParts>(p, pf);

    // Values: dims n D/16 + j of tokens 8 g .. 8 g + 7.
    u32x4 vf[S::kOut];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float s0 = scale_arg(vscale[i >> 1] >> (16 * (i & 1)));
      const float s1 = scale_arg(vscale[i >> 1] >> (16 * (i & 1) + 8));
#pragma unroll
      for (int d = 0; d < S::kOut / 2; ++d) {
        const uint32_t u0 = decode_pair<FMT>(vw[2 * i][d / S::kPerWord], s0, d % S::kPerWord);
        const uint32_t u1 = decode_pair<FMT>(vw[2 * i + 1][d / S::kPerWord], s1, d % S::kPerWord);
        vf[2 * d][i] = __builtin_amdgcn_perm(u1, u0, 0x05040100u);
        vf[2 * d + 1][i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
      }
    }
    if (masked && a.causal) {
      // A NaN among the values of a key that only some of the rows see would reach the others as 0 * NaN:
      // it is taken out of the product, and the rows that do see it get NaN by a product of flags.
      bool any = false;
#pragma unroll
      for (int j = 0; j < S::kOut; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          any |= (vf[j][i] & 0x7fffu) > 0x7f80u || (vf[j][i] & 0x7fff0000u) > 0x7f800000u;
      if (__ballot(any) != 0) {
        u32x4 seen;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          seen[i] = (x[2 * i] != -__builtin_inff() ? 0x3f80u : 0u) |
                    (x[2 * i + 1] != -__builtin_inff() ? 0x3f800000u : 0u);
#pragma unroll
        for (int j = 0; j < S::kOut; ++j) {
          u32x4 flag;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool lo = (vf[j][i] & 0x7fffu) > 0x7f80u, hi = (vf[j][i] & 0x7fff0000u) > 0x7f800000u;
            flag[i] = (lo ? 0x3f80u : 0u) | (hi ? 0x3f800000u : 0u);
            vf[j][i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
          }
          const f32x4 hit = mfma(flag, seen, f32x4{0, 0, 0, 0});
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (hit[i] > 0.0f) acc[j][i] = __builtin_nanf("");
        }
      }
    }
#pragma unroll
    for (int j = 0; j < S::kOut; ++j)
#pragma unroll
      for (int q = S::kPParts - 1; q >= 0; --q) acc[j] = mfma(vf[j], pf[q], acc[j]);
  }

  if (share) {
    // Waves 2, 3 hand their sums to 0, 1, then 1 to 0, in the accumulators' own layout.
    __shared__ float buf[kWaves / 2][D / 4 + 2][64];
#pragma unroll
    for (int w = kWaves / 2; w >= 1; w >>= 1) {
      if (wave >= w && wave < 2 * w) {
#pragma unroll
        for (int j = 0; j < S::kOut; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) buf[wave - w][4 * j + i][lane] = acc[j][i];
        buf[wave - w][D / 4][lane] = m;
        buf[wave - w][D / 4 + 1][lane] = l;
      }
      __syncthreads();
      if (wave < w) {
        const float mo = buf[wave][D / 4][lane];
        const float next = __builtin_fmaxf(m, mo);
        const float f = __builtin_amdgcn_exp2f(m - next), fo = __builtin_amdgcn_exp2f(mo - next);
        m = next;
        l = l * f + buf[wave][D / 4 + 1][lane] * fo;
#pragma unroll
        for (int j = 0; j < S::kOut; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[j][i] = acc[j][i] * f + buf[wave][4 * j + i][lane] * fo;
      }
      __syncthreads();
    }
    if (wave != 0) return;
  }
  l = across_g(l, true);
  if (!row_ok) return;
  const int64_t orow = tok * a.q_heads + head;
  if (active > 1) {
    float* po = a.part_o + (orow * a.splits + split) * D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < S::kOut; ++j) po[(4 * g + i) * S::kOut + j] = acc[j][i];
    if (g == 0) {
      a.part_ml[(orow * a.splits + split) * 2] = m;
      a.part_ml[(orow * a.splits + split) * 2 + 1] = l;
    }
    return;
  }
  const bool empty = l == 0.0f;
  const float inv = empty ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < S::kOut; ++j)
      Codec<DT>::store1(a.out, orow * D + (4 * g + i) * S::kOut + j, empty ? 0.0f : acc[j][i] * inv);
  if (a.lse != nullptr && g == 0)
    a.lse[orow] = empty ? -__builtin_inff() : (m + log2f(l)) * 0.693147180559945309f;
}

// ------------------------------------------------------------------------------------------
// Few rows a sequence: single and drafted tokens.
// ------------------------------------------------------------------------------------------
// A workgroup's four waves take the same 16 NQ query rows, each a quarter of the split's keys in one run,
// and add up at the end through LDS.  A wave reads its keys' codes straight into registers, one step of 32
// ahead of the products.  Page numbers come from one load of a lane each for 64 groups of 8 keys (512
// keys), and reach the addresses as scalars: a step's two halves of 16 keys lie on one page each.
constexpr int kRunGroups = 64;
constexpr int kRunKeys = 8 * kRunGroups;

template <int D, int FMT>
struct KeyTile {
  using S = Shape<D, FMT, VELOGRAD_DTYPE_BF16>;
  static constexpr int kWordsK = S::kKBytes / 4;
  static constexpr int kWordsV = S::kVBytes < 4 ? 1 : S::kVBytes / 4;
  uint32_t kw[2][kWordsK];
  uint32_t ks[2][S::kKScales];
  uint32_t vw[8][kWordsV];
  u32x2 vs;
};

struct CacheView {
  const uint8_t *kc, *ks, *vc, *vs;  // of the head
  int64_t code_page, scale_page;     // bytes of a page, all heads
  int32_t page_shift;
};

// Keys t .. t + 31, whose halves lie on pages p0 and p1 (places a0 and a1 of them).
template <int D, int FMT>
__device__ __forceinline__ void load_tile(const CacheView& c, int32_t p0, int32_t a0, int32_t p1, int32_t a1,
                                          int32_t n, int32_t g, KeyTile<D, FMT>& t) {
  using S = typename KeyTile<D, FMT>::S;
  const int64_t c0 = p0 * c.code_page + (int64_t)a0 * S::kRowBytes, c1 = p1 * c.code_page + (int64_t)a1 * S::kRowBytes;
  const int64_t s0 = p0 * c.scale_page + a0, s1 = p1 * c.scale_page + a1;
  const int32_t gk = n >> 2;  // the lane's group of 8 keys, as a row of K
  const uint8_t* kp = c.kc + (gk & 2 ? c1 : c0) + (8 * (gk & 1) + (n & 3)) * S::kRowBytes + g * S::kKBytes;
  const uint8_t* kq = c.ks + (gk & 2 ? s1 : s0) + (((g * (D / 4)) / 32) << c.page_shift) + 8 * (gk & 1) + (n & 3);
  const uint8_t* vp = c.vc + (g & 2 ? c1 : c0) + 8 * (g & 1) * S::kRowBytes + n * S::kVBytes;
  const uint8_t* vq = c.vs + (g & 2 ? s1 : s0) + (((n * (D / 16)) / 32) << c.page_shift) + 8 * (g & 1);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    load_words<S::kKBytes>(kp + 4 * u * S::kRowBytes, t.kw[u]);
#pragma unroll
    for (int b = 0; b < S::kKScales; ++b) t.ks[u][b] = kq[((int64_t)b << c.page_shift) + 4 * u];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) load_words<S::kVBytes>(vp + i * S::kRowBytes, t.vw[i]);
  t.vs = *reinterpret_cast<const u32x2*>(vq);
}

// S^T of the tile for one query tile: x[i] is the score of key 8 g + i, unscaled.
template <int D, int FMT, int PARTS>
__device__ __forceinline__ void decode_keys(const KeyTile<D, FMT>& t, u32x4 (*kf)[D / 32]) {
  using S = typename KeyTile<D, FMT>::S;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float scale[S::kKScales];
#pragma unroll
    for (int b = 0; b < S::kKScales; ++b) scale[b] = scale_arg(t.ks[u][b]);
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pair = 4 * s + i;  // of the lane's D/8 pairs
        kf[u][s][i] = decode_pair<FMT>(t.kw[u][pair / S::kPerWord], scale[pair / 16 % S::kKScales], pair % S::kPerWord);
      }
  }
}

// V^T of the tile: fragment j is dim n D/16 + j of keys 8 g .. 8 g + 7.
template <int D, int FMT>
__device__ __forceinline__ void decode_values(const KeyTile<D, FMT>& t, u32x4* vf) {
  using S = typename KeyTile<D, FMT>::S;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // The conversion reads its scale's exponent alone, so the bits around the byte may be anything.
    const uint32_t w = t.vs[i >> 1];
    const float s0 = __builtin_bit_cast(float, i & 1 ? w << 7 : w << 23);
    const float s1 = __builtin_bit_cast(float, i & 1 ? w >> 1 : w << 15);
#pragma unroll
    for (int d = 0; d < S::kOut / 2; ++d) {
      const uint32_t u0 = decode_pair<FMT>(t.vw[2 * i][d / S::kPerWord], s0, d % S::kPerWord);
      const uint32_t u1 = decode_pair<FMT>(t.vw[2 * i + 1][d / S::kPerWord], s1, d % S::kPerWord);
      vf[2 * d][i] = __builtin_amdgcn_perm(u1, u0, 0x05040100u);
      vf[2 * d + 1][i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
    }
  }
}

// One query tile's running state: rows in lanes (column n), keys or dims in registers.
template <int D>
struct RowState {
  f32x4 acc[D / 16];
  float m, l;
};

// x becomes the probabilities' exponents' arguments less the maximum; updates m, l, acc.
template <int D>
__device__ __forceinline__ void softmax_step(float* x, RowState<D>& r) {
  float top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(x[0], x[1]), __builtin_fmaxf(x[2], x[3])),
                              __builtin_fmaxf(__builtin_fmaxf(x[4], x[5]), __builtin_fmaxf(x[6], x[7])));
  // The running maximum moves only when a row's new maximum passes it by 8 (p stays below 2^8, which
  // costs fp32 nothing): most steps rescale nothing.
  if (__ballot(top > r.m + 8.0f) != 0) {
    top = across_g(top, false);
    const float next = top > r.m + 8.0f ? top : r.m;  // for each row by itself
    const float f = __builtin_amdgcn_exp2f(r.m - next);
    r.m = next;
    r.l *= f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) r.acc[j] *= f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(x[i] - r.m);
  r.l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
}

// Bytes of w that are 0xFF (scales: a block marked NaN), or 0x7F with any sign (e4m3's NaN): bit 7 of each.
__device__ __forceinline__ uint32_t nan_scales(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u; }
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

template <int D, int FMT>
__device__ __forceinline__ bool any_nan(const KeyTile<D, FMT>& t) {
  uint32_t any = nan_scales(t.vs[0]) | nan_scales(t.vs[1]);
  if constexpr (FMT == VELOGRAD_MX_E4M3)
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int w = 0; w < KeyTile<D, FMT>::kWordsV; ++w) any |= nan_codes(t.vw[i][w]);
  return __ballot(any != 0) != 0;
}

// A NaN among the values of a key that only some of the rows see would reach the others as 0 * NaN: its
// codes are taken out of the tile, and the rows that do see it get NaN by a product of flags.
template <int D, int FMT, int NQ>
__device__ __forceinline__ void keep_nan_apart(KeyTile<D, FMT>& t, const float (*x)[8], RowState<D>* rows) {
  constexpr int kOut = D / 16;
  constexpr int kEach = FMT == VELOGRAD_MX_E4M3 ? kOut : 1;  // e2m1 has no NaN of its own: blocks only
  u32x4 seen[NQ], blocks;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = t.vs[i >> 1] >> (16 * (i & 1));
    blocks[i] = ((w & 0xffu) == 0xffu ? 0x3f80u : 0u) | ((w & 0xff00u) == 0xff00u ? 0x3f800000u : 0u);
#pragma unroll
    for (int q = 0; q < NQ; ++q)
      seen[q][i] = (x[q][2 * i] != -__builtin_inff() ? 0x3f80u : 0u) |
                   (x[q][2 * i + 1] != -__builtin_inff() ? 0x3f800000u : 0u);
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    u32x4 f = blocks;
    if constexpr (FMT == VELOGRAD_MX_E4M3) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w0 = nan_codes(t.vw[2 * i][e >> 2]) >> (8 * (e & 3) + 7);
        const uint32_t w1 = nan_codes(t.vw[2 * i + 1][e >> 2]) >> (8 * (e & 3) + 7);
        f[i] |= (w0 & 1u) * 0x3f80u | (w1 & 1u) * 0x3f800000u;
      }
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const f32x4 hit = mfma(f, seen[q], f32x4{0, 0, 0, 0});
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < kOut; ++j)
          if (kEach == 1 || j == e) rows[q].acc[j][i] = hit[i] > 0.0f ? __builtin_nanf("") : rows[q].acc[j][i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool block = ((t.vs[i >> 2] >> (8 * (i & 3))) & 0xffu) == 0xffu;
#pragma unroll
    for (int w = 0; w < KeyTile<D, FMT>::kWordsV; ++w) {
      if constexpr (FMT == VELOGRAD_MX_E4M3) t.vw[i][w] &= ~((nan_codes(t.vw[i][w]) >> 7) * 0xffu);
      if (block) t.vw[i][w] = 0;
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) t.vs[i] &= ~(nan_scales(t.vs[i]));  // 0xFF -> 0x7F
}

// A row's result, unnormalised sums to the workspace where the keys are split, else out and lse.
template <int D, int DT>
__device__ __forceinline__ void store_row(const AttnArgs& a, const RowState<D>& r, int64_t orow, int32_t split,
                                          bool partial, int32_t g) {
  constexpr int kOut = D / 16;
  if (partial) {
    float* po = a.part_o + (orow * a.splits + split) * D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kOut; j += 4)
        *reinterpret_cast<f32x4*>(po + (4 * g + i) * kOut + j) =
            f32x4{r.acc[j][i], r.acc[j + 1][i], r.acc[j + 2][i], r.acc[j + 3][i]};
    if (g == 0) {
      a.part_ml[(orow * a.splits + split) * 2] = r.m;
      a.part_ml[(orow * a.splits + split) * 2 + 1] = r.l;
    }
    return;
  }
  const bool empty = r.l == 0.0f;
  const float inv = empty ? 0.0f : 1.0f / r.l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[kOut];
#pragma unroll
    for (int j = 0; j < kOut; ++j) f[j] = empty ? 0.0f : r.acc[j][i] * inv;
    const int64_t e = orow * D + (4 * g + i) * kOut;
    if constexpr (kOut >= Codec<DT>::kVec) {
#pragma unroll
      for (int j = 0; j < kOut; j += Codec<DT>::kVec) store16<DT>(a.out, e + j, Codec<DT>::pack(f + j));
    } else {
#pragma unroll
      for (int j = 0; j < kOut; ++j) Codec<DT>::store1(a.out, e + j, f[j]);
    }
  }
  if (a.lse != nullptr && g == 0)
    a.lse[orow] = empty ? -__builtin_inff() : (r.m + log2f(r.l)) * 0.693147180559945309f;
}

// A query row's fragments: dims g D/4 + 8 s .. + 7 for product s; zeros for a row that is none.
template <int D, int DT>
__device__ __forceinline__ void load_query(const AttnArgs& a, int64_t e, bool ok,
                                           u32x4 (*qf)[Shape<D, VELOGRAD_MX_E2M1, DT>::kQParts]) {
  using S = Shape<D, VELOGRAD_MX_E2M1, DT>;
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) {
    float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (ok) {
      Codec<DT>::unpack(load16_any<DT>(a.q, e + 8 * s), f);
      if constexpr (DT == VELOGRAD_DTYPE_F32) Codec<DT>::unpack(load16_any<DT>(a.q, e + 8 * s + 4), f + 4);
    }
    split_parts<S::kQParts>(f, qf[s]);
  }
}

// Waves of a SIMD that the registers are held to: as many as take no spills.
constexpr int step_occupancy(int dim, int fmt, int dtype) {
  const bool small = fmt == VELOGRAD_MX_E2M1, plain = dtype == VELOGRAD_DTYPE_BF16;
  return dim == 64 ? (small || plain ? 4 : 3) : dim == 128 ? (small && plain ? 3 : 2) : 1;
}

template <int D, int FMT, int DT, int NQ>
__global__ __launch_bounds__(kWaves * 64, step_occupancy(D, FMT, DT)) void mx_attention_step_kernel(const AttnArgs a) {
  using S = Shape<D, FMT, DT>;
  constexpr int kTileRows = kRows * NQ;
  // Heads fastest, then row tiles, then splits.
  const uint32_t tile_split = blockIdx.x / (uint32_t)a.kv_heads;
  const int32_t h = (int32_t)(blockIdx.x - tile_split * (uint32_t)a.kv_heads);
  const int32_t split = (int32_t)(tile_split / (uint32_t)a.row_tiles);
  const RowTile r = find_tile(a, (int32_t)(tile_split - (uint32_t)split * (uint32_t)a.row_tiles), kTileRows);
  if (r.row0 < 0 || r.row0 >= r.rows) return;
  const int32_t last = (r.row0 + kTileRows < r.rows ? r.row0 + kTileRows : r.rows) - 1;
  const int32_t most = row_limit(a, r, last / a.group);      // keys that the tile's last row sees,
  const int32_t clear = row_limit(a, r, r.row0 / a.group);   // and that all its rows see
  const int32_t active = splits_of(a, most);
  if (split >= active) return;
  const int32_t wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;

  // The wave's keys: a quarter of the split's steps.
  const int32_t from = split * a.chunk;
  const int32_t till = from + a.chunk < most ? from + a.chunk : most;
  const int32_t steps = (till - from + kTile - 1) / kTile;
  const int32_t begin = from + (steps * wave / kWaves) * kTile;
  int32_t end = from + (steps * (wave + 1) / kWaves) * kTile;
  if (end > till) end = till;

  bool row_ok[NQ];
  int32_t limit[NQ];
  int64_t orow[NQ];
  u32x4 qf[NQ][S::kSteps][S::kQParts];
  RowState<D> rows[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int32_t row = r.row0 + kRows * q + n;
    row_ok[q] = row < r.rows;
    const int32_t fresh = row_ok[q] ? row / a.group : 0;
    const int32_t head = h * a.group + (row_ok[q] ? row - fresh * a.group : 0);
    limit[q] = row_ok[q] ? row_limit(a, r, fresh) : 0;
    const int64_t tok = r.tok0 + fresh;
    orow[q] = tok * a.q_heads + head;
    load_query<D, DT>(a, tok * a.q_t + head * a.q_h + g * (D / 4), row_ok[q], qf[q]);
#pragma unroll
    for (int j = 0; j < S::kOut; ++j) rows[q].acc[j] = f32x4{0, 0, 0, 0};
    rows[q].m = -3.0e38f;
    rows[q].l = 0.0f;
  }

  const int32_t* table = a.table + (int64_t)(r.seq < 0 ? 0 : r.seq) * a.table_stride;
  const int32_t page_mask = (1 << a.page_shift) - 1;
  CacheView c;
  c.page_shift = a.page_shift;
  c.code_page = (int64_t)a.kv_heads * S::kRowBytes << a.page_shift;
  c.scale_page = (int64_t)a.kv_heads * (D / 32) << a.page_shift;
  c.kc = a.kc + ((int64_t)h * S::kRowBytes << a.page_shift);
  c.vc = a.vc + ((int64_t)h * S::kRowBytes << a.page_shift);
  c.ks = a.ks + ((int64_t)h * (D / 32) << a.page_shift);
  c.vs = a.vs + ((int64_t)h * (D / 32) << a.page_shift);

  for (int32_t run = begin; run < end; run += kRunKeys) {
    const int32_t run_end = run + kRunKeys < end ? run + kRunKeys : end;
    int32_t at = (run + 8 * lane) >> a.page_shift;
    if (at >= a.width) at = a.width - 1;
    int32_t page = table[at];
    const bool none = (uint32_t)page >= (uint32_t)a.pages;
    if (none) page = 0;
    const uint64_t missing = __ballot(none);

    auto fetch = [&](int32_t t0, KeyTile<D, FMT>& t) {
      const int32_t i = (t0 - run) >> 3;
      const int32_t p0 = __builtin_amdgcn_readlane(page, i), p1 = __builtin_amdgcn_readlane(page, i + 2);
      load_tile<D, FMT>(c, p0, t0 & page_mask, p1, (t0 + 16) & page_mask, n, g, t);
    };
    auto use = [&](int32_t t0, KeyTile<D, FMT>& t) {
      float x[NQ][8];
      {
        u32x4 kf[2][S::kSteps];
        decode_keys<D, FMT, S::kQParts>(t, kf);
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            f32x4 sc = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
              for (int p = S::kQParts - 1; p >= 0; --p) sc = mfma(kf[u][s], qf[q][s][p], sc);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[q][4 * u + i] = sc[i] * a.scale_log2;
          }
      }
      const uint32_t gone = (uint32_t)(missing >> ((t0 - run) >> 3)) & 0xfu;
      const bool masked = t0 + kTile > clear || gone != 0;
      if (masked) {
        const bool bad = (gone >> g) & 1u;
        // Of the lane's 8 keys: how many there are, and how many the row sees.
        const int32_t here = bad ? 0 : r.length - t0 - 8 * g;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const int32_t see = bad ? 0 : limit[q] - t0 - 8 * g;
#pragma unroll
          for (int i = 0; i < 8; ++i) x[q][i] = i < see ? x[q][i] : -__builtin_inff();
        }
        // What lies behind the sequence's end may be anything: it is taken as zeros.
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int w = 0; w < KeyTile<D, FMT>::kWordsV; ++w) t.vw[i][w] = i < here ? t.vw[i][w] : 0;
          const uint32_t m = 0xffu << (8 * (i & 3));
          t.vs[i >> 2] = i < here ? t.vs[i >> 2] : (t.vs[i >> 2] & ~m) | (0x7f7f7f7fu & m);
        }
      }
      if (masked && clear < most && any_nan<D, FMT>(t)) keep_nan_apart<D, FMT, NQ>(t, x, rows);
      u32x4 vf[S::kOut];
      decode_values<D, FMT>(t, vf);
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        softmax_step<D>(x[q], rows[q]);
        u32x4 pf[S::kPParts];
        split_probs<S::kPParts>(x[q], pf);
#pragma unroll
        for (int p = S::kPParts - 1; p >= 0; --p)
#pragma unroll
          for (int j = 0; j < S::kOut; ++j) rows[q].acc[j] = mfma(vf[j], pf[p], rows[q].acc[j]);
      }
    };
    // Each step's loads are issued a step before, without a branch around them (past the run's end the last
    // step's again): the wait for one step's codes then leaves the next one's in flight.
    const int32_t final = run + (run_end - 1 - run) / kTile * kTile;
    KeyTile<D, FMT> t0, t1;
    fetch(run, t0);
    for (int32_t t = run;; t += 2 * kTile) {
      fetch(t + kTile < final ? t + kTile : final, t1);
      use(t, t0);
      if (t >= final) break;
      fetch(t + 2 * kTile < final ? t + 2 * kTile : final, t0);
      use(t + kTile, t1);
      if (t + kTile >= final) break;
    }
  }

  // Waves 2, 3 hand their sums to 0, 1, then 1 to 0, in the accumulators' own layout.
  __shared__ float buf[kWaves / 2][D / 4 + 2][64];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
#pragma unroll
    for (int w = kWaves / 2; w >= 1; w >>= 1) {
      if (wave >= w && wave < 2 * w) {
#pragma unroll
        for (int j = 0; j < S::kOut; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) buf[wave - w][4 * j + i][lane] = rows[q].acc[j][i];
        buf[wave - w][D / 4][lane] = rows[q].m;
        buf[wave - w][D / 4 + 1][lane] = rows[q].l;
      }
      __syncthreads();
      if (wave < w) {
        const float mo = buf[wave][D / 4][lane];
        const float next = __builtin_fmaxf(rows[q].m, mo);
        const float f = __builtin_amdgcn_exp2f(rows[q].m - next), fo = __builtin_amdgcn_exp2f(mo - next);
        rows[q].m = next;
        rows[q].l = rows[q].l * f + buf[wave][D / 4 + 1][lane] * fo;
#pragma unroll
        for (int j = 0; j < S::kOut; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            rows[q].acc[j][i] = rows[q].acc[j][i] * f + buf[wave][4 * j + i][lane] * fo;
      }
      __syncthreads();
    }
  }
  if (wave != 0) return;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    rows[q].l = across_g(rows[q].l, true);
    if (row_ok[q]) store_row<D, DT>(a, rows[q], orow[q], split, active > 1, g);
  }
}

// Joins the splits of one (token, head) row; rows of tiles that had one split are left alone.  D/4 lanes
// hold the row, the workgroup's other lanes take other splits, and LDS adds them up.
template <int D, int DT>
__global__ __launch_bounds__(256) void mx_attention_join_kernel(const AttnArgs a) {
  constexpr int kLanes = D / 4, kSets = 256 / kLanes;
  const int64_t orow = blockIdx.x;
  const int32_t tok = (int32_t)(orow / a.q_heads), head = (int32_t)(orow - (int64_t)tok * a.q_heads);
  RowTile r;
  if (a.starts == nullptr) {
    r.seq = r.tok0 = tok;
    r.fresh = 1;
  } else {
    const int32_t i = find_bound(a, 1, 1, false, tok);
    r.tok0 = row_bound(a, i);
    r.fresh = row_bound(a, i + 1) - r.tok0;
    r.seq = i - 1 < a.batch ? i - 1 : -1;
  }
  r.rows = r.fresh * a.group;
  r.length = held_tokens(a, r.seq);
  const int32_t row = (tok - r.tok0) * a.group + head % a.group;
  int32_t last = row - row % a.tile_rows + a.tile_rows;
  if (last > r.rows) last = r.rows;
  const int32_t active = splits_of(a, row_limit(a, r, (last - 1) / a.group));
  if (active <= 1) return;

  const float* ml = a.part_ml + orow * a.splits * 2;
  const int32_t d = threadIdx.x % kLanes, set = threadIdx.x / kLanes;
  const float* po = a.part_o + orow * a.splits * D + 4 * d;
  float m = -3.0e38f;
  for (int32_t s = threadIdx.x & 63; s < active; s += 64) m = __builtin_fmaxf(m, ml[2 * s]);
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) m = __builtin_fmaxf(m, __shfl_xor(m, w));
  float l = 0.0f;
  f32x4 o = {0, 0, 0, 0};
  for (int32_t s = set; s < active; s += kSets) {
    const float f = __builtin_amdgcn_exp2f(ml[2 * s] - m);
    l += ml[2 * s + 1] * f;
    o += *reinterpret_cast<const f32x4*>(po + (int64_t)s * D) * f;
  }
  __shared__ float sums[kSets][D + 4];
#pragma unroll
  for (int i = 0; i < 4; ++i) sums[set][4 * d + i] = o[i];
  if (d == 0) sums[set][D] = l;
  __syncthreads();
  const int32_t e = threadIdx.x;
  if (e >= D) return;
  float total = 0.0f, x = 0.0f;
#pragma unroll
  for (int i = 0; i < kSets; ++i) {
    total += sums[i][D];
    x += sums[i][e];
  }
  const bool empty = total == 0.0f;
  Codec<DT>::store1(a.out, orow * D + e, empty ? 0.0f : x / total);
  if (a.lse != nullptr && e == 0)
    a.lse[orow] = empty ? -__builtin_inff() : (m + log2f(total)) * 0.693147180559945309f;
}

// How a call is laid out: workgroups over row tiles, heads and splits of the keys.
struct AttnPlan {
  int64_t row_tiles;
  int32_t tile_rows;
  int32_t query_tiles;  // of 16 rows a wave, in the kernel for few rows; 0: the kernel for many
  int32_t chunk, splits;
};

AttnPlan plan_attention(int64_t q_tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, bool ragged,
                        int64_t most, int cus) {
  AttnPlan p;
  const int64_t group = q_heads / kv_heads;
  // Rows of a sequence, on average.
  const int64_t rows = ragged ? q_tokens * group / (batch > 0 ? batch : 1) : group;
  p.query_tiles = rows <= 64 ? 1 : 0;
  p.tile_rows = p.query_tiles > 0 ? kRows * p.query_tiles : kWaves * kRows;
  p.row_tiles = ragged ? q_tokens * group / p.tile_rows + batch + 2
                       : batch * ((group + p.tile_rows - 1) / p.tile_rows);
  // Splits of the keys, so that there are about eight workgroups for each CU: sequences differ in length, and
  // many short workgroups even that out.
  const int64_t base = p.row_tiles * kv_heads;
  const int64_t want = (kStepGroups * (int64_t)cus + base - 1) / base;
  int64_t chunk = (most + want - 1) / want;
  chunk = (chunk + kWaves * kTile - 1) / (kWaves * kTile) * (kWaves * kTile);
  const int64_t least = kWaves * kTile * 2;
  if (chunk < least) chunk = least;
  p.chunk = (int32_t)chunk;
  p.splits = (int32_t)((most + chunk - 1) / chunk);
  if (p.splits < 1) p.splits = 1;
  return p;
}

template <int D, int FMT, int DT>
void launch_attention(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
  const dim3 grid((uint32_t)(a.kv_heads * p.row_tiles * a.splits));
  if (p.query_tiles == 1)
    hipLaunchKernelGGL((mx_attention_step_kernel<D, FMT, DT, 1>), grid, dim3(kWaves * 64), 0, st, a);
  else
    hipLaunchKernelGGL((mx_attention_kernel<D, FMT, DT>), grid, dim3(kWaves * 64), 0, st, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((mx_attention_join_kernel<D, DT>), dim3((uint32_t)a.q_tokens * (uint32_t)a.q_heads),
                       dim3(256), 0, st, a);
}

template <int FMT, int DT>
void launch_dim(const AttnArgs& a, const AttnPlan& p, int64_t dim, hipStream_t st) {
  if (dim == 64)
    launch_attention<64, FMT, DT>(a, p, st);
  else if (dim == 128)
    launch_attention<128, FMT, DT>(a, p, st);
  else
    launch_attention<256, FMT, DT>(a, p, st);
}

template <int DT>
void launch_fmt(const AttnArgs& a, const AttnPlan& p, int64_t dim, int fmt, hipStream_t st) {
  if (fmt == VELOGRAD_MX_E4M3)
    launch_dim<VELOGRAD_MX_E4M3, DT>(a, p, dim, st);
  else
    launch_dim<VELOGRAD_MX_E2M1, DT>(a, p, dim, st);
}

int32_t check_attention(const char* what, int64_t q_tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                        int64_t head_dim, int64_t table_width, int64_t page_size, bool ragged) {
  if (q_tokens < 0 || batch < 0 || q_heads < 1 || q_heads % kv_heads != 0)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT,
                "%s: invalid shape q_tokens=%lld sequences=%lld q_heads=%lld kv_heads=%lld", what,
                (long long)q_tokens, (long long)batch, (long long)q_heads, (long long)kv_heads);
  if (!ragged && q_tokens != batch)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT,
                "%s: without q_starts every sequence has one query token: q_tokens=%lld, sequences=%lld", what,
                (long long)q_tokens, (long long)batch);
  if (table_width < 0 || table_width > (1 << 30) / page_size)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: a sequence of %lld pages is too long", what,
                (long long)table_width);
  if (q_tokens > INT32_MAX / q_heads || batch > INT32_MAX / 2 || q_heads > INT32_MAX / head_dim)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: q_tokens=%lld, q_heads=%lld are too many", what,
                (long long)q_tokens, (long long)q_heads);
  return 0;
}

}  // namespace

extern "C" {

VELOGRAD_API size_t velograd_mx_cache_attention_workspace_bytes(int64_t q_tokens, int64_t sequences,
                                                                int64_t q_heads, int64_t kv_heads,
                                                                int64_t head_dim, int64_t table_width,
                                                                int64_t page_size, int32_t ragged,
                                                                int32_t device) {
  const char* what = "velograd_mx_cache_attention_workspace_bytes";
  if (check_mx_cache(what, kv_heads, head_dim, 0, page_size, VELOGRAD_MX_E2M1) != 0 ||
      check_attention(what, q_tokens, sequences, q_heads, kv_heads, head_dim, table_width, page_size,
                      ragged != 0) != 0)
    return 0;
  const int cus = cu_count(device);
  if (cus <= 0 || q_tokens == 0) return 0;
  const AttnPlan p = plan_attention(q_tokens, sequences, q_heads, kv_heads, ragged != 0,
                                    table_width * page_size, cus);
  if (p.splits <= 1) return 0;
  return (size_t)q_tokens * (size_t)q_heads * (size_t)p.splits * (size_t)(head_dim + 2) * sizeof(float);
}

VELOGRAD_API int32_t velograd_mx_cache_attention(
    const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
    const int32_t* block_table, const int32_t* lengths, const int32_t* q_starts, void* out, float* lse,
    void* workspace, size_t ws_bytes, int64_t q_tokens, int64_t sequences, int64_t q_heads, int64_t kv_heads,
    int64_t head_dim, int64_t q_token_stride, int64_t q_head_stride, int64_t table_stride, int64_t table_width,
    int64_t pages, int64_t page_size, float scale, int32_t causal, int32_t dtype, int32_t mx_format,
    void* hip_stream) {
  const char* what = "velograd_mx_cache_attention";
  if (elem_bytes_of(dtype) == 0)
    return fail(VELOGRAD_ERR_UNSUPPORTED_DTYPE, "%s: unsupported dtype %d", what, (int)dtype);
  if (const int32_t rc = check_mx_cache(what, kv_heads, head_dim, pages, page_size, mx_format)) return rc;
  const bool ragged = q_starts != nullptr;
  if (const int32_t rc = check_attention(what, q_tokens, sequences, q_heads, kv_heads, head_dim, table_width,
                                         page_size, ragged))
    return rc;
  if (!__builtin_isfinite(scale))
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: scale must be finite", what);
  if (q_tokens == 0) {
    clear_error();
    return 0;
  }
  if (q == nullptr || out == nullptr || (sequences > 0 && lengths == nullptr))
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: q, out and lengths must not be NULL", what);
  // An empty cache or table: every page is outside the cache and no key is read.
  const bool any = sequences > 0 && table_width > 0;
  if (any && (block_table == nullptr || (pages > 0 && (k_codes == nullptr || k_scales == nullptr ||
                                                       v_codes == nullptr || v_scales == nullptr))))
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: the cache and block_table must not be NULL", what);
  if (!aligned16(k_codes) || !aligned16(k_scales) || !aligned16(v_codes) || !aligned16(v_scales) ||
      !aligned16(out))
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: the cache and out must be 16-byte aligned", what);
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess)
    return fail(VELOGRAD_ERR_DEVICE_QUERY, "%s: hipGetDevice failed", what);
  const int cus = cu_count(device);
  if (cus <= 0) return fail(VELOGRAD_ERR_DEVICE_QUERY, "%s: cannot query device %d", what, device);
  const AttnPlan p = plan_attention(q_tokens, sequences, q_heads, kv_heads, ragged,
                                    pages > 0 ? table_width * page_size : 0, cus);
  const size_t rows = (size_t)q_tokens * (size_t)q_heads * (size_t)p.splits;
  if (p.splits > 1 && (workspace == nullptr || ws_bytes < rows * (size_t)(head_dim + 2) * sizeof(float)))
    return fail(VELOGRAD_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes,
                rows * (size_t)(head_dim + 2) * sizeof(float));
  if (p.row_tiles > INT32_MAX / p.splits || p.row_tiles * p.splits > INT32_MAX / kv_heads)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: %lld row tiles exceed the grid limit", what,
                (long long)p.row_tiles);

  AttnArgs a;
  a.q = q;
  a.kc = static_cast<const uint8_t*>(k_codes);
  a.ks = static_cast<const uint8_t*>(k_scales);
  a.vc = static_cast<const uint8_t*>(v_codes);
  a.vs = static_cast<const uint8_t*>(v_scales);
  a.table = block_table;
  a.lengths = lengths;
  a.starts = q_starts;
  a.out = out;
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o == nullptr ? nullptr : a.part_o + rows * (size_t)head_dim;
  a.q_t = q_token_stride;
  a.q_h = q_head_stride;
  a.table_stride = table_stride;
  a.q_tokens = (int32_t)q_tokens;
  a.batch = (int32_t)sequences;
  a.q_heads = (int32_t)q_heads;
  a.kv_heads = (int32_t)kv_heads;
  a.group = (int32_t)(q_heads / kv_heads);
  a.width = pages > 0 ? (int32_t)table_width : 0;
  a.pages = (int32_t)pages;
  a.page_shift = 0;
  while (((int64_t)1 << a.page_shift) < page_size) ++a.page_shift;
  a.causal = causal != 0 ? 1 : 0;
  a.row_tiles = (int32_t)p.row_tiles;
  a.tile_rows = p.tile_rows;
  a.chunk = p.chunk;
  a.splits = p.splits;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634074);
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  switch (dtype) {
    case VELOGRAD_DTYPE_F32: launch_fmt<VELOGRAD_DTYPE_F32>(a, p, head_dim, mx_format, st); break;
    case VELOGRAD_DTYPE_F16: launch_fmt<VELOGRAD_DTYPE_F16>(a, p, head_dim, mx_format, st); break;
    default: launch_fmt<VELOGRAD_DTYPE_BF16>(a, p, head_dim, mx_format, st); break;
  }
  return check_launch(what);
}

}  // extern "C"
