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
// most 2^-16, where the output's own half step is 2^-8 or 2^-11) and to 3 for fp32 outputs (2^-24); in chunks
// of bf16 to 1 (chunk_parts).  Maxima, sums and outputs are held in fp32.
//
// Few rows are bound by the codes' bytes: the step kernel's waves each take an equal share of all keys and stream them
// through LDS, and a second launch joins the pieces; where all is small, the item kernel does both.  Many rows are
// bound by the products and the exponentials: the chunk kernel decodes keys once for all its waves.
//
// The products are laid out so that nothing crosses lanes.  A lane is (n = lane % 16, g = lane / 16).
//   S^T = K Q^T: A = K, row n of half u of a 32-key tile is key 16 u + n; the contraction's order is free, so
//     lane g takes chunks of 16 bytes g, g + 4, ..: each within an MX block, and four lanes' load contiguous.
//     B = Q^T, column n = query row.  The result's lane holds query row n and keys 16 u + 4 g + (0..3):
//   O^T = V^T P^T: which is B's layout, P^T: column n, with the contraction's 8 positions of lane g those
//     keys.  A = V^T: fragment j's row n is dim n D/16 + j, so a lane decodes D/16 consecutive dims of its 8
//     keys, and pairs keys by one byte permutation for each two elements.
//   A query row's maximum, sum and rescaling are its lane's own (the four g's share the maximum).
#include <type_traits>

#include "mx_device.h"

namespace {

using namespace vg;

constexpr int kTile = 32;   // keys of one step
constexpr int kWaves = 4;   // waves of a workgroup
constexpr int kRows = 16;   // query rows of a wave
// Query tiles of a wave at most, so that its rows and their sums fit the registers.
constexpr int most_tiles(int dim, int dtype) {
  const int tiles = dtype == VELOGRAD_DTYPE_BF16 || dtype == VELOGRAD_DTYPE_F16 ? 4 : 2;
  return dim == 256 ? (dtype == VELOGRAD_DTYPE_BF16 ? 2 : 1) : dim == 128 && dtype == VELOGRAD_DTYPE_F16 ? 2 : tiles;
}
// Parts of a probability in chunks: the products count there, and one part of 8 bits is off by at most 2^-8 of each
// probability, the half step that the bf16 output is rounded by anyway.
constexpr int chunk_parts(int dtype) {
  return dtype == VELOGRAD_DTYPE_BF16 ? 1 : dtype == VELOGRAD_DTYPE_F16 ? 2 : 3;
}

// Query tiles of a wave of the chunk kernel, so that its rows, their sums and a step's scores fit 256 registers.  4096
// new tokens of 6000, 32 heads, e2m1, at 1, 2 and 3 tiles: bf16 of 64 dims 262, 197 and (at 4) 320 us, of 128 dims 364,
// 279 and 665, fp16 of 128 dims 465 and 391, fp32 of 64 dims 382, 336 and 460; of 256 dims 1 and 2 bf16 358 and 647.
constexpr int chunk_tiles(int dim, int dtype) {
  return dim == 64 ? 2 : dim == 128 && dtype != VELOGRAD_DTYPE_F32 ? 2 : 1;
}

// Steps of a wave's share at least: one decode step over 2000 keys takes 12.2 us at 1, 11.0 at 2, 12.7 at 4, 14.6 at
// 8 (fewer shares are joined faster, but last longer).
constexpr int kLeastSteps = 2;
// Steps that the beginning of an item counts for: 24 e4m3 sequences take 35.4 us at 0, 31.5 at 4, 30.7 at 6, 30.0 at
// 10; 64 ragged ones 79.0, 77.5, 76.9 and 79.2.
constexpr int kBeginSteps = 6;

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
  float* part_o;           // [workers, 2, tile_rows, dim]: unfinished sums
  float* part_ml;          // [workers, 2, tile_rows, 2]: their maximum and sum
  int32_t* joins;          // [q_tokens * q_heads, 2]: where a row's sums begin, and how many there are
  int64_t q_t, q_h;        // strides of q in elements
  int64_t table_stride;
  int32_t q_tokens, batch, q_heads, kv_heads, group;
  int32_t width;           // pages of a row of the table
  int32_t pages, page_shift;
  int32_t causal;
  int32_t workers;         // waves of the step kernel
  int32_t least_steps;     // its smallest share
  int32_t begin_steps;     // what the beginning of an item counts for
  int32_t step_rows;       // sequences of more rows are the chunk kernel's
  float scale_log2;        // |scale| * log2(e), or 1
  float q_factor;          // what queries are multiplied by: the scale's sign, or 0
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

__device__ inline int32_t held_tokens(const AttnArgs& a, int32_t seq) {
  if (seq < 0 || seq >= a.batch) return 0;
  const int64_t most = (int64_t)a.width << a.page_shift;
  const int64_t x = a.lengths[seq];
  return (int32_t)(x < 0 ? 0 : (x > most ? most : x));
}

// Sequence i of a call as the kernels count them: with q_starts, i = 0 and i = batch + 1 are the rows before
// the first sequence and behind the last.
__device__ inline int32_t sequences(const AttnArgs& a) { return a.starts == nullptr ? a.batch : a.batch + 2; }

__device__ inline RowTile sequence_rows(const AttnArgs& a, int32_t i) {
  RowTile r;
  if (a.starts == nullptr) {
    r.seq = r.tok0 = i;
    r.fresh = 1;
  } else {
    r.seq = i - 1 < a.batch ? i - 1 : -1;
    r.tok0 = row_bound(a, i);
    r.fresh = row_bound(a, i + 1) - r.tok0;
    if (r.fresh < 0) r.fresh = 0;  // starts that fall: no rows
  }
  r.row0 = 0;
  r.rows = r.fresh * a.group;
  r.length = held_tokens(a, r.seq);
  return r;
}

// Whether q_starts falls behind sequence i: no call that the entry point's contract allows.  The kernels then leave rows
// out, but stay inside their buffers: a share's steps are counted in 32 bits, which only disjoint rows cannot exceed.
__device__ __forceinline__ bool falls(const AttnArgs& a, int32_t i) {
  return a.starts != nullptr && i < sequences(a) && row_bound(a, i + 1) < row_bound(a, i);
}

// Keys that new token i of the tile's sequence sees.
__device__ inline int32_t row_limit(const AttnArgs& a, const RowTile& r, int32_t i) {
  int32_t x = a.causal ? r.length - r.fresh + i + 1 : r.length;
  if (x > r.length) x = r.length;
  return x < 0 ? 0 : x;
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
  uint32_t w = __builtin_bit_cast(uint32_t, p);
  asm("" : "+v"(w));  // one conversion: the halves that are taken out of w again are not converted anew
  return w;
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
  static constexpr int kKBytes = kRowBytes / 4;                      // a lane's bytes of a key,
  static constexpr int kChunkBytes = kKBytes < 16 ? kKBytes : 16;    // in chunks, 4 lanes' side by side
  static constexpr int kChunks = kKBytes / kChunkBytes;
  static constexpr int kChunkElems = FMT == VELOGRAD_MX_E2M1 ? 2 * kChunkBytes : kChunkBytes;  // 16 or 32
  static constexpr int kVBytes = kRowBytes / 16;                     // a lane's bytes of a value
  static constexpr int kPerWord = FMT == VELOGRAD_MX_E2M1 ? 4 : 2;   // pairs in a word of codes
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

// ------------------------------------------------------------------------------------------
// Few rows a sequence: single and drafted tokens.
// ------------------------------------------------------------------------------------------
// Every wave works by itself, on 16 NQ query rows of one kv head and a run of keys at a time, and reads the
// keys' codes straight into registers, one step of 32 ahead of the products.  Pages are looked up once for
// 1024 keys, by each lane for the 16 keys of a half step, which one page holds; a step takes its two halves'
// offsets from those lanes as scalars.
constexpr int kHalf = kTile / 2;
constexpr int kRunKeys = 64 * kHalf;

template <int D, int FMT>
struct KeyTile {
  using S = Shape<D, FMT, VELOGRAD_DTYPE_BF16>;
  static constexpr int kWordsK = S::kKBytes / 4;
  static constexpr int kWordsV = S::kVBytes < 4 ? 1 : S::kVBytes / 4;
  uint32_t kw[2][kWordsK];       // key n of each half: a lane's parts
  uint32_t ks[2][S::kChunks];    // and their scales
  uint32_t vw[8][kWordsV];       // values 4 g + (0..3) of each half
  u32x2 vs;
};

// A tile comes by way of LDS: copied there without passing registers, 16 bytes a lane from whole lines (past
// the caches that nothing else reads it from), kStages - 1 tiles ahead, into a ring of the wave's own.
template <int D, int FMT>
struct Stage {
  using S = typename KeyTile<D, FMT>::S;
  static constexpr int kHalfBytes = kHalf * S::kRowBytes;       // codes of a half's keys, or values
  static constexpr int kScaleWords = D / 2;                     // of both, [keys or values][half][block][key / 4]
  static constexpr int kScaleLoads = (kScaleWords + 63) / 64;
  static constexpr int kCodes = 4 * kHalfBytes;                 // keys, then values, each half by half
  static constexpr int kBytes = kCodes + 256 * kScaleLoads;
  static constexpr int kCodeLoads = kCodes / 1024;
  static constexpr int kLoads = kCodeLoads + kScaleLoads;
};

typedef __attribute__((address_space(3))) void LdsVoid;
typedef const __attribute__((address_space(1))) void GlobalVoid;

// An address that is the same for the wave, kept in scalar registers: the loads add the lane's own 32 bits.
typedef const __attribute__((address_space(1))) uint8_t GlobalByte;
__device__ __forceinline__ GlobalByte* scalar(const uint8_t* p) {
  GlobalByte* q = (GlobalByte*)p;
  asm("" : "+s"(q));
  return q;
}

// To lane l's 16 (or 4) bytes behind `to`.  Codes come in whole lines, which are not kept (nt, the last argument);
// scales in parts of lines, which the next steps find in the caches.
__device__ __forceinline__ void copy16_to_lds(GlobalByte* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((GlobalVoid*)from, (LdsVoid*)to, 16, 0, 2);
}
__device__ __forceinline__ void copy4_to_lds(GlobalByte* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((GlobalVoid*)from, (LdsVoid*)to, 4, 0, 0);
}

// Lets at most N loads stay in flight, in order, and LDS reads none.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "the counter has 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
  asm volatile("" ::: "memory");
}

template <int D, int FMT>
__device__ __forceinline__ void stage_tile(const AttnArgs& a, int64_t code0, int64_t code1, int64_t scale0,
                                           int64_t scale1, uint8_t* to) {
  using T = Stage<D, FMT>;
  const int32_t lane = threadIdx.x & 63;
  if constexpr (T::kHalfBytes >= 1024) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < T::kHalfBytes / 1024; ++i) {
        const uint32_t at = 16 * lane;
        copy16_to_lds(scalar(a.kc + (u == 0 ? code0 : code1) + 1024 * i) + at, to + u * T::kHalfBytes + 1024 * i);
        copy16_to_lds(scalar(a.vc + (u == 0 ? code0 : code1) + 1024 * i) + at, to + (2 + u) * T::kHalfBytes + 1024 * i);
      }
  } else {  // 512 bytes: both halves in one
    const int64_t at = (lane < 32 ? code0 : code1) + 16 * (lane & 31);
    copy16_to_lds((GlobalByte*)a.kc + at, to);
    copy16_to_lds((GlobalByte*)a.vc + at, to + 2 * T::kHalfBytes);
  }
#pragma unroll
  for (int i = 0; i < T::kScaleLoads; ++i) {
    const int32_t w = (64 * i + lane) % T::kScaleWords;  // lanes past the last word load it again
    const int64_t at = (w / (D / 8) & 1 ? scale1 : scale0) + (((w / 4) % (D / 32)) << a.page_shift) + 4 * (w & 3);
    copy4_to_lds((GlobalByte*)(w < D / 4 ? a.ks : a.vs) + at, to + T::kCodes + 256 * i);
  }
}

template <int D, int FMT>
__device__ __forceinline__ void read_stage(const uint8_t* from, int32_t n, int32_t g, KeyTile<D, FMT>& t) {
  using S = typename KeyTile<D, FMT>::S;
  using T = Stage<D, FMT>;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int i = 0; i < S::kChunks; ++i) {
      load_words<S::kChunkBytes>(from + u * T::kHalfBytes + n * S::kRowBytes + (4 * i + g) * S::kChunkBytes,
                                 t.kw[u] + i * (S::kChunkBytes / 4));
      t.ks[u][i] = from[T::kCodes + (u * (D / 32) + ((4 * i + g) * S::kChunkElems) / 32) * kHalf + n];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      load_words<S::kVBytes>(from + (2 + u) * T::kHalfBytes + (4 * g + i) * S::kRowBytes + n * S::kVBytes, t.vw[4 * u + i]);
    t.vs[u] = *reinterpret_cast<const uint32_t*>(from + T::kCodes + ((2 + u) * (D / 32) + (n * (D / 16)) / 32) * kHalf + 4 * g);
  }
}

// K of the tile: fragment s of half u holds elements 8 s .. 8 s + 7 of the lane's part of key n.
template <int D, int FMT>
__device__ __forceinline__ void decode_keys(const KeyTile<D, FMT>& t, u32x4 (*kf)[D / 32]) {
  using S = typename KeyTile<D, FMT>::S;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float scale[S::kChunks];
#pragma unroll
    for (int b = 0; b < S::kChunks; ++b) scale[b] = scale_arg(t.ks[u][b]);
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pair = 4 * s + i;  // of the lane's D/8 pairs
        kf[u][s][i] = decode_pair<FMT>(t.kw[u][pair / S::kPerWord], scale[8 * s / S::kChunkElems], pair % S::kPerWord);
      }
  }
}

// Fragments 2 d and 2 d + 1 of V^T of the tile: dims n D/16 + 2 d, + 1 of the lane's 8 keys.
template <int D, int FMT>
__device__ __forceinline__ void decode_values(const KeyTile<D, FMT>& t, int d, u32x4* vf) {
  using S = typename KeyTile<D, FMT>::S;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // The conversion reads its scale's exponent alone, so the bits around the byte may be anything.
    const uint32_t w = t.vs[i >> 1];
    const float s0 = __builtin_bit_cast(float, i & 1 ? w << 7 : w << 23);
    const float s1 = __builtin_bit_cast(float, i & 1 ? w >> 1 : w << 15);
    const uint32_t u0 = decode_pair<FMT>(t.vw[2 * i][d / S::kPerWord], s0, d % S::kPerWord);
    const uint32_t u1 = decode_pair<FMT>(t.vw[2 * i + 1][d / S::kPerWord], s1, d % S::kPerWord);
    vf[0][i] = __builtin_amdgcn_perm(u1, u0, 0x05040100u);
    vf[1][i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
  }
}

// One query tile's running state: rows in lanes (column n), keys or dims in registers.
template <int D>
struct RowState {
  f32x4 acc[D / 16];
  float m, l;
};

template <int N>
__device__ __forceinline__ float largest(const float* x) {
  if constexpr (N == 1) return x[0];
  else return __builtin_fmaxf(largest<N / 2>(x), largest<N / 2>(x + N / 2));
}
template <int N>
__device__ __forceinline__ float sum(const float* x) {
  if constexpr (N == 1) return x[0];
  else return sum<N / 2>(x) + sum<N / 2>(x + N / 2);
}

// A row's running maximum moves to `next`.
template <int D>
__device__ __forceinline__ void set_max(float next, RowState<D>& r) {
  const float f = __builtin_amdgcn_exp2f(r.m - next);
  r.m = next;
  r.l *= f;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) r.acc[j] *= f;
}

// Probabilities of N scores; returns their sum.  `c` > 0 is the scale times log2(e).
template <int N>
__device__ __forceinline__ float probabilities(const float* x, float* p, float c, float m) {
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c, -m));
  return sum<N>(p);
}

// N scores x become probabilities; updates m, l, acc.
template <int D, int N>
__device__ __forceinline__ void softmax_step(float* x, float c, RowState<D>& r) {
  float top = largest<N>(x) * c;
  // The running maximum moves only when a row's new maximum passes it by 8 (p stays below 2^8, which
  // costs fp32 nothing): most steps rescale nothing.
  if (__ballot(top > r.m + 8.0f) != 0) {
    top = across_g(top, false);
    set_max<D>(top > r.m + 8.0f ? top : r.m, r);  // for each row by itself
  }
  r.l += probabilities<N>(x, x, c, r.m);
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
// x0: where the tile's 8 scores lie in a row's N.
template <int D, int FMT, int NQ, int N>
__device__ __forceinline__ void keep_nan_apart(KeyTile<D, FMT>& t, const float (*x)[N], int x0, RowState<D>* rows) {
  constexpr int kOut = D / 16;
  constexpr int kEach = FMT == VELOGRAD_MX_E4M3 ? kOut : 1;  // e2m1 has no NaN of its own: blocks only
  u32x4 seen[NQ], blocks;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = t.vs[i >> 1] >> (16 * (i & 1));
    blocks[i] = ((w & 0xffu) == 0xffu ? 0x3f80u : 0u) | ((w & 0xff00u) == 0xff00u ? 0x3f800000u : 0u);
#pragma unroll
    for (int q = 0; q < NQ; ++q)
      seen[q][i] = (x[q][x0 + 2 * i] != -__builtin_inff() ? 0x3f80u : 0u) |
                   (x[q][x0 + 2 * i + 1] != -__builtin_inff() ? 0x3f800000u : 0u);
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

// A row's unfinished sums, into row `at` of the workspace's [.., tile_rows, D].
template <int D>
__device__ __forceinline__ void store_part(const AttnArgs& a, const RowState<D>& r, int64_t at, int32_t g) {
  constexpr int kOut = D / 16;
  float* po = a.part_o + at * D;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < kOut; j += 4)
      *reinterpret_cast<f32x4*>(po + (4 * g + i) * kOut + j) =
          f32x4{r.acc[j][i], r.acc[j + 1][i], r.acc[j + 2][i], r.acc[j + 3][i]};
  if (g == 0) {
    a.part_ml[at * 2] = r.m;
    a.part_ml[at * 2 + 1] = r.l;
  }
}

// A row's out and lse.
template <int D, int DT>
__device__ __forceinline__ void store_row(const AttnArgs& a, const RowState<D>& r, int64_t orow, int32_t g) {
  constexpr int kOut = D / 16;
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

// A query row's fragments, in the order of decode_keys; zeros for a row that is none.
template <int D, int FMT, int DT, int CHUNK>
__device__ __forceinline__ void load_query(const AttnArgs& a, int64_t e, int32_t g, bool ok,
                                           u32x4 (*qf)[Shape<D, FMT, DT>::kQParts]) {
  using S = Shape<D, FMT, DT>;
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) {
    const int64_t at = e + (4 * (8 * s / CHUNK) + g) * CHUNK + 8 * s % CHUNK;
    if constexpr (S::kQParts == 1) {
      qf[s][0] = u32x4{0u, 0u, 0u, 0u};
      if (ok) qf[s][0] = load16_any<DT>(a.q, at);
      if (a.q_factor != 1.0f) {
        float f[8];
        Codec<DT>::unpack(qf[s][0], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= a.q_factor;
        qf[s][0] = Codec<DT>::pack(f);
      }
      continue;
    }
    float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (ok) {
      Codec<DT>::unpack(load16_any<DT>(a.q, at), f);
      if constexpr (DT == VELOGRAD_DTYPE_F32) Codec<DT>::unpack(load16_any<DT>(a.q, at + 4), f + 4);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= a.q_factor;
    split_parts<S::kQParts>(f, qf[s]);
  }
}

__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ int64_t take_lane(int64_t v, int32_t lane) {
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  const u32x2 r = {(uint32_t)__builtin_amdgcn_readlane((int)w[0], lane),
                   (uint32_t)__builtin_amdgcn_readlane((int)w[1], lane)};
  return __builtin_bit_cast(int64_t, r);
}

// Steps of an item: a tile of rows of one kv head over everything its sequence holds.
// Beginning an item (queries, pages, the first codes) takes a wave as long as several steps do, and is counted as
// such: a wave whose share holds the beginnings of several items gets fewer keys.
__device__ inline int32_t item_steps(const AttnArgs& a, int32_t length) {
  return a.begin_steps + (length <= kTile ? 1 : (length + kTile - 1) / kTile);
}

// Row tiles of a sequence in the step kernel; rows of no sequence are all its own.
__device__ __forceinline__ int32_t row_tiles(const AttnArgs& a, const RowTile& r, int32_t tile_rows) {
  return r.seq >= 0 && r.rows > a.step_rows ? 0 : (r.rows + tile_rows - 1) / tile_rows;
}

__device__ __forceinline__ int32_t sequence_steps(const AttnArgs& a, const RowTile& r, int32_t tile_rows) {
  return row_tiles(a, r, tile_rows) * item_steps(a, r.length);
}

// Inclusive sums over the wave's lanes.
__device__ __forceinline__ int32_t wave_scan(int32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, :2, :4, :8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

__device__ __forceinline__ RowTile sequence_rows_or_none(const AttnArgs& a, int32_t i) {
  if (i < sequences(a)) return sequence_rows(a, i);
  return RowTile{-1, 0, 0, 0, 0, 0};
}

// A wave's share of a head's steps, in the order sequence, row tile, step.
struct Share {
  int32_t sequence, tile, step;  // where it begins
  int32_t steps;                 // how many it has; 0: none
  int32_t each;                  // how many every share but the last has
  RowTile rows;                  // of the sequence
};

// Sequences differ in length, so a head's steps are dealt out in equal shares of consecutive ones, each to one
// wave, whatever items they belong to; wave w takes head w % kv_heads, so neighbouring waves read the same
// pages.  Every wave adds up all sequences' steps, 64 at a time, and finds the one that its share begins in.
__device__ __forceinline__ Share find_share(const AttnArgs& a, int32_t tile_rows, int32_t worker) {
  const int32_t lane = threadIdx.x & 63, count = sequences(a);
  RowTile r = sequence_rows_or_none(a, lane);
  int32_t mine = sequence_steps(a, r, tile_rows);
  int32_t upto = wave_scan(mine);
  int32_t total = __builtin_amdgcn_readlane(upto, 63);
  bool fall = falls(a, lane);
  if (count > 64) {
    int32_t more = 0;
    for (int32_t i = lane + 64; i < count; i += 64) {
      more += sequence_steps(a, sequence_rows(a, i), tile_rows);
      fall |= falls(a, i);
    }
    total += __builtin_amdgcn_readlane(wave_scan(more), 63);
  }
  if (__ballot(fall) != 0) total = 0;
  const int32_t shares = a.workers / a.kv_heads;  // of a head
  Share s;
  s.each = (int32_t)(((uint32_t)total + (uint32_t)shares - 1) / (uint32_t)shares);
  if (s.each < a.least_steps) s.each = a.least_steps;
  const int64_t from = (int64_t)s.each * (worker / a.kv_heads);
  s.steps = 0;
  if (from >= total) return s;
  s.steps = total - (int32_t)from < s.each ? total - (int32_t)from : s.each;
  int32_t before = 0;
  for (int32_t i0 = 0;; i0 += 64) {
    if (i0 > 0) {
      r = sequence_rows_or_none(a, i0 + lane);
      mine = sequence_steps(a, r, tile_rows);
      upto = wave_scan(mine);
    }
    const uint64_t here = __ballot((int32_t)from < before + upto);
    if (here != 0) {
      const int32_t l = __builtin_ctzll(here);  // the first sequence whose steps reach past `from`
      const int32_t in = (int32_t)from - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l));
      s.sequence = i0 + l;
      s.rows.seq = a.starts == nullptr ? s.sequence : s.sequence - 1 < a.batch ? s.sequence - 1 : -1;
      s.rows.tok0 = __builtin_amdgcn_readlane(r.tok0, l);
      s.rows.fresh = __builtin_amdgcn_readlane(r.fresh, l);
      s.rows.rows = __builtin_amdgcn_readlane(r.rows, l);
      s.rows.length = __builtin_amdgcn_readlane(r.length, l);
      s.tile = (int32_t)((uint32_t)in / (uint32_t)item_steps(a, s.rows.length));
      s.step = in - s.tile * item_steps(a, s.rows.length);
      return s;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
}

// A wave's query rows: 16 NQ rows of a tile, each in a lane's column.
template <int D, int FMT, int DT, int NQ>
struct QueryRows {
  bool ok[NQ];
  int32_t limit[NQ];   // keys that the row sees
  int64_t orow[NQ];    // its row of the output
  u32x4 frag[NQ][D / 32][Shape<D, FMT, DT>::kQParts];
  RowState<D> state[NQ];
};

template <int CHUNK, int D, int FMT, int DT, int NQ>
__device__ __forceinline__ void begin_rows(const AttnArgs& a, const RowTile& r, int32_t h,
                                           QueryRows<D, FMT, DT, NQ>& w) {
  const int32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int32_t row = r.row0 + kRows * q + n;
    w.ok[q] = row < r.rows;
    const int32_t fresh = w.ok[q] ? row / a.group : 0;
    const int32_t head = h * a.group + (w.ok[q] ? row - fresh * a.group : 0);
    w.limit[q] = w.ok[q] ? row_limit(a, r, fresh) : 0;
    const int64_t tok = r.tok0 + fresh;
    w.orow[q] = tok * a.q_heads + head;
    load_query<D, FMT, DT, CHUNK>(a, tok * a.q_t + head * a.q_h, g, w.ok[q], w.frag[q]);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) w.state[q].acc[j] = f32x4{0, 0, 0, 0};
    w.state[q].m = -3.0e38f;
    w.state[q].l = 0.0f;
  }
}

// Keys from .. end - 1 (from a multiple of 32) of the tile's sequence and kv head h.  All rows see the keys
// below `clear`, the last of them those below `most`.  PARTS: of the probabilities.
// TILES of 32 keys make a step, STAGES steps the ring in LDS.
template <int D, int FMT, int DT, int NQ, int PARTS, int TILES, int STAGES>
__device__ __forceinline__ void attend(const AttnArgs& a, const RowTile& r, int32_t h, int32_t from, int32_t end,
                                       int32_t clear, int32_t most, QueryRows<D, FMT, DT, NQ>& rows, uint8_t* ring) {
  constexpr int kStep = TILES * kTile;
  using S = Shape<D, FMT, DT>;
  const int32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int32_t page_mask = (1 << a.page_shift) - 1;
  const int32_t* table = a.table + (int64_t)(r.seq < 0 ? 0 : r.seq) * a.table_stride;

  for (int32_t run = from; run < end; run += kRunKeys) {
    const int32_t run_end = run + kRunKeys < end ? run + kRunKeys : end;
    int32_t at = (run + kHalf * lane) >> a.page_shift;
    if (at >= a.width) at = a.width - 1;
    int32_t page = table[at];
    const bool none = (uint32_t)page >= (uint32_t)a.pages;
    if (none) page = 0;
    const uint64_t missing = __ballot(none);
    const int64_t paged = (int64_t)page * a.kv_heads + h;
    const int32_t place = (run + kHalf * lane) & page_mask;
    const int64_t code = ((paged << a.page_shift) + place) * S::kRowBytes;
    const int64_t scale = ((paged * (D / 32)) << a.page_shift) + place;

    auto use = [&](int32_t t0, KeyTile<D, FMT>* t) {
      float x[NQ][8 * TILES];
#pragma unroll
      for (int j = 0; j < TILES; ++j) {
        u32x4 kf[2][S::kSteps];
        decode_keys<D, FMT>(t[j], kf);
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            f32x4 sc = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
              for (int p = S::kQParts - 1; p >= 0; --p) sc = mfma(kf[u][s], rows.frag[q][s][p], sc);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[q][8 * j + 4 * u + i] = sc[i];
          }
      }
      const uint32_t gone = (uint32_t)(missing >> ((t0 - run) / kHalf)) & ((1u << 2 * TILES) - 1u);
      const bool masked = t0 + kStep > (clear < end ? clear : end) || gone != 0;
      if (masked) {
#pragma unroll
        for (int u = 0; u < 2 * TILES; ++u) {
          const bool bad = (gone >> u) & 1u;
          const int32_t first = t0 + kHalf * u + 4 * g;
          KeyTile<D, FMT>& k = t[u / 2];
          // Of the lane's 4 keys: how many there are, and how many the row sees.
          const int32_t here = bad ? 0 : (r.length < end ? r.length : end) - first;
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            const int32_t see = bad ? 0 : (rows.limit[q] < end ? rows.limit[q] : end) - first;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[q][4 * u + i] = i < see ? x[q][4 * u + i] : -__builtin_inff();
          }
          // What lies behind the sequence's end (or another wave's beginning) is taken as zeros.
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 4 * (u & 1) + i;
#pragma unroll
            for (int w = 0; w < KeyTile<D, FMT>::kWordsV; ++w) k.vw[at][w] = i < here ? k.vw[at][w] : 0;
            const uint32_t m = 0xffu << (8 * i);
            k.vs[u & 1] = i < here ? k.vs[u & 1] : (k.vs[u & 1] & ~m) | (0x7f7f7f7fu & m);
          }
        }
        if (clear < most) {
#pragma unroll
          for (int j = 0; j < TILES; ++j)
            if (any_nan<D, FMT>(t[j])) keep_nan_apart<D, FMT, NQ, 8 * TILES>(t[j], x, 8 * j, rows.state);
        }
      }
      u32x4 pf[NQ][TILES][PARTS];
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        softmax_step<D, 8 * TILES>(x[q], a.scale_log2, rows.state[q]);
#pragma unroll
        for (int j = 0; j < TILES; ++j) split_probs<PARTS>(x[q] + 8 * j, pf[q][j]);
      }
#pragma unroll
      for (int d = 0; d < S::kOut / 2; ++d)
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
          u32x4 vf[2];
          decode_values<D, FMT>(t[j], d, vf);
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                rows.state[q].acc[2 * d + e] = mfma(vf[e], pf[q][j][p], rows.state[q].acc[2 * d + e]);
        }
    };
    const int32_t final = run + (run_end - 1 - run) / kTile * kTile;
    using T = Stage<D, FMT>;
    constexpr uint32_t kBytes = TILES * T::kBytes;
    uint32_t put = 0, get = 0;  // bytes into the ring
    auto stage = [&](int32_t t0) {
#pragma unroll
      for (int j = 0; j < TILES; ++j) {
        const int32_t t1 = t0 + j * kTile < final ? t0 + j * kTile : final, i = (t1 - run) / kHalf;
        stage_tile<D, FMT>(a, take_lane(code, i), take_lane(code, i + 1), take_lane(scale, i),
                           take_lane(scale, i + 1), ring + put + j * T::kBytes);
      }
      put = put == (STAGES - 1) * kBytes ? 0 : put + kBytes;
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) stage(run + i * kStep);
    for (int32_t t = run; t <= final; t += kStep) {
      // Past the run's end its last tile is copied again, so that the count of loads is the same for all.
      stage(t + (STAGES - 1) * kStep);
      wait_loads<(STAGES - 1) * TILES * T::kLoads>();
      KeyTile<D, FMT> tiles[TILES];
#pragma unroll
      for (int j = 0; j < TILES; ++j) read_stage<D, FMT>(ring + get + j * T::kBytes, n, g, tiles[j]);
      get = get == (STAGES - 1) * kBytes ? 0 : get + kBytes;
      use(t, tiles);
      // The next copy overwrites what was read here.
      wait_loads<(STAGES - 1) * TILES * T::kLoads>();
    }
    wait_loads<0>();
  }
}

__device__ __forceinline__ RowTile uniform_rows(const AttnArgs& a, int32_t i) {
  RowTile r = sequence_rows(a, i);
  r.tok0 = uniform(r.tok0);
  r.fresh = uniform(r.fresh);
  r.rows = uniform(r.rows);
  r.length = uniform(r.length);
  return r;
}

// Tiles of a step: two where a ring of two steps leaves LDS for the card's waves (step_occupancy) and the
// registers hold them.
constexpr int step_tiles(int dim, int fmt, int query_tiles) {
  return dim * (fmt == VELOGRAD_MX_E4M3 ? 64 : 32) <= 4096 && query_tiles <= 2 ? 2 : 1;
}

// Waves of a SIMD that the step kernel's registers are held to (and its LDS allows).
constexpr int step_occupancy(int dim, int fmt, int dtype, int query_tiles) {
  const bool small = fmt == VELOGRAD_MX_E2M1, plain = dtype == VELOGRAD_DTYPE_BF16;
  if (query_tiles == 4) return 1;
  if (query_tiles == 2) return dim == 64 || (dim == 128 && plain) ? 2 : 1;
  return dim < 256 || (small && dtype != VELOGRAD_DTYPE_F32) ? 2 : 1;
}

// A wave takes its share of a head's steps: whole items, and at either end a piece of one.  Bound by HBM: e2m1, bf16, 8
// kv heads of 128 dims, 2 sequences of 131072 keys 56.7 us = 5.0 TB/s of codes and scales (a kernel that only reads
// them so 47.6), 64 sequences of 300 to 12001 76.6 us = 5.6 TB/s.  Loads straight into registers, a tile ahead, took 71
// and 95; scales read past the caches 57 and 80.
template <int D, int FMT, int DT, int NQ>
__global__ __launch_bounds__(kWaves * 64, step_occupancy(D, FMT, DT, NQ)) void mx_attention_step_kernel(const AttnArgs a) {
  using S = Shape<D, FMT, DT>;
  constexpr int kTileRows = kRows * NQ;
  constexpr int kStages = 2, kTiles = step_tiles(D, FMT, NQ);
  __shared__ __attribute__((aligned(16))) uint8_t rings[kWaves][kStages * kTiles * Stage<D, FMT>::kBytes];
  const int32_t wave = uniform((int)threadIdx.x >> 6), worker = (int32_t)blockIdx.x * kWaves + wave;
  const int32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  uint8_t* ring = rings[wave];

  const Share share = find_share(a, kTileRows, worker);
  const int32_t h = worker % a.kv_heads;
  int32_t at = share.sequence, tile = share.tile, step = share.step, left = share.steps;
  RowTile r = share.rows;
  while (left > 0) {
    if (tile >= row_tiles(a, r, kTileRows)) {
      r = uniform_rows(a, ++at);
      tile = step = 0;
      continue;
    }
    r.row0 = tile * kTileRows;
    const int32_t all = item_steps(a, r.length);
    const int32_t take = all - step < left ? all - step : left;
    const int32_t last = (r.row0 + kTileRows < r.rows ? r.row0 + kTileRows : r.rows) - 1;
    const int32_t most = row_limit(a, r, last / a.group);      // keys that the tile's last row sees,
    const int32_t clear = row_limit(a, r, r.row0 / a.group);   // and that all its rows see
    const int32_t from = step > a.begin_steps ? (step - a.begin_steps) * kTile : 0;
    const int32_t till = step + take > a.begin_steps ? (step + take - a.begin_steps) * kTile : 0;
    const int32_t end = till < most ? till : most;
    QueryRows<D, FMT, DT, NQ> rows;
    begin_rows<S::kChunkElems>(a, r, h, rows);
    attend<D, FMT, DT, NQ, S::kPParts, kTiles, kStages>(a, r, h, from, end, clear, most, rows, ring);

    const bool whole = take == all;
    const int64_t part = ((int64_t)worker * 2 + (step > 0 ? 0 : 1)) * kTileRows;
    const int32_t pieces = 1 + (all - take + share.each - 1) / share.each;  // of the item, from its first piece
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      rows.state[q].l = across_g(rows.state[q].l, true);
      if (!rows.ok[q]) continue;
      if (whole)
        store_row<D, DT>(a, rows.state[q], rows.orow[q], g);
      else
        store_part<D>(a, rows.state[q], part + kRows * q + n, g);
      if (step == 0 && g == 0) {
        a.joins[rows.orow[q] * 2] = worker;
        a.joins[rows.orow[q] * 2 + 1] = pieces << 8 | (kRows * q + n);
      }
    }
    left -= take;
    step = 0;
    ++tile;
  }
}

// Row tile `tile` of a grid that has room for every sequence's last, short tile: tiles of sequence i begin at
// floor(row bound / tile rows) + i.  False where there is none.
__device__ __forceinline__ bool find_tile(const AttnArgs& a, int32_t tile, int32_t tile_rows, RowTile& r) {
  if (a.starts == nullptr) {
    const int32_t per = (a.group + tile_rows - 1) / tile_rows;
    r = uniform_rows(a, tile / per);
    r.row0 = tile % per * tile_rows;
    return true;
  }
  const int32_t lane = threadIdx.x & 63;
  int32_t i = -1;
  for (int32_t i0 = 0; i0 < sequences(a); i0 += 64) {
    const bool below = i0 + lane < sequences(a) && row_bound(a, i0 + lane) * a.group / tile_rows + i0 + lane <= tile;
    i += __popcll(__ballot(below));
  }
  i = uniform(i);
  r = uniform_rows(a, i);
  r.row0 = (tile - (r.tok0 * a.group / tile_rows + i)) * tile_rows;
  return r.row0 >= 0 && r.row0 < r.rows;
}

// ------------------------------------------------------------------------------------------
// Few rows and short sequences: one launch.
// ------------------------------------------------------------------------------------------
// A workgroup takes 16 query rows of one kv head and all their keys, its waves a run of them each, and adds up
// through LDS: where the card has room for all of them, and the keys are few, that saves the joining launch.
constexpr int item_waves(int dim, int fmt) { return dim == 256 && fmt == VELOGRAD_MX_E4M3 ? 4 : 8; }

template <int D, int FMT, int DT>
__global__ __launch_bounds__(item_waves(D, FMT) * 64) void mx_attention_item_kernel(const AttnArgs a) {
  using S = Shape<D, FMT, DT>;
  constexpr int kAll = item_waves(D, FMT), kTiles = step_tiles(D, FMT, 1), kStages = 2;
  constexpr int kRing = kStages * kTiles * Stage<D, FMT>::kBytes, kSums = D / 4 + 2;
  static_assert(kAll / 2 * kSums * 256 <= kAll * kRing, "the sums reuse the rings");
  __shared__ __attribute__((aligned(16))) uint8_t rings[kAll * kRing];
  const int32_t wave = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4;
  const int32_t h = (int32_t)(blockIdx.x % (uint32_t)a.kv_heads);
  RowTile r;
  if (!find_tile(a, (int32_t)(blockIdx.x / (uint32_t)a.kv_heads), kRows, r)) return;
  const int32_t last = (r.row0 + kRows < r.rows ? r.row0 + kRows : r.rows) - 1;
  const int32_t most = row_limit(a, r, last / a.group), clear = row_limit(a, r, r.row0 / a.group);
  const int32_t steps = (most + kTile - 1) / kTile;
  const int32_t from = steps * wave / kAll * kTile, till = steps * (wave + 1) / kAll * kTile;
  QueryRows<D, FMT, DT, 1> rows;
  begin_rows<S::kChunkElems>(a, r, h, rows);
  attend<D, FMT, DT, 1, S::kPParts, kTiles, kStages>(a, r, h, from, till < most ? till : most, clear, most, rows,
                                                     rings + wave * kRing);
  // The upper half of the waves hands its sums to the lower, in the accumulators' own layout, until one is left.
  RowState<D>& mine = rows.state[0];
  float* buf = reinterpret_cast<float*>(rings);
#pragma unroll
  for (int w = kAll / 2; w >= 1; w >>= 1) {
    __syncthreads();
    if (wave >= w && wave < 2 * w) {
      float* to = buf + (wave - w) * kSums * 64 + lane;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) to[(4 * j + i) * 64] = mine.acc[j][i];
      to[D / 4 * 64] = mine.m;
      to[(D / 4 + 1) * 64] = mine.l;
    }
    __syncthreads();
    if (wave < w) {
      const float* at = buf + wave * kSums * 64 + lane;
      const float mo = at[D / 4 * 64], next = __builtin_fmaxf(mine.m, mo);
      const float f = __builtin_amdgcn_exp2f(mine.m - next), fo = __builtin_amdgcn_exp2f(mo - next);
      mine.m = next;
      mine.l = mine.l * f + at[(D / 4 + 1) * 64] * fo;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine.acc[j][i] = mine.acc[j][i] * f + at[(4 * j + i) * 64] * fo;
    }
  }
  if (wave != 0) return;
  mine.l = across_g(mine.l, true);
  if (rows.ok[0]) store_row<D, DT>(a, mine, rows.orow[0], g);
}

// ------------------------------------------------------------------------------------------
// Many rows a sequence: prefill chunks.
// ------------------------------------------------------------------------------------------
// A workgroup takes 128 NQ consecutive rows of one kv head over all the keys they see, a wave 16 NQ of them.  All
// waves decode a step's keys together, a thread 16 elements of a key and 4 dims of 4 values, into LDS in the order
// of the products' operands; each step's codes are loaded a step before they are decoded, so one barrier a step is
// left.  Bound by instructions: matrix products and vector work (an exponential for each score, the decoding, the
// operands' way out of LDS) add up more than they overlap on a SIMD.  4096 new tokens of 16383, 32 heads of 128 dims,
// bf16: 830 us a pass = 1.16 PFLOP/s; in a kernel trace 1022 us, where decoding in every wave for itself (64 rows a wave,
// one wave a SIMD) took 1112, a maximum taken in every step 1103 for 1086, waves half a step apart 1083 and 4 waves of 64
// rows 1462.  The row tiles of one head go to one XCD where the heads divide so.  Later tiles see more keys and go first.
constexpr int kChunkWaves = 8;

// The codes of a thread's keys and values of one step.
template <int D, int FMT>
struct ChunkCodes {
  static constexpr int kWordsK = FMT == VELOGRAD_MX_E2M1 ? 2 : 4;
  uint32_t kw[kWordsK], vw[4], ks, vs;
  bool bad;  // the keys' page is not in the cache
};

template <int D, int FMT>
struct ChunkPlace {
  static constexpr int kKeys = 16 * kChunkWaves * 64 / D;  // of a step
  static constexpr int kLanes = D / 4;                     // threads of 4 keys
  int32_t quad, c;      // first of the 4 keys in the step; dims 4 c .. of the values
  int32_t key, chunk;   // its key and the 16 elements of it
  int32_t h;
};

template <int D, int FMT>
__device__ __forceinline__ void load_codes(const AttnArgs& a, const ChunkPlace<D, FMT>& w, int32_t page, int32_t t0,
                                           ChunkCodes<D, FMT>& t) {
  constexpr int kRowBytes = FMT == VELOGRAD_MX_E2M1 ? D / 2 : D;
  t.bad = (uint32_t)page >= (uint32_t)a.pages;
  const int64_t base = (int64_t)(t.bad ? 0 : page) * a.kv_heads + w.h;
  const int32_t place = (t0 + w.quad) & ((1 << a.page_shift) - 1);
  const int64_t code = ((base << a.page_shift) + place) * kRowBytes;
  const int64_t scale = ((base * (D / 32)) << a.page_shift) + place;
  const uint8_t* kc = a.kc + code + (w.key - w.quad) * kRowBytes + w.chunk * (16 * kRowBytes / D);
  const uint8_t* vc = a.vc + code + w.c * (4 * kRowBytes / D);
  if constexpr (FMT == VELOGRAD_MX_E2M1) {
    const u32x2 k = *reinterpret_cast<const u32x2*>(kc);
    t.kw[0] = k[0];
    t.kw[1] = k[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) t.vw[i] = *reinterpret_cast<const uint16_t*>(vc + i * kRowBytes);
  } else {
    const u32x4 k = *reinterpret_cast<const u32x4*>(kc);
#pragma unroll
    for (int i = 0; i < 4; ++i) t.kw[i] = k[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) t.vw[i] = *reinterpret_cast<const uint32_t*>(vc + i * kRowBytes);
  }
  t.ks = a.ks[scale + ((int64_t)(w.chunk / 2) << a.page_shift) + (w.key - w.quad)];
  t.vs = *reinterpret_cast<const uint32_t*>(a.vs + scale + ((int64_t)(w.c / 8) << a.page_shift));
}

// Of a step's keys in LDS: the operands of S^T and of O^T, and for each 16 keys whether their page is missing.
template <int D>
struct ChunkStage {
  static constexpr int kKeys = 16 * kChunkWaves * 64 / D, kTiles = kKeys / kTile;
  u32x4 k[kTiles][2][D / 32][64];
  u32x4 v[kTiles][D / 16][64];
  uint8_t gone[16];
};

// Keys from `end` on, and those of missing pages, are decoded to zeros.
template <int D, int FMT>
__device__ __forceinline__ void put_codes(const ChunkPlace<D, FMT>& w, ChunkCodes<D, FMT>& t, int32_t t0, int32_t end,
                                          ChunkStage<D>& st) {
  constexpr int kOut = D / 16, kPerWord = FMT == VELOGRAD_MX_E2M1 ? 4 : 2;
  if (t0 + ChunkStage<D>::kKeys > end || __ballot(t.bad) != 0) {
    const int32_t here = t.bad ? 0 : end - t0;
    if (w.key >= here) {
#pragma unroll
      for (int i = 0; i < ChunkCodes<D, FMT>::kWordsK; ++i) t.kw[i] = 0;
      t.ks = 127;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = 0xffu << (8 * i);
      if (w.quad + i >= here) {
        t.vw[i] = 0;
        t.vs = (t.vs & ~m) | (0x7f7f7f7fu & m);
      }
    }
  }
  if (w.c == 0 && w.quad % kHalf == 0) st.gone[w.quad / kHalf] = t.bad ? 1 : 0;
  const float ks = scale_arg(t.ks);
  u32x4 e[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i / 4][i % 4] = decode_pair<FMT>(t.kw[i / kPerWord], ks, i % kPerWord);
  // Lane (n, g) of step s reads column n ^ (4 s + (g & 2)): threads of one key would write to the same banks.
  u32x4* k = st.k[w.key / kTile][w.key / kHalf % 2][w.chunk / 2];
  const int32_t g = w.chunk % 2 * 2, n = (w.key % kHalf) ^ (w.chunk * 2 & 15);
  k[16 * g + n] = e[0];
  k[16 * g + 16 + n] = e[1];
  u32x2 x[4];  // 4 dims of 4 keys: pairs of keys
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float s0 = __builtin_bit_cast(float, i == 0 ? t.vs << 23 : t.vs << 7);
    const float s1 = __builtin_bit_cast(float, i == 0 ? t.vs << 15 : t.vs >> 1);
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const uint32_t u0 = decode_pair<FMT>(t.vw[2 * i], s0, d), u1 = decode_pair<FMT>(t.vw[2 * i + 1], s1, d);
      x[2 * d][i] = __builtin_amdgcn_perm(u1, u0, 0x05040100u);
      x[2 * d + 1][i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
    }
  }
  const int32_t lane = 16 * (w.quad / 4 % 4) + 4 * w.c / kOut, half = w.quad / kHalf % 2;
#pragma unroll
  for (int d = 0; d < 4; ++d)
    reinterpret_cast<u32x2*>(&st.v[w.quad / kTile][4 * w.c % kOut + d][lane])[half] = x[d];
}

// A barrier for what lies in LDS: loads into registers stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int D, int FMT, int DT, int NQ>
__global__ __launch_bounds__(kChunkWaves * 64, 2) void mx_attention_chunk_kernel(const AttnArgs a) {
  using S = Shape<D, FMT, DT>;
  using T = ChunkStage<D>;
  constexpr int kTileRows = kRows * NQ, kGroupRows = kChunkWaves * kTileRows, kOut = D / 16;
  constexpr int kGroup = T::kTiles < 2 ? T::kTiles : 2;  // tiles whose scores are held at a time
  constexpr int kParts = chunk_parts(DT);
  __shared__ T stages[2];
  const int32_t tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4, wave = uniform(tid >> 6);
  ChunkPlace<D, FMT> w;
  w.h = (int32_t)(blockIdx.x % (uint32_t)a.kv_heads);
  w.quad = tid / w.kLanes * 4;
  w.c = tid % w.kLanes;
  w.key = w.quad + w.c / kOut;
  w.chunk = w.c % kOut;
  const int32_t item = (int32_t)((gridDim.x - 1 - blockIdx.x) / (uint32_t)a.kv_heads);
  RowTile r;
  if (!find_tile(a, item, kGroupRows, r) || r.seq < 0 || r.rows <= a.step_rows) return;
  const int32_t group_last = (r.row0 + kGroupRows < r.rows ? r.row0 + kGroupRows : r.rows) - 1;
  const int32_t end = row_limit(a, r, group_last / a.group);  // keys that any row of the group sees
  r.row0 += wave * kTileRows;
  int32_t most = 0, clear = 0;  // of the wave's rows: the last sees, all see
  if (r.row0 < r.rows) {
    const int32_t last = (r.row0 + kTileRows < r.rows ? r.row0 + kTileRows : r.rows) - 1;
    most = row_limit(a, r, last / a.group);
    clear = row_limit(a, r, r.row0 / a.group);
  }
  QueryRows<D, FMT, DT, NQ> rows;
  begin_rows<8>(a, r, w.h, rows);

  const int32_t* table = a.table + (int64_t)r.seq * a.table_stride;
  auto find_page = [&](int32_t t0) {
    const int32_t at = (t0 + w.quad) >> a.page_shift;
    return table[at < a.width ? at : a.width - 1];
  };
  auto use = [&](const T& st, int32_t t0, int32_t j0, uint32_t gone, auto masked_step) {
    constexpr bool kMasked = decltype(masked_step)::value;
    // Operands are read from LDS in batches of 4, each while the products of the one before run.
    constexpr int kBatchesK = kGroup * S::kSteps / 2, kBatchesV = kGroup * kOut / 4;
    u32x4 kf[2][2][2], vf[2][4];
    auto read_keys = [&](int b) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int s = b % (S::kSteps / 2) * 2 + i;
          kf[b & 1][i][u] = st.k[j0 + b / (S::kSteps / 2)][u][s][16 * g + (n ^ ((4 * s + (g & 2)) & 15))];
        }
    };
    auto read_values = [&](int b) {
#pragma unroll
      for (int i = 0; i < 4; ++i) vf[b & 1][i] = st.v[j0 + b / (kOut / 4)][b % (kOut / 4) * 4 + i][lane];
    };
    float x[NQ][8 * kGroup];
    f32x4 sc[NQ][2];
    read_keys(0);
#pragma unroll
    for (int b = 0; b < kBatchesK; ++b) {
      const int s0 = b % (S::kSteps / 2) * 2, j = b / (S::kSteps / 2);
      if (b + 1 < kBatchesK) read_keys(b + 1);
      else read_values(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int p = S::kQParts - 1; p >= 0; --p)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int q = 0; q < NQ; ++q)
              sc[q][u] = mfma(kf[b & 1][i][u], rows.frag[q][s0 + i][p],
                              s0 + i == 0 && p == S::kQParts - 1 ? f32x4{0, 0, 0, 0} : sc[q][u]);
      if (s0 + 2 == S::kSteps)
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[q][8 * j + i] = sc[q][i / 4][i % 4];
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kMasked) {
#pragma unroll
      for (int u = 0; u < 2 * kGroup; ++u)
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const int32_t see = (gone >> 8 * u & 1u) != 0 ? 0 : rows.limit[q] - (t0 + kHalf * u + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[q][4 * u + i] = i < see ? x[q][4 * u + i] : -__builtin_inff();
        }
    }
    // Probabilities by the running maximum as it is: it has to move only where their sum passes 2^8, which a maximum
    // behind by 8 brings about by itself, so that no maximum is taken in most steps.
    float p[NQ][8 * kGroup], l[NQ];
    bool moves = false;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      l[q] = probabilities<8 * kGroup>(x[q], p[q], a.scale_log2, rows.state[q].m);
      moves |= l[q] > 256.0f;
    }
    if (__ballot(moves) != 0) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const float top = across_g(largest<8 * kGroup>(x[q]) * a.scale_log2, false);
        const bool own = across_g(l[q], false) > 256.0f;  // each row by itself: its bits do not depend on others'
        set_max<D>(own ? __builtin_fmaxf(top, rows.state[q].m) : rows.state[q].m, rows.state[q]);
        l[q] = probabilities<8 * kGroup>(x[q], p[q], a.scale_log2, rows.state[q].m);
      }
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q) rows.state[q].l += l[q];
    u32x4 pf[NQ][kParts];
#pragma unroll
    for (int b = 0; b < kBatchesV; ++b) {
      const int j = b / (kOut / 4);
      if (b + 1 < kBatchesV) read_values(b + 1);
      if (b % (kOut / 4) == 0)
#pragma unroll
        for (int q = 0; q < NQ; ++q) split_probs<kParts>(p[q] + 8 * j, pf[q]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kMasked) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // A NaN among the values that only some of the rows see would reach the others as 0 * NaN: it is taken
          // out, and the rows that do see it get NaN by a product of flags.
          const int d = b % (kOut / 4) * 4 + e;
          u32x4& v = vf[b & 1][e];
          u32x4 flags;
          uint32_t any = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool low = (v[i] & 0x7fffu) > 0x7f80u, high = (v[i] & 0x7fffffffu) > 0x7f80ffffu;
            flags[i] = (low ? 0x3f80u : 0u) | (high ? 0x3f800000u : 0u);
            v[i] &= (low ? 0u : 0xffffu) | (high ? 0u : 0xffff0000u);
            any |= flags[i];
          }
          if (__ballot(any != 0) == 0) continue;
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            u32x4 seen;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int u = 2 * j + i / 2;
              const int32_t see =
                  (gone >> 8 * u & 1u) != 0 ? 0 : rows.limit[q] - (t0 + kHalf * u + 4 * g + 2 * (i & 1));
              seen[i] = (see > 0 ? 0x3f80u : 0u) | (see > 1 ? 0x3f800000u : 0u);
            }
            const f32x4 hit = mfma(flags, seen, f32x4{0, 0, 0, 0});
#pragma unroll
            for (int i = 0; i < 4; ++i)
              rows.state[q].acc[d][i] = hit[i] > 0.0f ? __builtin_nanf("") : rows.state[q].acc[d][i];
          }
        }
      }
#pragma unroll
      for (int i = kParts - 1; i >= 0; --i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            f32x4& acc = rows.state[q].acc[b % (kOut / 4) * 4 + e];
            acc = mfma(vf[b & 1][e], pf[q][i], acc);
          }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  ChunkCodes<D, FMT> codes;
  if (end > 0) {
    load_codes<D, FMT>(a, w, find_page(0), 0, codes);
    put_codes<D, FMT>(w, codes, 0, end, stages[0]);
    load_codes<D, FMT>(a, w, find_page(T::kKeys), T::kKeys, codes);
  }
  int32_t page = end > 0 ? find_page(2 * T::kKeys) : 0;
  int32_t t = 0, at = 0;
  // A step begins: its keys lie in LDS, those of the one before may be overwritten.  Whether pages are missing
  // (for each 16 keys a byte of `gone`).
  constexpr int kWords = (2 * T::kTiles + 3) / 4;
  constexpr uint32_t kEvery = T::kTiles == 1 ? 0xffffu : 0xffffffffu;
  uint32_t gone[kWords];
  auto begin_step = [&]() {
    lds_barrier();
    // Past the end the loads go on over the table's last page; nothing uses them.
    put_codes<D, FMT>(w, codes, t + T::kKeys, end, stages[at ^ 1]);
    load_codes<D, FMT>(a, w, page, t + 2 * T::kKeys, codes);
    page = find_page(t + 3 * T::kKeys);
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      gone[i] = (uint32_t)uniform(*reinterpret_cast<const int32_t*>(stages[at].gone + 4 * i)) & kEvery;
    return kWords == 2 ? (gone[0] | gone[1]) != 0 : gone[0] != 0;
  };
  // All rows see all keys of the first steps.  The rest, and all from a missing page on, is masked.  Every wave
  // begins one step more than there are, whichever loop ends its walk.
  bool any_gone = end > 0 && begin_step();
  while (t + T::kKeys <= clear && !any_gone) {
#pragma unroll
    for (int j = 0; j < T::kTiles; j += kGroup) use(stages[at], t + j * kTile, j, 0, std::false_type{});
    t += T::kKeys;
    at ^= 1;
    any_gone = begin_step();
  }
  while (t < end) {
#pragma unroll
    for (int j = 0; j < T::kTiles; j += kGroup)
      if (t + j * kTile < most) use(stages[at], t + j * kTile, j, gone[j / 2], std::true_type{});
    t += T::kKeys;
    at ^= 1;
    begin_step();
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    rows.state[q].l = across_g(rows.state[q].l, true);
    if (!rows.ok[q]) continue;
    store_row<D, DT>(a, rows.state[q], rows.orow[q], g);
    if (a.joins != nullptr && g == 0) a.joins[rows.orow[q] * 2 + 1] = 1 << 8;
  }
}

// Joins the pieces of the (token, head) rows that have several: a row's first is the last of its wave's share,
// the others are the first of the shares that follow in the head.  D/4 lanes hold the row, the workgroup's
// other lanes take other pieces, and LDS adds them up.  A workgroup's rows lie a grid apart, so that a sequence's rows,
// split or not split together, go to many workgroups.
constexpr int kMostPieces = 2048;

template <int D, int DT>
__global__ __launch_bounds__(256) void mx_attention_join_kernel(const AttnArgs a, int32_t tile_rows, int32_t rows) {
  constexpr int kLanes = D / 4, kSets = 256 / kLanes;
  __shared__ float weight[kMostPieces + 1];
  __shared__ float sums[kSets][D];
  __shared__ float wave_top[4], wave_sum[4];
  __shared__ int32_t found[256];
  __shared__ int32_t count;
  const int32_t tid = threadIdx.x, d = tid % kLanes, set = tid / kLanes;
  const int64_t all = (int64_t)a.q_tokens * a.q_heads;
  if (tid == 0) count = 0;
  __syncthreads();
  const int64_t mine = blockIdx.x + (int64_t)tid * gridDim.x;
  if (tid < rows && mine < all && (a.joins[mine * 2 + 1] >> 8) > 1) found[atomicAdd(&count, 1)] = tid;
  __syncthreads();
  for (int32_t k = 0; k < count; ++k) {
    const int64_t orow = blockIdx.x + (int64_t)found[k] * gridDim.x;
    // In bounds whatever rows that no kernel took left there (falls).
    const int32_t packed = a.joins[orow * 2 + 1];
    int32_t first = a.joins[orow * 2], in_tile = packed & 0xff;
    first = first < 0 ? 0 : first < a.workers ? first : a.workers - 1;
    in_tile = in_tile < tile_rows ? in_tile : tile_rows - 1;
    const int32_t most = (a.workers - 1 - first) / a.kv_heads + 1, active = packed >> 8 < most ? packed >> 8 : most;
    auto place = [&](int32_t s) {
      return ((int64_t)(first + s * a.kv_heads) * 2 + (s == 0 ? 1 : 0)) * tile_rows + in_tile;
    };
    float m = -3.0e38f;
    for (int32_t s = tid; s < active; s += 256) m = __builtin_fmaxf(m, a.part_ml[place(s) * 2]);
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) m = __builtin_fmaxf(m, __shfl_xor(m, w));
    if ((tid & 63) == 0) wave_top[tid >> 6] = m;
    __syncthreads();
    m = __builtin_fmaxf(__builtin_fmaxf(wave_top[0], wave_top[1]), __builtin_fmaxf(wave_top[2], wave_top[3]));
    float l = 0.0f;
    for (int32_t s = tid; s < active; s += 256) {
      const float f = __builtin_amdgcn_exp2f(a.part_ml[place(s) * 2] - m);
      weight[s] = f;
      l += a.part_ml[place(s) * 2 + 1] * f;
    }
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) l += __shfl_xor(l, w);
    if ((tid & 63) == 0) wave_sum[tid >> 6] = l;
    __syncthreads();
    l = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
    f32x4 o = {0, 0, 0, 0};
#pragma unroll 4
    for (int32_t s = set; s < active; s += kSets)
      o += *reinterpret_cast<const f32x4*>(a.part_o + place(s) * D + 4 * d) * weight[s];
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[set][4 * d + i] = o[i];
    __syncthreads();
    if (tid < D) {
      float x = 0.0f;
#pragma unroll
      for (int i = 0; i < kSets; ++i) x += sums[i][tid];
      const bool empty = l == 0.0f;
      Codec<DT>::store1(a.out, orow * D + tid, empty ? 0.0f : x / l);
      if (a.lse != nullptr && tid == 0)
        a.lse[orow] = empty ? -__builtin_inff() : (m + log2f(l)) * 0.693147180559945309f;
    }
    __syncthreads();
  }
}

// How a call is laid out.
struct AttnPlan {
  int32_t query_tiles;  // of a wave of the step kernel: 1, 2 or 4
  int32_t workers;      // its waves
  int32_t least_steps, begin_steps;
  int32_t step_rows;    // sequences of more rows go to the chunk kernel
  int64_t chunk_tiles;  // its workgroups for each kv head; 0: not launched
  int64_t items;        // workgroups of the item kernel, which then runs alone; or 0
};

AttnPlan plan_attention(int64_t q_tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                        int32_t fmt, int32_t dtype, bool ragged, int64_t table_keys, int cus) {
  AttnPlan p;
  const int64_t group = q_heads / kv_heads, tiles = most_tiles((int)head_dim, dtype);
  const int64_t chunk_rows = kChunkWaves * kRows * chunk_tiles((int)head_dim, dtype);
  p.chunk_tiles = 0;
  p.step_rows = INT32_MAX;
  // Chunks where their workgroups fill much of the card; the step kernel splits the keys where they do not, but decodes
  // them for every wave.  32 heads of 128 dims, e2m1, new tokens of all, chunk and step kernel: bf16 512 of 8000 (a
  // quarter of the card) 234 and 162 us, 1024 of 8000 (half) 235 and 262, 4 x 256 of 4000 129 and 168, 1536 of 8000 236
  // and 392; fp16 1024 of 8000 354 and 264, 1536 of 8000 356 and 429; fp32 512 of 8000 (half) 281 and 216, 1024 of 8000
  // 291 and 345.
  const int64_t quarters = dtype == VELOGRAD_DTYPE_BF16 && chunk_tiles((int)head_dim, dtype) == 2 ? 2 : 3;
  if (ragged && q_tokens * q_heads * 4 >= quarters * chunk_rows * cus) {
    p.chunk_tiles = q_tokens * group / chunk_rows + batch + 2;
    p.step_rows = kRows * 4;
  }
  // Rows of a sequence, on average.
  const int64_t rows = ragged ? q_tokens * group / (batch > 0 ? batch : 1) : group;
  p.query_tiles = p.chunk_tiles > 0 || rows <= kRows || tiles < 2 ? 1 : rows <= 2 * kRows || tiles < 4 ? 2 : 4;
  // As many waves as the card holds at once: every one runs from the start, with an equal share.
  p.workers = cus * step_occupancy((int)head_dim, fmt, dtype, p.query_tiles) * kWaves;
  if (p.workers > kMostPieces) p.workers = kMostPieces;
  // At least one share for each head.
  if (p.workers < kv_heads) p.workers = (int32_t)((kv_heads + kWaves - 1) / kWaves * kWaves);
  p.least_steps = kLeastSteps;
  p.begin_steps = kBeginSteps;
  // One launch, where the card takes all items in few turns and a wave's run of the keys is short: the second launch
  // costs 4 us, a run of 128 keys of 128 dims as much.  With more items the split's shares grow as well, and with several
  // row tiles a sequence so do its pieces.  One sequence, 8 kv heads: 500 keys 11.0 us split and 8.1 in one launch,
  // 1000 11.6 and 10.7, 2000 11.5 and 14.8; 16 sequences: 500 keys 14.7 and 8.9, 2000 20.1 and 15.6; 64: 2000 37.8 and
  // 35.1; 128: 1000 43.9 and 47.7.  Rows of 36 tokens of 8 sequences of 1348 keys 53.8 and 38.8, of 128 tokens of 2 of
  // 6000 78.9 and 63.2; 8 tokens of 32 of 2000, 2 kv heads of 256 e4m3 dims, 71.7 and 77.9.
  const bool wide = rows > kRows;
  const int64_t items = (ragged ? q_tokens * group / kRows + batch + 2 : batch * ((group + kRows - 1) / kRows)) * kv_heads;
  const int64_t wave_keys = 128 + (wide ? 2 * items : items < cus ? items : cus);
  const bool short_runs = table_keys * head_dim <= item_waves((int)head_dim, fmt) * 128 * wave_keys;
  p.items = p.chunk_tiles == 0 && items <= (wide ? 4 : 2) * cus && short_runs ? items : 0;
  return p;
}

size_t workspace_bytes(const AttnPlan& p, int64_t q_tokens, int64_t q_heads, int64_t head_dim) {
  if (p.items > 0) return 0;
  return (size_t)p.workers * 2 * kRows * (size_t)p.query_tiles * (size_t)(head_dim + 2) * sizeof(float) +
         (size_t)q_tokens * (size_t)q_heads * 2 * sizeof(int32_t);
}

template <int D, int FMT, int DT>
void launch_attention(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
  constexpr int kMost = most_tiles(D, DT);
  const dim3 block(kWaves * 64), steps((uint32_t)p.workers / kWaves);
  if (p.items > 0) {
    hipLaunchKernelGGL((mx_attention_item_kernel<D, FMT, DT>), dim3((uint32_t)p.items), dim3(item_waves(D, FMT) * 64), 0, st, a);
    return;
  }
  if (p.chunk_tiles > 0)
    hipLaunchKernelGGL((mx_attention_chunk_kernel<D, FMT, DT, chunk_tiles(D, DT)>),
                       dim3((uint32_t)(p.chunk_tiles * a.kv_heads)), dim3(kChunkWaves * 64), 0, st, a);
  if (p.query_tiles == 4) {
    if constexpr (kMost >= 4) hipLaunchKernelGGL((mx_attention_step_kernel<D, FMT, DT, 4>), steps, block, 0, st, a);
  } else if (p.query_tiles == 2) {
    if constexpr (kMost >= 2) hipLaunchKernelGGL((mx_attention_step_kernel<D, FMT, DT, 2>), steps, block, 0, st, a);
  } else {
    hipLaunchKernelGGL((mx_attention_step_kernel<D, FMT, DT, 1>), steps, block, 0, st, a);
  }
  const int64_t all = (int64_t)a.q_tokens * a.q_heads;
  // Of 288 tokens of 32 heads all rows are joined: 53.8 us a call at one row a workgroup, 68.7 at 16.  Of 6216 of 32, a
  // hundredth: 5.8 us in the join at 64, 7.6 at 16.
  const int64_t rows = all <= 16384 ? 1 : all <= 65536 ? 4 : all <= 262144 ? 64 : 256;
  hipLaunchKernelGGL((mx_attention_join_kernel<D, DT>), dim3((uint32_t)((all + rows - 1) / rows)), dim3(256), 0, st,
                     a, kRows * p.query_tiles, (int32_t)rows);
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

VELOGRAD_API size_t velograd_mx_cache_attention_workspace_bytes(
    int64_t q_tokens, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
    int64_t table_width, int64_t page_size, int32_t ragged, int32_t dtype, int32_t mx_format, int32_t device) {
  const char* what = "velograd_mx_cache_attention_workspace_bytes";
  if (elem_bytes_of(dtype) == 0 || check_mx_cache(what, kv_heads, head_dim, 0, page_size, mx_format) != 0 ||
      check_attention(what, q_tokens, sequences, q_heads, kv_heads, head_dim, table_width, page_size,
                      ragged != 0) != 0)
    return 0;
  const int cus = cu_count(device);
  if (cus <= 0 || q_tokens == 0) return 0;
  const AttnPlan p = plan_attention(q_tokens, sequences, q_heads, kv_heads, head_dim, mx_format,
                                    dtype, ragged != 0, table_width * page_size, cus);
  return workspace_bytes(p, q_tokens, q_heads, head_dim);
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
  const AttnPlan p = plan_attention(q_tokens, sequences, q_heads, kv_heads, head_dim, mx_format, dtype, ragged,
                                    table_width * page_size, cus);
  // The waves count steps in 32 bits: those of the sequences that the step kernel takes.
  const int64_t step_tiles = p.chunk_tiles > 0 ? sequences * ((p.step_rows + kRows - 1) / kRows)
                                               : q_tokens * (q_heads / kv_heads) / kRows + sequences;
  const int64_t most_steps = table_width * page_size / kTile + 1 + p.begin_steps;
  if (step_tiles + q_tokens * (q_heads / kv_heads) / kRows + 2 > INT32_MAX / most_steps)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: %lld tokens over %lld pages are too many", what,
                (long long)q_tokens, (long long)table_width);
  if (p.chunk_tiles > INT32_MAX / kv_heads)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: %lld row tiles exceed the grid limit", what,
                (long long)p.chunk_tiles);
  const size_t need = workspace_bytes(p, q_tokens, q_heads, head_dim);
  if (need > 0 && (workspace == nullptr || ws_bytes < need))
    return fail(VELOGRAD_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, need);
  if (!aligned16(workspace))
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);

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
  const size_t part_rows = (size_t)p.workers * 2 * kRows * (size_t)p.query_tiles;
  a.part_ml = a.part_o + part_rows * (size_t)head_dim;
  a.joins = reinterpret_cast<int32_t*>(a.part_ml + part_rows * 2);
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
  a.workers = p.workers;
  a.least_steps = p.least_steps;
  a.begin_steps = p.begin_steps;
  a.step_rows = p.step_rows;
  a.scale_log2 = scale == 0.0f ? 1.0f : (float)(__builtin_fabs((double)scale) * 1.4426950408889634074);
  a.q_factor = scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : 0.0f;
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  switch (dtype) {
    case VELOGRAD_DTYPE_F32: launch_fmt<VELOGRAD_DTYPE_F32>(a, p, head_dim, mx_format, st); break;
    case VELOGRAD_DTYPE_F16: launch_fmt<VELOGRAD_DTYPE_F16>(a, p, head_dim, mx_format, st); break;
    default: launch_fmt<VELOGRAD_DTYPE_BF16>(a, p, head_dim, mx_format, st); break;
  }
  return check_launch(what);
}

}  // extern "C"
