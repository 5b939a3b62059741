// A paged cache of keys and values in the OCP MX block formats: writing new tokens' head vectors
// into it (rotated on the way where asked), and reading tokens back.
//
// Layout (all bytes), for fmt E2M1 with R = head_dim / 2 bytes a head vector, E4M3 with R = head_dim:
//   codes   [pages, kv_heads, page_size, R]
//   scales  [pages, kv_heads, head_dim / 32, page_size]
// A token's slot is page * page_size + place.  A head's vectors of consecutive tokens are contiguous,
// so the attention reads whole lines; its scales lie token by token, so those of the 4 consecutive tokens
// that a lane takes are one word.
//
// Quantisation is the norms' MX epilogue: per 32 elements a = max|x|, s = floor(log2 a) - emax clamped
// to [-127, 127], codes RNE(x * 2^-s) saturating, scale code s + 127; a block whose maximum is not
// finite takes scale 0xFF and zero codes (it reads back as NaN).
//
// Rotation (rotate half, the pairing of velograd_rope): (x_j, x_{j + D/2}) -> (x_j c - x_{j+D/2} s,
// x_j s + x_{j+D/2} c), c and s from row `position` of a float32 table [max_positions, D] that holds
// D/2 cosines, then D/2 sines.  Every product and sum rounds to fp32, and the rotated key is rounded to
// its own type before it is quantised, so the cache holds exactly what rotating first and writing then
// would give.  A position outside the table rotates by NaN: the query row is NaN and the key's blocks
// are marked NaN.
//
// Both kernels are bound by HBM (a few operations for each element): rotating and writing 8191 tokens (bf16, e2m1, 32
// query and 8 kv heads of 128 dims) takes 38.6 us = 4.7 TB/s, reading 66000 tokens back 58.8 us = 5.8 TB/s.  Small
// calls are bound by their launches: 8 tokens 3.5 us written, 2.6 read.
#include "mx_device.h"

namespace {

using namespace vg;

constexpr int kMxBlock = 256;  // threads of a workgroup

typedef float f32x2 __attribute__((ext_vector_type(2)));

struct WriteArgs {
  const void *q, *k, *v;
  void* q_out;
  const float* cos_sin;
  const int64_t* positions;
  const int64_t* slots;
  uint8_t *kc, *ks, *vc, *vs;
  int64_t tokens;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;  // strides of tokens and heads, in elements
  int64_t max_pos;
  int64_t capacity;  // pages * page_size
  int32_t q_heads, kv_heads;
  int32_t dim;
  int32_t lane_shift;  // log2(dim / 16): lanes of one head vector
  int32_t page_shift;
};

// Eight consecutive elements as fp32, from any element.
template <int DT>
__device__ inline void load8(const void* p, int64_t e, float* f) {
  Codec<DT>::unpack(load16_any_stream<DT>(p, e), f);
  if constexpr (DT == VELOGRAD_DTYPE_F32)
    Codec<DT>::unpack(load16_any_stream<DT>(p, e + 4), f + 4);
}

// f rounded to DT and back.
template <int DT>
__device__ inline void round8(float* f) {
  if constexpr (DT != VELOGRAD_DTYPE_F32) Codec<DT>::unpack(Codec<DT>::pack(f), f);
}

template <int DT>
__device__ inline void store8(void* p, int64_t e, const float* f) {
  store16_stream<DT>(p, e, Codec<DT>::pack(f));
  if constexpr (DT == VELOGRAD_DTYPE_F32) store16_stream<DT>(p, e + 4, Codec<DT>::pack(f + 4));
}

// Codes of eight elements; the block's 32 lie in 4 neighbouring lanes.  `scale` gets the block's code.
template <int FMT>
__device__ inline u32x2 encode8(const float* f, uint32_t& scale) {
  constexpr int kEmax = FMT == VELOGRAD_MX_E4M3 ? vg_mx::kEmaxE4M3 : vg_mx::kEmaxE2M1;
  uint32_t am = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) am = umax(am, __builtin_bit_cast(uint32_t, f[i]) & 0x7fffffffu);
  am = lane_group_max<4>(am);
  const bool finite = am < 0x7f800000u;
  const float m = finite ? vg_mx::inverse_scale(vg_mx::shared_exp(am, kEmax)) : 0.0f;
  scale = vg_mx::scale_code(am, kEmax);
  u32x2 w = {0u, 0u};
  if constexpr (FMT == VELOGRAD_MX_E4M3) {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      q[i] = __builtin_fminf(__builtin_fmaxf(f[i] * m, -vg_fp8::kE4M3Max), vg_fp8::kE4M3Max);
    if (finite) {
      w[0] = e4m3x4(q[0], q[1], q[2], q[3]);
      w[1] = e4m3x4(q[4], q[5], q[6], q[7]);
    }
  } else {
    uint32_t word = 0;
    word = e2m1x2<0>(word, f[0] * m, f[1] * m);
    word = e2m1x2<1>(word, f[2] * m, f[3] * m);
    word = e2m1x2<2>(word, f[4] * m, f[5] * m);
    word = e2m1x2<3>(word, f[6] * m, f[7] * m);
    if (finite) w[0] = word;
  }
  return w;
}

// A lane owns two chunks of 8 elements of one head vector, c and c + dim / 16: the two halves of 8
// rotation pairs.  dim / 16 lanes hold a head vector, a workgroup 4096 / dim consecutive tokens of one
// head, so a workgroup's stores into one page are one contiguous run.
template <int DT, int FMT, bool ROPE>
__global__ __launch_bounds__(kMxBlock) void mx_write_kernel(const WriteArgs a) {
  const int32_t heads = (ROPE ? a.q_heads : 0) + 2 * a.kv_heads;
  const int64_t group = blockIdx.x / (uint32_t)heads;
  int32_t h = (int32_t)(blockIdx.x - (uint32_t)group * (uint32_t)heads);
  const int32_t lanes = 1 << a.lane_shift;
  const int64_t t = group * (kMxBlock >> a.lane_shift) + (threadIdx.x >> a.lane_shift);
  if (t >= a.tokens) return;
  const int32_t e = (int32_t)(threadIdx.x & (lanes - 1)) * 8;
  const int32_t half = a.dim >> 1;

  const bool is_q = ROPE && h < a.q_heads;
  if (ROPE && !is_q) h -= a.q_heads;
  const bool is_k = !is_q && h < a.kv_heads;
  if (!is_q && !is_k) h -= a.kv_heads;
  int64_t slot = 0;
  if (!is_q) {
    slot = a.slots[t];
    if (slot < 0 || slot >= a.capacity) return;
  }
  const void* src = is_q ? a.q : is_k ? a.k : a.v;
  const int64_t from = is_q ? t * a.q_t + h * a.q_h : is_k ? t * a.k_t + h * a.k_h : t * a.v_t + h * a.v_h;
  float lo[8], hi[8];
  load8<DT>(src, from + e, lo);
  load8<DT>(src, from + half + e, hi);
  if constexpr (ROPE) {
    if (is_q || is_k) {
      const int64_t pos = a.positions[t];
      const bool ok = pos >= 0 && pos < a.max_pos;
      float c[8], s[8];
      if (ok) {
        const float* row = a.cos_sin + pos * a.dim;
        Codec<VELOGRAD_DTYPE_F32>::unpack(load16_any<VELOGRAD_DTYPE_F32>(row, e), c);
        Codec<VELOGRAD_DTYPE_F32>::unpack(load16_any<VELOGRAD_DTYPE_F32>(row, e + 4), c + 4);
        Codec<VELOGRAD_DTYPE_F32>::unpack(load16_any<VELOGRAD_DTYPE_F32>(row, half + e), s);
        Codec<VELOGRAD_DTYPE_F32>::unpack(load16_any<VELOGRAD_DTYPE_F32>(row, half + e + 4), s + 4);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = s[i] = __builtin_nanf("");
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = lo[i], y = hi[i];
        lo[i] = x * c[i] - y * s[i];
        hi[i] = x * s[i] + y * c[i];
      }
      if (is_q) {
        const int64_t to = (t * a.q_heads + h) * (int64_t)a.dim;
        store8<DT>(a.q_out, to + e, lo);
        store8<DT>(a.q_out, to + half + e, hi);
        return;
      }
      round8<DT>(lo);
      round8<DT>(hi);
    }
  }
  uint32_t slo, shi;
  const u32x2 wlo = encode8<FMT>(lo, slo);
  const u32x2 whi = encode8<FMT>(hi, shi);
  const int64_t page = slot >> a.page_shift;
  const int64_t place = slot & (((int64_t)1 << a.page_shift) - 1);
  const int64_t ph = page * a.kv_heads + h;
  const int32_t row_bytes = FMT == VELOGRAD_MX_E4M3 ? a.dim : half;
  uint8_t* codes = (is_k ? a.kc : a.vc) + ((ph << a.page_shift) + place) * row_bytes;
  if constexpr (FMT == VELOGRAD_MX_E4M3) {
    *reinterpret_cast<u32x2*>(codes + e) = wlo;
    *reinterpret_cast<u32x2*>(codes + half + e) = whi;
  } else {
    *reinterpret_cast<uint32_t*>(codes + (e >> 1)) = wlo[0];
    *reinterpret_cast<uint32_t*>(codes + ((half + e) >> 1)) = whi[0];
  }
  if ((threadIdx.x & 3) == 0) {
    uint8_t* scales = (is_k ? a.ks : a.vs) + ((ph * (a.dim >> 5)) << a.page_shift) + place;
    scales[(int64_t)(e >> 5) << a.page_shift] = (uint8_t)slo;
    scales[(int64_t)((half + e) >> 5) << a.page_shift] = (uint8_t)shi;
  }
}

struct ReadArgs {
  const uint8_t *kc, *ks, *vc, *vs;
  const int64_t* slots;
  void *k, *v;
  int64_t items;     // tokens * kv_heads * dim / 8
  int64_t capacity;
  int32_t kv_heads;
  int32_t dim;
  int32_t chunk_shift;  // log2(dim / 8)
  int32_t page_shift;
};

template <int FMT>
__device__ inline void decode8(const uint8_t* p, float scale, float* f) {
  if constexpr (FMT == VELOGRAD_MX_E4M3) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
      const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
      f[4 * i] = a[0] * scale;
      f[4 * i + 1] = a[1] * scale;
      f[4 * i + 2] = b[0] * scale;
      f[4 * i + 3] = b[1] * scale;
    }
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    f[0] = a[0] * scale;
    f[1] = a[1] * scale;
    f[2] = b[0] * scale;
    f[3] = b[1] * scale;
    f[4] = c[0] * scale;
    f[5] = c[1] * scale;
    f[6] = d[0] * scale;
    f[7] = d[1] * scale;
  }
}

// 2^(code - 127) as fp32 (code 0 is the subnormal 2^-127), NaN for code 0xFF.
__device__ inline float scale_value(uint32_t code) {
  const uint32_t b = code == 0 ? 0x00400000u : code << 23;
  return code == vg_mx::kScaleNaN ? __builtin_nanf("") : __builtin_bit_cast(float, b);
}

// One thread: 8 elements of one token's head vector, of the keys and of the values.  Consecutive
// threads write consecutive outputs.
template <int DT, int FMT>
__global__ __launch_bounds__(kMxBlock) void mx_read_kernel(const ReadArgs a) {
  const int64_t i = (int64_t)blockIdx.x * kMxBlock + threadIdx.x;
  if (i >= a.items) return;
  const int64_t th = i >> a.chunk_shift;
  const int32_t c = (int32_t)(i & ((1 << a.chunk_shift) - 1));
  const int64_t t = th / a.kv_heads;
  const int32_t h = (int32_t)(th - t * a.kv_heads);
  const int64_t slot = a.slots[t];
  float kf[8], vf[8];
  if (slot >= 0 && slot < a.capacity) {
    const int64_t page = slot >> a.page_shift;
    const int64_t place = slot & (((int64_t)1 << a.page_shift) - 1);
    const int64_t ph = page * a.kv_heads + h;
    const int32_t row_bytes = FMT == VELOGRAD_MX_E4M3 ? a.dim : a.dim >> 1;
    const int64_t code = ((ph << a.page_shift) + place) * row_bytes +
                         (FMT == VELOGRAD_MX_E4M3 ? c * 8 : c * 4);
    const int64_t scale = ((ph * (a.dim >> 5) + (c >> 2)) << a.page_shift) + place;
    decode8<FMT>(a.kc + code, scale_value(a.ks[scale]), kf);
    decode8<FMT>(a.vc + code, scale_value(a.vs[scale]), vf);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) kf[j] = vf[j] = 0.0f;
  }
  store8<DT>(a.k, i * 8, kf);
  store8<DT>(a.v, i * 8, vf);
}

int log2_exact(int64_t v) {
  int s = 0;
  while (((int64_t)1 << s) < v) ++s;
  return s;
}

template <int DT, int FMT>
void launch_write(const WriteArgs& a, uint32_t blocks, bool rope, hipStream_t st) {
  if (rope)
    hipLaunchKernelGGL((mx_write_kernel<DT, FMT, true>), dim3(blocks), dim3(kMxBlock), 0, st, a);
  else
    hipLaunchKernelGGL((mx_write_kernel<DT, FMT, false>), dim3(blocks), dim3(kMxBlock), 0, st, a);
}

template <int DT>
void launch_write_fmt(const WriteArgs& a, int fmt, uint32_t blocks, bool rope, hipStream_t st) {
  if (fmt == VELOGRAD_MX_E4M3)
    launch_write<DT, VELOGRAD_MX_E4M3>(a, blocks, rope, st);
  else
    launch_write<DT, VELOGRAD_MX_E2M1>(a, blocks, rope, st);
}

template <int DT>
void launch_read_fmt(const ReadArgs& a, int fmt, uint32_t blocks, hipStream_t st) {
  if (fmt == VELOGRAD_MX_E4M3)
    hipLaunchKernelGGL((mx_read_kernel<DT, VELOGRAD_MX_E4M3>), dim3(blocks), dim3(kMxBlock), 0, st, a);
  else
    hipLaunchKernelGGL((mx_read_kernel<DT, VELOGRAD_MX_E2M1>), dim3(blocks), dim3(kMxBlock), 0, st, a);
}

}  // namespace

extern "C" {

VELOGRAD_API int32_t velograd_mx_cache_write(
    const void* q, const void* k, const void* v, void* q_out, const float* cos_sin,
    const int64_t* positions, const int64_t* slots, void* k_codes, void* k_scales, void* v_codes,
    void* v_scales, int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
    int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
    int64_t v_token_stride, int64_t v_head_stride, int64_t max_positions, int64_t pages,
    int64_t page_size, int32_t dtype, int32_t mx_format, void* hip_stream) {
  const char* what = "velograd_mx_cache_write";
  if (elem_bytes_of(dtype) == 0)
    return fail(VELOGRAD_ERR_UNSUPPORTED_DTYPE, "%s: unsupported dtype %d", what, (int)dtype);
  if (const int32_t rc = check_mx_cache(what, kv_heads, head_dim, pages, page_size, mx_format)) return rc;
  const bool rope = positions != nullptr;
  if (tokens < 0 || q_heads < 0 || q_heads > INT32_MAX / 4 || (!rope && q_heads != 0))
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: invalid shape tokens=%lld q_heads=%lld", what,
                (long long)tokens, (long long)q_heads);
  if (tokens == 0) {
    clear_error();
    return 0;
  }
  if (k == nullptr || v == nullptr || slots == nullptr || k_codes == nullptr || k_scales == nullptr ||
      v_codes == nullptr || v_scales == nullptr ||
      (rope && (cos_sin == nullptr || (q_heads > 0 && (q == nullptr || q_out == nullptr)))))
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: a required pointer must not be NULL", what);
  if (!aligned16(k_codes) || !aligned16(k_scales) || !aligned16(v_codes) || !aligned16(v_scales) ||
      (q_heads > 0 && !aligned16(q_out)))
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: the cache and q_out must be 16-byte aligned", what);
  if (rope && max_positions < 0)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: max_positions=%lld", what, (long long)max_positions);

  WriteArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.cos_sin = cos_sin;
  a.positions = positions;
  a.slots = slots;
  a.kc = static_cast<uint8_t*>(k_codes);
  a.ks = static_cast<uint8_t*>(k_scales);
  a.vc = static_cast<uint8_t*>(v_codes);
  a.vs = static_cast<uint8_t*>(v_scales);
  a.tokens = tokens;
  a.q_t = q_token_stride;
  a.q_h = q_head_stride;
  a.k_t = k_token_stride;
  a.k_h = k_head_stride;
  a.v_t = v_token_stride;
  a.v_h = v_head_stride;
  a.max_pos = max_positions;
  a.capacity = pages * page_size;
  a.q_heads = (int32_t)q_heads;
  a.kv_heads = (int32_t)kv_heads;
  a.dim = (int32_t)head_dim;
  a.lane_shift = log2_exact(head_dim / 16);
  a.page_shift = log2_exact(page_size);
  const int64_t per_block = kMxBlock >> a.lane_shift;
  const int64_t blocks = (tokens + per_block - 1) / per_block * (q_heads + 2 * kv_heads);
  if (blocks > INT32_MAX)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: %lld tokens exceed the grid limit", what,
                (long long)tokens);
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  switch (dtype) {
    case VELOGRAD_DTYPE_F32:
      launch_write_fmt<VELOGRAD_DTYPE_F32>(a, mx_format, (uint32_t)blocks, rope, st);
      break;
    case VELOGRAD_DTYPE_F16:
      launch_write_fmt<VELOGRAD_DTYPE_F16>(a, mx_format, (uint32_t)blocks, rope, st);
      break;
    default:
      launch_write_fmt<VELOGRAD_DTYPE_BF16>(a, mx_format, (uint32_t)blocks, rope, st);
      break;
  }
  return check_launch(what);
}

VELOGRAD_API int32_t velograd_mx_cache_read(
    const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
    const int64_t* slots, void* k, void* v, int64_t tokens, int64_t kv_heads, int64_t head_dim,
    int64_t pages, int64_t page_size, int32_t dtype, int32_t mx_format, void* hip_stream) {
  const char* what = "velograd_mx_cache_read";
  if (elem_bytes_of(dtype) == 0)
    return fail(VELOGRAD_ERR_UNSUPPORTED_DTYPE, "%s: unsupported dtype %d", what, (int)dtype);
  if (const int32_t rc = check_mx_cache(what, kv_heads, head_dim, pages, page_size, mx_format)) return rc;
  if (tokens < 0 || tokens > INT64_MAX / (kv_heads * head_dim))
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: invalid shape tokens=%lld", what, (long long)tokens);
  if (tokens == 0) {
    clear_error();
    return 0;
  }
  if (k == nullptr || v == nullptr || slots == nullptr || k_codes == nullptr || k_scales == nullptr ||
      v_codes == nullptr || v_scales == nullptr)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: a required pointer must not be NULL", what);
  if (!aligned16(k_codes) || !aligned16(k_scales) || !aligned16(v_codes) || !aligned16(v_scales) ||
      !aligned16(k) || !aligned16(v))
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: the cache and the outputs must be 16-byte aligned", what);

  ReadArgs a;
  a.kc = static_cast<const uint8_t*>(k_codes);
  a.ks = static_cast<const uint8_t*>(k_scales);
  a.vc = static_cast<const uint8_t*>(v_codes);
  a.vs = static_cast<const uint8_t*>(v_scales);
  a.slots = slots;
  a.k = k;
  a.v = v;
  a.items = tokens * kv_heads * (head_dim / 8);
  a.capacity = pages * page_size;
  a.kv_heads = (int32_t)kv_heads;
  a.dim = (int32_t)head_dim;
  a.chunk_shift = log2_exact(head_dim / 8);
  a.page_shift = log2_exact(page_size);
  const int64_t blocks = (a.items + kMxBlock - 1) / kMxBlock;
  if (blocks > INT32_MAX)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: %lld tokens exceed the grid limit", what,
                (long long)tokens);
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  switch (dtype) {
    case VELOGRAD_DTYPE_F32: launch_read_fmt<VELOGRAD_DTYPE_F32>(a, mx_format, (uint32_t)blocks, st); break;
    case VELOGRAD_DTYPE_F16: launch_read_fmt<VELOGRAD_DTYPE_F16>(a, mx_format, (uint32_t)blocks, st); break;
    default: launch_read_fmt<VELOGRAD_DTYPE_BF16>(a, mx_format, (uint32_t)blocks, st); break;
  }
  return check_launch(what);
}

}  // extern "C"
