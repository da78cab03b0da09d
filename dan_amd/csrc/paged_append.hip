// Appending new tokens to a paged key-value cache on gfx950 (MI355X, CDNA4):
// per-head RMS norm and rotate-half RoPE of q and k, q written token-major, k
// and v written into their pages.
//
//   n = x | w x / sqrt(mean x^2 + eps) | (1 + w) x / sqrt(mean x^2 + eps)
//   o_i = n_i cos_i - n_{i+R/2} sin_i  (i < R/2),  n_i cos_i + n_{i-R/2} sin_i  (R/2 <= i < R)
//
// in fp32 with one rounding, at the store (the front end of the prefill path,
// qkv_front.hip, rounds after each of the eager ops that it stands for: its keys
// differ from these by up to two roundings).
//
// HBM-bound: q, k, v, cos and sin are read once, q and the cache rows written
// once. A work group takes one token, so its place, page and rotary row are looked up by the scalar
// unit, and cos, sin and the norm weights are loaded once for all heads. A head vector (one head of
// q, k or v: D values) takes D / 8 lanes, 16 bytes each, so rows move as whole lines;
// each lane takes up to kVecs of them at a time, all loaded before any math. (Vectors dealt out over work
// groups whatever their token, as the front end does, cost about 200 vector instructions each,
// most of them addresses and a 64-bit division, and were bound by those.) 8192 tokens of 32 + 2 x 8
// heads of 128 with norm: 41.7 us (205 MB, 4.9 TB/s, as a large copy); where every call's q goes into the same memory 38.2, dealt
// out 47.2, on an e4m3 cache 40.0 against 49.4. One token: 3.1.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dan_paged.h"
#include "paged_index.h"

namespace dan {
int fail(int status, const char *fmt, ...);  // tree_attn.hip: sets the thread's last-error message
bool finite_nonnegative(float x);             // tree_attn.hip: decided from the float's bits
extern thread_local char g_err[512];
}  // namespace dan

namespace dan_append {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

#define DAN_GLOBAL __attribute__((address_space(1)))

template <typename T>
struct V;
template <>
struct V<__bf16> {
  typedef bf16x8 x8;
};
template <>
struct V<_Float16> {
  typedef f16x8 x8;
};

template <typename T>
__device__ inline f32x8 to_f32(u32x4 raw) {
  return __builtin_convertvector(__builtin_bit_cast(typename V<T>::x8, raw), f32x8);
}
template <typename T>
__device__ inline u32x4 from_f32(f32x8 x) {
  return __builtin_bit_cast(u32x4, __builtin_convertvector(x, typename V<T>::x8));
}
template <typename T>
__device__ inline u32x4 load16(const T *p) {
  return *(const DAN_GLOBAL u32x4 *)p;
}

// Sum of v over the L consecutive lanes of a vector (L = 8, 16 or 32), in every one of them.
#define DAN_DPP(x, ctrl) __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), ctrl, 0xF, 0xF, false))
template <int L>
__device__ inline float vec_sum(float v) {
  v += DAN_DPP(v, 0xB1);   // quad_perm 1, 0, 3, 2
  v += DAN_DPP(v, 0x4E);   // quad_perm 2, 3, 0, 1
  v += DAN_DPP(v, 0x141);  // row_half_mirror
  if constexpr (L >= 16) v += DAN_DPP(v, 0x140);  // row_mirror
  if constexpr (L >= 32) v += __shfl_xor(v, 16, 32);
  return v;
}

// x / scale, rounded once (the quotient by the reciprocal, and what is left of it: right to the last
// bit where nothing under- or overflows), beyond +-448 the largest e4m3 value; NaN stays NaN.
struct Scale {
  float s, inv;
};
__device__ inline float to_code_range(float x, Scale c) {
  const float q = x * c.inv, y = __builtin_fmaf(__builtin_fmaf(-q, c.s, x), c.inv, q);
  return q > 448.0f ? 448.0f : q < -448.0f ? -448.0f : y;
}
__device__ inline u32x2 to_e4m3(f32x8 x, Scale c) {
  u32x2 out;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(to_code_range(x[4 * i], c), to_code_range(x[4 * i + 1], c), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(to_code_range(x[4 * i + 2], c), to_code_range(x[4 * i + 3], c), w, true);
    out[i] = (uint32_t)w;
  }
  return out;
}

struct Params {
  const void *q, *k, *v, *cos, *sin, *qw, *kw;
  void *qo, *kc, *vc;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, cs_st, qo_st, qo_sh, kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;
  const float *ks, *vs;
  dan::PageTable table;
  const int32_t *places, *seqs, *rope_rows;
  int32_t N, H, Hkv, R, rope_count;
  float eps;
};

constexpr int kVecs = 3;

template <typename T, int D, int NORM, bool FP8, bool CS32>
__global__ __launch_bounds__(256) void append_kernel(const Params p) {
  constexpr int L = D / 8;  // lanes per head vector
  const int vpb = blockDim.x / L, slot = threadIdx.x / L, j = threadIdx.x % L;
  const int HV = p.H + 2 * p.Hkv, t = blockIdx.x;
  const dan::PageRow to = dan::find_row(p.table, p.seqs ? p.seqs[t] : t, p.places[t]);
  const int rope = p.rope_rows ? p.rope_rows[t] : t;
  const bool there = (uint32_t)rope < (uint32_t)p.rope_count;
  const T *q = static_cast<const T *>(p.q) + t * p.q_st, *k = static_cast<const T *>(p.k) + t * p.k_st, *v = static_cast<const T *>(p.v) + t * p.v_st;
  const int64_t krow = to.page * p.kc_sp + to.row * p.kc_st, vrow = to.page * p.vc_sp + to.row * p.vc_st;
  Scale ks = {1, 1}, vs = {1, 1};
  if constexpr (FP8) {
    ks = {*p.ks, 1.0f / *p.ks};
    vs = {*p.vs, 1.0f / *p.vs};
  }
  f32x8 cs = 0, sn = 0, qw = 0, kw = 0;
  const bool turns = 8 * j < p.R;
  const int half = p.R / 16;  // lanes per rotary half
  const int partner = j < half ? j + half : j - half;
  if (turns) {
    const int64_t off = (there ? rope : 0) * p.cs_st + 8 * j;
    if constexpr (CS32) {
      const float *c = static_cast<const float *>(p.cos) + off, *s = static_cast<const float *>(p.sin) + off;
      const f32x4 c0 = *(const DAN_GLOBAL f32x4 *)c, c1 = *(const DAN_GLOBAL f32x4 *)(c + 4);
      const f32x4 s0 = *(const DAN_GLOBAL f32x4 *)s, s1 = *(const DAN_GLOBAL f32x4 *)(s + 4);
      cs = __builtin_shufflevector(c0, c1, 0, 1, 2, 3, 4, 5, 6, 7);
      sn = __builtin_shufflevector(s0, s1, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      cs = to_f32<T>(load16(static_cast<const T *>(p.cos) + off));
      sn = to_f32<T>(load16(static_cast<const T *>(p.sin) + off));
    }
    if (j < half) sn = -sn;
    if (!there) cs = __builtin_nanf("");
  }
  if constexpr (NORM != DAN_FRONT_NORM_NONE) {
    if (p.H > 0) qw = to_f32<T>(load16(static_cast<const T *>(p.qw) + 8 * j));
    kw = to_f32<T>(load16(static_cast<const T *>(p.kw) + 8 * j));
    if constexpr (NORM == DAN_FRONT_NORM_RMS_ZERO_CENTERED) {
      qw += 1.0f;
      kw += 1.0f;
    }
  }
  for (int first = slot; first < HV; first += kVecs * vpb) {  // whole vectors go round together
    u32x4 raw[kVecs];
#pragma unroll
    for (int z = 0; z < kVecs; ++z) {
      const int hv = min(first + z * vpb, HV - 1);
      const bool isq = hv < p.H, isk = hv < p.H + p.Hkv;
      raw[z] = load16((isq ? q + hv * p.q_sh : isk ? k + (hv - p.H) * p.k_sh : v + (hv - p.H - p.Hkv) * p.v_sh) + 8 * j);
    }
#pragma unroll
    for (int z = 0; z < kVecs; ++z) {
      const int hv = first + z * vpb;
      if (hv >= HV) break;
      const bool isq = hv < p.H, isk = !isq && hv < p.H + p.Hkv;
      f32x8 o = to_f32<T>(raw[z]);
      if (isq || isk) {
        if constexpr (NORM != DAN_FRONT_NORM_NONE) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(o[i], o[i], ss);
          const float r = rsqrtf(vec_sum<L>(ss) * (1.0f / (float)D) + p.eps);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = o[i] * r * (isq ? qw[i] : kw[i]);
        }
        if (turns) {
          f32x8 y;
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(o[i], cs[i], __shfl(o[i], partner, L) * sn[i]);  // lane `partner` of this vector's L lanes
          o = y;
        }
      }
      if (isq) {
        *(DAN_GLOBAL u32x4 *)(static_cast<T *>(p.qo) + t * p.qo_st + hv * p.qo_sh + 8 * j) = from_f32<T>(o);
      } else if (to.page >= 0) {
        const int64_t at = (isk ? krow + (hv - p.H) * p.kc_sh : vrow + (hv - p.H - p.Hkv) * p.vc_sh) + 8 * j;
        if constexpr (FP8) *(DAN_GLOBAL u32x2 *)(static_cast<uint8_t *>(isk ? p.kc : p.vc) + at) = to_e4m3(o, {isk ? ks.s : vs.s, isk ? ks.inv : vs.inv});
        else *(DAN_GLOBAL u32x4 *)(static_cast<T *>(isk ? p.kc : p.vc) + at) = from_f32<T>(o);
      }
    }
  }
}

// Of a token's work group.
int threads_of(int h, int hkv, int d) {
  const int64_t lanes = ((int64_t)h + 2 * (int64_t)hkv) * (d / 8);
  return lanes < 256 ? (int)(lanes + 63) / 64 * 64 : 256;
}

template <typename T, int D, bool FP8, bool CS32>
void by_norm(const Params &p, int norm, hipStream_t s) {
  const dim3 grid((unsigned)p.N), block(threads_of(p.H, p.Hkv, D));
  if (norm == DAN_FRONT_NORM_RMS) hipLaunchKernelGGL((append_kernel<T, D, DAN_FRONT_NORM_RMS, FP8, CS32>), grid, block, 0, s, p);
  else if (norm == DAN_FRONT_NORM_RMS_ZERO_CENTERED)
    hipLaunchKernelGGL((append_kernel<T, D, DAN_FRONT_NORM_RMS_ZERO_CENTERED, FP8, CS32>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((append_kernel<T, D, DAN_FRONT_NORM_NONE, FP8, CS32>), grid, block, 0, s, p);
}

template <typename T, int D>
void by_types(const Params &p, int norm, bool fp8, bool cs32, hipStream_t s) {
  if (fp8) cs32 ? by_norm<T, D, true, true>(p, norm, s) : by_norm<T, D, true, false>(p, norm, s);
  else cs32 ? by_norm<T, D, false, true>(p, norm, s) : by_norm<T, D, false, false>(p, norm, s);
}

template <typename T>
void by_dim(const Params &p, int d, int norm, bool fp8, bool cs32, hipStream_t s) {
  if (d == 64) by_types<T, 64>(p, norm, fp8, cs32, s);
  else if (d == 128) by_types<T, 128>(p, norm, fp8, cs32, s);
  else by_types<T, 256>(p, norm, fp8, cs32, s);
}

}  // namespace dan_append

extern "C" {

int dan_paged_abi_version(void) { return DAN_PAGED_ABI_VERSION; }

int dan_paged_append(const DanPagedAppendArgs *a, void *stream) {
  using namespace dan_append;
  using dan::fail;
  dan::g_err[0] = 0;
  if (!a) return fail(DAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->abi_version != DAN_PAGED_ABI_VERSION)
    return fail(DAN_ERR_VERSION, "abi_version %d, paged cache speaks %d", a->abi_version, DAN_PAGED_ABI_VERSION);
  const int N = a->num_tokens, H = a->num_heads, Hkv = a->num_kv_heads, D = a->head_dim, R = a->rotary_dim;
  if (N < 0 || H < 0 || Hkv <= 0) return fail(DAN_ERR_INVALID_ARGUMENT, "need num_tokens >= 0, num_heads >= 0 and num_kv_heads > 0");
  if (D != 64 && D != 128 && D != 256) return fail(DAN_ERR_UNSUPPORTED, "head_dim %d: only 64, 128 and 256 are built", D);
  if (a->dtype != DAN_DTYPE_BF16 && a->dtype != DAN_DTYPE_F16) return fail(DAN_ERR_UNSUPPORTED, "dtype %d: bf16 or f16", a->dtype);
  const bool fp8 = a->cache_dtype == DAN_DTYPE_E4M3, cs32 = a->table_dtype == DAN_DTYPE_F32;
  if (!fp8 && a->cache_dtype != a->dtype) return fail(DAN_ERR_UNSUPPORTED, "cache_dtype %d: dtype's own or e4m3", a->cache_dtype);
  if (!cs32 && a->table_dtype != a->dtype) return fail(DAN_ERR_UNSUPPORTED, "table_dtype %d: dtype's own or f32", a->table_dtype);
  if (R < 0 || R > D || R % 16) return fail(DAN_ERR_INVALID_ARGUMENT, "rotary_dim %d must be a multiple of 16 in [0, %d]", R, D);
  if (a->norm < DAN_FRONT_NORM_NONE || a->norm > DAN_FRONT_NORM_RMS_ZERO_CENTERED)
    return fail(DAN_ERR_INVALID_ARGUMENT, "norm %d is not a DanFrontNorm", a->norm);
  if (a->norm != DAN_FRONT_NORM_NONE && ((H > 0 && !a->q_norm_weight) || !a->k_norm_weight || !dan::finite_nonnegative(a->eps)))
    return fail(DAN_ERR_INVALID_ARGUMENT, "a norm needs q_norm_weight, k_norm_weight and a finite eps >= 0");
  if (a->page_size <= 0 || a->page_size % DAN_PAGED_KEY_BLOCK)
    return fail(DAN_ERR_INVALID_ARGUMENT, "page_size %d must be a positive multiple of %d", a->page_size, DAN_PAGED_KEY_BLOCK);
  if (a->num_pages < 0 || a->table_width < 0 || a->num_seqs < 0 || a->num_rope_rows < 0)
    return fail(DAN_ERR_INVALID_ARGUMENT, "num_pages, table_width, num_seqs and num_rope_rows must be >= 0");
  if (R > 0 && !a->rope_rows && a->num_rope_rows < N)
    return fail(DAN_ERR_INVALID_ARGUMENT, "%d rows of cos and sin for %d tokens", a->num_rope_rows, N);
  if (N == 0) return DAN_OK;
  if ((H > 0 && (!a->q || !a->q_out)) || !a->k || !a->v || !a->places || (R > 0 && (!a->cos || !a->sin)) ||
      (a->num_pages > 0 && (!a->k_cache || !a->v_cache)) || (a->table_width > 0 && a->num_seqs > 0 && !a->table))
    return fail(DAN_ERR_INVALID_ARGUMENT, "NULL tensor pointer");
  if (R > 0 && a->num_rope_rows == 0) return fail(DAN_ERR_INVALID_ARGUMENT, "cos and sin have no rows");
  if (fp8 && (!a->k_scale || !a->v_scale)) return fail(DAN_ERR_INVALID_ARGUMENT, "an e4m3 cache needs k_scale and v_scale");
  if (R > 0 && a->cs_stride_tok < R) return fail(DAN_ERR_INVALID_ARGUMENT, "cs_stride_tok %lld < rotary_dim", (long long)a->cs_stride_tok);
  const int64_t strides[] = {H > 0 ? a->q_stride_tok : 0, H > 0 ? a->q_stride_head : 0, a->k_stride_tok, a->k_stride_head, a->v_stride_tok,
                             a->v_stride_head, H > 0 ? a->qo_stride_tok : 0, H > 0 ? a->qo_stride_head : 0, R > 0 ? a->cs_stride_tok : 0};
  for (int64_t st : strides)
    if (st % 8) return fail(DAN_ERR_INVALID_ARGUMENT, "strides must be multiples of 8 elements (16-byte rows)");
  for (int64_t st : {a->kc_stride_page, a->kc_stride_head, a->kc_stride_tok, a->vc_stride_page, a->vc_stride_head, a->vc_stride_tok})
    if (st % (fp8 ? 16 : 8)) return fail(DAN_ERR_INVALID_ARGUMENT, "cache strides must be multiples of 16 bytes");
  const void *ptrs[] = {H > 0 ? a->q : nullptr, H > 0 ? a->q_out : nullptr, a->k, a->v, R > 0 ? a->cos : nullptr, R > 0 ? a->sin : nullptr,
                        a->q_norm_weight, a->k_norm_weight, a->k_cache, a->v_cache};
  for (const void *ptr : ptrs)
    if ((uintptr_t)ptr & 15) return fail(DAN_ERR_INVALID_ARGUMENT, "tensor pointers must be 16-byte aligned");
  if ((int64_t)H + 2 * (int64_t)Hkv >= (int64_t)1 << 30) return fail(DAN_ERR_INVALID_ARGUMENT, "too many heads");
  if ((int64_t)N * threads_of(H, Hkv, D) >= (int64_t)1 << 32) return fail(DAN_ERR_INVALID_ARGUMENT, "%d tokens: too many for one launch", N);

  Params p;
  p.q = a->q; p.k = a->k; p.v = a->v; p.cos = a->cos; p.sin = a->sin; p.qw = a->q_norm_weight; p.kw = a->k_norm_weight;
  p.qo = a->q_out; p.kc = a->k_cache; p.vc = a->v_cache;
  p.q_st = a->q_stride_tok; p.q_sh = a->q_stride_head; p.k_st = a->k_stride_tok; p.k_sh = a->k_stride_head;
  p.v_st = a->v_stride_tok; p.v_sh = a->v_stride_head; p.cs_st = a->cs_stride_tok; p.qo_st = a->qo_stride_tok; p.qo_sh = a->qo_stride_head;
  p.kc_sp = a->kc_stride_page; p.kc_sh = a->kc_stride_head; p.kc_st = a->kc_stride_tok;
  p.vc_sp = a->vc_stride_page; p.vc_sh = a->vc_stride_head; p.vc_st = a->vc_stride_tok;
  p.ks = a->k_scale; p.vs = a->v_scale;
  p.table = {a->table, a->table_stride, a->num_seqs, a->table_width, a->page_size, a->num_pages}; p.places = a->places; p.seqs = a->seqs; p.rope_rows = a->rope_rows;
  p.N = N; p.H = H; p.Hkv = Hkv; p.R = R; p.rope_count = a->num_rope_rows; p.eps = a->eps;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == DAN_DTYPE_BF16) by_dim<__bf16>(p, D, a->norm, fp8, cs32, s);
  else by_dim<_Float16>(p, D, a->norm, fp8, cs32, s);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(DAN_ERR_LAUNCH, "append launch failed: %s", hipGetErrorString(err));
  return DAN_OK;
}

}  // extern "C"
