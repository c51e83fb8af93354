// Block-scaled ("microscaled") rows: quantisation to mx4 / mx8, reading them back, and the gated activation whose backward pass
// reads an mx8 checkpoint.
//
// A row of `cols` values is ceil(cols / 32) blocks of 32 consecutive columns, the last one filled up with zeros.  A block with
// largest magnitude a has ONE power-of-two scale 2^e, kept as the byte e + 127:
//   mx4   e = max(floor(log2 a) - 2, -127), elements 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives (sign, 2 exponent bits, 1 mantissa
//         bit), two to a byte, the lower column in the lower half: x -> nearest(x / 2^e), ties to the even code, at most 6
//   mx8   e = max(floor(log2 a), -127), elements q / 64 with q = -127 .. 127: q = nearest_even(64 x / 2^e), at most 127
// A block with an infinity or a NaN gets the byte 255 and stands for NaN throughout.  Scaling by a power of two is exact, so the
// ONE rounding of an element is the format's own, by the block's scale and not by the element: small elements of a block may vanish.
// mx4: at most 2^e / 4 below 2 2^e, 2^e / 2 below 4 2^e and 2^e up to 6 2^e, above which values (a may reach 8 2^e) are held to 6 2^e, up to
// 2 2^e off; mx8: at most 2^e / 128, or 2^e / 64 for magnitudes past 127.5 / 64 2^e (a may reach 2 2^e), which are held to 127 / 64 2^e.
// Storage: elements row-major without gaps between blocks (16 / 32 bytes a block), scale bytes row-major with rows filled up
// with zeros to whole 32-bit words (mx_scale_stride), so that a matrix kernel can fetch four blocks' scales at once.
//
// Every kernel here is bound by HBM: one thread moves 8 columns (16 bytes of bf16), the four threads of a block share their
// maximum by two quad permutations (no LDS), U chunks of a thread are in flight at once.  Measured (a large copy moves 5.0 TB/s):
// float32 10240 x 1280 to mx4 10.9 us (59 MB, 5.5 TB/s) and back 13.1 us (4.5); bf16 32768 x 320 to mx8 9.0 us (32 MB, of which 2-3 us are
// the launch); gated activation of bf16 8192 x 2560 forward 30.1 us and backward 32.9 us (169 MB each, 5.6 and 5.1 TB/s).
#include "common.h"

namespace ldm {

// n / d for n < 2^31, d >= 1, by one multiplication: with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1 the quotient
// is (hi32(n m) + n) >> s (Granlund & Montgomery, "Division by invariant integers using multiplication")
struct FastDiv { unsigned d, m, s; };

static FastDiv fast_div(unsigned d) {
  FastDiv f{d, 0, 0};
  while ((1ull << f.s) < d) ++f.s;
  f.m = (unsigned)((((1ull << 32) * ((1ull << f.s) - d)) / d) + 1);
  return f;
}
__device__ __forceinline__ unsigned div_by(unsigned n, const FastDiv& f) {
  return ((unsigned)(((unsigned long long)n * f.m) >> 32) + n) >> f.s;
}

// largest of the four lanes 4i .. 4i+3 / of the two lanes 2i, 2i+1 (quad permutations [1,0,3,2] and [2,3,0,1])
__device__ __forceinline__ unsigned pair_max(unsigned v) {
  const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);
  return v > o ? v : o;
}
__device__ __forceinline__ unsigned quad_max(unsigned v) {
  v = pair_max(v);
  const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);
  return v > o ? v : o;
}

// bits of the largest magnitude of 8 floats: as integers magnitudes order like the floats do, with NaN above infinity
__device__ __forceinline__ unsigned top_bits(const float (&v)[8]) {
  unsigned t = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const unsigned b = __float_as_uint(v[e]) & 0x7fffffffu;
    t = t > b ? t : b;
  }
  return t;
}

// scale byte of a block from the bits of its largest magnitude (subnormal magnitudes have exponent field 0: e = -127)
template <int FMT>
__device__ __forceinline__ int scale_code(unsigned top) {
  if (top >= 0x7f800000u) return 255;
  const int f = (int)(top >> 23);
  return FMT == LDM_MX4 ? (f > 2 ? f - 2 : 0) : f;
}

// 8 elements of mx4 in the 4 bytes they are stored in; the conversion takes the scale's exponent field as it is (0 means 2^-127),
// rounds to nearest even and holds to 6
__device__ __forceinline__ unsigned encode4(const float (&v)[8], int code) {
  if (code == 255) return 0;
  const float s = __uint_as_float((unsigned)code << 23);
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
  return w;
}

// 8 elements of mx8.  ldexp: 2^(133 - code) itself need not exist in float32.  Adding 1.5 * 2^23 rounds to nearest even and
// leaves the whole number, in two's complement, in the low bits.
__device__ __forceinline__ uint2 encode8(const float (&v)[8], int code) {
  if (code == 255) return make_uint2(0, 0);
  unsigned b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = fminf(fmaxf(ldexpf(v[e], 133 - code), -127.0f), 127.0f);
    b[e] = __float_as_uint(y + 12582912.0f) & 0xffu;
  }
  return make_uint2(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24);
}

// 2^(code - 133), the value of one step of mx8 (subnormal for the smallest codes), NaN for code 255
__device__ __forceinline__ float step8(int code) {
  return code == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(1.0f, code - 133);
}
__device__ __forceinline__ void decode8(uint2 w, float step, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = (float)((int)(w.x << (24 - 8 * e)) >> 24) * step;
    v[e + 4] = (float)((int)(w.y << (24 - 8 * e)) >> 24) * step;
  }
}
__device__ __forceinline__ void decode4(unsigned w, int code, float (&v)[8]) {
  const float s = __uint_as_float((unsigned)code << 23);      // code 255 reads as NaN
  const f32x2_hw_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
  const f32x2_hw_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
}

// 8 floats of a row that may start at any element
__device__ __forceinline__ void load8_any(const bf16_t* p, float (&v)[8]) {
  const uint4 r = load16_any(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8_any(const float* p, float (&v)[8]) {
  const uint4 a = load16_any(p), b = load16_any(p + 4);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void store8_any(bf16_t* p, const float (&v)[8]) {
  store16_any(p, make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])));
}
__device__ __forceinline__ void store8_any(float* p, const float (&v)[8]) {
  store16_any(p, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
  store16_any(p + 4, make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])));
}

// ---------------------------------------------------------------------------------------------------------------- quantise
constexpr int MX_U = 4;        // chunks a thread has in flight

struct MxParams {
  const void* src;
  void* dst;
  void* data;                  // elements
  unsigned char* scale;
  long long ld;                // elements between rows of the float matrix
  unsigned total;              // chunks of this launch
  FastDiv cpr;                 // chunks a row
  int cols, blocks, sstride;
};

// Chunks are counted over rows filled up to whole scale words, so the threads of a row's padding write its padding bytes.
template <typename T, int FMT>
__global__ void __launch_bounds__(256)
mx_quantize_kernel(const MxParams p) {
  float v[MX_U][8];
  unsigned row[MX_U], ch[MX_U];
  const unsigned first = blockIdx.x * (256u * MX_U) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < MX_U; ++u) {
    const unsigned idx = first + u * 256u;
    row[u] = div_by(idx, p.cpr);
    ch[u] = idx - row[u] * p.cpr.d;
    const int col = (int)ch[u] * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[u][e] = 0.f;
    if (idx >= p.total || col >= p.cols) continue;
    const T* src = static_cast<const T*>(p.src) + (long long)row[u] * p.ld + col;
    if (col + 8 <= p.cols) {
      load8_any(src, v[u]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < p.cols) v[u][e] = Elem<T>::ld(src + e);
    }
  }
#pragma unroll
  for (int u = 0; u < MX_U; ++u) {
    const unsigned idx = first + u * 256u;
    if (idx >= p.total) break;                                     // whole quads: chunks a row are a multiple of 16
    const int code = scale_code<FMT>(quad_max(top_bits(v[u])));
    const int blk = (int)(ch[u] >> 2);
    if (blk < p.blocks) {
      if constexpr (FMT == LDM_MX4)
        *reinterpret_cast<unsigned*>(static_cast<char*>(p.data) + ((long long)row[u] * p.blocks * 4 + ch[u]) * 4) = encode4(v[u], code);
      else
        *reinterpret_cast<uint2*>(static_cast<char*>(p.data) + ((long long)row[u] * p.blocks * 4 + ch[u]) * 8) = encode8(v[u], code);
    }
    if ((ch[u] & 3) == 0) p.scale[(long long)row[u] * p.sstride + blk] = (unsigned char)(blk < p.blocks ? code : 0);
  }
}

template <typename T, int FMT>
__global__ void __launch_bounds__(256)
mx_dequantize_kernel(const MxParams p) {
  uint2 w[MX_U];
  int code[MX_U];
  unsigned row[MX_U], ch[MX_U];
  const unsigned first = blockIdx.x * (256u * MX_U) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < MX_U; ++u) {
    const unsigned idx = first + u * 256u;
    row[u] = div_by(idx, p.cpr);
    ch[u] = idx - row[u] * p.cpr.d;
    w[u] = make_uint2(0, 0);
    code[u] = 0;
    if (idx >= p.total) continue;
    code[u] = p.scale[(long long)row[u] * p.sstride + (ch[u] >> 2)];
    const long long at = (long long)row[u] * p.blocks * 4 + ch[u];
    if constexpr (FMT == LDM_MX4) w[u].x = *reinterpret_cast<const unsigned*>(static_cast<const char*>(p.data) + at * 4);
    else w[u] = *reinterpret_cast<const uint2*>(static_cast<const char*>(p.data) + at * 8);
  }
#pragma unroll
  for (int u = 0; u < MX_U; ++u) {
    const unsigned idx = first + u * 256u;
    if (idx >= p.total) break;
    float v[8];
    if constexpr (FMT == LDM_MX4) decode4(w[u].x, code[u], v);
    else decode8(w[u], step8(code[u]), v);
    const int col = (int)ch[u] * 8;
    T* dst = static_cast<T*>(p.dst) + (long long)row[u] * p.ld + col;
    if (col + 8 <= p.cols) {
      store8_any(dst, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < p.cols) Elem<T>::st(dst + e, v[e]);
    }
  }
}

// out[k][n] = value of mx4 element (n, k) in bf16, n filled up with zeros to `ld` columns: the filter of the input-gradient
// product.  A workgroup turns 64 rows n x 128 columns k through LDS: a thread decodes 16 columns of two neighbouring rows and
// writes them as 16 pairs (n, n + 1); the rows of the turned image then leave as 16-byte pieces.
constexpr int MXT_PITCH = 64 + 2;        // bf16 elements between the image's rows: 33 words, so 16 consecutive k hit 16 banks

__global__ void __launch_bounds__(256)
mx4_dequantize_t_kernel(const unsigned char* __restrict__ data, const unsigned char* __restrict__ scale, bf16_t* __restrict__ out, int rows,
                        int cols, int blocks, int sstride, int ld) {
  __shared__ __attribute__((aligned(16))) uint32_t img[128 * (MXT_PITCH / 2)];
  const int tid = threadIdx.x;
  const int k0 = blockIdx.x * 128, n0 = blockIdx.y * 64;
  {
    const int half = tid & 7, np = tid >> 3;               // 16 columns, a pair of rows
    const int blk = (k0 >> 5) + (half >> 1);
    float v[2][16];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = n0 + 2 * np + i;
      uint2 w = make_uint2(0, 0);
      int code = 0;
      if (n < rows && blk < blocks) {
        w = *reinterpret_cast<const uint2*>(data + ((long long)n * blocks + blk) * 16 + (half & 1) * 8);
        code = scale[(long long)n * sstride + blk];
      }
      float a[8], b[8];
      decode4(w.x, code, a);
      decode4(w.y, code, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) { v[i][e] = a[e]; v[i][e + 8] = b[e]; }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) img[(half * 16 + e) * (MXT_PITCH / 2) + np] = pack_bf16x2(v[0][e], v[1][e]);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = (tid >> 3) + 32 * j, n = (tid & 7) * 8;
    if (k0 + k < cols && n0 + n < ld) {                    // ld is a multiple of 8
      const uint32_t* s = img + k * (MXT_PITCH / 2) + n / 2;
      *reinterpret_cast<uint4*>(out + (long long)(k0 + k) * ld + n0 + n) = make_uint4(s[0], s[1], s[2], s[3]);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------ pad
// rows of `cols` bf16 -> rows of ld (a multiple of 8), zeros behind: 16 bytes a thread, one pass (a clear and a copy would be two)
__global__ void __launch_bounds__(256)
pad_columns_kernel(const bf16_t* __restrict__ x, bf16_t* __restrict__ out, long long rows, int cols, int ld) {
  const int c = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (c >= ld) return;
  for (long long r = blockIdx.y; r < rows; r += gridDim.y) {
    const bf16_t* src = x + r * cols + c;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (c + 8 <= cols) {
      v = load16_any(src);
    } else {
      uint32_t h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = c + e < cols ? src[e] : 0;
      v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
    *reinterpret_cast<uint4*>(out + r * ld + c) = v;
  }
}

// --------------------------------------------------------------------------------------------------- gated activation
// h: (rows, 2 ff) with columns in the paired order of ldm_pack_weight(glu_pairs): blocks of 16 values, then their 16 gates -- an mx8
// block is exactly one such pair of blocks, so two threads hold a block: each 8 values and their 8 gates.
//   forward   out = v a(g), and h in mx8 (a: erf-GELU or SiLU)
//   backward  dv = dout a(g), dg = dout v a'(g) with v, g read from the mx8 form alone; optionally out again
// float32: erfcf, expf.  bf16: the one-instruction exponential and reciprocal, and erfc(z) = t P(t) exp(-z^2) with t = 1 / (1 + 0.407 z) and a
// polynomial of degree 5 fitted for this so that for z up to 9.6, where float32 ends, the error is below 7e-8 and below 2^-12 of the value
// both (4e-7 at small z with float32's own roundings): far in the negative tail the result is as near as bf16 holds it, too.  (The
// polynomial of the GEMM epilogues has the absolute bound alone: off by 1.5 % at x = -9.)
template <typename T, bool GELU>
__device__ __forceinline__ void gate_act(float x, float& a, float& da) {
  if constexpr (GELU) {
    float cdf, e;
    if constexpr (sizeof(T) == 2) {
      const float z = fabsf(x) * 0.70710678118654752440f;
      const float t = __builtin_amdgcn_rcpf(fmaf(0.407f, z, 1.0f));
      float q = fmaf(t, -0.18516022f, 0.61275858f);
      q = fmaf(q, t, -0.24113482f);
      q = fmaf(q, t, 0.38995084f);
      q = fmaf(q, t, 0.19068530f);
      q = fmaf(q, t, 0.23290025f);
      e = __builtin_amdgcn_exp2f(-1.44269504088896341f * z * z);
      const float half_erfc = 0.5f * q * t * e;                    // Phi(-|x|), no cancellation in the tail
      cdf = x >= 0.0f ? 1.0f - half_erfc : half_erfc;
    } else {
      cdf = 0.5f * erfcf(-x * 0.70710678118654752440f);
      e = expf(-0.5f * x * x);
    }
    a = x * cdf;
    da = fmaf(x * 0.39894228040143267794f, e, cdf);
  } else {
    float s;
    if constexpr (sizeof(T) == 2) s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * x));
    else s = 1.0f / (1.0f + expf(-x));
    a = x * s;
    da = s * fmaf(x, 1.0f - s, 1.0f);
  }
}

struct GluMx8Params {
  const void* h;
  const void* dout;
  void* out;
  void* dh;
  unsigned char* data;
  unsigned char* scale;
  unsigned total;              // 8-column chunks of out in this launch
  FastDiv cpr;                 // chunks a row: ff / 8
  int ff, sstride;
};

constexpr int GLU_U = 2;

template <typename T, bool GELU>
__global__ void __launch_bounds__(256)
glu_fwd_mx8_kernel(const GluMx8Params p) {
  float v[GLU_U][8], g[GLU_U][8];
  unsigned row[GLU_U], ch[GLU_U];
  const unsigned first = blockIdx.x * (256u * GLU_U) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < GLU_U; ++u) {
    const unsigned idx = first + u * 256u;
    if (idx >= p.total) break;
    row[u] = div_by(idx, p.cpr);
    ch[u] = idx - row[u] * p.cpr.d;
    const T* src = static_cast<const T*>(p.h) + (long long)row[u] * (2 * p.ff) + (ch[u] >> 1) * 32 + (ch[u] & 1) * 8;
    load8(src, v[u]);
    load8(src + 16, g[u]);
  }
#pragma unroll
  for (int u = 0; u < GLU_U; ++u) {
    const unsigned idx = first + u * 256u;
    if (idx >= p.total) break;                             // whole pairs: ff / 8 is even
    const unsigned tv = top_bits(v[u]), tg = top_bits(g[u]);
    const int code = scale_code<LDM_MX8>(pair_max(tv > tg ? tv : tg));
    const int blk = (int)(ch[u] >> 1);
    unsigned char* d = p.data + (long long)row[u] * (2 * p.ff) + blk * 32 + (ch[u] & 1) * 8;
    *reinterpret_cast<uint2*>(d) = encode8(v[u], code);
    *reinterpret_cast<uint2*>(d + 16) = encode8(g[u], code);
    if ((ch[u] & 1) == 0) {
      unsigned char* s = p.scale + (long long)row[u] * p.sstride;
      s[blk] = (unsigned char)code;
      if (blk == (p.ff >> 4) - 1)
        for (int b = blk + 1; b < p.sstride; ++b) s[b] = 0;
    }
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float a, da;
      gate_act<T, GELU>(g[u][e], a, da);
      o[e] = v[u][e] * a;
    }
    store8(static_cast<T*>(p.out) + (long long)row[u] * p.ff + ch[u] * 8, o);
  }
}

template <typename T, bool GELU, bool OUT>
__global__ void __launch_bounds__(256)
glu_bwd_mx8_kernel(const GluMx8Params p) {
  uint2 wv[GLU_U], wg[GLU_U];
  int code[GLU_U];
  float d[GLU_U][8];
  unsigned row[GLU_U], ch[GLU_U];
  const unsigned first = blockIdx.x * (256u * GLU_U) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < GLU_U; ++u) {
    const unsigned idx = first + u * 256u;
    if (idx >= p.total) break;
    row[u] = div_by(idx, p.cpr);
    ch[u] = idx - row[u] * p.cpr.d;
    const unsigned char* s = p.data + (long long)row[u] * (2 * p.ff) + (ch[u] >> 1) * 32 + (ch[u] & 1) * 8;
    wv[u] = *reinterpret_cast<const uint2*>(s);
    wg[u] = *reinterpret_cast<const uint2*>(s + 16);
    code[u] = p.scale[(long long)row[u] * p.sstride + (ch[u] >> 1)];
    load8(static_cast<const T*>(p.dout) + (long long)row[u] * p.ff + ch[u] * 8, d[u]);
  }
#pragma unroll
  for (int u = 0; u < GLU_U; ++u) {
    const unsigned idx = first + u * 256u;
    if (idx >= p.total) break;
    const float step = step8(code[u]);
    float v[8], g[8], dv[8], dg[8], o[8];
    decode8(wv[u], step, v);
    decode8(wg[u], step, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float a, da;
      gate_act<T, GELU>(g[e], a, da);
      dv[e] = d[u][e] * a;
      dg[e] = d[u][e] * v[e] * da;
      o[e] = v[e] * a;
    }
    T* dh = static_cast<T*>(p.dh) + (long long)row[u] * (2 * p.ff) + (ch[u] >> 1) * 32 + (ch[u] & 1) * 8;
    store8(dh, dv);
    store8(dh + 16, dg);
    if constexpr (OUT) store8(static_cast<T*>(p.out) + (long long)row[u] * p.ff + ch[u] * 8, o);
  }
}

// Rows of one launch: the kernels count chunks in 31 bits
static long long rows_a_launch(long long chunks_a_row) { return 0x7ff00000LL / chunks_a_row; }

template <typename T, int FMT>
static void launch_quantize(const MxParams& p, hipStream_t st) {
  hipLaunchKernelGGL((mx_quantize_kernel<T, FMT>), dim3((p.total + 256u * MX_U - 1) / (256u * MX_U)), dim3(256), 0, st, p);
}
template <typename T, int FMT>
static void launch_dequantize(const MxParams& p, hipStream_t st) {
  hipLaunchKernelGGL((mx_dequantize_kernel<T, FMT>), dim3((p.total + 256u * MX_U - 1) / (256u * MX_U)), dim3(256), 0, st, p);
}

}  // namespace ldm

using namespace ldm;

static int mx_check(const char* what, int dtype, int fmt, long long rows, int cols, long long ld) {
  LDM_REQUIRE(dtype_ok(dtype), "%s: bad dtype %d", what, dtype);
  LDM_REQUIRE(fmt == LDM_MX4 || fmt == LDM_MX8, "%s: bad format %d", what, fmt);
  LDM_REQUIRE(rows >= 0 && cols >= 1 && cols <= (1 << 30) && ld >= cols, "%s: bad sizes (rows=%lld cols=%d ld=%lld)", what, rows, cols, ld);
  return LDM_OK;
}

extern "C" int ldm_mx_quantize(const void* x, int dtype, long long rows, int cols, long long ld, int fmt, void* data, void* scale,
                               void* stream) {
  if (int rc = mx_check("ldm_mx_quantize", dtype, fmt, rows, cols, ld)) return rc;
  if (rows == 0) return LDM_OK;
  LDM_REQUIRE(x && data && scale && aligned16(data) && (reinterpret_cast<uintptr_t>(scale) & 3) == 0 &&
                  reinterpret_cast<uintptr_t>(x) % dtype_size(dtype) == 0, "ldm_mx_quantize: null or unaligned pointer");
  const size_t es = dtype_size(dtype);
  MxParams p;
  p.ld = ld; p.cols = cols; p.blocks = mx_blocks(cols); p.sstride = mx_scale_stride(cols); p.dst = nullptr;
  p.cpr = fast_div((unsigned)p.sstride * 4u);
  const long long step = rows_a_launch((long long)p.sstride * 4), bytes = fmt == LDM_MX4 ? 16 : 32;
  for (long long r = 0; r < rows; r += step) {
    const long long n = rows - r < step ? rows - r : step;
    p.src = static_cast<const char*>(x) + r * ld * es;
    p.data = static_cast<char*>(data) + r * p.blocks * bytes;
    p.scale = static_cast<unsigned char*>(scale) + r * p.sstride;
    p.total = (unsigned)(n * p.sstride * 4);
    if (dtype == LDM_BF16) fmt == LDM_MX4 ? launch_quantize<bf16_t, LDM_MX4>(p, (hipStream_t)stream) : launch_quantize<bf16_t, LDM_MX8>(p, (hipStream_t)stream);
    else fmt == LDM_MX4 ? launch_quantize<float, LDM_MX4>(p, (hipStream_t)stream) : launch_quantize<float, LDM_MX8>(p, (hipStream_t)stream);
    LDM_HIP_CHECK_LAUNCH("ldm_mx_quantize");
  }
  return LDM_OK;
}

extern "C" int ldm_mx_dequantize(const void* data, const void* scale, int fmt, long long rows, int cols, void* out, int dtype,
                                 long long ld, void* stream) {
  if (int rc = mx_check("ldm_mx_dequantize", dtype, fmt, rows, cols, ld)) return rc;
  if (rows == 0) return LDM_OK;
  LDM_REQUIRE(out && data && scale && aligned16(data) && (reinterpret_cast<uintptr_t>(scale) & 3) == 0 &&
                  reinterpret_cast<uintptr_t>(out) % dtype_size(dtype) == 0, "ldm_mx_dequantize: null or unaligned pointer");
  const size_t es = dtype_size(dtype);
  MxParams p;
  p.ld = ld; p.cols = cols; p.blocks = mx_blocks(cols); p.sstride = mx_scale_stride(cols); p.src = nullptr;
  const int chunks = (cols + 7) / 8;
  p.cpr = fast_div((unsigned)chunks);
  const long long step = rows_a_launch(chunks), bytes = fmt == LDM_MX4 ? 16 : 32;
  for (long long r = 0; r < rows; r += step) {
    const long long n = rows - r < step ? rows - r : step;
    p.dst = static_cast<char*>(out) + r * ld * es;
    p.data = const_cast<char*>(static_cast<const char*>(data) + r * p.blocks * bytes);
    p.scale = const_cast<unsigned char*>(static_cast<const unsigned char*>(scale) + r * p.sstride);
    p.total = (unsigned)(n * chunks);
    if (dtype == LDM_BF16) fmt == LDM_MX4 ? launch_dequantize<bf16_t, LDM_MX4>(p, (hipStream_t)stream) : launch_dequantize<bf16_t, LDM_MX8>(p, (hipStream_t)stream);
    else fmt == LDM_MX4 ? launch_dequantize<float, LDM_MX4>(p, (hipStream_t)stream) : launch_dequantize<float, LDM_MX8>(p, (hipStream_t)stream);
    LDM_HIP_CHECK_LAUNCH("ldm_mx_dequantize");
  }
  return LDM_OK;
}

extern "C" int ldm_mx4_dequantize_t(const void* data, const void* scale, int rows, int cols, void* out, int ld, void* stream) {
  LDM_REQUIRE(rows >= 1 && cols >= 1 && cols <= (1 << 30) && ld >= rows && ld % 8 == 0 && (ld + 63) / 64 <= 65535,
              "ldm_mx4_dequantize_t: bad sizes (rows=%d cols=%d ld=%d)", rows, cols, ld);
  LDM_REQUIRE(out && data && scale && aligned16(out) && aligned16(data), "ldm_mx4_dequantize_t: null or unaligned pointer");
  hipLaunchKernelGGL(mx4_dequantize_t_kernel, dim3((cols + 127) / 128, (ld + 63) / 64), dim3(256), 0, (hipStream_t)stream,
                     static_cast<const unsigned char*>(data), static_cast<const unsigned char*>(scale), static_cast<bf16_t*>(out), rows, cols,
                     mx_blocks(cols), mx_scale_stride(cols), ld);
  LDM_HIP_CHECK_LAUNCH("ldm_mx4_dequantize_t");
  return LDM_OK;
}

extern "C" int ldm_pad_columns_bf16(const void* x, void* out, long long rows, int cols, int ld, void* stream) {
  LDM_REQUIRE(rows >= 0 && cols >= 1 && ld >= cols && ld % 8 == 0 && ld <= (1 << 30), "ldm_pad_columns_bf16: bad sizes (rows=%lld cols=%d ld=%d)", rows,
              cols, ld);
  if (rows == 0) return LDM_OK;
  LDM_REQUIRE(x && out && aligned16(out) && (reinterpret_cast<uintptr_t>(x) & 1) == 0, "ldm_pad_columns_bf16: null or unaligned pointer");
  hipLaunchKernelGGL(pad_columns_kernel, dim3((ld / 8 + 255) / 256, (unsigned)(rows < 65535 ? rows : 65535)), dim3(256), 0, (hipStream_t)stream,
                     static_cast<const bf16_t*>(x), static_cast<bf16_t*>(out), rows, cols, ld);
  LDM_HIP_CHECK_LAUNCH("ldm_pad_columns_bf16");
  return LDM_OK;
}

static int glu_mx8_check(const char* what, int dtype, long long rows, int ff) {
  LDM_REQUIRE(dtype_ok(dtype), "%s: bad dtype %d", what, dtype);
  LDM_REQUIRE(rows >= 0 && ff >= 16 && ff % 16 == 0 && ff <= (1 << 28), "%s: ff must be a multiple of 16 (rows=%lld ff=%d)", what, rows, ff);
  return LDM_OK;
}

template <typename T>
static void launch_glu_fwd(const GluMx8Params& p, int gelu, hipStream_t st) {
  const dim3 grid((p.total + 256u * GLU_U - 1) / (256u * GLU_U));
  if (gelu) hipLaunchKernelGGL((glu_fwd_mx8_kernel<T, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((glu_fwd_mx8_kernel<T, false>), grid, dim3(256), 0, st, p);
}
template <typename T>
static void launch_glu_bwd(const GluMx8Params& p, int gelu, hipStream_t st) {
  const dim3 grid((p.total + 256u * GLU_U - 1) / (256u * GLU_U));
  if (p.out) {
    if (gelu) hipLaunchKernelGGL((glu_bwd_mx8_kernel<T, true, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((glu_bwd_mx8_kernel<T, false, true>), grid, dim3(256), 0, st, p);
  } else {
    if (gelu) hipLaunchKernelGGL((glu_bwd_mx8_kernel<T, true, false>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((glu_bwd_mx8_kernel<T, false, false>), grid, dim3(256), 0, st, p);
  }
}

extern "C" int ldm_glu_forward_mx8(const void* h, void* out, void* data, void* scale, int dtype, long long rows, int ff, int gelu,
                                   void* stream) {
  if (int rc = glu_mx8_check("ldm_glu_forward_mx8", dtype, rows, ff)) return rc;
  if (rows == 0) return LDM_OK;
  LDM_REQUIRE(h && out && data && scale && aligned16(h) && aligned16(out) && aligned16(data), "ldm_glu_forward_mx8: null or unaligned pointer");
  GluMx8Params p{};
  p.ff = ff; p.sstride = mx_scale_stride(2 * ff); p.cpr = fast_div((unsigned)ff / 8u);
  const long long step = rows_a_launch(ff / 8), es = (long long)dtype_size(dtype);
  for (long long r = 0; r < rows; r += step) {
    const long long n = rows - r < step ? rows - r : step;
    p.h = static_cast<const char*>(h) + r * 2 * ff * es;
    p.out = static_cast<char*>(out) + r * ff * es;
    p.data = static_cast<unsigned char*>(data) + r * 2 * ff;
    p.scale = static_cast<unsigned char*>(scale) + r * p.sstride;
    p.total = (unsigned)(n * (ff / 8));
    if (dtype == LDM_BF16) launch_glu_fwd<bf16_t>(p, gelu, (hipStream_t)stream);
    else launch_glu_fwd<float>(p, gelu, (hipStream_t)stream);
    LDM_HIP_CHECK_LAUNCH("ldm_glu_forward_mx8");
  }
  return LDM_OK;
}

extern "C" int ldm_glu_backward_mx8(const void* data, const void* scale, const void* dout, void* dh, void* out, int dtype, long long rows,
                                    int ff, int gelu, void* stream) {
  if (int rc = glu_mx8_check("ldm_glu_backward_mx8", dtype, rows, ff)) return rc;
  if (rows == 0) return LDM_OK;
  LDM_REQUIRE(data && scale && dout && dh && aligned16(data) && aligned16(dout) && aligned16(dh) && aligned16(out),
              "ldm_glu_backward_mx8: null or unaligned pointer");
  GluMx8Params p{};
  p.ff = ff; p.sstride = mx_scale_stride(2 * ff); p.cpr = fast_div((unsigned)ff / 8u);
  const long long step = rows_a_launch(ff / 8), es = (long long)dtype_size(dtype);
  for (long long r = 0; r < rows; r += step) {
    const long long n = rows - r < step ? rows - r : step;
    p.data = const_cast<unsigned char*>(static_cast<const unsigned char*>(data)) + r * 2 * ff;
    p.scale = const_cast<unsigned char*>(static_cast<const unsigned char*>(scale)) + r * p.sstride;
    p.dout = static_cast<const char*>(dout) + r * ff * es;
    p.dh = static_cast<char*>(dh) + r * 2 * ff * es;
    p.out = out ? static_cast<char*>(out) + r * ff * es : nullptr;
    p.total = (unsigned)(n * (ff / 8));
    if (dtype == LDM_BF16) launch_glu_bwd<bf16_t>(p, gelu, (hipStream_t)stream);
    else launch_glu_bwd<float>(p, gelu, (hipStream_t)stream);
    LDM_HIP_CHECK_LAUNCH("ldm_glu_backward_mx8");
  }
  return LDM_OK;
}
