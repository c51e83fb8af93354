// Products with block-scaled operands on the gfx950 matrix cores: linear layers with mx4 (4-bit) weights.
//
//   out[m][n] = bias[n] + sum_k x[m][k] w[n][k]
//
// mx4_gemm_kernel: both operands mx4, on v_mfma_scale_f32_32x32x64_f8f6f4.  A lane's operand is 32 consecutive k of one row -- one
// block, 16 bytes as stored -- and its scale byte; products and sums are float32 inside the instruction, so nothing is
// rounded before the output.  The weights are the instruction's first operand: a lane then holds four consecutive n of one m.
// mx4_rows_kernel: few rows of x, where the weights' bytes are what counts (see there).
#include "common.h"

#include <type_traits>
#include <utility>

namespace ldm {

typedef __attribute__((ext_vector_type(8))) short bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;

struct Mx4Params {
  const unsigned char* x;      // mx4 elements, or bf16
  const unsigned char* xs;
  const unsigned char* w;
  const unsigned char* ws;
  const float* bias;
  void* out;
  long long rows;              // M
  int n, k, blocks, sstride;   // N, K, blocks and scale bytes a row
  int nk;                      // steps of 128 columns
  int tiles_m, tiles_n;
  int vec_out;                 // 16-byte stores of the output are legal
};

// bijective XCD remap: workgroups b and b + 8 share an XCD; every XCD gets a contiguous run of tiles
__device__ __forceinline__ int mx_xcd_remap(int bid, int nblk) {
  const int q = nblk >> 3, r = nblk & 7, x = bid & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (bid >> 3);
}

__device__ __forceinline__ i32x8_t mx4_operand(uint4 v) { return i32x8_t{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0}; }

// 16 / 4 bytes a lane from a raw buffer (base, bytes) into LDS, lane-linear from `lds`; a lane offset past `bytes` gives zeros
__device__ __forceinline__ void mx_dma16(const void* base, unsigned bytes, unsigned char* lds, unsigned voff, int soff) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void mx_dma4(const void* base, unsigned bytes, unsigned char* lds, unsigned voff, int soff) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 4, voff, soff, 0, 0);
}

// Tile of BM (rows of x) x BN (rows of w) by WM x WN waves, 128 columns (64 bytes a row) a step, S slots of LDS: the LDS-DMA of S - 1
// steps is in flight.  16-byte chunks of a row are XOR-swizzled by (row >> 1) & 3 (the DMA writes lane-linear, so the swizzle is
// applied to the lane's SOURCE chunk and again on the read): eight consecutive rows then lie in eight different 16-byte
// columns of the 128-byte LDS line.  A chunk IS a block, so chunks past the last block are fetched from beyond the descriptor's end
// (zeros), and rows past the end likewise.
//
// Scales: one 32-bit word a row and step.  From four steps on, 16 bytes (four steps) a row at a time in one DMA instruction, the last
// ones ending with the row (a fetch never passes its row); with fewer steps word by word, once.
template <int BM, int BN, int WM, int WN, int S, typename OUT>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN == 8 ? 2 : 2)
mx4_gemm_kernel(const Mx4Params p) {
  constexpr int NT = 64 * WM * WN, ROWS = BM + BN;
  constexpr int IT = ROWS * 4 / NT;                        // tile DMA instructions of a wave a step
  constexpr int SIT = ROWS / NT;                           // scale DMA instructions of a wave (16 bytes a row)
  static_assert(ROWS * 4 % NT == 0 && ROWS % NT == 0 && BM % 64 == 0, "tile / threads mismatch");
  constexpr int STAGE = ROWS * 64;
  constexpr int SCALES = ROWS * 16;                        // one group of four steps
  constexpr int WTM = BM / WM, WTN = BN / WN, MI = WTM / 32, NI = WTN / 32;
  constexpr unsigned OOB = 0x80000000u;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane & 31, fh = lane >> 5;

  const int tile = mx_xcd_remap(blockIdx.x, gridDim.x);
  // bands of 8 tile rows walked column by column: the tiles in flight on one XCD share their operands in its L2
  const int band = 8 * p.tiles_n, g8 = tile / band, in = tile - g8 * band;
  const int brows = min(p.tiles_m - g8 * 8, 8);
  const int tn = in / brows, tm = g8 * 8 + (in - tn * brows);
  const long long m0 = (long long)tm * BM;
  const int n0 = tn * BN;

  const int rb = p.blocks * 16;
  const int mrows = (int)min((long long)BM, p.rows - m0), nrows = min(BN, p.n - n0);
  const unsigned char* xbase = p.x + m0 * rb;
  const unsigned char* wbase = p.w + (long long)n0 * rb;
  const unsigned char* xsbase = p.xs + m0 * p.sstride;
  const unsigned char* wsbase = p.ws + (long long)n0 * p.sstride;
  const unsigned xbytes = (unsigned)mrows * rb, wbytes = (unsigned)nrows * rb;
  const unsigned xsbytes = (unsigned)mrows * p.sstride, wsbytes = (unsigned)nrows * p.sstride;


  // lane's part of tile instruction `it`: chunk q = it * NT + tid of the stage image (x rows, then w rows; four chunks a row)
  unsigned voff[IT];
  int chunk[IT];
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int row = (it * NT + tid) >> 2;
    chunk[it] = (tid & 3) ^ ((row >> 1) & 3);
    voff[it] = (unsigned)(row < BM ? row : row - BM) * rb + chunk[it] * 16;
  }
  const int nk = p.nk;
  const bool word_scales = nk < 4;
  unsigned char* const scales = smem + S * STAGE;

  // word j of row r of scale group g lies at group_base + r * row_step + (j - first word) * word_step
  auto group_first = [&](int g) { return word_scales ? 0 : min(g * 4, nk - 4); };
  auto stage_scales = [&](int g) {
    unsigned char* dst = scales + (g & 1) * SCALES;
    if (word_scales) {
      for (int j = 0; j < nk; ++j)
#pragma unroll
        for (int it = 0; it < SIT; ++it) {
          const int r0 = it * NT + wave * 64, row = r0 + lane;
          if (r0 < BM) mx_dma4(xsbase, xsbytes, dst + (j * ROWS + r0) * 4, (unsigned)row * p.sstride, j * 4);
          else mx_dma4(wsbase, wsbytes, dst + (j * ROWS + r0) * 4, (unsigned)(row - BM) * p.sstride, j * 4);
        }
    } else {
      const int first = group_first(g) * 4;
#pragma unroll
      for (int it = 0; it < SIT; ++it) {
        const int r0 = it * NT + wave * 64, row = r0 + lane;
        if (r0 < BM) mx_dma16(xsbase, xsbytes, dst + r0 * 16, (unsigned)row * p.sstride, first);
        else mx_dma16(wsbase, wsbytes, dst + r0 * 16, (unsigned)(row - BM) * p.sstride, first);
      }
    }
  };
  auto stage = [&](int kt) {
    if ((kt & 3) == 0) stage_scales(kt >> 2);
    unsigned char* dst = smem + (kt % S) * STAGE;
    const bool tail = kt == nk - 1;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int q0 = it * NT + wave * 64;                  // the instruction's first chunk: 16 whole rows, all of one operand
      const unsigned vo = tail && kt * 4 + chunk[it] >= p.blocks ? OOB : voff[it];
      if (q0 < BM * 4) mx_dma16(xbase, xbytes, dst + q0 * 16, vo, kt * 64);
      else mx_dma16(wbase, wbytes, dst + q0 * 16, vo, kt * 64);
    }
  };

  f32x16_t acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  auto compute = [&](int kt) {
    const unsigned char* img = smem + (kt % S) * STAGE;
    const int g = kt >> 2, word = kt - group_first(g);
    const unsigned char* sc = scales + (g & 1) * SCALES + word * (word_scales ? ROWS * 4 : 4);
    const int sstep = word_scales ? 4 : 16;
    // byte 0: this half's block of the step's first 64 columns, byte 2: of the second
    int sx[MI], sw[NI];
#pragma unroll
    for (int i = 0; i < MI; ++i) sx[i] = (int)(*reinterpret_cast<const unsigned*>(sc + (wm * WTM + i * 32 + fr) * sstep) >> (8 * fh));
#pragma unroll
    for (int j = 0; j < NI; ++j) sw[j] = (int)(*reinterpret_cast<const unsigned*>(sc + (BM + wn * WTN + j * 32 + fr) * sstep) >> (8 * fh));
    [&]<int... HI>(std::integer_sequence<int, HI...>) {
      ([&] {
        constexpr int H = HI;
        i32x8_t xf[MI], wf[NI];
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const int row = wm * WTM + i * 32 + fr;
          xf[i] = mx4_operand(*reinterpret_cast<const uint4*>(img + row * 64 + (((2 * H + fh) ^ ((row >> 1) & 3)) << 4)));
        }
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const int row = BM + wn * WTN + j * 32 + fr;
          wf[j] = mx4_operand(*reinterpret_cast<const uint4*>(img + row * 64 + (((2 * H + fh) ^ ((row >> 1) & 3)) << 4)));
        }
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[j], xf[i], acc[i][j], 4, 4, 2 * H, sw[j], 2 * H, sx[i]);
      }(), ...);
    }(std::integer_sequence<int, 0, 1>{});
  };

  // one barrier a step: wait until this wave's DMA of step kt has landed (that of the S - 2 steps behind it may be in flight; a scale
  // fetch among them only makes the wait stricter), barrier, refill the slot of step kt - 1, multiply
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < nk) stage(s);
  for (int kt = 0; kt < nk; ++kt) {
    const int ahead = nk - 1 - kt;
    if (ahead >= S - 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * IT) : "memory");
    else if (S > 3 && ahead == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(IT) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (kt + S - 1 < nk) stage(kt + S - 1);
    compute(kt);
  }
  __syncthreads();                                         // the slots become the epilogue's

  // ---- epilogue: 32 rows of the wave's tile at a time through its own LDS, then whole 16-byte pieces of rows
  constexpr int PITCH = WTN * (int)sizeof(OUT) + 16;
  constexpr int EPR = 16 / (int)sizeof(OUT);               // elements of a piece
  static_assert(WM * WN * 32 * PITCH <= S * STAGE + 2 * SCALES, "epilogue image");
  unsigned char* const cst = smem + wave * 32 * PITCH;
  float bv[NI][4][4];
#pragma unroll
  for (int j = 0; j < NI; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + wn * WTN + j * 32 + 8 * q + 4 * fh + e;
        bv[j][q][e] = p.bias != nullptr && n < p.n ? p.bias[n] : 0.f;
      }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e] + bv[j][q][e];
        unsigned char* d = cst + fr * PITCH + (j * 32 + 8 * q + 4 * fh) * (int)sizeof(OUT);
        if constexpr (sizeof(OUT) == 2) *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        else *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
      }
    LDM_LOCKSTEP();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    constexpr int PPR = WTN / EPR;                         // pieces a row
#pragma unroll
    for (int t = 0; t < 32 * PPR / 64; ++t) {
      const int piece = t * 64 + lane, r = piece / PPR, c = (piece - r * PPR) * EPR;
      const long long m = m0 + wm * WTM + i * 32 + r;
      const int n = n0 + wn * WTN + c;
      if (m >= p.rows || n >= p.n) continue;
      OUT* dst = static_cast<OUT*>(p.out) + m * p.n + n;
      const unsigned char* s = cst + r * PITCH + c * (int)sizeof(OUT);
      if (p.vec_out) {                                     // n is a multiple of the piece: no piece passes the row
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(s);
      } else {
        for (int e = 0; e < EPR && n + e < p.n; ++e) dst[e] = reinterpret_cast<const OUT*>(s)[e];
      }
    }
    LDM_LOCKSTEP();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// --------------------------------------------------------------------------------------------------------- few rows
// 16 NF rows of w and 16 MT rows of x a workgroup; its 8 waves take every 8th step of 128 columns and add up through LDS in a fixed
// order.  Operands go straight from memory to registers (nothing is used twice by a wave), several steps' loads at once.
//   MX  true: x in mx4, v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds row l % 16, block l / 16 of the step
//       false: x in bf16; the lane's block of w is widened to bf16 (exact: 2 significant bits) and multiplied by
//              v_mfma_f32_16x16x32_bf16 in four pieces.  Piece s takes columns 32 (l / 16) + 8 s .. + 7 of the step from BOTH
//              operands: a permutation of the contraction index, which the sum does not see.
template <bool MX, int MT, int NF, bool VEC, typename OUT>
__global__ void __launch_bounds__(512)
mx4_rows_kernel(const Mx4Params p) {
  constexpr int NW = 8;
  constexpr int U = MX ? 4 : (MT == 1 ? 4 : MT == 2 ? 2 : 1);   // steps whose loads are in flight
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float4* const red = reinterpret_cast<float4*>(smem);     // [wave][NF * MT][64]
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int n0 = blockIdx.x * (16 * NF);
  const long long m0 = (long long)blockIdx.y * (16 * MT);
  const int rb = p.blocks * 16;

  f32x4_t acc[NF][MT];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  for (int kt0 = wave; kt0 < p.nk; kt0 += NW * U) {
    uint4 wv[U][NF], xv[U][MT][MX ? 1 : 4];
    int wc[U][NF], xc[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int blk = (kt0 + u * NW) * 4 + fq;
      const bool live = blk < p.blocks;
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        const int n = n0 + i * 16 + fr;
        wv[u][i] = make_uint4(0, 0, 0, 0);
        wc[u][i] = 0;
        if (live && n < p.n) {
          wv[u][i] = *reinterpret_cast<const uint4*>(p.w + (long long)n * rb + blk * 16);
          wc[u][i] = p.ws[(long long)n * p.sstride + blk];
        }
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const long long m = m0 + j * 16 + fr;
        const bool ok = live && m < p.rows;
        xc[u][j] = 0;
        if constexpr (MX) {
          xv[u][j][0] = make_uint4(0, 0, 0, 0);
          if (ok) {
            xv[u][j][0] = *reinterpret_cast<const uint4*>(p.x + m * rb + blk * 16);
            xc[u][j] = p.xs[m * p.sstride + blk];
          }
        } else {
          const bf16_t* src = reinterpret_cast<const bf16_t*>(p.x) + m * p.k + blk * 32;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            xv[u][j][s] = make_uint4(0, 0, 0, 0);
            const int left = p.k - (blk * 32 + 8 * s);
            if (!ok || left <= 0) continue;
            if (VEC) {                                     // k is a multiple of 8
              xv[u][j][s] = *reinterpret_cast<const uint4*>(src + 8 * s);
            } else {
              uint32_t h[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) h[e] = e < left ? src[8 * s + e] : 0;
              xv[u][j][s] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
            }
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        if constexpr (MX) {
          const i32x8_t a = mx4_operand(wv[u][i]);
#pragma unroll
          for (int j = 0; j < MT; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, mx4_operand(xv[u][j][0]), acc[i][j], 4, 4, 0, wc[u][i], 0, xc[u][j]);
        } else {
          const float sc = __uint_as_float((unsigned)wc[u][i] << 23);
          const unsigned q[4] = {wv[u][i].x, wv[u][i].y, wv[u][i].z, wv[u][i].w};
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            uint4 b;
            b.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[s], sc, 0));
            b.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[s], sc, 1));
            b.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[s], sc, 2));
            b.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[s], sc, 3));
#pragma unroll
            for (int j = 0; j < MT; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, b), __builtin_bit_cast(bf16x8_t, xv[u][j][s]),
                                                                  acc[i][j], 0, 0, 0);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
      red[(wave * NF * MT + i * MT + j) * 64 + lane] = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
  __syncthreads();
  for (int t = tid; t < NF * MT * 64; t += 512) {
    const int f = t >> 6, l = t & 63, i = f / MT, j = f - i * MT;
    const int n = n0 + i * 16 + (l >> 4) * 4;
    const long long m = m0 + j * 16 + (l & 15);
    if (m >= p.rows || n >= p.n) continue;
    float4 s = red[t];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      const float4 o = red[w * NF * MT * 64 + t];
      s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
    }
    float v[4] = {s.x, s.y, s.z, s.w};
    OUT* dst = static_cast<OUT*>(p.out) + m * p.n + n;
    if (p.bias != nullptr)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += n + e < p.n ? p.bias[n + e] : 0.f;
    if (p.vec_out) {                                       // n a multiple of 4 elements
      if constexpr (sizeof(OUT) == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      else *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.n) Elem<OUT>::st(dst + e, v[e]);
    }
  }
}

template <typename K>
static int mx_allow_lds(const char* what, K kern, int bytes, bool& done) {
  if (done || bytes <= 64 * 1024) return LDM_OK;
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) { set_error("%s: hipFuncSetAttribute: %s", what, hipGetErrorString(e)); return LDM_EHIP; }
  done = true;
  return LDM_OK;
}

template <int BM, int BN, int WM, int WN, int S, typename OUT>
static int launch_mx4_gemm(Mx4Params& p, hipStream_t st) {
  p.tiles_m = (int)((p.rows + BM - 1) / BM);
  p.tiles_n = (p.n + BN - 1) / BN;
  constexpr int smem = (BM + BN) * (S * 64 + 2 * 16);
  auto kern = mx4_gemm_kernel<BM, BN, WM, WN, S, OUT>;
  static bool done = false;
  if (int rc = mx_allow_lds("ldm_mx4_linear", kern, smem, done)) return rc;
  hipLaunchKernelGGL(kern, dim3(p.tiles_m * p.tiles_n), dim3(64 * WM * WN), smem, st, p);
  return LDM_OK;
}

template <bool MX, int MT, int NF, bool VEC, typename OUT>
static int launch_mx4_rows(const Mx4Params& p, hipStream_t st) {
  constexpr int smem = 8 * NF * MT * 1024;
  auto kern = mx4_rows_kernel<MX, MT, NF, VEC, OUT>;
  static bool done = false;
  if (int rc = mx_allow_lds("ldm_mx4_linear", kern, smem, done)) return rc;
  hipLaunchKernelGGL(kern, dim3((p.n + 16 * NF - 1) / (16 * NF), (unsigned)((p.rows + 16 * MT - 1) / (16 * MT))), dim3(512), smem, st, p);
  return LDM_OK;
}

template <bool MX, bool VEC, typename OUT>
static int rows_by_size(const Mx4Params& p, hipStream_t st) {
  const bool wide = p.n >= 32 * 256;                       // two fragments of w a wave once every CU has a workgroup of them
  if (p.rows <= 16) return wide ? launch_mx4_rows<MX, 1, 2, VEC, OUT>(p, st) : launch_mx4_rows<MX, 1, 1, VEC, OUT>(p, st);
  if (p.rows <= 32) return launch_mx4_rows<MX, 2, 1, VEC, OUT>(p, st);
  return launch_mx4_rows<MX, 4, 1, VEC, OUT>(p, st);
}

template <typename OUT>
static int mx4_linear_out(Mx4Params& p, bool mx, bool vec_x, hipStream_t st) {
  if (!mx) return vec_x ? rows_by_size<false, true, OUT>(p, st) : rows_by_size<false, false, OUT>(p, st);
  if (p.rows <= 64) return rows_by_size<true, true, OUT>(p, st);
  const long long tiles = ((p.rows + 255) / 256) * ((p.n + 255) / 256);
  if (tiles >= 128) return launch_mx4_gemm<256, 256, 2, 4, 4, OUT>(p, st);
  return launch_mx4_gemm<128, 128, 2, 2, 4, OUT>(p, st);
}

}  // namespace ldm

using namespace ldm;

extern "C" int ldm_mx4_linear(const void* x, const void* x_scale, const void* w, const void* w_scale, const float* bias, void* out,
                              int out_dtype, long long rows, int n, int k, void* stream) {
  LDM_REQUIRE(dtype_ok(out_dtype), "ldm_mx4_linear: bad dtype %d", out_dtype);
  LDM_REQUIRE(rows >= 0 && n >= 1 && k >= 1 && k <= (1 << 22), "ldm_mx4_linear: bad sizes (rows=%lld n=%d k=%d)", rows, n, k);
  if (rows == 0) return LDM_OK;
  LDM_REQUIRE(x && w && w_scale && out, "ldm_mx4_linear: null pointer");
  const bool mx = x_scale != nullptr;
  const size_t es = dtype_size(out_dtype);
  LDM_REQUIRE(aligned16(w) && (reinterpret_cast<uintptr_t>(w_scale) & 3) == 0 && (!mx || (aligned16(x) && (reinterpret_cast<uintptr_t>(x_scale) & 3) == 0)) &&
                  (mx || (reinterpret_cast<uintptr_t>(x) & 1) == 0) && (reinterpret_cast<uintptr_t>(bias) & 3) == 0 &&
                  reinterpret_cast<uintptr_t>(out) % es == 0,
              "ldm_mx4_linear: unaligned pointer");
  Mx4Params p;
  p.x = static_cast<const unsigned char*>(x); p.xs = static_cast<const unsigned char*>(x_scale);
  p.w = static_cast<const unsigned char*>(w); p.ws = static_cast<const unsigned char*>(w_scale);
  p.bias = bias; p.out = out; p.rows = rows; p.n = n; p.k = k;
  p.blocks = mx_blocks(k); p.sstride = mx_scale_stride(k); p.nk = (p.blocks + 3) / 4;
  p.tiles_m = p.tiles_n = 0;
  p.vec_out = aligned16(out) && (n * es) % 16 == 0;
  LDM_REQUIRE(rows <= 64LL * 65535 || mx, "ldm_mx4_linear: %lld rows of bfloat16", rows);
  LDM_REQUIRE(((rows + 127) / 128) * ((n + 127LL) / 128) < (1LL << 31), "ldm_mx4_linear: too large (rows=%lld n=%d)", rows, n);
  hipStream_t st = (hipStream_t)stream;
  const bool vec_x = !mx && aligned16(x) && k % 8 == 0;
  const int rc = out_dtype == LDM_BF16 ? mx4_linear_out<bf16_t>(p, mx, vec_x, st) : mx4_linear_out<float>(p, mx, vec_x, st);
  if (rc) return rc;
  LDM_HIP_CHECK_LAUNCH("ldm_mx4_linear");
  return LDM_OK;
}
