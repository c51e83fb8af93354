// Products with block-scaled operands on the gfx950 matrix cores: linear layers with mx4 (4-bit) weights.
//
//   out[m][n] = bias[n] + sum_k x[m][k] w[n][k]
//
// Both operands mx4: v_mfma_scale_f32_32x32x64_f8f6f4.  A lane's operand is 32 consecutive k of one row -- one block, 16 bytes as stored --
// and its scale byte; products and sums are float32 inside the instruction, so nothing is rounded before the output.  The weights
// are the instruction's first operand: a lane then holds four consecutive n of one m.
//   mx4_gemm_kernel   large outputs.  8192^3: 310-340 us, 3.2-3.5 PFLOP/s (a loop of this instruction alone on random operands, without
//                     any loads: 6.4); 32768 x 2560, k = 320: 51 us, 168 MB of output at 3.3 TB/s.
//   mx_gemm_kernel    small and medium outputs, and plain bf16 operands (the product behind the widening of the weights): 8192 x 640, k =
//                     5120 in bf16: 60 us, 890 TFLOP/s; 154 x 768, k = 1312: 7.5 us.
//   mx4_rows_kernel   few rows of x, where the weights' bytes are what counts: 16 x 10240, k = 8192: 13 us, 3.3 TB/s.
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
  int vec_out;                 // four neighbours of a row can be stored at once (few rows)
};

// bijective XCD remap: workgroups b and b + 8 share an XCD; every XCD gets a contiguous run of tiles
__device__ __forceinline__ int mx_xcd_remap(int bid, int nblk) {
  const int q = nblk >> 3, r = nblk & 7, x = bid & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (bid >> 3);
}

// 16 / 4 bytes a lane from a raw buffer (base, bytes) into LDS, lane-linear from `lds`; a lane offset past `bytes` gives zeros
__device__ __forceinline__ void mx_dma16(const void* base, unsigned bytes, unsigned char* lds, unsigned voff, int soff) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void mx_dma4(const void* base, unsigned bytes, unsigned char* lds, unsigned voff, int soff) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 4, voff, soff, 0, 0);
}

// LDS reads that the caller waits for: around reads of its own the compiler would wait for every LDS-DMA in flight, also those of
// the steps ahead.
template <int OFF>
__device__ __forceinline__ void lds_read16(i32x4_t& v, unsigned addr) {
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void lds_read4(int& v, unsigned addr) {
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void lds_write16(unsigned addr, i32x4_t v) {
  asm volatile("ds_write_b128 %0, %1 offset:%2" ::"v"(addr), "v"(v), "n"(OFF) : "memory");
}
// no use of v moves above the wait in front of this
__device__ __forceinline__ void stay_below(i32x4_t& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void stay_below(int& v) { asm volatile("" : "+v"(v)); }

// A row's last block may be cut short, and so may its last word of scales.  What is stored behind them counts for nothing: the scale bytes
// behind the last block are left out where a lane's byte is taken from the word, and x's elements behind the last column -- that is
// enough, a product needs both of its factors -- are cleared in LDS once they have landed, behind branches that rows of whole blocks
// never take (in registers, in every step or behind branches, it cost 2-9 % of all products).
__device__ __forceinline__ unsigned scale_bytes(int blocks) { return blocks & 3 ? (1u << 8 * (blocks & 3)) - 1 : ~0u; }   // of the last word
// selector of byte `block` of a scale word whose last block is `last` (12: zero, as is the byte behind the last block)
__device__ __forceinline__ unsigned scale_pick(int block, int last) { return block <= last ? (unsigned)block : 12u; }
__device__ __forceinline__ int scale_take(int word, unsigned pick) { return (int)__builtin_amdgcn_perm(0u, (unsigned)word, pick); }
__device__ __forceinline__ int last_columns(const Mx4Params& p) { return p.k - (p.blocks - 1) * 32; }                    // of the last block
// x's elements, in LDS: row r's last block lies at image + r PITCH + 16 (chunk ^ swizzle(r)); THREADS share the rows, those left over take the
// last one again (which changes nothing), and the caller lets them meet afterwards
template <int ROWS, int PITCH, int THREADS, typename SWZ>
__device__ __forceinline__ void clear_behind(unsigned image, int chunk, int live, int thread, SWZ swizzle) {
#pragma unroll
  for (int r0 = 0; r0 < ROWS; r0 += THREADS) {
    const int r = min(r0 + thread, ROWS - 1);
    const unsigned at = image + r * PITCH + ((chunk ^ swizzle(r)) << 4);
    i32x4_t v;
    lds_read16<0>(v, at);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    stay_below(v);
#pragma unroll
    for (int d = 0; d < 4; ++d) {                          // columns 8 d .. + 7
      const int c = live - 8 * d;
      v[d] &= c >= 8 ? -1 : c <= 0 ? 0 : (1 << 4 * c) - 1;
    }
    lds_write16<0>(at, v);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

template <bool MX, int H>
__device__ __forceinline__ void mx_mfma(f32x16_t& c, i32x4_t a, i32x4_t b, int sa, int sb) {
  if constexpr (MX)
    c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(i32x8_t{a[0], a[1], a[2], a[3], 0, 0, 0, 0}, i32x8_t{b[0], b[1], b[2], b[3], 0, 0, 0, 0}, c, 4, 4,
                                                        2 * H, sa, 2 * H, sb);
  else
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// A wave's MI x NI tiles of 32 x 32 (register r of tile (i, j): column n0 + 32 j + 8 (r / 4) + 4 (lane / 32) + r % 4, row m0 + 32 i + lane % 32)
// plus bias into the output: 32 rows at a time through the wave's own LDS, then whole 16-byte pieces of rows.
template <int NI, typename OUT>
constexpr int store_pitch() { return NI * 32 * (int)sizeof(OUT) + 16; }
template <int MI, int NI, typename OUT>
__device__ __forceinline__ void store_tiles(const Mx4Params& p, const f32x16_t (&acc)[MI][NI], unsigned char* cst, long long m0, int n0, int lane) {
  constexpr int WTN = NI * 32;
  const int fr = lane & 31, fh = lane >> 5;
  constexpr int PITCH = store_pitch<NI, OUT>();
  constexpr int EPR = 16 / (int)sizeof(OUT);               // elements of a piece
  float bv[NI][4][4];
  if (p.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) bv[j][q][e] = p.bias[min(n0 + j * 32 + 8 * q + 4 * fh + e, p.n - 1)];
  } else {
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) bv[j][q][e] = 0.f;
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
#pragma unroll 4
    for (int t = 0; t < 32 * PPR / 64; ++t) {
      const int piece = t * 64 + lane, r = piece / PPR, c = (piece - r * PPR) * EPR;
      const long long m = m0 + i * 32 + r;
      const int n = n0 + c;
      if (m >= p.rows || n >= p.n) continue;
      OUT* dst = static_cast<OUT*>(p.out) + m * p.n + n;
      const unsigned char* s = cst + r * PITCH + c * (int)sizeof(OUT);
      if (n + EPR <= p.n) {
        store16_any(dst, *reinterpret_cast<const uint4*>(s));
      } else {                                             // the end of a row
#pragma unroll 1
        for (int e = 0; n + e < p.n; ++e) dst[e] = reinterpret_cast<const OUT*>(s)[e];
      }
    }
    LDM_LOCKSTEP();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// Large products: tile of BM (rows of x) x BN (rows of w) by WM x WN waves; a step is 64 bytes of every row (128 columns of mx4, four
// blocks), S slots of LDS.  16-byte chunks of a row are XOR-swizzled by (row >> 1) & 3 (the DMA writes lane-linear, so the
// swizzle is applied to the lane's SOURCE chunk and again on the read): eight consecutive rows then lie in eight different 16-byte
// columns of the 128-byte LDS line.  A chunk is a block, what a lane gives one matrix instruction, so chunks past the end
// of a row are fetched from beyond the descriptor's end (zeros), and rows past the end likewise.
//
// Each step has two halves, one matrix instruction deep; the registers of one are read while the other multiplies:
//   multiply half 0 | read half 1;  wait for the next step's DMA, barrier;  multiply half 1 | refill the slot, read the next half 0
// so the matrix cores wait for nothing but the skew at the one barrier a step.
//
// Scales: one 32-bit word a row and step.  From four steps on, 16 bytes (four steps) a row at a time in one DMA instruction, the last
// ones ending with the row (a fetch never passes its row); with fewer steps word by word, once.
template <int BM, int BN, int WM, int WN, int S, typename OUT>
__global__ void __launch_bounds__(64 * WM * WN, 2)
mx4_gemm_kernel(const Mx4Params p) {
  constexpr int NT = 64 * WM * WN, ROWS = BM + BN;
  constexpr int IT = ROWS * 4 / NT;                        // tile DMA instructions of a wave a step
  constexpr int SIT = (ROWS + NT - 1) / NT;                // scale DMA instructions of a wave (16 bytes a row)
  static_assert(BM * 4 % NT == 0 && BN * 4 % NT == 0 && BM % 64 == 0 && BN % 64 == 0, "tile / threads mismatch");
  constexpr int STAGE = ROWS * 64;
  constexpr int SCALES = ROWS * 16;              // one group of four steps
  constexpr int WTM = BM / WM, WTN = BN / WN, MI = WTM / 32, NI = WTN / 32;
  constexpr unsigned OOB = 0x80000000u;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane & 31, fh = lane >> 5;

  const int tile = mx_xcd_remap(blockIdx.x, gridDim.x);
  // bands of 4 tile rows walked column by column: the tiles in flight on one XCD share their operands in its L2 (bands of 8: 3 % slower
  // at 8192 x 8192 x 8192)
  const int band = 4 * p.tiles_n, g4 = tile / band, in = tile - g4 * band;
  const int brows = min(p.tiles_m - g4 * 4, 4);
  const int tn = in / brows, tm = g4 * 4 + (in - tn * brows);
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
  const int chunk = (tid & 3) ^ ((tid >> 3) & 3);          // NT / 4 rows on, the swizzle is the same
  static_assert(NT / 4 % 8 == 0, "swizzle period");
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int row = (it * NT + tid) >> 2;
    voff[it] = (unsigned)(row < BM ? row : row - BM) * rb + chunk * 16;
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
          if (r0 >= ROWS) continue;
          if (r0 < BM) mx_dma4(xsbase, xsbytes, dst + (j * ROWS + r0) * 4, (unsigned)row * p.sstride, j * 4);
          else mx_dma4(wsbase, wsbytes, dst + (j * ROWS + r0) * 4, (unsigned)(row - BM) * p.sstride, j * 4);
        }
    } else {
      const int first = group_first(g) * 4;
#pragma unroll
      for (int it = 0; it < SIT; ++it) {
        const int r0 = it * NT + wave * 64, row = r0 + lane;
        if (r0 >= ROWS) continue;
        if (r0 < BM) mx_dma16(xsbase, xsbytes, dst + r0 * 16, (unsigned)row * p.sstride, first);
        else mx_dma16(wsbase, wsbytes, dst + r0 * 16, (unsigned)(row - BM) * p.sstride, first);
      }
    }
  };
  // a step past the last one is fetched like any other (zeros, into a slot that nobody reads): the loop needs no case for its end
  auto stage = [&](int kt) {
    if ((kt & 3) == 0 && kt < nk) stage_scales(kt >> 2);
    unsigned char* dst = smem + (kt % S) * STAGE + wave * 1024;
    const bool past = kt * 4 + chunk >= p.blocks;
#pragma unroll
    for (int it = 0; it < IT; ++it) {                      // 16 whole rows a wave and instruction, all of one operand
      const unsigned vo = past ? OOB : voff[it];
      if (it * NT < BM * 4) mx_dma16(xbase, xbytes, dst + it * NT * 16, vo, kt * 64);
      else mx_dma16(wbase, wbytes, dst + it * NT * 16, vo, kt * 64);
    }
  };

  f32x16_t acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  // fragments of the two halves; scales of this step (shifted: byte 0 this lane's block of half 0, byte 2 of half 1) and of the next
  i32x4_t xf[2][MI], wf[2][NI];
  int sx[MI], sw[NI], nsx[MI], nsw[NI];
#pragma unroll
  for (int i = 0; i < MI; ++i) sx[i] = nsx[i] = 0;
#pragma unroll
  for (int j = 0; j < NI; ++j) sw[j] = nsw[j] = 0;
  const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const int swz = (fr >> 1) & 3;
  const unsigned xaddr = lds + (wm * WTM + fr) * 64 + ((fh ^ swz) << 4), waddr = lds + (BM + wn * WTN + fr) * 64 + ((fh ^ swz) << 4);
  const int sstep = word_scales ? 4 : 16;
  const unsigned xsaddr = lds + S * STAGE + (wm * WTM + fr) * sstep, wsaddr = lds + S * STAGE + (BM + wn * WTN + fr) * sstep;

  // q-th read of half H of the step whose image starts at `slot`: the scale words come with half 0
  constexpr int READS = MI + NI;
  static_assert(READS <= MI * NI, "one read behind each instruction");
  auto read = [&]<int H, int Q>(std::integral_constant<int, H>, std::integral_constant<int, Q>, unsigned slot) {
    constexpr int i = Q < MI ? Q : 0, j = Q < MI ? 0 : Q - MI;
    if constexpr (Q < MI) lds_read16<i * 2048>(xf[H][i], (xaddr ^ (H * 32)) + slot);
    else lds_read16<j * 2048>(wf[H][j], (waddr ^ (H * 32)) + slot);
  };
  auto read_scales = [&](int kt) {
    const int g = kt >> 2, word = kt - group_first(g);
    const unsigned o = (g & 1) * SCALES + word * (word_scales ? ROWS * 4 : 4);
    const unsigned step = 32 * sstep;
#pragma unroll
    for (int i = 0; i < MI; ++i) lds_read4<0>(nsx[i], xsaddr + o + i * step);
#pragma unroll
    for (int j = 0; j < NI; ++j) lds_read4<0>(nsw[j], wsaddr + o + j * step);
  };
  auto landed = [&]<int H>(std::integral_constant<int, H>, unsigned pick) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < MI; ++i) asm volatile("" : "+v"(xf[H][i]));   // no use moves above the wait
#pragma unroll
    for (int j = 0; j < NI; ++j) asm volatile("" : "+v"(wf[H][j]));
    if constexpr (H == 0) {
#pragma unroll
      for (int i = 0; i < MI; ++i) { asm volatile("" : "+v"(nsx[i])); sx[i] = scale_take(nsx[i], pick); }
#pragma unroll
      for (int j = 0; j < NI; ++j) { asm volatile("" : "+v"(nsw[j])); sw[j] = scale_take(nsw[j], pick); }
    }
  };
  // half H of this step on the matrix cores; behind each of the first instructions a read of the other half (of `slot`)
  auto multiply = [&]<int H>(std::integral_constant<int, H>, unsigned slot) {
    [&]<int... Q>(std::integer_sequence<int, Q...>) {
      ([&] {
        constexpr int q = Q, i = q / NI, j = q % NI;
        mx_mfma<true, H>(acc[i][j], wf[H][j], xf[H][i], sw[j], sx[i]);
        if constexpr (q < READS) read(std::integral_constant<int, 1 - H>{}, std::integral_constant<int, q>{}, slot);
        __builtin_amdgcn_sched_barrier(0);
      }(), ...);
    }(std::make_integer_sequence<int, MI * NI>{});
  };
  // until this wave's DMA of the next step has landed; that of the S - 2 steps behind it may be in flight (a fetch of scales among them
  // only makes the wait stricter)
  auto dma_landed = [&] { asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * IT) : "memory"); };
  // bytes 0 and 2: this lane's scales of a step's two halves
  const unsigned whole = scale_pick(fh, 3) | scale_pick(fh + 2, 3) << 16;
  const unsigned ends = scale_pick(fh, (p.blocks - 1) & 3) | scale_pick(fh + 2, (p.blocks - 1) & 3) << 16;
  auto scales_of = [&](int kt) { return kt == nk - 1 ? ends : whole; };
  const int cut_step = (p.k & 31) ? nk - 1 : -1;
  auto cut = [&] {                                         // the last step has landed
    clear_behind<BM, 64, NT>(lds + (unsigned)((nk - 1) % S) * STAGE, (p.blocks - 1) & 3, last_columns(p), tid, [](int r) { return (r >> 1) & 3; });
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  constexpr std::integral_constant<int, 0> H0{};
  constexpr std::integral_constant<int, 1> H1{};

#pragma unroll
  for (int s = 0; s < S - 1; ++s) stage(s);
  dma_landed();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (__builtin_expect(cut_step == 0, 0)) cut();
  stage(S - 1);
  read_scales(0);
  [&]<int... Q>(std::integer_sequence<int, Q...>) {
    (read(H0, std::integral_constant<int, Q>{}, 0u), ...);
  }(std::make_integer_sequence<int, READS>{});
  landed(H0, scales_of(0));
  for (int kt = 0; kt < nk; ++kt) {
    multiply(H0, (unsigned)(kt % S) * STAGE);
    landed(H1, 0u);
    const int next = min(kt + 1, nk - 1);                  // behind the last step itself once more, unused
    dma_landed();
    __builtin_amdgcn_s_barrier();                          // every wave has read slot kt, and its part of the next step is there
    asm volatile("" ::: "memory");
    if (__builtin_expect(kt + 1 == cut_step, 0)) cut();
    stage(kt + S);
    read_scales(next);
    multiply(H1, (unsigned)(next % S) * STAGE);
    landed(H0, scales_of(next));
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();                                         // the slots become the epilogue's

  static_assert(WM * WN * 32 * store_pitch<NI, OUT>() <= S * STAGE + 2 * SCALES, "epilogue image");
  store_tiles<MI, NI, OUT>(p, acc, smem + wave * 32 * store_pitch<NI, OUT>(), m0 + wm * WTM, n0 + wn * WTN, lane);
}

// Tile of BM (rows of x) x BN (rows of w).  A step is 128 bytes of every row (MX: 256 columns of mx4, eight blocks; else 64 columns of
// bf16): the chip's L2 hands out lines of 128 bytes, and LDS-DMA of 64 of them a row gets half the rate (17 against 29 TB/s over all CUs).
// 16-byte chunks of a row are XOR-swizzled by row & 7 (the DMA writes lane-linear, so the swizzle is applied to the lane's SOURCE chunk
// and again on the read): eight consecutive rows then lie in eight different 16-byte columns of LDS.  A chunk is what a lane gives one
// matrix instruction -- a block, or 8 columns of bf16 -- so chunks past the end of a row are fetched from beyond the descriptor's end
// (zeros), rows past the end likewise, and steps past the end too: their number is rounded up to an even one.
//
// S slots of LDS.  The registers of a whole step -- four rounds of matrix instructions -- are read while the step before multiplies, reads and
// DMA spread between the instructions, one barrier a step.  What bounds the loop is LDS: a wave's tile of 64 x 64 reads 0.031 rows of
// operands a product, which takes as long as its instructions; the 64 x 160 of the 256 x 160 tile reads 0.022, but the 32 x 160 of the
// 128 x 160 tile 0.0375.
//   KW == 1: WM x WN waves share the tile.
//   KW > 1:  few tiles, where a launch is as long as one workgroup's chain of steps: the KW waves of a workgroup each take a contiguous part
//            of the columns of the whole tile, with a ring of their own and no barrier, and add up through LDS in a fixed order.
//
// Scales (MX): two 32-bit words a row and step.  From four words a row on, 16 bytes (two steps) a row at a time in one DMA instruction, the
// last ones ending with the row (a fetch never passes its row); with fewer words one by one, once.  Words past the end count as zero: what
// LDS holds there may be another row's NaN.
template <int BM, int BN, int WM, int WN, int KW, int S, bool MX, typename OUT>
__global__ void __launch_bounds__(64 * WM * WN * KW, KW > 1 || BM * BN > 16384 ? 1 : 2)
mx_gemm_kernel(const Mx4Params p) {
  static_assert(KW == 1 || (WM == 1 && WN == 1), "a wave of its own tile or of its own columns");
  constexpr int NT = 64 * WM * WN, ROWS = BM + BN;
  constexpr int IT = ROWS * 8 / NT;                        // DMA instructions of a wave a step
  constexpr int STAGE = ROWS * 128;
  constexpr int SROWS = (ROWS + 63) / 64 * 64, SCALES = MX ? SROWS * 16 : 0;   // one group of two steps
  constexpr int RING = S * STAGE + 2 * SCALES;
  constexpr int WTM = BM / WM, WTN = BN / WN, MI = WTM / 32, NI = WTN / 32;
  constexpr unsigned OOB = 0x80000000u;
  static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0 && BM % 64 == 0 && (S - 2) * IT < 64, "tile / threads mismatch");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = KW > 1 ? wave : 0, gw = KW > 1 ? 0 : wave;
  const int gt = KW > 1 ? lane : tid;                      // thread of the group that shares a ring
  const int wm = gw / WN, wn = gw % WN;
  const int fr = lane & 31, fh = lane >> 5;

  const int tile = mx_xcd_remap(blockIdx.x, gridDim.x);
  // bands of 4 tile rows walked column by column: the tiles in flight on one XCD share their operands in its L2
  const int band = 4 * p.tiles_n, g4 = tile / band, in = tile - g4 * band;
  const int brows = min(p.tiles_m - g4 * 4, 4);
  const int tn = in / brows, tm = g4 * 4 + (in - tn * brows);
  const long long m0 = (long long)tm * BM;
  const int n0 = tn * BN;

  const int rb = MX ? p.blocks * 16 : p.k * 2, chunks = rb >> 4;
  const int mrows = (int)min((long long)BM, p.rows - m0), nrows = min(BN, p.n - n0);
  const unsigned char* xbase = p.x + m0 * rb;
  const unsigned char* wbase = p.w + (long long)n0 * rb;
  const unsigned xbytes = (unsigned)mrows * rb, wbytes = (unsigned)nrows * rb;
  const int chunk = (gt & 7) ^ ((gt >> 3) & 7);
  const unsigned voff = (unsigned)(gt >> 3) * rb + chunk * 16;

  const int per = ((p.nk + KW - 1) / KW + 1) & ~1, s0 = kw * per;
  unsigned char* const ring = smem + kw * RING;

  const int nwords = p.sstride >> 2;                       // scale words a row
  const bool word_scales = nwords < 4;
  // word w of row r of group g lies at group + r * row_step + (w - first word of the group) * word_step
  auto group_first = [&](int kt) { return word_scales ? 0 : min((s0 + (kt & ~1)) * 2, nwords - 4); };
  auto stage_scales = [&](int kt) {                        // of steps kt and kt + 1, kt even
    unsigned char* dst = ring + S * STAGE + ((kt >> 1) & 1) * SCALES;
    const unsigned char* xs = p.xs + m0 * p.sstride;
    const unsigned char* ws = p.ws + (long long)n0 * p.sstride;
    const unsigned xsb = (unsigned)mrows * p.sstride, wsb = (unsigned)nrows * p.sstride;
#pragma unroll
    for (int it = 0; it < (SROWS + NT - 1) / NT; ++it) {
      const int r0 = it * NT + gw * 64;
      if (r0 >= SROWS) continue;
      const bool isx = r0 < BM;
      const unsigned vo = (unsigned)(r0 - (isx ? 0 : BM) + lane) * p.sstride;
      if (word_scales) {
        for (int j = 0; j < nwords; ++j) mx_dma4(isx ? xs : ws, isx ? xsb : wsb, dst + (j * SROWS + r0) * 4, vo, j * 4);
      } else {
        mx_dma16(isx ? xs : ws, isx ? xsb : wsb, dst + r0 * 16, vo, group_first(kt) * 4);
      }
    }
  };
  auto stage_part = [&](int kt, int it) {                  // instruction `it` of step s0 + kt
    unsigned char* dst = ring + (kt % S) * STAGE + gw * 1024 + it * NT * 16;
    const bool past = kt >= per || (s0 + kt) * 8 + chunk >= chunks;
    const int so = (s0 + kt) * 128;
    if (it * NT < BM * 8) mx_dma16(xbase, xbytes, dst, past ? OOB : voff + it * (NT / 8) * rb, so);
    else mx_dma16(wbase, wbytes, dst, past ? OOB : voff + (it * (NT / 8) - BM) * rb, so);
  };
  auto stage_begin = [&](int kt) {
    if constexpr (MX)
      if ((kt & 1) == 0 && kt < per) stage_scales(kt);
  };
  auto stage = [&](int kt) {
    stage_begin(kt);
#pragma unroll
    for (int it = 0; it < IT; ++it) stage_part(kt, it);
  };

  f32x16_t acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  i32x4_t xf[2][4][MI], wf[2][4][NI];                      // [set][round of the step]
  // scale words of rounds 0, 1 and 2, 3: as read, and shifted so that byte 0 / byte 2 is this lane's block of the even / odd round
  int rx[2][MI], rw[2][NI], sx[2][MI], sw[2][NI];
#pragma unroll
  for (int o = 0; o < 2; ++o) {
#pragma unroll
    for (int i = 0; i < MI; ++i) rx[o][i] = sx[o][i] = 0;
#pragma unroll
    for (int j = 0; j < NI; ++j) rw[o][j] = sw[o][j] = 0;
  }
  const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)ring;
  const int swz = fr & 7;
  const unsigned xaddr = lds + (wm * WTM + fr) * 128 + ((fh ^ swz) << 4), waddr = lds + (BM + wn * WTN + fr) * 128 + ((fh ^ swz) << 4);
  constexpr int READS = 4 * (MI + NI), MM = 4 * MI * NI;
  static_assert(READS <= 2 * MM, "every read has its place");
  auto read = [&]<int SET, int Q>(std::integral_constant<int, SET>, std::integral_constant<int, Q>, unsigned slot) {
    constexpr int h = Q / (MI + NI), q = Q % (MI + NI), i = q < MI ? q : 0, j = q < MI ? 0 : q - MI;
    if constexpr (q < MI) lds_read16<i * 4096>(xf[SET][h][i], (xaddr ^ (h * 32)) + slot);
    else lds_read16<j * 4096>(wf[SET][h][j], (waddr ^ (h * 32)) + slot);
  };
  const int row_step = word_scales ? 4 : 16, word_step = word_scales ? SROWS * 4 : 4;
  auto read_scales = [&](int kt) {
    if constexpr (MX) {
      const unsigned base = lds + S * STAGE + ((kt >> 1) & 1) * SCALES;
      const int w = (s0 + kt) * 2 - group_first(kt);
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const unsigned at = base + min(w + o, 3) * word_step;
#pragma unroll
        for (int i = 0; i < MI; ++i) lds_read4<0>(rx[o][i], at + (wm * WTM + i * 32 + fr) * row_step);
#pragma unroll
        for (int j = 0; j < NI; ++j) lds_read4<0>(rw[o][j], at + (BM + wn * WTN + j * 32 + fr) * row_step);
      }
    }
  };
  auto landed = [&]<int SET>(std::integral_constant<int, SET>, int kt) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int h = 0; h < 4; ++h) {
#pragma unroll
      for (int i = 0; i < MI; ++i) stay_below(xf[SET][h][i]);
#pragma unroll
      for (int j = 0; j < NI; ++j) stay_below(wf[SET][h][j]);
    }
    if constexpr (MX) {
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const int word = (s0 + kt) * 2 + o;
        const unsigned there = word < nwords - 1 ? ~0u : word == nwords - 1 ? scale_bytes(p.blocks) : 0u;
#pragma unroll
        for (int i = 0; i < MI; ++i) { stay_below(rx[o][i]); sx[o][i] = (int)(((unsigned)rx[o][i] & there) >> (8 * fh)); }
#pragma unroll
        for (int j = 0; j < NI; ++j) { stay_below(rw[o][j]); sw[o][j] = (int)(((unsigned)rw[o][j] & there) >> (8 * fh)); }
      }
    }
  };
  auto next_here = [&] {                                   // the next step's DMA has landed, and the slot of this one is free
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * IT) : "memory");   // a fetch of scales behind it only makes the wait stricter
    if constexpr (KW == 1) __builtin_amdgcn_s_barrier();
    else LDM_LOCKSTEP();
    asm volatile("" ::: "memory");
  };
  const int cut_step = MX && (p.k & 31) ? p.nk - 1 - s0 : -1;
  auto cut = [&](int kt) {                                 // step kt has landed
    if constexpr (MX) {
      if (__builtin_expect(kt != cut_step, 1)) return;
      clear_behind<BM, 128, NT>(lds + (unsigned)(kt % S) * STAGE, (p.blocks - 1) & 7, last_columns(p), gt, [](int r) { return r & 7; });
      if constexpr (KW == 1) __builtin_amdgcn_s_barrier();
      else LDM_LOCKSTEP();
      asm volatile("" ::: "memory");
    }
  };
  // step kt from register set SET; the next one's reads, and the DMA into the slot that is free now, between the matrix instructions
  auto step = [&]<int SET>(std::integral_constant<int, SET>, int kt) {
    next_here();
    cut(kt + 1);
    stage_begin(kt + S);
    read_scales(kt + 1);
    const unsigned slot = (unsigned)((kt + 1) % S) * STAGE;
    [&]<int... Q>(std::integer_sequence<int, Q...>) {
      ([&] {
        constexpr int q = Q, h = q / (MI * NI), i = q / NI % MI, j = q % NI;
        mx_mfma<MX, h & 1>(acc[i][j], wf[SET][h][j], xf[SET][h][i], sw[h >> 1][j], sx[h >> 1][i]);
        if constexpr (2 * q < READS) read(std::integral_constant<int, 1 - SET>{}, std::integral_constant<int, 2 * q>{}, slot);
        if constexpr (2 * q + 1 < READS) read(std::integral_constant<int, 1 - SET>{}, std::integral_constant<int, 2 * q + 1>{}, slot);
#pragma unroll
        for (int it = q * IT / MM; it < (q + 1) * IT / MM; ++it) stage_part(kt + S, it);
        __builtin_amdgcn_sched_barrier(0);
      }(), ...);
    }(std::make_integer_sequence<int, MM>{});
    landed(std::integral_constant<int, 1 - SET>{}, kt + 1);
  };
  constexpr std::integral_constant<int, 0> SET0{};
  constexpr std::integral_constant<int, 1> SET1{};

#pragma unroll
  for (int t = 0; t < S - 1; ++t) stage(t);
  next_here();
  cut(0);
  stage(S - 1);
  read_scales(0);
  [&]<int... Q>(std::integer_sequence<int, Q...>) {
    (read(SET0, std::integral_constant<int, Q>{}, 0u), ...);
  }(std::make_integer_sequence<int, READS>{});
  landed(SET0, 0);
  for (int kt = 0; kt < per; kt += 2) {
    step(SET0, kt);
    step(SET1, kt + 1);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if constexpr (KW == 1) {
    __syncthreads();                                       // the slots become the epilogue's
    static_assert(KW > 1 || WM * WN * 32 * store_pitch<NI, OUT>() <= RING, "epilogue image");
    store_tiles<MI, NI, OUT>(p, acc, smem + wave * 32 * store_pitch<NI, OUT>(), m0 + wm * WTM, n0 + wn * WTN, lane);
  } else {
    // tile t of the MI NI of this output tile is wave t's to add up and store
    static_assert(KW == 1 || (MI * NI == KW && MI * NI * 4096 <= RING && 32 * store_pitch<1, OUT>() <= RING), "a tile a wave");
    LDM_LOCKSTEP();
#pragma unroll
    for (int t = 0; t < MI * NI; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        reinterpret_cast<float4*>(ring)[(t * 4 + q) * 64 + lane] = make_float4(acc[t / NI][t % NI][4 * q], acc[t / NI][t % NI][4 * q + 1],
                                                                               acc[t / NI][t % NI][4 * q + 2], acc[t / NI][t % NI][4 * q + 3]);
    __syncthreads();
    f32x16_t sum[1][1];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float4 v = reinterpret_cast<const float4*>(smem)[(wave * 4 + q) * 64 + lane];
#pragma unroll
      for (int w = 1; w < KW; ++w) {
        const float4 o = reinterpret_cast<const float4*>(smem + w * RING)[(wave * 4 + q) * 64 + lane];
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      sum[0][0][4 * q] = v.x; sum[0][0][4 * q + 1] = v.y; sum[0][0][4 * q + 2] = v.z; sum[0][0][4 * q + 3] = v.w;
    }
    __syncthreads();
    store_tiles<1, 1, OUT>(p, sum, ring, m0 + wave / NI * 32, n0 + wave % NI * 32, lane);
  }
}

// --------------------------------------------------------------------------------------------------------- few rows
// 16 NF rows of w and 16 MT rows of x a workgroup; its NW waves take a contiguous part of the columns each, 128 a step, and add up through
// LDS in a fixed order.  What is to be had is the weights' bytes at the memory's rate, so every wave keeps S steps of its own in LDS
// by LDS-DMA (no barrier: no wave reads another's), four or more consecutive lanes to a row.  Loading the matrix instructions'
// fragments straight into registers -- consecutive lanes, different rows -- gives the address unit 16 bytes of every line at a
// time: 31 us instead of 14 at 16 x 8192 x 10240 (42 MB of weights; 9 us at the rate of a large copy).
//   MX  true: x in mx4, v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds row l % 16, block l / 16 of the step
//       false: x in bf16, four v_mfma_f32_16x16x32_bf16 a step.  Lane l holds row l % 16 again; the s-th takes columns 8 s .. + 7 of the
//              lane's block l / 16, which are dword s of its weights, widened to bf16 (exact: 2 significant bits) two at a time by the
//              conversion that takes the scale along, and chunk 4 (l / 16) + s of the 16 in the step's 256 bytes of x.
// Chunks of a row are XOR-swizzled as in the tiles above: weights (64 bytes a row) by (row >> 1) & 3, x in bf16 (256) by row & 15.
// DMAX: x can be fetched in 16-byte chunks (k a multiple of 8, x aligned); otherwise it goes through registers, zeros past the row's end.
// until the LDS-DMA of all but the newest min(N, behind) steps of PER instructions has landed
template <int N, int PER>
__device__ __forceinline__ void wait_steps(int behind) {
  if constexpr (N == 0) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  } else {
    if (behind >= N) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N * PER) : "memory");
    else wait_steps<N - 1, PER>(behind);
  }
}

template <bool MX, int MT, int NF, int NW, int S, bool DMAX, typename OUT>
__global__ void __launch_bounds__(64 * NW)
mx4_rows_kernel(const Mx4Params p) {
  constexpr int XI = MX ? MT : 4 * MT;                     // x instructions of a step
  constexpr int SLOT = (NF + XI) * 1024;
  constexpr int SCALES = MX ? 2048 : 1024;                 // a group of four steps: 16 bytes a row
  constexpr int WAVE = S * SLOT + 2 * SCALES;
  constexpr int PER = NF + (DMAX ? XI : 0);                // LDS-DMA instructions of a step
  constexpr unsigned OOB = 0x80000000u;
  static_assert(NF * MT * 1024 <= WAVE && (S - 1) * PER < 64, "LDS image");
  // scales have room for two groups of four steps: step 4 g + 3 fetches step 4 g + 2 + S, which must not be of group g + 2
  static_assert(S <= 5, "scale groups");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int n0 = blockIdx.x * (16 * NF);
  const long long m0 = (long long)blockIdx.y * (16 * MT);
  const int nk = p.nk, rb = p.blocks * 16, xb = MX ? rb : p.k * 2;
  const int mrows = (int)min((long long)(16 * MT), p.rows - m0), nrows = min(16 * NF, p.n - n0);
  const unsigned char* wbase = p.w + (long long)n0 * rb;
  const unsigned char* wsbase = p.ws + (long long)n0 * p.sstride;
  const unsigned char* xbase = p.x + m0 * xb;
  const unsigned char* xsbase = MX ? p.xs + m0 * p.sstride : nullptr;
  const unsigned wbytes = (unsigned)nrows * rb, xbytes = (unsigned)mrows * xb;
  const unsigned wsbytes = (unsigned)nrows * p.sstride, xsbytes = (unsigned)mrows * p.sstride;

  const int per = (nk + NW - 1) / NW, s0 = wave * per, s1 = min(s0 + per, nk);
  const bool word_scales = nk < 4;                         // rows of less than 16 bytes of scales: a step at a time
  unsigned char* const mine = smem + wave * WAVE;
  const int wchunk = (lane & 3) ^ ((lane >> 3) & 3);
  const unsigned wvoff = (unsigned)(lane >> 2) * rb + wchunk * 16;
  const int srow = 16 * NF;

  auto stage = [&](int kt) {
    if (((kt - s0) & 3) == 0) {
      unsigned char* dst = mine + S * SLOT + (((kt - s0) >> 2) & 1) * SCALES;
      const unsigned wo = lane < srow ? (unsigned)lane * p.sstride : OOB, xo = lane < 16 * MT ? (unsigned)lane * p.sstride : OOB;
      if (word_scales) {
        mx_dma4(wsbase, wsbytes, dst, wo, kt * 4);
        if constexpr (MX) mx_dma4(xsbase, xsbytes, dst + 1024, xo, kt * 4);
      } else {
        const int first = min(kt, nk - 4) * 4;             // the last fetch ends with the row
        mx_dma16(wsbase, wsbytes, dst, wo, first);
        if constexpr (MX) mx_dma16(xsbase, xsbytes, dst + 1024, xo, first);
      }
    }
    unsigned char* dst = mine + (kt - s0) % S * SLOT;
    const bool past = kt * 4 + wchunk >= p.blocks;
#pragma unroll
    for (int i = 0; i < NF; ++i) mx_dma16(wbase, wbytes, dst + i * 1024, past ? OOB : wvoff + i * 16 * rb, kt * 64);
    dst += NF * 1024;
    if constexpr (MX) {
#pragma unroll
      for (int j = 0; j < MT; ++j) mx_dma16(xbase, xbytes, dst + j * 1024, past ? OOB : wvoff + j * 16 * rb, kt * 64);
    } else {
#pragma unroll
      for (int t = 0; t < XI; ++t) {
        const int row = 4 * t + fq, chunk = fr ^ (row & 15), col = kt * 128 + chunk * 8;
        if constexpr (DMAX) {
          mx_dma16(xbase, xbytes, dst + t * 1024, col >= p.k ? OOB : (unsigned)row * xb + chunk * 16, kt * 256);
        } else {
          uint4 v = make_uint4(0, 0, 0, 0);
          const int left = row >= mrows ? 0 : p.k - col;
          const bf16_t* src = reinterpret_cast<const bf16_t*>(xbase + (long long)row * xb) + col;
          if (left >= 8) {
            v = load16_any(src);
          } else if (left > 0) {
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = e < left ? src[e] : 0;
            v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
          }
          *reinterpret_cast<uint4*>(dst + t * 1024 + lane * 16) = v;
        }
      }
    }
  };

  f32x4_t acc[NF][MT];
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)mine;
  const unsigned waddr = lds + fr * 64 + ((fq ^ ((fr >> 1) & 3)) << 4);
  unsigned xaddr[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) xaddr[s] = lds + NF * 1024 + fr * 256 + (((4 * fq + s) ^ fr) << 4);
  const int sstep = word_scales ? 4 : 16;
  const unsigned saddr = lds + S * SLOT + fr * sstep;
  const int cut_step = (p.k & 31) ? nk - 1 : -1;           // MX: a last block that is not whole
  const unsigned whole = scale_pick(fq, 3) | 0x0c0c0c00u, ends = scale_pick(fq, (p.blocks - 1) & 3) | 0x0c0c0c00u;   // byte 0: this lane's scale

#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s0 + s < s1) stage(s0 + s);
  for (int kt = s0; kt < s1; ++kt) {
    if (kt + S - 1 < s1) stage(kt + S - 1);                // into the slot of the step before this one
    wait_steps<S - 1, PER>(s1 - 1 - kt);
    LDM_LOCKSTEP();
    const unsigned slot = (unsigned)((kt - s0) % S) * SLOT;
    const int g = (kt - s0) >> 2, word = word_scales ? 0 : kt - min(s0 + 4 * g, nk - 4);
    const unsigned sa = saddr + (g & 1) * SCALES + word * 4;
    if constexpr (MX) {
      if (__builtin_expect(kt == cut_step, 0)) {
        clear_behind<16 * MT, 64, 64>(lds + slot + NF * 1024, (p.blocks - 1) & 3, last_columns(p), lane, [](int r) { return (r >> 1) & 3; });
        LDM_LOCKSTEP();
      }
    }
    i32x4_t wv[NF], xv[MT][MX ? 1 : 4];
    int wc[NF], xc[MT];
#pragma unroll
    for (int i = 0; i < NF; ++i) lds_read4<0>(wc[i], sa + i * 16 * sstep);
    if constexpr (MX) {
#pragma unroll
      for (int j = 0; j < MT; ++j) lds_read4<1024>(xc[j], sa + j * 16 * sstep);
    }
    [&]<int... I>(std::integer_sequence<int, I...>) {
      (lds_read16<I * 1024>(wv[I], waddr + slot), ...);
    }(std::make_integer_sequence<int, NF>{});
    [&]<int... J>(std::integer_sequence<int, J...>) {
      ([&] {
        constexpr int j = J;
        if constexpr (MX) {
          lds_read16<(NF + j) * 1024>(xv[j][0], waddr + slot);
        } else {
          lds_read16<j * 4096>(xv[j][0], xaddr[0] + slot);
          lds_read16<j * 4096>(xv[j][1], xaddr[1] + slot);
          lds_read16<j * 4096>(xv[j][2], xaddr[2] + slot);
          lds_read16<j * 4096>(xv[j][3], xaddr[3] + slot);
        }
      }(), ...);
    }(std::make_integer_sequence<int, MT>{});
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < NF; ++i) asm volatile("" : "+v"(wv[i]), "+v"(wc[i]));   // no use moves above the wait
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      if constexpr (MX) asm volatile("" : "+v"(xc[j]));
#pragma unroll
      for (int s = 0; s < (MX ? 1 : 4); ++s) asm volatile("" : "+v"(xv[j][s]));
    }
    const unsigned pick = kt == nk - 1 ? ends : whole;
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      const unsigned code = (unsigned)scale_take(wc[i], pick);
      if constexpr (MX) {
        const i32x8_t a{wv[i][0], wv[i][1], wv[i][2], wv[i][3], 0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const i32x8_t b{xv[j][0][0], xv[j][0][1], xv[j][0][2], xv[j][0][3], 0, 0, 0, 0};
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc[i][j], 4, 4, 0, (int)code, 0, scale_take(xc[j], pick));
        }
      } else {
        const float sc = __uint_as_float(code << 23);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const unsigned q = (unsigned)wv[i][s];
          uint4 b;
          b.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, sc, 0));
          b.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, sc, 1));
          b.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, sc, 2));
          b.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, sc, 3));
#pragma unroll
          for (int j = 0; j < MT; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, b), __builtin_bit_cast(bf16x8_t, xv[j][s]), acc[i][j],
                                                                0, 0, 0);
        }
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  LDM_LOCKSTEP();
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
      reinterpret_cast<float4*>(mine)[(i * MT + j) * 64 + lane] = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
  __syncthreads();
  for (int t = tid; t < NF * MT * 64; t += 64 * NW) {
    const int f = t >> 6, l = t & 63, i = f / MT, j = f - i * MT;
    const int n = n0 + i * 16 + (l >> 4) * 4;
    const long long m = m0 + j * 16 + (l & 15);
    if (m >= p.rows || n >= p.n) continue;
    float4 s = reinterpret_cast<const float4*>(smem)[t];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      const float4 o = reinterpret_cast<const float4*>(smem + w * WAVE)[t];
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

// A launch's threads are counted in 32 bits.
static bool mx_launchable(long long workgroups, int threads) { return workgroups * threads < (1LL << 32); }
// The tile kernels launch no more than tiles of 128 x 128 by 256 threads would: smaller tiles are taken only where there are few.
static bool mx_tiles_launchable(long long rows, long long n) { return mx_launchable(((rows + 127) / 128) * ((n + 127) / 128), 256); }

template <int BM, int BN, int WM, int WN, int S, typename OUT>
static int launch_mx4_gemm(Mx4Params& p, hipStream_t st) {
  p.tiles_m = (int)((p.rows + BM - 1) / BM);
  p.tiles_n = (p.n + BN - 1) / BN;
  p.nk = (p.blocks + 3) / 4;
  constexpr int smem = (BM + BN) * (S * 64 + 2 * 16);
  auto kern = mx4_gemm_kernel<BM, BN, WM, WN, S, OUT>;
  static bool done = false;
  if (int rc = mx_allow_lds("ldm_mx4_linear", kern, smem, done)) return rc;
  hipLaunchKernelGGL(kern, dim3(p.tiles_m * p.tiles_n), dim3(64 * WM * WN), smem, st, p);
  return LDM_OK;
}

template <int BM, int BN, int WM, int WN, int KW, int S, bool MX, typename OUT>
static int launch_mx_gemm(Mx4Params& p, hipStream_t st) {
  p.tiles_m = (int)((p.rows + BM - 1) / BM);
  p.tiles_n = (p.n + BN - 1) / BN;
  p.nk = (MX ? p.blocks + 7 : p.k / 8 + 7) / 8;
  constexpr int smem = KW * (S * (BM + BN) * 128 + (MX ? 2 * ((BM + BN + 63) / 64 * 64) * 16 : 0));
  static_assert(smem <= 160 * 1024, "LDS of a CU");
  auto kern = mx_gemm_kernel<BM, BN, WM, WN, KW, S, MX, OUT>;
  static bool done = false;
  if (int rc = mx_allow_lds("mx product", kern, smem, done)) return rc;
  hipLaunchKernelGGL(kern, dim3(p.tiles_m * p.tiles_n), dim3(64 * WM * WN * KW), smem, st, p);
  return LDM_OK;
}

template <bool MX, int MT, int NF, int NW, int S, bool DMAX, typename OUT>
static int launch_mx4_rows(const Mx4Params& p, hipStream_t st) {
  constexpr int smem = NW * (S * (NF + (MX ? MT : 4 * MT)) * 1024 + (MX ? 4096 : 2048));
  const dim3 grid((p.n + 16 * NF - 1) / (16 * NF), (unsigned)((p.rows + 16 * MT - 1) / (16 * MT)));
  LDM_REQUIRE(mx_launchable((long long)grid.x * grid.y, 64 * NW), "ldm_mx4_linear: %lld x %d outputs are too many", p.rows, p.n);
  auto kern = mx4_rows_kernel<MX, MT, NF, NW, S, DMAX, OUT>;
  static bool done = false;
  if (int rc = mx_allow_lds("ldm_mx4_linear", kern, smem, done)) return rc;
  hipLaunchKernelGGL(kern, grid, dim3(64 * NW), smem, st, p);
  return LDM_OK;
}

template <bool MX, bool DMAX, typename OUT>
static int rows_by_size(const Mx4Params& p, hipStream_t st) {
  // Fragments of w a workgroup: as many as leave every CU one workgroup of its own (n = 8192 / 10240, 16 rows, k = 8192: 12.4 / 14.3 us;
  // with two fragments throughout 12.4 / 19.2, since some CUs then have two workgroups and some one).  Waves and steps: what LDS holds.
  const int nf = (p.n + 4095) / 4096;
  if (p.rows <= 16) {
    if (nf == 1) return launch_mx4_rows<MX, 1, 1, 8, 2, DMAX, OUT>(p, st);
    if (nf == 2) return launch_mx4_rows<MX, 1, 2, 8, 3, DMAX, OUT>(p, st);
    if (nf == 3) return launch_mx4_rows<MX, 1, 3, 8, 2, DMAX, OUT>(p, st);
    if (nf == 4) return launch_mx4_rows<MX, 1, 4, 8, 2, DMAX, OUT>(p, st);
    return launch_mx4_rows<MX, 1, 2, 4, 3, DMAX, OUT>(p, st);   // several rounds of workgroups: two a CU at a time
  }
  if (p.rows <= 32) {
    if (nf == 1) return launch_mx4_rows<MX, 2, 1, 8, 2, DMAX, OUT>(p, st);
    return launch_mx4_rows<MX, 2, 2, 4, 3, DMAX, OUT>(p, st);
  }
  if (nf == 1) return launch_mx4_rows<MX, 4, 1, MX ? 8 : 4, MX ? 3 : 2, DMAX, OUT>(p, st);
  return launch_mx4_rows<MX, 4, 2, 4, MX ? 4 : 2, DMAX, OUT>(p, st);
}

static float tile_rounds(const Mx4Params& p, int bm, int bn) {
  return (float)((((p.rows + bm - 1) / bm) * ((p.n + bn - 1) / bn) + 255) / 256);
}

template <typename OUT>
static int mx4_linear_out(Mx4Params& p, bool mx, hipStream_t st) {
  if (!mx) return p.k % 8 == 0 && aligned16(p.x) ? rows_by_size<false, true, OUT>(p, st) : rows_by_size<false, false, OUT>(p, st);
  // few rows, or few enough outputs that each CU has at most one workgroup of the few-row kernel (k = 128 .. 8192: 128 x 1280 3.4 .. 8.8 us
  // against 6.2 .. 12.1 in tiles, 1024 x 256 3.4 .. 10.6 / 6.2 .. 12.4); with two a CU its re-reading of the operands loses for longer sums
  // (128 x 4096: k = 320 5.0 / 6.4, k = 1280 6.5 / 6.3, k = 8192 18.4 / 12.5)
  if (p.rows <= 64 || ((p.rows + 63) / 64) * ((p.n + 15) / 16) <= 256) return rows_by_size<true, true, OUT>(p, st);
  // rounds of one workgroup a CU x the time of 256 columns of the tile (us: 64 x 64 with its columns split 0.55, 128 x 128 1, 256 x 256
  // 2.3).  8192^3: 715, 464 and 341 us; 2048^3: 21.5, 11.5, 12.3; 154 x 2560 (k = 2560): 7.3, 10.4, 12.0
  const float a = tile_rounds(p, 64, 64) * 0.55f, b = tile_rounds(p, 128, 128), c = tile_rounds(p, 256, 256) * 2.3f;
  if (a <= b && a <= c) return launch_mx_gemm<64, 64, 1, 1, 4, 2, true, OUT>(p, st);
  if (b <= c) return launch_mx_gemm<128, 128, 2, 2, 1, 3, true, OUT>(p, st);
  // Short sums: two workgroups a CU, one's output and first loads behind the other's products (8192 x 5120, k = 640: 34.3 us against 37.2,
  // 2048 x 10240, k = 1280: 31.0 / 32.9); long ones: the larger tile's fewer operand reads (k = 4096: 52.3 / 49.8, 8192: 353 / 310).
  if (p.k < 2048) return launch_mx4_gemm<256, 128, 2, 2, 2, OUT>(p, st);
  return launch_mx4_gemm<256, 256, 2, 4, 4, OUT>(p, st);
}

template <typename OUT>
static int linear_bf16_out(Mx4Params& p, hipStream_t st) {
  // rounds of one workgroup a CU x the time of a step of the tile (us, measured at full chips: 64 x 64 with its columns split 0.27,
  // 128 x 128 0.5, 128 x 160 0.7, 256 x 160 1.1).  8192 x 640 (k = 5120): 83 us with 128 x 128, 65 with 128 x 160; 32768 x 320 (k = 2560):
  // 89, 77 and 62 with 256 x 160; 154 x 768 (k = 1312): 11.7 with 128 x 128, 6.8 with 64 x 64.
  const float a = tile_rounds(p, 64, 64) * 0.27f, b = tile_rounds(p, 128, 128) * 0.5f, c = tile_rounds(p, 128, 160) * 0.7f,
              d = tile_rounds(p, 256, 160) * 1.1f;
  if (a <= b && a <= c && a <= d) return launch_mx_gemm<64, 64, 1, 1, 4, 2, false, OUT>(p, st);
  if (b <= c && b <= d) return launch_mx_gemm<128, 128, 2, 2, 1, 3, false, OUT>(p, st);
  if (c <= d) return launch_mx_gemm<128, 160, 4, 1, 1, 3, false, OUT>(p, st);
  return launch_mx_gemm<256, 160, 4, 1, 1, 3, false, OUT>(p, st);
}

}  // namespace ldm

using namespace ldm;

extern "C" int ldm_mx4_linear(const void* x, const void* x_scale, const void* w, const void* w_scale, const float* bias, void* out,
                              int out_dtype, long long rows, int n, int k, void* stream) {
  LDM_REQUIRE(dtype_ok(out_dtype), "ldm_mx4_linear: bad dtype %d", out_dtype);
  LDM_REQUIRE(rows >= 0 && n >= 1 && n <= (1 << 30) && k >= 1 && k <= (1 << 22), "ldm_mx4_linear: bad sizes (rows=%lld n=%d k=%d)", rows, n, k);
  LDM_REQUIRE(rows < (1LL << 40) && mx_tiles_launchable(rows, n), "ldm_mx4_linear: %lld x %d outputs are too many", rows, n);
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
  hipStream_t st = (hipStream_t)stream;
  const int rc = out_dtype == LDM_BF16 ? mx4_linear_out<bf16_t>(p, mx, st) : mx4_linear_out<float>(p, mx, st);
  if (rc) return rc;
  LDM_HIP_CHECK_LAUNCH("ldm_mx4_linear");
  return LDM_OK;
}

extern "C" int ldm_linear_bf16(const void* x, const void* w, const float* bias, void* out, int out_dtype, long long rows, int n, int k, void* stream) {
  LDM_REQUIRE(dtype_ok(out_dtype), "ldm_linear_bf16: bad dtype %d", out_dtype);
  LDM_REQUIRE(rows >= 0 && n >= 1 && n <= (1 << 30) && k >= 8 && k % 8 == 0 && k <= (1 << 21),
              "ldm_linear_bf16: bad sizes (rows=%lld n=%d k=%d; k a multiple of 8)", rows, n, k);
  LDM_REQUIRE(rows < (1LL << 40) && mx_tiles_launchable(rows, n), "ldm_linear_bf16: %lld x %d outputs are too many", rows, n);
  if (rows == 0) return LDM_OK;
  LDM_REQUIRE(x && w && out && aligned16(x) && aligned16(w) && (reinterpret_cast<uintptr_t>(bias) & 3) == 0 &&
                  reinterpret_cast<uintptr_t>(out) % dtype_size(out_dtype) == 0,
              "ldm_linear_bf16: null or unaligned pointer");
  Mx4Params p{};
  p.x = static_cast<const unsigned char*>(x); p.w = static_cast<const unsigned char*>(w);
  p.bias = bias; p.out = out; p.rows = rows; p.n = n; p.k = k;
  p.nk = (k + 63) / 64;
  const int rc = out_dtype == LDM_BF16 ? linear_bf16_out<bf16_t>(p, (hipStream_t)stream) : linear_bf16_out<float>(p, (hipStream_t)stream);
  if (rc != LDM_OK) return rc;
  LDM_HIP_CHECK_LAUNCH("ldm_linear_bf16");
  return LDM_OK;
}

// *x: rows that the product can fetch, in the front of the workspace if they have to be laid out for it; *wide: the place of the widened weights
// behind them.  Everything that the steps after this one could refuse has been looked at: a refused call launches nothing.
static int mx_rows_for_product(const char* what, const void** x, const void* w, const void* w_scale, const void* bias, const void* out, int out_dtype,
                               long long rows, int cols, int ld, long long outer, void* workspace, long long workspace_bytes, void** wide, void* stream) {
  LDM_REQUIRE(dtype_ok(out_dtype), "%s: bad dtype %d", what, out_dtype);
  LDM_REQUIRE(*x && w && w_scale && out && (reinterpret_cast<uintptr_t>(*x) & 1) == 0 && aligned16(w) &&
                  (reinterpret_cast<uintptr_t>(w_scale) & 3) == 0 && (reinterpret_cast<uintptr_t>(bias) & 3) == 0 &&
                  reinterpret_cast<uintptr_t>(out) % dtype_size(out_dtype) == 0,
              "%s: null or unaligned pointer", what);
  LDM_REQUIRE(rows < (1LL << 40) && outer <= (1 << 30) && mx_tiles_launchable(rows, outer), "%s: %lld x %lld outputs are too many", what, rows, outer);
  const bool pad = ld != cols || !aligned16(*x);
  const long long need = (outer + (pad ? rows : 0)) * ld * 2;
  LDM_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= need, "%s: workspace of %lld bytes needed (got %lld)", what, need,
              workspace_bytes);
  *wide = workspace;
  if (!pad) return LDM_OK;
  const int rc = ldm_pad_columns_bf16(*x, workspace, rows, cols, ld, stream);
  *x = workspace;
  *wide = static_cast<bf16_t*>(workspace) + rows * ld;
  return rc;
}

extern "C" int ldm_mx4_linear_wide(const void* x, const void* w, const void* w_scale, const float* bias, void* out, int out_dtype, long long rows, int n,
                                   int k, void* workspace, long long workspace_bytes, void* stream) {
  LDM_REQUIRE(rows >= 0 && n >= 1 && k >= 1 && k <= (1 << 21), "ldm_mx4_linear_wide: bad sizes (rows=%lld n=%d k=%d)", rows, n, k);
  if (rows == 0) return LDM_OK;
  const int kp = (k + 7) & ~7;
  void* wide = nullptr;
  if (int rc = mx_rows_for_product("ldm_mx4_linear_wide", &x, w, w_scale, bias, out, out_dtype, rows, k, kp, n, workspace, workspace_bytes, &wide, stream))
    return rc;
  if (int rc = ldm_mx_dequantize(w, w_scale, LDM_MX4, n, kp, wide, LDM_BF16, kp, stream)) return rc;
  return ldm_linear_bf16(x, wide, bias, out, out_dtype, rows, n, kp, stream);
}

extern "C" int ldm_mx4_linear_dgrad(const void* dy, const void* w, const void* w_scale, void* dx, long long rows, int n, int k, void* workspace,
                                    long long workspace_bytes, void* stream) {
  LDM_REQUIRE(rows >= 0 && n >= 1 && n <= (1 << 21) && k >= 1, "ldm_mx4_linear_dgrad: bad sizes (rows=%lld n=%d k=%d)", rows, n, k);
  if (rows == 0) return LDM_OK;
  const int np = (n + 7) & ~7;
  void* wide = nullptr;
  if (int rc = mx_rows_for_product("ldm_mx4_linear_dgrad", &dy, w, w_scale, nullptr, dx, LDM_BF16, rows, n, np, k, workspace, workspace_bytes, &wide, stream))
    return rc;
  if (int rc = ldm_mx4_dequantize_t(w, w_scale, n, k, wide, np, stream)) return rc;
  return ldm_linear_bf16(dy, wide, nullptr, dx, LDM_BF16, rows, k, np, stream);
}
