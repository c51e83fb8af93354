// Weight gradient of a linear layer whose input was kept as an mx8 checkpoint:
//
//   dW[n][k] = sum_m dY[m][n] x[m][k]         dY bf16, x = 8-bit elements under one power-of-two scale per 32 columns
//
// An mx8 value has at most 7 significant bits, so it IS a bf16 value: the checkpoint is widened without rounding on its way into
// LDS and the product is the bf16 one (v_mfma_f32_16x16x32_bf16, float32 sums).  Read at 8.25 bits a value, the checkpoint costs half
// of what the bf16 activation would.
//
// The contraction runs over the rows of both operands.  A workgroup of 8 waves owns T0 columns of dY x T1 columns of x and walks its
// share of the rows 32 a step: dY goes to LDS by LDS-DMA (two steps ahead), x through registers -- loaded two steps ahead, widened
// and written one step ahead, once per workgroup, under the MFMAs -- and both operands' fragments are read transposed
// (ds_read_b64_tr_b16, the same permutation of the rows on both sides).  One barrier a step, three slots.  The rows are split over
// blockIdx.y where there are few tiles; the partial tiles are added by a second kernel in a fixed order (no atomics).
#include "common.h"

#include <type_traits>
#include <utility>

namespace ldm {

typedef __attribute__((ext_vector_type(8))) short bf16x8_t;
typedef __attribute__((ext_vector_type(4))) short bf16x4_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

struct WgradMx8Params {
  const unsigned char* x;
  const unsigned char* xs;
  const char* dy;
  float* out;                  // dw, or partial tiles [splits][n][k]
  long long rows;
  int n, k, blocks, sstride;
  int tiles_n, tiles_k;
  int steps_per_split, splits;
  int accumulate;              // direct form only
};

constexpr int WM8_MS = 32;     // rows a step: one MFMA contraction block

// 16-byte chunks of an image row are swizzled in pairs by row so that the eight rows a transposed read touches lie in eight different
// 32-byte columns of the LDS line: rows of 512 bytes all start at bank 0 (flip by row & 7), rows of 640 bytes alternate between
// the line's halves (flip by (row >> 1) & 3, inside aligned groups of eight chunks)
template <int T>
__device__ __forceinline__ int wm8_swz(int row) { return T == 256 ? (row & 7) << 1 : ((row >> 1) & 3) << 1; }

__device__ __forceinline__ void wm8_dma16(const void* base, int bytes, unsigned char* lds, unsigned voff) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
}

template <int T0, int T1, int W0, int W1>
__global__ void __launch_bounds__(512)
linear_wgrad_mx8_kernel(const WgradMx8Params p) {
  constexpr unsigned OOB = 0x80000000u;
  constexpr int F0 = T0 / W0 / 16, F1 = T1 / W1 / 16;
  constexpr int IMG0 = WM8_MS * T0 * 2, IMG1 = WM8_MS * T1 * 2, SLOT = IMG0 + IMG1;
  constexpr int NI0 = IMG0 / 1024;                         // DMA instructions of the workgroup a step
  constexpr int JMAX = (NI0 + 7) / 8, JMIN = NI0 / 8;
  constexpr int UPR = T1 / 16;                             // units of 16 columns (half a block) a row of x
  constexpr int UMAX = (WM8_MS * UPR + 511) / 512;         // units a thread stages a step
  constexpr int UFULL = WM8_MS * UPR / 512;
  static_assert(W0 * W1 == 8 && (WM8_MS * UPR) % 64 == 0, "tile / waves mismatch");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int w0 = wave / W1, w1 = wave % W1;
  const int tn = blockIdx.x % p.tiles_n, tk = blockIdx.x / p.tiles_n;
  const int n0 = tn * T0, k0 = tk * T1;
  const int total_steps = (int)((p.rows + WM8_MS - 1) / WM8_MS);
  const int step_begin = blockIdx.y * p.steps_per_split;
  const int nsteps = min(step_begin + p.steps_per_split, total_steps) - step_begin;

  // dY: the descriptor moves 32 rows a step and ends with the matrix (rows past it read as zeros); lane offsets are constant
  unsigned dvoff[JMAX];
#pragma unroll
  for (int j = 0; j < JMAX; ++j) {
    const int c = (j * 8 + wave) * 64 + lane, row = c / (T0 / 8), phys = c - row * (T0 / 8);
    const int col = n0 + (phys ^ wm8_swz<T0>(row)) * 8;
    dvoff[j] = col < p.n ? ((unsigned)row * p.n + col) * 2u : OOB;
  }
  const long long dy_step = (long long)WM8_MS * p.n * 2;
  const char* dy_ptr = p.dy + (long long)step_begin * dy_step;
  long long dy_left = (p.rows - (long long)step_begin * WM8_MS) * p.n * 2;
  auto stage_dy = [&](int slot) {
    const int bytes = dy_left > 0x7fffffffLL ? 0x7fffffff : (int)dy_left;
#pragma unroll
    for (int j = 0; j < JMAX; ++j) {
      const int q = j * 8 + wave;
      if (j < JMIN || q < NI0) wm8_dma16(dy_ptr, bytes, smem + slot * SLOT + q * 1024, dvoff[j]);   // wave-uniform
    }
    dy_ptr += dy_step;
    dy_left -= dy_step;
  };

  // x: a thread's unit is 16 elements of one row and their block's scale byte
  int urow[UMAX];
  unsigned udst[UMAX];
  bool uok[UMAX];
  long long udata[UMAX], uscale[UMAX];
#pragma unroll
  for (int u = 0; u < UMAX; ++u) {
    const int id = u * 512 + tid, row = id / UPR, half = id - row * UPR;
    const int blk = (k0 >> 5) + (half >> 1);
    urow[u] = row;
    uok[u] = (u < UFULL || id < WM8_MS * UPR) && blk < p.blocks;
    udst[u] = IMG0 + row * (T1 * 2) + (((2 * half) ^ wm8_swz<T1>(row)) << 4);
    udata[u] = ((long long)row * p.blocks + blk) * 32 + (half & 1) * 16;
    uscale[u] = (long long)row * p.sstride + blk;
  }
  long long x_row = (long long)step_begin * WM8_MS;        // first row of the step to load next
  uint4 raw[UMAX];
  int code[UMAX];
  auto load_x = [&]() {
    const unsigned char* xb = p.x + x_row * p.blocks * 32;
    const unsigned char* sb = p.xs + x_row * p.sstride;
#pragma unroll
    for (int u = 0; u < UMAX; ++u) {
      raw[u] = make_uint4(0, 0, 0, 0);
      code[u] = 0;
      if (u >= UFULL && wave * 64 + u * 512 >= WM8_MS * UPR) continue;     // wave-uniform
      if (uok[u] && x_row + urow[u] < p.rows) {
        raw[u] = *reinterpret_cast<const uint4*>(xb + udata[u]);
        code[u] = sb[uscale[u]];
      }
    }
    x_row += WM8_MS;
  };
  auto widen_x = [&](int slot) {
#pragma unroll
    for (int u = 0; u < UMAX; ++u) {
      if (u >= UFULL && wave * 64 + u * 512 >= WM8_MS * UPR) continue;
      const float step = code[u] == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(1.0f, code[u] - 133);
      const unsigned w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
      uint32_t o[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)((int)(w[q] << (24 - 8 * e)) >> 24) * step;
        o[2 * q] = pack_bf16x2(v[0], v[1]);
        o[2 * q + 1] = pack_bf16x2(v[2], v[3]);
      }
      uint4* d = reinterpret_cast<uint4*>(smem + slot * SLOT + udst[u]);
      d[0] = make_uint4(o[0], o[1], o[2], o[3]);
      d[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  };

  f32x4_t acc[F0][F1];
#pragma unroll
  for (int i = 0; i < F0; ++i)
#pragma unroll
    for (int j = 0; j < F1; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  // transposed fragments: lane -> row 4 fq + tq (and 16 further down, where the swizzle is the same), chunk 2 ct + (tp >> 1), half tp & 1
  const int fr = lane & 15, fq = lane >> 4, tq = fr >> 2, tp = fr & 3;
  const int frow = 4 * fq + tq;
  const unsigned lds_base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  unsigned off0[F0], off1[F1];
#pragma unroll
  for (int i = 0; i < F0; ++i)
    off0[i] = frow * (T0 * 2) + (((2 * (w0 * F0 + i) + (tp >> 1)) ^ wm8_swz<T0>(frow)) << 4) + ((tp & 1) << 3);
#pragma unroll
  for (int j = 0; j < F1; ++j)
    off1[j] = IMG0 + frow * (T1 * 2) + (((2 * (w1 * F1 + j) + (tp >> 1)) ^ wm8_swz<T1>(frow)) << 4) + ((tp & 1) << 3);

  if (nsteps > 0) {
    // In memory order: x(s + 1) in registers, then dY(s + 1) to LDS -- a wait that leaves only this wave's youngest DMA batch in flight
    // has dY(s) in LDS and x(s + 1) in registers, whether or not the x loads were issued.
    load_x();
    stage_dy(0);
    widen_x(0);
    if (nsteps > 1) { load_x(); stage_dy(1); }
    const bool three = JMAX > JMIN && (JMIN * 8 + wave) < NI0;
    int slot = 0;
    for (int s = 0; s < nsteps; ++s) {
      if (s + 1 < nsteps) {
        if (three) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(JMAX) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(JMIN) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this wave's widened x(s) is in LDS
      __builtin_amdgcn_s_barrier();                        // everybody's is; the slot of step s - 1 is free
      asm volatile("" ::: "memory");
      const unsigned sbase = lds_base + slot * SLOT;
      const int next = slot == 2 ? 0 : slot + 1, after = next == 2 ? 0 : next + 1;
      bf16x4_t lo0[F0], hi0[F0], lo1[F1], hi1[F1];
      constexpr bool OUT0 = F0 >= F1;                      // the longer fragment list is the outer loop of the MFMAs
      constexpr int NOUT = OUT0 ? F0 : F1;
      auto read0 = [&](int i) {
        asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(lo0[i]) : "v"(sbase + off0[i]) : "memory");
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(hi0[i]) : "v"(sbase + off0[i]), "n"(16 * T0 * 2) : "memory");
      };
      auto read1 = [&](int j) {
        asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(lo1[j]) : "v"(sbase + off1[j]) : "memory");
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(hi1[j]) : "v"(sbase + off1[j]), "n"(16 * T1 * 2) : "memory");
      };
      if constexpr (OUT0) {
#pragma unroll
        for (int j = 0; j < F1; ++j) read1(j);
#pragma unroll
        for (int i = 0; i < F0; ++i) read0(i);
      } else {
#pragma unroll
        for (int i = 0; i < F0; ++i) read0(i);
#pragma unroll
        for (int j = 0; j < F1; ++j) read1(j);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int i = 0; i < F0; ++i) asm volatile("" : "+v"(lo0[i]), "+v"(hi0[i]));   // no use of a fragment moves above the wait
#pragma unroll
      for (int j = 0; j < F1; ++j) asm volatile("" : "+v"(lo1[j]), "+v"(hi1[j]));
      if (s + 1 < nsteps) widen_x(next);
      if (s + 2 < nsteps) { load_x(); stage_dy(after); }
      auto join = [](const bf16x4_t& lo, const bf16x4_t& hi) {
        return bf16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      };
#pragma unroll
      for (int g = 0; g < NOUT; ++g) {
        if constexpr (OUT0) {
#pragma unroll
          for (int j = 0; j < F1; ++j) acc[g][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(join(lo0[g], hi0[g]), join(lo1[j], hi1[j]), acc[g][j], 0, 0, 0);
        } else {
#pragma unroll
          for (int i = 0; i < F0; ++i) acc[i][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(join(lo0[i], hi0[i]), join(lo1[g], hi1[g]), acc[i][g], 0, 0, 0);
        }
      }
      slot = next;
    }
  }

  // C[row = n = 4 fq + r][column = k = fr]
  float* out = p.out + (long long)blockIdx.y * p.n * p.k;
#pragma unroll
  for (int i = 0; i < F0; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + (w0 * F0 + i) * 16 + fq * 4 + r;
      if (n >= p.n) continue;
#pragma unroll
      for (int j = 0; j < F1; ++j) {
        const int k = k0 + (w1 * F1 + j) * 16 + fr;
        if (k >= p.k) continue;
        float* d = out + (long long)n * p.k + k;
        *d = p.accumulate ? *d + acc[i][j][r] : acc[i][j][r];
      }
    }
}

// dw (+)= the partial tiles, in order
__global__ void __launch_bounds__(256)
wgrad_mx8_fold_kernel(const float* __restrict__ partial, float* __restrict__ dw, long long total, int splits, int accumulate) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  float v = accumulate ? dw[i] : 0.f;
  for (int s = 0; s < splits; ++s) v += partial[(long long)s * total + i];
  dw[i] = v;
}

// Tile shape with the least padded work (channel counts of this model family are multiples of 320), then enough splits of the rows for
// one workgroup on every CU, at least 16 steps each
static int wgrad_mx8_plan(long long rows, int n, int k, WgradMx8Params& p) {
  static const int shapes[3][2] = {{256, 256}, {320, 256}, {256, 320}};
  long long best = -1;
  int cfg = 0;
  for (int c = 0; c < 3; ++c) {
    const long long tn = (n + shapes[c][0] - 1) / shapes[c][0], tk = (k + shapes[c][1] - 1) / shapes[c][1];
    const long long padded = tn * shapes[c][0] * tk * shapes[c][1];
    if (best < 0 || padded < best) { best = padded; cfg = c; p.tiles_n = (int)tn; p.tiles_k = (int)tk; }
  }
  const int steps = (int)((rows + WM8_MS - 1) / WM8_MS);
  const long long tiles = (long long)p.tiles_n * p.tiles_k;
  long long splits = tiles >= 256 ? 1 : 256 / tiles;
  if (splits > steps / 16) splits = steps / 16;
  if (splits < 1) splits = 1;
  p.steps_per_split = (int)((steps + splits - 1) / splits);
  p.splits = (steps + p.steps_per_split - 1) / p.steps_per_split;
  return cfg;
}

template <int T0, int T1, int W0, int W1>
static int launch_wgrad_mx8(const WgradMx8Params& p, hipStream_t st) {
  constexpr int smem = 3 * WM8_MS * (T0 + T1) * 2;
  auto kern = linear_wgrad_mx8_kernel<T0, T1, W0, W1>;
  static bool done = false;
  if (!done) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != hipSuccess) { set_error("ldm_linear_wgrad_mx8: hipFuncSetAttribute: %s", hipGetErrorString(e)); return LDM_EHIP; }
    done = true;
  }
  hipLaunchKernelGGL(kern, dim3(p.tiles_n * p.tiles_k, p.splits), dim3(512), smem, st, p);
  return LDM_OK;
}

}  // namespace ldm

using namespace ldm;

static bool wgrad_mx8_sizes_ok(long long rows, int n, int k) {
  return rows >= 1 && rows <= 32LL * 0x7fffffff && n >= 1 && k >= 1 && n <= (1 << 24) && k <= (1 << 24) && (long long)n * k < (1LL << 38);
}

extern "C" long long ldm_linear_wgrad_mx8_workspace_bytes(long long rows, int n, int k) {
  if (!wgrad_mx8_sizes_ok(rows, n, k)) return 0;
  WgradMx8Params p;
  wgrad_mx8_plan(rows, n, k, p);
  return p.splits > 1 ? (long long)p.splits * n * k * 4 : 0;
}

extern "C" int ldm_linear_wgrad_mx8(const void* x8, const void* x8_scale, const void* dy, float* dw, long long rows, int n, int k,
                                    int accumulate, void* workspace, long long workspace_bytes, void* stream) {
  LDM_REQUIRE(wgrad_mx8_sizes_ok(rows, n, k) && n % 8 == 0, "ldm_linear_wgrad_mx8: bad sizes (rows=%lld n=%d k=%d; n a multiple of 8)", rows, n, k);
  LDM_REQUIRE(x8 && x8_scale && dy && dw && aligned16(x8) && aligned16(dy), "ldm_linear_wgrad_mx8: null or unaligned pointer");
  WgradMx8Params p;
  const int cfg = wgrad_mx8_plan(rows, n, k, p);
  const long long need = p.splits > 1 ? (long long)p.splits * n * k * 4 : 0;
  LDM_REQUIRE(need == 0 || (workspace != nullptr && aligned16(workspace) && workspace_bytes >= need),
              "ldm_linear_wgrad_mx8: workspace of %lld bytes needed (got %lld)", need, workspace_bytes);
  LDM_REQUIRE((long long)p.tiles_n * p.tiles_k < (1LL << 31) && p.splits <= 65535, "ldm_linear_wgrad_mx8: too large");
  p.x = static_cast<const unsigned char*>(x8); p.xs = static_cast<const unsigned char*>(x8_scale); p.dy = static_cast<const char*>(dy);
  p.rows = rows; p.n = n; p.k = k; p.blocks = mx_blocks(k); p.sstride = mx_scale_stride(k);
  p.out = need ? static_cast<float*>(workspace) : dw;
  p.accumulate = need ? 0 : accumulate;
  hipStream_t st = (hipStream_t)stream;
  const int rc = cfg == 0 ? launch_wgrad_mx8<256, 256, 2, 4>(p, st) : cfg == 1 ? launch_wgrad_mx8<320, 256, 2, 4>(p, st) : launch_wgrad_mx8<256, 320, 4, 2>(p, st);
  if (rc) return rc;
  LDM_HIP_CHECK_LAUNCH("ldm_linear_wgrad_mx8");
  if (need) {
    const long long total = (long long)n * k;
    hipLaunchKernelGGL(wgrad_mx8_fold_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st, p.out, dw, total, p.splits, accumulate);
    LDM_HIP_CHECK_LAUNCH("ldm_linear_wgrad_mx8(fold)");
  }
  return LDM_OK;
}
