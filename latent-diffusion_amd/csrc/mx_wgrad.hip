// Weight gradient of a linear layer whose input was kept as an mx8 checkpoint:
//
//   dW[n][k] = sum_m dY[m][n] x[m][k]         dY bf16, x = 8-bit elements under one power-of-two scale per 32 columns
//
// An mx8 value has at most 7 significant bits, so it IS a bf16 value: the checkpoint is widened without rounding on its way into
// LDS and the product is the bf16 one (v_mfma_f32_16x16x32_bf16, float32 sums).  Read at 8.25 bits a value, the checkpoint costs half
// of what the bf16 activation would.
//
// The contraction runs over the rows of both operands.  A workgroup of 8 waves owns T0 columns of dY x T1 columns of x and walks its
// share of the rows 64 a step, double-buffered: dY goes to LDS by LDS-DMA; x goes there by LDS-DMA as it is stored, and the thread that
// fetched 16 of its elements widens them into the bf16 image one step ahead.  Both operands' fragments are read transposed
// (ds_read_b64_tr_b16, the same permutation of the rows on both sides), each block of 32 rows while the block before multiplies.  The
// rows are split over workgroups where there are few tiles; the partial tiles are added by a second kernel in a fixed order (no
// atomics).
//
// 32768 rows, 2560 x 320 (54 GFLOP, 180 MB): 68 us + 9 us for the 16 partial tiles, 700 TFLOP/s; a large bf16 matrix product reaches
// 1220.  Parts left out one at a time: the partial tiles' stores 10 us, dY's loads 13, the widening 2 (6 without dY's loads), the
// fragments' reads 4; the products alone take 26.
#include "common.h"

#include <type_traits>
#include <utility>

namespace ldm {

typedef __attribute__((ext_vector_type(8))) short bf16x8_t;
typedef __attribute__((ext_vector_type(4))) short bf16x4_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;

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

constexpr int WM8_MS = 64;     // rows a step: two MFMA contraction blocks

// 16-byte chunks of an image row are swizzled in pairs by row so that the eight rows a transposed read touches lie in eight different
// 32-byte columns of the 256-byte LDS line.  Rows of a multiple of 256 bytes all start at its first column (flip the pair by row & 7);
// rows of 128 bytes more alternate between its halves (by (row >> 1) & 3, inside aligned groups of four pairs); rows of 64 bytes more
// start at every second column in turn (by (row >> 2) & 1, inside groups of two).
template <int T>
__device__ __forceinline__ int wm8_swz(int row) {
  return T % 128 == 0 ? (row & 7) << 1 : T % 64 == 0 ? ((row >> 1) & 3) << 1 : ((row >> 2) & 1) << 1;
}
// pairs in a group that the swizzle stays inside of: fragment i of a row is fragment i % that many, and whole groups further on
template <int T, int F>
constexpr int wm8_distinct() { return T % 128 == 0 ? F : T % 64 == 0 ? 4 : 2; }

__device__ __forceinline__ void wm8_dma16(const void* base, int bytes, unsigned char* lds, unsigned voff) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
}

__device__ __forceinline__ void wm8_dma4(const void* base, int bytes, unsigned char* lds, unsigned voff) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 4, voff, 0, 0, 0);
}
// LDS accesses in assembly; the caller waits before it uses what it reads.  In front of reads and writes of its own the compiler waits for
// every LDS-DMA in flight -- here for the next step's, which had just been issued: 86 us instead of 76 at 32768 x 2560 x 320.
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
// transposed
template <int OFF>
__device__ __forceinline__ void tr_read(bf16x4_t& v, unsigned addr) {
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF) : "memory");
}

// min(4, left) values to (or added to) dst.  The adding form is kept out of line: 25 copies of it would be fetched once each from far memory.
__device__ __attribute__((noinline)) void wm8_add(float* dst, int left, f32x4_t v) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) dst[e] += v[e];
}
__device__ __forceinline__ void wm8_store(float* dst, int left, f32x4_t v, int accumulate) {
  if (left <= 0) return;
  if (accumulate) {
    wm8_add(dst, left, v);
  } else if (left >= 4) {
    store16_any(dst, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
  } else {                                                 // the end of a row
    dst[0] = v[0];
    if (left > 1) dst[1] = v[1];
    if (left > 2) dst[2] = v[2];
  }
}

template <int T0, int T1, int W0, int W1>
__global__ void __launch_bounds__(512)
linear_wgrad_mx8_kernel(const WgradMx8Params p) {
  constexpr unsigned OOB = 0x80000000u;
  constexpr int F0 = T0 / W0 / 16, F1 = T1 / W1 / 16;
  constexpr int IMG0 = WM8_MS * T0 * 2, IMG1 = WM8_MS * T1 * 2, SLOT = IMG0 + IMG1;
  constexpr int ND = IMG0 / 1024 / 8;                      // dY DMA instructions of a wave a step
  constexpr int UPR = T1 / 16;                             // units of 16 columns (half a block) a row of x
  constexpr int UNITS = WM8_MS * UPR, UMAX = (UNITS + 511) / 512, UFULL = UNITS / 512;
  constexpr int RAW = UNITS * 20;
  static_assert(W0 * W1 == 8 && IMG0 % 8192 == 0 && UNITS % 64 == 0 && UMAX <= 2, "tile / waves mismatch");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int w0 = wave / W1, w1 = wave % W1;
  // Workgroups b and b + 8 share an XCD.  Every XCD gets a contiguous run of (split, tile): the tiles of one range of rows then share its
  // rows of dY and x in one L2 (spread over the XCDs, x came over the fabric once for each of them: 265 MB for 180 MB of operands)
  const int blocks = gridDim.x, q8 = blocks >> 3, r8 = blocks & 7, xcd = blockIdx.x & 7;
  const int work = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + ((int)blockIdx.x >> 3);
  const int tiles = p.tiles_n * p.tiles_k, split = work / tiles, tile = work - split * tiles;
  const int tn = tile % p.tiles_n, tk = tile / p.tiles_n;
  const int n0 = tn * T0, k0 = tk * T1;
  const int total_steps = (int)((p.rows + WM8_MS - 1) / WM8_MS);
  const int step_begin = split * p.steps_per_split;
  const int nsteps = min(step_begin + p.steps_per_split, total_steps) - step_begin;

  // ---- loads.  dY: the descriptor moves 64 rows a step and ends with the matrix (rows past it read as zeros); lane offsets are constant.
  // x: units of 16 elements of one row, and the 32-bit word with their block's scale byte, into a place of the thread's own (two steps'
  // worth); rows past the end and blocks past the row read as zeros.
  unsigned dvoff[ND];
#pragma unroll
  for (int j = 0; j < ND; ++j) {
    const int c = (j * 8 + wave) * 64 + lane, row = c / (T0 / 8), phys = c - row * (T0 / 8);
    const int col = n0 + (phys ^ wm8_swz<T0>(row)) * 8;
    dvoff[j] = col < p.n ? ((unsigned)row * p.n + col) * 2u : OOB;
  }
  const int dy_row = p.n * 2, xd_row = p.blocks * 32;
  auto rows_of = [&](int step) {                           // rows of a step inside the matrix
    if (step >= step_begin + nsteps) return 0;             // fetched like any other: zeros that nobody reads
    return step == total_steps - 1 ? (int)(p.rows - (long long)step * WM8_MS) : WM8_MS;
  };
  // the loads of the step being issued: set up once a step, then issued one instruction at a time between MFMAs
  const char* dy_ptr = p.dy + (long long)step_begin * WM8_MS * dy_row;
  int dy_step = step_begin, dy_bytes = 0;
  unsigned char* dy_dst = nullptr;
  auto begin_dy = [&](int slot) {
    dy_bytes = rows_of(dy_step) * dy_row;
    dy_dst = smem + slot * SLOT + wave * 1024;
  };
  auto issue_dy = [&](int j) { wm8_dma16(dy_ptr, dy_bytes, dy_dst + j * 8192, dvoff[j]); };
  auto end_dy = [&]() {
    dy_ptr += (long long)WM8_MS * dy_row;
    ++dy_step;
  };
  auto has_unit = [&](int u) { return u < UFULL || u * 512 + wave * 64 < UNITS; };        // wave-uniform
  unsigned char* const raw = smem + 2 * SLOT;
  unsigned udata[UMAX], uscale[UMAX];
#pragma unroll
  for (int u = 0; u < UMAX; ++u) {
    const int id = u * 512 + tid, row = id / UPR, half = id - row * UPR, blk = (k0 >> 5) + (half >> 1);
    udata[u] = blk < p.blocks ? (unsigned)row * xd_row + blk * 32u + (half & 1) * 16u : OOB;
    uscale[u] = blk < p.blocks ? (unsigned)row * p.sstride + (blk & ~3) : OOB;
  }
  const unsigned char* xd_ptr = p.x + (long long)step_begin * WM8_MS * xd_row;
  const unsigned char* xs_ptr = p.xs + (long long)step_begin * WM8_MS * p.sstride;
  int x_step = step_begin;
  auto load_x = [&](int place) {
    const int rows = rows_of(x_step);
    unsigned char* const dst = raw + place * RAW;
#pragma unroll
    for (int u = 0; u < UMAX; ++u)
      if (has_unit(u)) {
        wm8_dma16(xd_ptr, rows * xd_row, dst + (u * 8 + wave) * 1024, udata[u]);
        wm8_dma4(xs_ptr, rows * p.sstride, dst + UNITS * 16 + (u * 8 + wave) * 256, uscale[u]);
      }
    xd_ptr += (long long)WM8_MS * xd_row;
    xs_ptr += (long long)WM8_MS * p.sstride;
    ++x_step;
  };

  // ---- widening: this thread's units
  unsigned udst[UMAX];
  int ubyte[UMAX];
#pragma unroll
  for (int u = 0; u < UMAX; ++u) {
    const int id = u * 512 + tid, row = id / UPR, half = id - row * UPR;
    udst[u] = IMG0 + row * (T1 * 2) + (((2 * half) ^ wm8_swz<T1>(row)) << 4);
    ubyte[u] = 8 * (((k0 >> 5) + (half >> 1)) & 3);
  }
  const unsigned lds_base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  i32x4_t xraw[UMAX];
  int xcode[UMAX];
  auto read_raw = [&](int place) {
#pragma unroll
    for (int u = 0; u < UMAX; ++u) {
      xraw[u] = i32x4_t{0, 0, 0, 0};
      xcode[u] = 0;
      if (has_unit(u)) {
        lds_read16<0>(xraw[u], lds_base + 2 * SLOT + place * RAW + (u * 512 + tid) * 16);
        lds_read4<UNITS * 16>(xcode[u], lds_base + 2 * SLOT + place * RAW + (u * 512 + tid) * 4);
      }
    }
  };
  auto raw_here = [&] {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int u = 0; u < UMAX; ++u) { stay_below(xraw[u]); stay_below(xcode[u]); }
  };
  uint32_t wide[8];
  float one = 0.f;
  auto widen_begin = [&](auto unit) {
    constexpr int u = decltype(unit)::value;
    const int code = (xcode[u] >> ubyte[u]) & 255;
    one = code == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(1.0f, code - 133);
  };
  auto widen_word = [&](auto unit, auto word) {            // four elements
    constexpr int u = decltype(unit)::value, i = decltype(word)::value;
    const unsigned w = (unsigned)xraw[u][i];
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)((int)(w << (24 - 8 * e)) >> 24) * one;
    wide[2 * i] = pack_bf16x2(v[0], v[1]);
    wide[2 * i + 1] = pack_bf16x2(v[2], v[3]);
  };
  auto widen = [&](auto unit) {
    widen_begin(unit);
    [&]<int... I>(std::integer_sequence<int, I...>) { (widen_word(unit, std::integral_constant<int, I>{}), ...); }(std::make_integer_sequence<int, 4>{});
  };
  auto write_wide = [&](auto unit, int slot) {
    constexpr int u = decltype(unit)::value;
    if (has_unit(u)) {
      const unsigned d = lds_base + slot * SLOT + udst[u];
      lds_write16<0>(d, i32x4_t{(int)wide[0], (int)wide[1], (int)wide[2], (int)wide[3]});
      lds_write16<16>(d, i32x4_t{(int)wide[4], (int)wide[5], (int)wide[6], (int)wide[7]});
    }
  };
  using First = std::integral_constant<int, 0>;
  using Last = std::integral_constant<int, UMAX - 1>;

  f32x4_t acc[F0][F1];
#pragma unroll
  for (int i = 0; i < F0; ++i)
#pragma unroll
    for (int j = 0; j < F1; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  // transposed fragments: lane -> row 4 fq + tq (and 16, 32, 48 further down, where the swizzle is the same), chunk 2 ct + (tp >> 1),
  // half tp & 1
  const int fr = lane & 15, fq = lane >> 4, tq = fr >> 2, tp = fr & 3;
  const int frow = 4 * fq + tq;
  constexpr int NO0 = wm8_distinct<T0, F0>(), NO1 = wm8_distinct<T1, F1>();
  unsigned off0[NO0], off1[NO1];
#pragma unroll
  for (int i = 0; i < NO0; ++i)
    off0[i] = lds_base + frow * (T0 * 2) + (((2 * (w0 * F0 + i) + (tp >> 1)) ^ wm8_swz<T0>(frow)) << 4) + ((tp & 1) << 3);
#pragma unroll
  for (int j = 0; j < NO1; ++j)
    off1[j] = lds_base + IMG0 + frow * (T1 * 2) + (((2 * (w1 * F1 + j) + (tp >> 1)) ^ wm8_swz<T1>(frow)) << 4) + ((tp & 1) << 3);

  struct Frags { bf16x4_t lo0[F0], hi0[F0], lo1[F1], hi1[F1]; };
  // fragment Q (dY's, then x's) of 32-row block B of a slot
  auto read_fragment = [&]<int B, int Q>(std::integral_constant<int, B>, std::integral_constant<int, Q>, Frags& f, unsigned sbase) {
    if constexpr (Q < F0) {
      constexpr int i = Q;
      tr_read<i / NO0 * (NO0 * 32) + B * 32 * T0 * 2>(f.lo0[i], sbase + off0[i % NO0]);
      tr_read<i / NO0 * (NO0 * 32) + (B * 32 + 16) * T0 * 2>(f.hi0[i], sbase + off0[i % NO0]);
    } else {
      constexpr int j = Q - F0;
      tr_read<j / NO1 * (NO1 * 32) + B * 32 * T1 * 2>(f.lo1[j], sbase + off1[j % NO1]);
      tr_read<j / NO1 * (NO1 * 32) + (B * 32 + 16) * T1 * 2>(f.hi1[j], sbase + off1[j % NO1]);
    }
  };
  auto here = [&](Frags& f) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < F0; ++i) asm volatile("" : "+v"(f.lo0[i]), "+v"(f.hi0[i]));   // no use of a fragment moves above the wait
#pragma unroll
    for (int j = 0; j < F1; ++j) asm volatile("" : "+v"(f.lo1[j]), "+v"(f.hi1[j]));
  };
  // a block's products; behind the first of them the reads of block B into `ahead`, behind the others -- with DY -- dY's loads
  auto multiply = [&]<int B, bool DY>(const Frags& f, Frags& ahead, unsigned sbase, std::integral_constant<int, B> block, std::integral_constant<bool, DY>) {
    auto join = [](const bf16x4_t& lo, const bf16x4_t& hi) {
      return bf16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    __builtin_amdgcn_sched_barrier(0);
    [&]<int... Q>(std::integer_sequence<int, Q...>) {
      ([&] {
        constexpr int q = Q, i = q / F1, j = q % F1, FF = F0 + F1, MM = F0 * F1;
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(join(f.lo1[j], f.hi1[j]), join(f.lo0[i], f.hi0[i]), acc[i][j], 0, 0, 0);
        if constexpr (q < FF) read_fragment(block, std::integral_constant<int, q>{}, ahead, sbase);
        if constexpr (DY) {
#pragma unroll
          for (int d = q * ND / MM; d < (q + 1) * ND / MM; ++d) issue_dy(d);
        }
        __builtin_amdgcn_sched_barrier(0);
      }(), ...);
    }(std::make_integer_sequence<int, F0 * F1>{});
  };
  static_assert(F0 + F1 <= F0 * F1, "a read behind each product");
  constexpr std::integral_constant<int, 0> B0{};
  constexpr std::integral_constant<int, 1> B1{};

  if (nsteps > 0) {
    auto arrive = [&]() {                                  // what this wave loaded and wrote is there, and then everybody's is
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    auto load_dy = [&](int slot) {
      begin_dy(slot);
#pragma unroll
      for (int j = 0; j < ND; ++j) issue_dy(j);
      end_dy();
    };
    auto next_x = [&](int slot) {
      widen(First{});
      write_wide(First{}, slot);
      if constexpr (UMAX > 1) { widen(Last{}); write_wide(Last{}, slot); }
    };
    Frags f0, f1;
    load_x(0);
    load_dy(0);
    load_x(1);
    arrive();
    read_raw(0);
    raw_here();
    next_x(0);
    load_dy(1);
    load_x(0);
    arrive();
    read_raw(1);
    [&]<int... Q>(std::integer_sequence<int, Q...>) {
      (read_fragment(B0, std::integral_constant<int, Q>{}, f0, 0u), ...);
    }(std::make_integer_sequence<int, F0 + F1>{});
    here(f0);
    raw_here();
    // At the top of step s: block 0 of slot s & 1 in f0, the stored x(s + 1) in registers, x(s + 2) in place s & 1, dY(s + 1) in or on its way to
    // the other slot.  The barrier in the middle frees the step's slot (its block 1 is in registers) and says that the next one is
    // whole; x(s + 1) is widened in front of block 0 by waves 4 .. 7 and behind it by waves 0 .. 3 -- the other wave of each SIMD -- so
    // that the SIMD's matrix core works for one while the other converts.
    for (int s = 0; s < nsteps; ++s) {
      const int cur = s & 1, next = cur ^ 1;
      if (wave >= 4) next_x(next);
      multiply(f0, f1, (unsigned)cur * SLOT, B1, std::false_type{});
      if (wave < 4) next_x(next);
      here(f1);
      arrive();
      read_raw(cur);
      begin_dy(cur);
      load_x(next);
      multiply(f1, f0, (unsigned)next * SLOT, B0, std::true_type{});
      end_dy();
      here(f0);
      raw_here();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }

  // x is the instruction's first operand: a lane has four consecutive k (rows 4 fq .. + 3 of the fragment) of one n (column fr)
  float* out = p.out + (long long)split * p.n * p.k;
#pragma unroll
  for (int i = 0; i < F0; ++i) {
    const int n = n0 + (w0 * F0 + i) * 16 + fr;
    float* row = out + (long long)n * p.k + k0 + w1 * (T1 / W1) + fq * 4;
    const int left = n < p.n ? p.k - (k0 + w1 * (T1 / W1) + fq * 4) : 0;
#pragma unroll
    for (int j = 0; j < F1; ++j) wm8_store(row + j * 16, left - j * 16, acc[i][j], p.accumulate);
  }
}

// dw (+)= the partial tiles, in order.  The loads of eight are under way at a time: one by one they would wait for each other.
__global__ void __launch_bounds__(256)
wgrad_mx8_fold_kernel(const float* __restrict__ partial, float* __restrict__ dw, long long total, int splits, int accumulate) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  float v = accumulate ? dw[i] : 0.f;
  int s = 0;
  for (; s + 8 <= splits; s += 8) {
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = partial[(long long)(s + j) * total + i];
#pragma unroll
    for (int j = 0; j < 8; ++j) v += o[j];
  }
  for (; s < splits; ++s) v += partial[(long long)s * total + i];
  dw[i] = v;
}

// Tile shape: least padded work (channel counts of this model family are multiples of 320), then the larger one.  Enough splits of the
// rows for one workgroup on every CU but no second round, at least 4 steps each.
static int wgrad_mx8_plan(long long rows, int n, int k, WgradMx8Params& p) {
  static const int shapes[4][2] = {{320, 160}, {256, 192}, {256, 160}, {256, 128}};
  long long best = -1;
  int cfg = 0;
  for (int c = 0; c < 4; ++c) {
    const long long tn = (n + shapes[c][0] - 1) / shapes[c][0], tk = (k + shapes[c][1] - 1) / shapes[c][1];
    const long long padded = tn * shapes[c][0] * tk * shapes[c][1];
    if (best < 0 || padded < best) { best = padded; cfg = c; p.tiles_n = (int)tn; p.tiles_k = (int)tk; }
  }
  const int steps = (int)((rows + WM8_MS - 1) / WM8_MS);
  const long long tiles = (long long)p.tiles_n * p.tiles_k;
  long long splits = tiles >= 256 ? 1 : 256 / tiles;
  if (splits > steps / 4) splits = steps / 4;
  if (splits < 1) splits = 1;
  p.steps_per_split = (int)((steps + splits - 1) / splits);
  p.splits = (steps + p.steps_per_split - 1) / p.steps_per_split;
  return cfg;
}

template <int T0, int T1, int W0, int W1>
static int launch_wgrad_mx8(const WgradMx8Params& p, hipStream_t st) {
  constexpr int smem = 2 * WM8_MS * ((T0 + T1) * 2 + (T1 / 16) * 20);
  static_assert(smem <= 160 * 1024, "LDS");
  auto kern = linear_wgrad_mx8_kernel<T0, T1, W0, W1>;
  static bool done = false;
  if (!done) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != hipSuccess) { set_error("ldm_linear_wgrad_mx8: hipFuncSetAttribute: %s", hipGetErrorString(e)); return LDM_EHIP; }
    done = true;
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)(p.tiles_n * p.tiles_k * p.splits)), dim3(512), smem, st, p);
  return LDM_OK;
}

}  // namespace ldm

using namespace ldm;

// n, k: 64 rows of dY and of the checkpoint lie under descriptors of less than 2^31 bytes
static bool wgrad_mx8_sizes_ok(long long rows, int n, int k) {
  return rows >= 1 && rows <= 32LL * 0x7fffffff && n >= 1 && k >= 1 && n <= (1 << 24) - 8 && k <= (1 << 24) && (long long)n * k < (1LL << 38);
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
  LDM_REQUIRE(x8 && x8_scale && dy && dw && aligned16(x8) && aligned16(dy) && (reinterpret_cast<uintptr_t>(x8_scale) & 3) == 0,
              "ldm_linear_wgrad_mx8: null or unaligned pointer");
  WgradMx8Params p;
  const int cfg = wgrad_mx8_plan(rows, n, k, p);
  const long long need = p.splits > 1 ? (long long)p.splits * n * k * 4 : 0;
  LDM_REQUIRE(need == 0 || (workspace != nullptr && aligned16(workspace) && workspace_bytes >= need),
              "ldm_linear_wgrad_mx8: workspace of %lld bytes needed (got %lld)", need, workspace_bytes);
  LDM_REQUIRE((long long)p.tiles_n * p.tiles_k * p.splits < (1LL << 31), "ldm_linear_wgrad_mx8: too large");
  p.x = static_cast<const unsigned char*>(x8); p.xs = static_cast<const unsigned char*>(x8_scale); p.dy = static_cast<const char*>(dy);
  p.rows = rows; p.n = n; p.k = k; p.blocks = mx_blocks(k); p.sstride = mx_scale_stride(k);
  p.out = need ? static_cast<float*>(workspace) : dw;
  p.accumulate = need ? 0 : accumulate;
  hipStream_t st = (hipStream_t)stream;
  const int rc = cfg == 0   ? launch_wgrad_mx8<320, 160, 4, 2>(p, st)
                 : cfg == 1 ? launch_wgrad_mx8<256, 192, 4, 2>(p, st)
                 : cfg == 2 ? launch_wgrad_mx8<256, 160, 4, 2>(p, st)
                            : launch_wgrad_mx8<256, 128, 4, 2>(p, st);
  if (rc) return rc;
  LDM_HIP_CHECK_LAUNCH("ldm_linear_wgrad_mx8");
  if (need) {
    const long long total = (long long)n * k;
    hipLaunchKernelGGL(wgrad_mx8_fold_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st, p.out, dw, total, p.splits, accumulate);
    LDM_HIP_CHECK_LAUNCH("ldm_linear_wgrad_mx8(fold)");
  }
  return LDM_OK;
}
