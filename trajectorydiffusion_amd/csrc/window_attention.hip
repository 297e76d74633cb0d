// Attention with a window and a few first tokens that stay visible (tdx_window_attention), forward and backward.
//
// Which key a row sees: p = i + k_len - q_len;  j < k_len,  j <= p + right,  j >= p - left or j < sinks.
//
// Layout of every kernel.  The Hq / Hkv query heads that read one key head are packed into the rows of a tile: row r of (batch, key
// head) is query r / G, head r % G of the group, so the keys are loaded once for the group and a 32-row tile spans only 32 / G
// positions of the window.  A wave owns 32 rows as the COLUMNS of its products (32x32 matrix instructions):
//   S^T (keys x rows) = K Q^T, the accumulator of lane (n = lane & 31, h = lane >> 5) then holds, for row n, the scores of the keys
//   8 g + 4 h + r (g, r = 0..3): softmax statistics are one number per lane (and its partner n + 32), and the probabilities are
//   already where the second product wants its right operand, O^T (channels x rows) = V^T P^T, once its contraction index is
//   taken in the order the scores are held in.  V^T then has to be read from LDS along the keys: 16-bit tiles by the transposing
//   LDS read, which hands lane i of 16 lanes column i of a 4 x 16 tile; fp32 tiles (few rows) by plain 4-byte reads (one key per lane half).
// K and V tiles are staged in LDS as they lie in memory (direct loads, 16 bytes a lane); the 16-byte pieces of a row are permuted
// (swz) so that neither the row reads nor the transposed ones meet in a bank.
#include "tdx_common.h"

#include <algorithm>
#include <bit>
#include <cmath>
#include <type_traits>

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4_t;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4_t;
typedef __attribute__((address_space(3))) float lds_f32_t;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4_t;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kFar = 1 << 30;         // a limit no position reaches (lengths stay below 2^28)
constexpr uint32_t kOutside = 0x80000000u;

struct WaArgs {
  const void *q, *k, *v;
  void* out;
  __bf16* out_lo;                     // or null: what the rounding of out left, (B, Tq, Hq, D)
  float* lse;
  long q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, o_bs, o_ts, o_hs;
  int B, Tq, Tk, Hkv, G, D;
  int left, right, sinks;
  float scale, down, up;              // exponentials are taken 2^down smaller, up = 2^down (see softmax_exp)
  const int *q_lens, *k_lens;
  int ntiles, nsplit;                 // row (backward: or key) tiles of a (batch, key head); key (backward: row) splits
  float* ws;
  // backward
  const void* dout;
  void *dq, *dk, *dv;
  long do_bs, do_ts, do_hs, dq_bs, dq_ts, dq_hs, dk_bs, dk_ts, dk_hs, dv_bs, dv_ts, dv_hs;
  float *stat, *part, *near;          // per 32 rows kStat numbers (see there); shares of the sinks' gradients; of all rows' (nkey > 1), then of all keys' (nrow > 1)
  int ntiles32, nparts, sink_rows;    // row tiles of 32; shares; sinks rounded up to 32 (0: no separate pass over the sinks)
  int nrow, nkey;                     // shares that the rows of a key tile (dK / dV) and the keys of a row tile (dQ) are cut into
};

// ---- geometry of a staged tile ------------------------------------------------------------------------------------------------
template <typename T, int DP>
struct Geo {
  static constexpr int ES = sizeof(T), PITCH = DP * ES, CH = PITCH / 16, ND = DP / 32, RPI = 1024 / PITCH;
};
// Permutation of the 16-byte pieces of row `row`.  Row reads (16 rows, one piece): the bank groups must differ over 16 rows.
// Transposed reads: bf16 takes 4 rows x 64 bytes at a time (rows 4a .. 4a+3 must differ in the 64-byte block), fp32 the 128 bytes of
// rows R and R + 4 (they must differ in the 128-byte block).
template <typename T, int DP>
__device__ __forceinline__ int swz(int row) {
  constexpr int CH = Geo<T, DP>::CH;
  if constexpr (CH == 4) return (row >> 2) & 3;
  else if constexpr (CH == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  else if constexpr (sizeof(T) == 2) return ((row & 3) << 2) | ((row >> 2) & 3);
  else return (row & 3) | (((row >> 2) & 1) << 3) | (((row >> 3) & 1) << 2);
}

__device__ __forceinline__ u32x4 lds_ld16(uint32_t a) { return *reinterpret_cast<lds_u32x4_t*>(a); }
__device__ __forceinline__ float lds_ld4(uint32_t a) { return *reinterpret_cast<lds_f32_t*>(a); }

__device__ __forceinline__ u32x4 make_srd(const void* base) {
  const uint64_t a = (uint64_t)base;
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu);
  r[2] = 0x7fffffffu;
  r[3] = 0x00020000u;
  return r;
}
// 64 lanes x 16 B from srd[voff] to LDS[lds_addr + 16 * lane]; lanes with voff >= 2^31 - 1 write zeros.  Issued from asm so that the
// compiler does not order later LDS reads behind it: the kernels wait for their loads themselves (vmcnt, then a barrier).
__device__ __forceinline__ void dma16(uint32_t lds_addr, uint32_t voff, const u32x4& srd) {
  uint32_t keep;
  lds_addr = __builtin_amdgcn_readfirstlane(lds_addr);
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "s"(lds_addr), "v"(voff), "s"(srd)
      : "memory");
}
// The same N times, 4096 bytes of LDS apart
template <int N>
__device__ __forceinline__ void dma16n(uint32_t lds_addr, const uint32_t (&voff)[N], const u32x4& srd) {
  uint32_t keep;
  lds_addr = __builtin_amdgcn_readfirstlane(lds_addr);
  if constexpr (N == 4) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %2, %6, 0 offen lds\n\t"
        "s_add_u32 m0, m0, 4096\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %3, %6, 0 offen lds\n\t"
        "s_add_u32 m0, m0, 4096\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %4, %6, 0 offen lds\n\t"
        "s_add_u32 m0, m0, 4096\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %5, %6, 0 offen lds\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "s"(lds_addr), "v"(voff[0]), "v"(voff[1]), "v"(voff[2]), "v"(voff[3]), "s"(srd)
        : "memory", "scc");
  } else if constexpr (N == 2) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %2, %4, 0 offen lds\n\t"
        "s_add_u32 m0, m0, 4096\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %3, %4, 0 offen lds\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "s"(lds_addr), "v"(voff[0]), "v"(voff[1]), "s"(srd)
        : "memory", "scc");
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n) dma16(lds_addr + 4096 * n, voff[n], srd);
  }
}
template <int N>
__device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// every wave's LDS traffic is complete, then the barrier (without a release fence, which would wait for the direct loads in flight)
__device__ __forceinline__ void wg_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Stages `ROWS` rows (row 0 at `base`, `stride` bytes apart) by NW waves; rows from `valid` on and channels from `dbytes` on are zeros.
template <typename T, int DP, int ROWS, int NW>
__device__ __forceinline__ void stage_rows(uint32_t lds, const char* base, uint32_t stride, int valid, int dbytes, int wave, int lane) {
  using G = Geo<T, DP>;
  constexpr int TOTAL = ROWS * G::PITCH / 1024;
  const u32x4 srd = make_srd(base);
#pragma unroll
  for (int n = 0; n < (TOTAL + NW - 1) / NW; ++n) {
    const int it = wave + n * NW;
    if (TOTAL % NW == 0 || it < TOTAL) {
      const int row = it * G::RPI + lane / G::CH;
      const int chunk = (lane % G::CH) ^ swz<T, DP>(row);
      const bool ok = row < valid && chunk * 16 < dbytes;
      dma16(lds + it * 1024, ok ? (uint32_t)row * stride + chunk * 16 : kOutside, srd);
    }
  }
}

// ---- matrix steps ---------------------------------------------------------------------------------------------------------------
// acc[dt] (channels 32 dt .. + 31 x 32 columns) += (tile rows [row0, row0 + 32))^T p, p as few_scores left it: element i of a lane is tile
// row row0 + 8 (i / 4) + 4 h + i % 4
template <int DP>
__device__ __forceinline__ void cols_times(f32x16 (&acc)[DP / 32], uint32_t tile, int row0, const float (&p)[16], int lane, __bf16) {
  using G = Geo<__bf16, DP>;
  const int rl = 4 * (lane >> 5) + ((lane >> 2) & 3);              // the row this lane addresses inside a group of 8
  const int piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);      // and the 16-byte piece inside the 64 bytes of 32 channels
#pragma unroll
  for (int s = 0; s < 2; ++s) {                                     // 16 tile rows a step
    float pe[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) pe[j] = p[8 * s + j];
    const bf16x8 b = __builtin_bit_cast(bf16x8, Elem<__bf16>::pack(pe));
    const int ra = row0 + 16 * s + rl, rb = ra + 8;
#pragma unroll
    for (int dt = 0; dt < G::ND; ++dt) {
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<lds_s16x4_t*>(tile + ra * G::PITCH + (((4 * dt + piece) ^ swz<__bf16, DP>(ra)) << 4) + 8 * (lane & 1)));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<lds_s16x4_t*>(tile + rb * G::PITCH + (((4 * dt + piece) ^ swz<__bf16, DP>(rb)) << 4) + 8 * (lane & 1)));
      const bf16x8 a = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc[dt], 0, 0, 0);
    }
  }
}
template <int DP>
__device__ __forceinline__ void cols_times(f32x16 (&acc)[DP / 32], uint32_t tile, int row0, const float (&p)[16], int lane, float) {
  using G = Geo<float, DP>;
  constexpr int STEPS = 16 * G::ND, AHEAD = 6, RING = AHEAD + 1;     // two tile rows a step, one for each lane half
  float r[RING];
  auto read = [&](int k) {
    const int i = k / G::ND, d = 32 * (k % G::ND) + (lane & 31);
    const int row = row0 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
    r[k % RING] = lds_ld4(tile + row * G::PITCH + (((d >> 2) ^ swz<float, DP>(row)) << 4) + 4 * (d & 3));
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) read(k);
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    if (k + AHEAD < STEPS) read(k + AHEAD);
    __builtin_amdgcn_sched_barrier(0);
    acc[k % G::ND] = __builtin_amdgcn_mfma_f32_32x32x2f32(r[k % RING], p[k / G::ND], acc[k % G::ND], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
}

__device__ __forceinline__ float half_max(float v) {   // with the partner lane of the other half
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// ---- tiles in 16 bits: bf16 as it is, fp32 as three bf16 planes ------------------------------------------------------------------------
// The many-row kernels multiply fp32 as sums of bf16 products: x = hi + mid + lo, each the bf16 nearest to what the ones before it leave, holds
// all 24 bits, and of the nine products the six down to 2^-16 are taken (the three others are below 2^-25 of |x y| together: less than the
// sum's own rounding in 32 bits).  Six 32x32x16 instructions at 16 times the fp32 rate are 2.7 times as fast as the fp32 matrix instructions.
template <typename T>
struct Planes {
  static constexpr int N = sizeof(T) == 4 ? 3 : 1;
};
template <int DP>
struct G16 {
  static constexpr int PITCH = DP * 2, CH = PITCH / 16, NC = DP / 16, ND = DP / 32;
};
template <int N, int DP>
using Frags16 = bf16x8[N][G16<DP>::NC];

// LDS offsets of a lane, the same for every tile: what differs between tiles, stages and planes is an immediate of the read
template <int DP>
struct LaneOff {
  uint32_t row[G16<DP>::NC];          // row lane & 31, piece 2 c + lane half
  uint32_t lo[G16<DP>::ND], hi[G16<DP>::ND];   // transposed reads of rows 4 h .. 4 h + 3 and 8 + 4 h .. (rows + 16: the same permutation)
  __device__ __forceinline__ LaneOff(uint32_t base, int lane) {
    using G = G16<DP>;
    const int r = lane & 31;
#pragma unroll
    for (int c = 0; c < G::NC; ++c) row[c] = base + r * G::PITCH + (((2 * c + (lane >> 5)) ^ swz<__bf16, DP>(r)) << 4);
    const int ra = 4 * (lane >> 5) + ((lane >> 2) & 3), piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
    for (int d = 0; d < G::ND; ++d) {
      lo[d] = base + ra * G::PITCH + (((4 * d + piece) ^ swz<__bf16, DP>(ra)) << 4) + 8 * (lane & 1);
      hi[d] = base + (ra + 8) * G::PITCH + (((4 * d + piece) ^ swz<__bf16, DP>(ra + 8)) << 4) + 8 * (lane & 1);
    }
  }
};

__device__ __forceinline__ f32x16 mfma16(const bf16x8& a, const bf16x8& b, const f32x16& c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
// SWAP: in the order that gives the bits of the product with a and b exchanged
template <int N, bool SWAP = false>
__device__ __forceinline__ void mma_planes(f32x16& acc, const bf16x8 (&a)[N], const bf16x8 (&b)[N]) {
  if constexpr (N == 3) {   // the smallest products first
    constexpr int X = SWAP ? 0 : 2, Y = 2 - X, Z = SWAP ? 0 : 1, W = 1 - Z;
    acc = mfma16(a[X], b[Y], acc);
    acc = mfma16(a[Y], b[X], acc);
    acc = mfma16(a[1], b[1], acc);
    acc = mfma16(a[Z], b[W], acc);
    acc = mfma16(a[W], b[Z], acc);
  }
  acc = mfma16(a[0], b[0], acc);
}
// Reads run AHEAD steps in front of the matrix instructions that take them, and vector work that is ready stands between these: the order
// is pinned, since left alone the compiler reads one fragment, waits for it and multiplies, and every step pays the read's latency
// (dK / dV, causal prompts of 4096 tokens, 16 / 4 heads of 128 channels, window 1024: 293 -> 241 us).
__device__ __forceinline__ void pin() {
  __builtin_amdgcn_sched_barrier(0);
}
struct Nothing {
  __device__ __forceinline__ void operator()(int) const {}
};
// acc (32 tile rows x 32 columns) = the 32 tile rows at IMM times the fragments b; planes of a tile are PLANE bytes apart.
// between(c) is called behind the instructions of step c < NC.  SWAP: see mma_planes.
template <int N, int DP, uint32_t IMM, uint32_t PLANE, bool SWAP = false, typename F = Nothing>
__device__ __forceinline__ void rows16(f32x16& acc, const LaneOff<DP>& off, const Frags16<N, DP>& b, F&& between = F()) {
  constexpr int NC = G16<DP>::NC, AHEAD = N == 3 ? 1 : NC < 4 ? NC : 4, RING = AHEAD + 1;
  bf16x8 a[RING][N];
  auto read = [&](int c) {
#pragma unroll
    for (int n = 0; n < N; ++n) a[c % RING][n] = __builtin_bit_cast(bf16x8, lds_ld16(off.row[c] + IMM + n * PLANE));
  };
#pragma unroll
  for (int c = 0; c < AHEAD; ++c) read(c);
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (c + AHEAD < NC) read(c + AHEAD);
    pin();
    bf16x8 bc[N];
#pragma unroll
    for (int n = 0; n < N; ++n) bc[n] = b[n][c];
    mma_planes<N, SWAP>(acc, a[c % RING], bc);
    between(c);
    pin();
  }
}
// x as N bf16 planes.  The first is bf16's largest number where fp32's are larger still, so that every number is the sum of its planes; an infinity
// has one that is NaN, and so have its products
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&p)[N]) {
  if constexpr (N == 1) {
    p[0] = __builtin_bit_cast(bf16x8, Elem<__bf16>::pack(x));
  } else {
    constexpr float most = 0x1.fep127f;
    float h[8], r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __builtin_amdgcn_fmed3f(x[i], -most, most);
    u32x4 w = Elem<__bf16>::pack(r);
    p[0] = __builtin_bit_cast(bf16x8, w);
    Elem<__bf16>::unpack(w, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i] - h[i];
    w = Elem<__bf16>::pack(r);
    p[1] = __builtin_bit_cast(bf16x8, w);
    Elem<__bf16>::unpack(w, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] -= h[i];
    p[2] = __builtin_bit_cast(bf16x8, Elem<__bf16>::pack(r));
  }
}
// the right operand of cols16: 32 rows' numbers as rows16 left them (element i of a lane is tile row 8 (i / 4) + 4 h + i % 4).  bf16 tensors: probabilities and
// score gradients are rounded to 16 bits here, which the instruction takes on both sides.  Each is off by 2^-9 at most, independently, so a result is off by 1.35
// to 1.45 times what rounding it once at the end leaves (measured against 64 bits: 0.0023 and 0.0017 of its size); a second plane would double the products with V.
template <int N>
__device__ __forceinline__ void pack16(bf16x8 (&b)[2][N], const float (&p)[16]) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    float pe[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) pe[j] = p[8 * s + j];
    split8<N>(pe, b[s]);
  }
}
// acc[dt] (channels 32 dt .. + 31 x 32 columns) += (the 32 tile rows at IMM)^T b.  between(k) is called behind the instructions of step
// k < 2 ND.
template <int N, int DP, uint32_t IMM, uint32_t PLANE, typename F = Nothing>
__device__ __forceinline__ void cols16(f32x16 (&acc)[DP / 32], const LaneOff<DP>& off, const bf16x8 (&b)[2][N], F&& between = F()) {
  using G = G16<DP>;
  constexpr int STEPS = 2 * G::ND, AHEAD = N == 3 ? 1 : STEPS < 3 ? STEPS : 3, RING = AHEAD + 1;
  bf16x8 a[RING][N];
  auto read = [&](int k) {
    const int s = k / G::ND, dt = k % G::ND;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint32_t at = IMM + n * PLANE + 16 * s * G::PITCH;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4_t*>(off.lo[dt] + at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4_t*>(off.hi[dt] + at));
      a[k % RING][n] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) read(k);
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    if (k + AHEAD < STEPS) read(k + AHEAD);
    pin();
    mma_planes<N>(acc[k % G::ND], a[k % RING], b[k / G::ND]);
    between(k);
    pin();
  }
}
// piece c of a 32-row operand from memory: channels 16 c + 8 h .. + 7 of the lane's row `row`, zero beyond the channels or when !ok
template <typename T>
__device__ __forceinline__ void load_piece16(bf16x8 (&f)[Planes<T>::N], const T* row, int c, bool ok, int D, int lane) {
  const int d = 16 * c + 8 * (lane >> 5);
  const bool in = ok && d < D;
  if constexpr (sizeof(T) == 2) {
    f[0] = __builtin_bit_cast(bf16x8, in ? *reinterpret_cast<const u32x4*>(row + d) : (u32x4){0u, 0u, 0u, 0u});
  } else {
    float x[8];
    const u32x4 a = in ? *reinterpret_cast<const u32x4*>(row + d) : (u32x4){0u, 0u, 0u, 0u};
    const u32x4 b = in ? *reinterpret_cast<const u32x4*>(row + d + 4) : (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(a[i]), x[4 + i] = __uint_as_float(b[i]);
    split8<3>(x, f);
  }
}
// a 32-row operand in registers
template <typename T, int DP>
__device__ __forceinline__ void load_frags16(Frags16<Planes<T>::N, DP>& f, const T* row, bool ok, int D, int lane) {
#pragma unroll
  for (int c = 0; c < G16<DP>::NC; ++c) {
    bf16x8 p[Planes<T>::N];
    load_piece16<T>(p, row, c, ok, D, lane);
#pragma unroll
    for (int n = 0; n < Planes<T>::N; ++n) f[n][c] = p[n];
  }
}
// The product of row `held` (the same for all lanes) with the lane's own row, both from memory, in the bits of rows16 with `held` in the tile (SWAP: the other
// row); lanes n and n + 32 have the same row.
template <typename T, bool SWAP = false>
__device__ __forceinline__ float row_times(const T* held, const T* row, bool ok, int D, int lane) {
  f32x16 acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int c = 0; 16 * c < D; ++c) {
    bf16x8 a[Planes<T>::N], b[Planes<T>::N];
    load_piece16<T>(a, held, c, true, D, lane);
    load_piece16<T>(b, row, c, ok, D, lane);
    mma_planes<Planes<T>::N, SWAP>(acc, a, b);
  }
  return acc[0];
}
// Uses the fragments, so that the compiler's wait for their loads stands here and not inside a loop, where it would also wait for the
// direct loads in flight.
template <int N, int M>
__device__ __forceinline__ void arrived16(bf16x8 (&f)[N][M]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int c = 0; c < M; ++c) {
      u32x4 w = __builtin_bit_cast(u32x4, f[n][c]);
      asm volatile("" : "+v"(w));
      f[n][c] = __builtin_bit_cast(bf16x8, w);
    }
}

// One thread's part of staging a ROWS-row tile by 256 threads: direct loads into LDS, whose addresses a lane keeps from tile to tile.  bf16 is
// used as it arrives; fp32 arrives in a buffer of its own, from which put() writes the planes.  (Held in registers across a tile instead,
// the numbers spill, and a spill waits for its load.)
template <typename T, int DP, int ROWS>
struct Stager;
template <int DP, int ROWS>
struct Stager<__bf16, DP, ROWS> {
  using G = G16<DP>;
  static constexpr int TOTAL = ROWS * G::PITCH / 1024, PER = (TOTAL + 3) / 4;
  uint32_t voff[PER];
  int row0;                            // row of this lane in the wave's first load
  __device__ __forceinline__ static int row_of(int n, int wave, int lane) { return (wave + 4 * n) * (1024 / G::PITCH) + lane / G::CH; }
  // rows `stride` bytes apart
  __device__ __forceinline__ void init(uint32_t stride, int dbytes, int wave, int lane) {
    row0 = row_of(0, wave, lane);
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int row = row_of(n, wave, lane), chunk = (lane % G::CH) ^ swz<__bf16, DP>(row);
      voff[n] = chunk * 16 < dbytes ? (uint32_t)row * stride + chunk * 16 : kOutside;
    }
  }
  __device__ __forceinline__ void load(uint32_t lds, const char* base, int valid, int wave) const {
    static_assert(TOTAL % 4 == 0, "whole loads for each of the 4 waves");
    const u32x4 srd = make_srd(base);
    if (valid >= ROWS) {
      dma16n<PER>(lds + wave * 1024, voff, srd);
    } else {
      uint32_t v[PER];
#pragma unroll
      for (int n = 0; n < PER; ++n) v[n] = row0 + 4 * n * (1024 / G::PITCH) < valid ? voff[n] : kOutside;
      dma16n<PER>(lds + wave * 1024, v, srd);
    }
  }
};
template <int DP, int ROWS>
struct Stager<float, DP, ROWS> {
  using G = G16<DP>;
  static constexpr int P32 = DP * 4, TOTAL = ROWS * P32 / 1024, PER = TOTAL / 4, ITEMS = ROWS * G::CH;
  static constexpr uint32_t PLANE = ROWS * G::PITCH, RAW = ROWS * P32;
  static_assert(TOTAL % 4 == 0, "whole loads for each of the 4 waves");
  uint32_t voff[PER];
  int row0;
  __device__ __forceinline__ static int row_of(int n, int wave, int lane) { return (wave + 4 * n) * (1024 / P32) + lane / (P32 / 16); }
  __device__ __forceinline__ void init(uint32_t stride, int dbytes, int wave, int lane) {
    row0 = row_of(0, wave, lane);
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int at = (lane % (P32 / 16)) * 16;
      voff[n] = at < dbytes ? (uint32_t)row_of(n, wave, lane) * stride + at : kOutside;
    }
  }
  __device__ __forceinline__ void load(uint32_t raw, const char* base, int valid, int wave) const {
    const u32x4 srd = make_srd(base);
    if (valid >= ROWS) {
      dma16n<PER>(raw + wave * 1024, voff, srd);
    } else {
      uint32_t v[PER];
#pragma unroll
      for (int n = 0; n < PER; ++n) v[n] = row0 + 4 * n * (1024 / P32) < valid ? voff[n] : kOutside;
      dma16n<PER>(raw + wave * 1024, v, srd);
    }
  }
  __device__ __forceinline__ void put(uint32_t lds, uint32_t raw) const {
#pragma unroll
    for (int n = 0; n < (ITEMS + 255) / 256; ++n) {
      const int item = threadIdx.x + 256 * n, row = item / G::CH, chunk = item % G::CH;
      if (ITEMS % 256 == 0 || item < ITEMS) {
        float x[8];
        const u32x4 u = lds_ld16(raw + item * 32), w = lds_ld16(raw + item * 32 + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(u[i]), x[4 + i] = __uint_as_float(w[i]);
        bf16x8 p[3];
        split8<3>(x, p);
        const uint32_t at = lds + row * G::PITCH + ((chunk ^ swz<__bf16, DP>(row)) << 4);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<lds_u32x4_t*>(at + k * PLANE) = __builtin_bit_cast(u32x4, p[k]);
      }
    }
  }
};

// acc (32 keys x 32 columns) = the 32 rows of a tile as it lies in memory (swz) times the fragments b, in the bits of rows16: fp32 rows are split into planes here
template <typename T, int DP>
__device__ __forceinline__ void few_scores(f32x16& acc, uint32_t tile, const Frags16<Planes<T>::N, DP>& b, int lane) {
  constexpr int N = Planes<T>::N, NC = G16<DP>::NC, AHEAD = N == 3 ? 1 : NC < 4 ? NC : 4, RING = AHEAD + 1, PIECES = N == 3 ? 2 : 1;   // 16-byte pieces of a step
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  const int row = lane & 31;
  const uint32_t a0 = tile + row * Geo<T, DP>::PITCH;
  const int c0 = (PIECES * (lane >> 5)) ^ swz<T, DP>(row);
  // reads run AHEAD steps in front of the instructions that take them (see rows16)
  u32x4 p[RING][PIECES];
  auto read = [&](int c) {
#pragma unroll
    for (int x = 0; x < PIECES; ++x) p[c % RING][x] = lds_ld16(a0 + ((c0 ^ (2 * PIECES * c + x)) << 4));
  };
#pragma unroll
  for (int c = 0; c < AHEAD; ++c) read(c);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (c + AHEAD < NC) read(c + AHEAD);
    pin();
    bf16x8 ac[N], bc[N];
    if constexpr (N == 1) {
      ac[0] = __builtin_bit_cast(bf16x8, p[c % RING][0]);
    } else {
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(p[c % RING][0][i]), x[4 + i] = __uint_as_float(p[c % RING][1][i]);
      split8<N>(x, ac);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) bc[n] = b[n][c];
    mma_planes<N>(acc, ac, bc);
    pin();
  }
}

// ---- one sequence ---------------------------------------------------------------------------------------------------------------
struct Seq {
  int ql, kl, shift;
};
__device__ __forceinline__ Seq seq_of(const WaArgs& a, int b) {
  Seq s;
  s.ql = a.q_lens ? min(max(a.q_lens[b], 0), a.Tq) : a.Tq;
  s.kl = a.k_lens ? min(max(a.k_lens[b], 0), a.Tk) : a.Tk;
  s.shift = s.kl - s.ql;
  return s;
}
// Key tiles of BN keys that rows at positions [p0, p1] may see: na tiles from key 0 (the sinks, when the window begins behind them),
// then nb tiles from key `start`.  No key lies in two tiles; the mask decides inside a tile.
struct Tiles {
  int na, nb, start;
};
__device__ __forceinline__ Tiles tiles_of(const WaArgs& a, const Seq& s, int p0, int p1, int bn) {
  Tiles t;
  const int hi = min(s.kl, p1 + a.right + 1);
  const int lo = max(0, p0 - a.left);
  const int sink = lo > 0 ? min(a.sinks, hi) : 0;
  t.na = sink > 0 ? (sink + bn - 1) / bn : 0;
  t.start = max(lo, t.na * bn);
  t.nb = hi > t.start ? (hi - t.start + bn - 1) / bn : 0;
  return t;
}
__device__ __forceinline__ int tile_start(const Tiles& t, int i, int bn) { return i < t.na ? i * bn : t.start + (i - t.na) * bn; }

// What the KEYS keys from j0 are to rows at positions [p0, p1]: 0 unseen, 1 seen in part, 2 seen by all
template <int KEYS = 32>
__device__ __forceinline__ int seen_class(const WaArgs& a, const Seq& s, int j0, int p0, int p1) {
  const int j1 = j0 + KEYS - 1;
  if (j0 >= s.kl || j0 > p1 + a.right || (j1 < p0 - a.left && j0 >= a.sinks)) return 0;
  return j1 < s.kl && j1 <= p0 + a.right && (j0 >= p1 - a.left || j1 < a.sinks) ? 2 : 1;
}

// ---- online softmax ----------------------------------------------------------------------------------------------------------------
// m is the running maximum of the raw scores that the exponents are taken against.  It follows the true maximum only when that is more
// than 8 powers of two above it: the terms stay below 2^8, nothing is lost in fp32 (nor in bf16, whose exponent is as wide), and the
// accumulators are rescaled in the first tiles of a row only.
__device__ __forceinline__ float softmax_slack(float c) { return fminf(8.0f / c, 3.4e38f); }   // (a number: a row without a maximum, m = -inf, is below every score)
// Takes the maximum t of new scores into m (rescaling l and o); returns m c, what the exponents are taken against
template <int ND>
__device__ __forceinline__ float softmax_follow(float t, float& m, float& l, f32x16 (&o)[ND], float c, float slack) {
  if (__ballot(t > m + slack)) {
    const float mn = fmaxf(m, t);
    const float f = mn == m ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c);
    m = mn;
    l *= f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] *= f;
  }
  return m == -INFINITY ? 0.f : m * c;
}
template <int ND>
__device__ __forceinline__ float softmax_max(const float (&s)[16], float& m, float& l, f32x16 (&o)[ND], float c, float slack) {
  float t = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) t = fmaxf(t, s[i]);
  return softmax_follow<ND>(half_max(t), m, l, o, c, slack);
}
// Every exponent is also lowered by a.down = 8 + log2 Tk, so that a row's exponentials sum to at most 1 before they are normalised too, and their sum with values
// next to the largest stays a number; at the other end values lose what lies below 2^(down - 149).
// exp2(s c - mc) in one fused step is exact enough while the rounding of mc = m c is small; beyond 2^22 the scores are moved by m first
template <int NS>
__device__ __forceinline__ void softmax_huge(float (&s)[NS][16], float m, float& mc) {
  if (__ballot(__builtin_fabsf(mc) > 4194304.f)) {
    const float me = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[n][i] -= me;
    mc = 0.f;
  }
}
// elements [A, B) of the scores become exponentials
template <int A, int B>
__device__ __forceinline__ void softmax_exp(float (&s)[16], float& l, float off, float c) {
  float sum = 0.f;
#pragma unroll
  for (int i = A; i < B; ++i) {
    s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -off));
    sum += s[i];
  }
  l += sum;
}
// log-sum-exp of a row that sees keys.  Below 32 bits it is their lowest number, -inf is for rows that see none.
__device__ __forceinline__ float log_sum(const WaArgs& a, float m, float l) {
  const float x = m * a.scale + __logf(l * a.up);
  return x < -3.4028235e38f ? -3.4028235e38f : x;
}
// scores of keys a row does not see become -inf (element i: key j0 + 8 (i / 4) + 4 h + i % 4)
__device__ __forceinline__ void mask_scores(float (&s)[16], const WaArgs& a, const Seq& q, int j0, int p, int lane) {
  asm volatile("");   // (a branch, not a select over all tiles)
  const int base = j0 + 4 * (lane >> 5);
  const int hi = min(p + a.right, q.kl - 1) - base, lo = p - a.left - base, sk = a.sinks - base;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int e = 8 * (i >> 2) + (i & 3);
    if (!(e <= hi && (e >= lo || e < sk))) s[i] = -INFINITY;
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]);
template <>
__device__ __forceinline__ void store4<float>(float* p, const float (&v)[4]) {
  *reinterpret_cast<f32x4*>(p) = (f32x4){v[0], v[1], v[2], v[3]};
}
template <>
__device__ __forceinline__ void store4<__bf16>(__bf16* p, const float (&v)[4]) {
  float e[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
  const u32x4 w = Elem<__bf16>::pack(e);
  *reinterpret_cast<u32x2*>(p) = (u32x2){w[0], w[1]};
}

// Four channels from d of the result of query i, head hq.  For the backward pass what bf16 leaves of it is stored too: delta = sum dO O from a
// rounded O alone is off by 2^-9 of |dO| |O|, which for rows that see a few keys is as much as all other roundings of dQ and dK together
// (their error goes from 2.3 to 1.5 times that of one rounding at two keys, from 1.5 to 1.45 at 64).  It costs the forward pass of a training
// step a second store: 91 -> 104 us at 33 MB of results.
template <typename T>
__device__ __forceinline__ void store_out(const WaArgs& a, int b, int i, long hq, int d, const float (&v)[4]) {
  store4<T>((T*)a.out + b * a.o_bs + (long)i * a.o_ts + hq * a.o_hs + d, v);
  if constexpr (sizeof(T) == 2) {
    if (a.out_lo) {
      float lo[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) lo[x] = v[x] - (float)(__bf16)v[x];
      store4<__bf16>(a.out_lo + (((long)b * a.Tq + i) * (a.Hkv * a.G) + hq) * a.D + d, lo);
    }
  }
}

// What is computed from `lane` from here on is computed here, not kept in registers from where the kernel's loops computed it
__device__ __forceinline__ void fresh(int& lane) { asm volatile("" : "+v"(lane)); }

// Whether a channel that this wave has stored is no number (the again-functions' channels to take: the others are right, and a channel that is NaN over what is
// seen stays so, which ends the walk)
template <typename T>
__device__ __forceinline__ bool no_number(const T* at, bool on) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  return on && !(__builtin_fabsf(Elem<T>::ld(at)) < INFINITY);
}

// A product over a tile also adds 0 times what stands at unseen keys, and 0 times an infinity is NaN.  A row whose sum of exponentials is
// a number but whose result is not is therefore taken again, over the keys it sees alone: one wave, 32 keys at a time, a running mean (its weights sum to 1 whatever
// the scores), the lanes split the channels.
template <typename T>
__device__ __forceinline__ void row_again(const WaArgs& a, const Seq& s, int b, int hk, int r, int lane) {
  fresh(lane);
  const int i = r / a.G, g = r - i * a.G;
  const T* q = (const T*)a.q + b * a.q_bs + i * a.q_ts + (long)(hk * a.G + g) * a.q_hs;
  const T* k = (const T*)a.k + b * a.k_bs + hk * a.k_hs;
  const T* v = (const T*)a.v + b * a.v_bs + hk * a.v_hs;
  const long hq = (long)(hk * a.G + g);
  T* o = (T*)a.out + b * a.o_bs + i * a.o_ts + hq * a.o_hs;
  const int p = i + s.shift, hi = min(p + a.right, s.kl - 1), lo = max(p - a.left, 0);
  const float c = a.scale * kLog2e;
  const Tiles t = tiles_of(a, s, p, p, 32);
  const int d0 = lane, d1 = lane + 64;
  const bool on0 = no_number<T>(o + min(d0, a.D - 1), d0 < a.D), on1 = no_number<T>(o + min(d1, a.D - 1), d1 < a.D);
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int it = 0; it < t.na + t.nb; ++it) {
    const int j0 = tile_start(t, it, 32), j = j0 + (lane & 31);
    const bool seen = j <= hi && (j >= lo || j < a.sinks);
    const float sc = row_times<T, true>(q, k + (long)j * a.k_ts, j < s.kl, a.D, lane);
    const float top = fmaxf(wave_max(seen ? sc : -INFINITY), m);
    if (top == -INFINITY) continue;
    float w = seen ? __builtin_amdgcn_exp2f((sc - top) * c) : 0.f;
    const float was = l * __builtin_amdgcn_exp2f((m - top) * c);
    l = was + 0.5f * wave_sum(w);                                          // (both lane halves hold the keys)
    m = top, w /= l, o0 *= was / l, o1 *= was / l;
    const uint32_t mask = (uint32_t)__ballot(seen);
#pragma unroll 4
    for (int n = 0; n < 32; ++n) {
      const T* vr = v + (long)(j0 + n) * a.v_ts;
      const bool in = mask >> n & 1;
      const float wn = __shfl(w, n, 64), v0 = in && on0 ? Elem<T>::ld(vr + d0) : 0.f, v1 = in && on1 ? Elem<T>::ld(vr + d1) : 0.f;
      o0 = fmaf(wn, v0, o0);
      o1 = fmaf(wn, v1, o1);
    }
    if (__all((!on0 || o0 != o0) && (!on1 || o1 != o1))) break;
  }
  if (on0) o[d0] = (T)o0;
  if (on1) o[d1] = (T)o1;
  if constexpr (sizeof(T) == 2) {
    if (a.out_lo) {
      __bf16* r = a.out_lo + (((long)b * a.Tq + i) * (a.Hkv * a.G) + hq) * a.D;
      if (on0) r[d0] = (__bf16)(o0 - (float)(__bf16)o0);
      if (on1) r[d1] = (__bf16)(o1 - (float)(__bf16)o1);
    }
  }
}

// Work item `block` of n = nbh x per -> (batch and key head, item of it), so that the items of one head, which read the same keys, run on one
// XCD (workgroups go round the 8 of them).  Heads go round the XCDs when their number allows it, since sequences differ in length (padded
// tracks: each XCD gets heads of every sequence); else each XCD takes a contiguous run of items.
struct Item {
  int bh, at;
};
__device__ __forceinline__ Item xcd_item(int block, int nbh, int per) {
  const int x = block & 7, y = block >> 3;
  if (nbh % 8 == 0) {
    const int g = y / per;
    return {g * 8 + x, y - g * per};
  }
  const int n = nbh * per, run = n >> 3, rest = n & 7, item = x * run + min(x, rest) + y, bh = item / per;
  return {bh, item - bh * per};
}

// What the many-row kernels walk over the key tiles with: BN keys a tile, bf16 in two stages of direct loads, fp32 in one stage of planes and
// one of numbers as they arrive (forward at 128 channels: 128 us with the numbers held in registers, 84 so; 64 keys a tile would leave a compute unit one workgroup)
template <typename T, int DP>
struct Walk {
  static constexpr int N = Planes<T>::N, BN = N == 1 ? 64 : 32, NSTAGE = N == 1 ? 2 : 1;
  static constexpr uint32_t PLANE = BN * G16<DP>::PITCH, TILE = N * PLANE, STAGE = 2 * TILE, RAW = N == 1 ? 0 : BN * DP * 4, LDS = NSTAGE * STAGE + 2 * RAW;
};
// Calls f(key, offset of the stage in LDS as a type) for the key tiles [first, n) of `t`, staged
// (ready() is called once the first tile's loads are on their way)
template <typename T, int DP, typename R, typename F>
__device__ __forceinline__ void walk_keys(const WaArgs& a, const Seq& s, const Tiles& t, int first, int n, const T* kb, const T* vb, uint32_t lds, int wave, int lane, R&& ready,
                                          F&& f) {
  using W = Walk<T, DP>;
  constexpr int ES = sizeof(T);
  Stager<T, DP, W::BN> sk, sv;
  sk.init(a.k_ts * ES, a.D * ES, wave, lane);
  sv.init(a.v_ts * ES, a.D * ES, wave, lane);
  auto load = [&](int it, uint32_t at) {
    const int j0 = tile_start(t, it, W::BN);
    sk.load(at, (const char*)(kb + (long)j0 * a.k_ts), s.kl - j0, wave);
    sv.load(at + (W::N == 1 ? W::TILE : W::RAW), (const char*)(vb + (long)j0 * a.v_ts), s.kl - j0, wave);
  };
  if (first < n) load(first, W::N == 1 ? lds : lds + W::STAGE);
  ready();
  if constexpr (W::N == 1) {
    for (int it = first; it < n; it += 2) {
      wait_vm<0>();
      wg_barrier();
      if (it + 1 < n) load(it + 1, lds + W::STAGE);
      f(tile_start(t, it, W::BN), std::integral_constant<uint32_t, 0>());
      if (it + 1 >= n) break;
      wait_vm<0>();
      wg_barrier();
      if (it + 2 < n) load(it + 2, lds);
      f(tile_start(t, it + 1, W::BN), std::integral_constant<uint32_t, W::STAGE>());
    }
  } else {
    for (int it = first; it < n; ++it) {
      wait_vm<0>();
      wg_barrier();                    // the numbers are there, the planes of the tile before have been read
      sk.put(lds, lds + W::STAGE);
      sv.put(lds + W::TILE, lds + W::STAGE + W::RAW);
      wg_barrier();
      if (it + 1 < n) load(it + 1, lds + W::STAGE);
      f(tile_start(t, it, W::BN), std::integral_constant<uint32_t, 0>());
    }
  }
}

// ---- forward, many rows: 4 waves x 32 rows ----------------------------------------------------------------------------------------------
// Bound by the SIMDs, which share their issue between matrix and vector work (a score costs as many cycles of exponential, mask, sum and rounding
// as of products at 64 channels, half at 128): what helps is waves enough to have both at hand, so registers are held to 2 waves a SIMD at 128
// channels, 3 or 4 below.  Measured, in a row of calls (alone, under the profiler): bf16, 2 x 4096 tokens, 16 / 4 heads of 128 channels, window 1024: 83 us (94 to
// 100), 720 TFLOP/s of what is seen (the matrix units are busy 35 % of the time, the vector units 41 %); 16384 tokens, 8 heads of 64 channels, window 1025:
// 56 us (63 to 67), 610 TFLOP/s; fp32, 8 x 1250 tokens and fewer, 8 heads of 64, window 257: 55 us (63), 93 TFLOP/s (560 of bf16 products).
template <typename T, int DP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DP == 128 ? 2 : sizeof(T) == 4 ? (DP == 64 ? 3 : 4) : 4))) void window_attn_kernel(const WaArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using W = Walk<T, DP>;
  constexpr int ND = DP / 32, N = W::N;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Item item = xcd_item(blockIdx.x, a.B * a.Hkv, a.ntiles);
  const int tile = item.at, bh = item.bh, hk = bh % a.Hkv, b = bh / a.Hkv;
  const Seq s = seq_of(a, b);
  const int R = a.Tq * a.G, r0 = tile * 128, rw = r0 + wave * 32;
  const int rend = min(r0 + 128, s.ql * a.G);            // rows of the tile that see anything at all
  const int r = rw + (lane & 31), i = r / a.G, g = r - i * a.G;
  const bool row_ok = r < s.ql * a.G;
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float c = a.scale * kLog2e, slack = softmax_slack(c);
  if (r0 < rend) {
    Frags16<N, DP> qf;
    load_frags16<T, DP>(qf, (const T*)a.q + b * a.q_bs + (long)i * a.q_ts + (long)(hk * a.G + g) * a.q_hs, row_ok, a.D, lane);
    const LaneOff<DP> off(lds, lane);
    const int p = i + s.shift;
    const int wp0 = rw / a.G + s.shift, wp1 = (min(rw + 32, rend) - 1) / a.G + s.shift;   // positions of this wave's rows
    const bool wave_ok = rw < rend;
    const Tiles t = tiles_of(a, s, r0 / a.G + s.shift, (rend - 1) / a.G + s.shift, W::BN);
    walk_keys<T, DP>(a, s, t, 0, t.na + t.nb, (const T*)a.k + b * a.k_bs + hk * a.k_hs, (const T*)a.v + b * a.v_bs + hk * a.v_hs, lds, wave, lane, [&] { arrived16(qf); },
                     [&](int j0, auto st) {
      // a tile is taken whole: with a path of its own for a half the accumulators would be copied where the paths meet
      constexpr uint32_t S0 = decltype(st)::value;
      constexpr int NS = W::BN / 32, STEPS = 2 * ND;
      const int cls = wave_ok ? seen_class<W::BN>(a, s, j0, wp0, wp1) : 0;
      if (!cls) return;
      float sc[NS][16];
      bf16x8 pb[2][N];
      if constexpr (NS == 2) {
        // (Taking the first half's exponentials against the maximum so far, between the second half's products, measured no faster at 128
        // channels and costs the fourth wave at 64.)
        constexpr uint32_t S1 = S0 + 32 * G16<DP>::PITCH;
        f32x16 acc;
        rows16<N, DP, S0, W::PLANE>(acc, off, qf);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[0][e] = acc[e];
        rows16<N, DP, S1, W::PLANE>(acc, off, qf);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[1][e] = acc[e];
        if (cls == 1) {
          mask_scores(sc[0], a, s, j0, p, lane);
          mask_scores(sc[1], a, s, j0 + 32, p, lane);
        }
        float t = sc[0][0];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) t = fmaxf(t, sc[n][e]);
        float mc = softmax_follow<ND>(half_max(t), m, l, o, c, slack);
        softmax_huge<2>(sc, m, mc);
        mc += a.down;
        softmax_exp<0, 16>(sc[0], l, mc, c);
        pack16<N>(pb, sc[0]);
        // the exponentials of the second half stand between the products of the first with V
        cols16<N, DP, S0 + W::TILE, W::PLANE>(o, off, pb, [&](int k) {
#pragma unroll
          for (int i = k * 16 / STEPS; i < (k + 1) * 16 / STEPS; ++i) {
            sc[1][i] = __builtin_amdgcn_exp2f(fmaf(sc[1][i], c, -mc));
            l += sc[1][i];
          }
        });
        pack16<N>(pb, sc[1]);
        cols16<N, DP, S1 + W::TILE, W::PLANE>(o, off, pb);
      } else {
        f32x16 acc;
        rows16<N, DP, S0, W::PLANE>(acc, off, qf);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[0][e] = acc[e];
        if (cls == 1) mask_scores(sc[0], a, s, j0, p, lane);
        float mc = softmax_max<ND>(sc[0], m, l, o, c, slack);
        softmax_huge<1>(sc, m, mc);
        mc += a.down;
        softmax_exp<0, 16>(sc[0], l, mc, c);
        pack16<N>(pb, sc[0]);
        cols16<N, DP, S0 + W::TILE, W::PLANE>(o, off, pb);
      }
    });
    l = half_sum(l);
  }
  // rows the sequence does not have: zero, like rows that see nothing
  const float inv = row_ok && l != 0.f ? 1.0f / l : 0.f;
  bool bad = false;
  if (r < R) {
    const int h4 = 4 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          v[x] = inv != 0.f ? o[d][4 * e + x] * inv : (l != l ? l : 0.f);
          bad |= v[x] != v[x];
        }
        if (32 * d + 8 * e + h4 < a.D) store_out<T>(a, b, i, hk * a.G + g, 32 * d + 8 * e + h4, v);
      }
    if (a.lse && lane < 32) a.lse[((long)b * a.Hkv * a.G + hk * a.G + g) * a.Tq + i] = row_ok && l != 0.f ? log_sum(a, m, l) : -INFINITY;
  }
  uint64_t again = __ballot(bad && row_ok && l == l);
  again = (again | (again >> 32)) & 0xffffffffull;
  while (again) {
    const int n = __builtin_ctzll(again);
    again &= again - 1;
    row_again<T>(a, s, b, hk, rw + n, lane);
  }
#endif
}

// ---- forward, few rows: one 32-row tile per workgroup, its waves (and the splits) share the keys -------------------------------------
// Single tokens over a cache are bound by the reads of K and V: every wave streams its own key tiles through LDS of its own, so a compute
// unit has up to 128 KB of direct loads in flight and no wave waits for another before the end.  bf16 has two stages a wave, fp32 one, whose halves
// are reloaded in turn, which leaves room for four waves at 128 channels too (8 x 4 heads over 8192 keys, window 4096: 75 -> 41 us).  Where a row tile sees two key
// tiles at most (short tracks) a workgroup is one wave and keeps its result in registers: more workgroups fit a compute unit, and there is
// nothing to join (64 x 8 heads x 13 tokens of 128 channels, fp32: 14 us, latency; 29 with two waves that join).  fp32 splits a tile into
// planes as it reads it for the scores, which so have the bits that the backward pass sees again (instead of fp32 instructions: 16 x 4 heads of 64 over 4096 keys 33 -> 31 us, 13 tokens of 128
// 13.1 -> 13.7); the product with V takes the fp32 matrix instructions: it is
// not what binds it, and a tile that is read once need not be split first.
// Measured: 64 streams of up to 8192 cached keys, 4 heads of 128 channels in bf16, window 4096: 98 us, 5.3 TB/s (a copy reaches 5.2); one stream of
// 32768, window 16384: 13 to 15 us and 4 to join, 2.4 TB/s.
template <typename T, int DP, bool ONE>
struct Few {
  using G = Geo<T, DP>;
  static constexpr int STAGE = 2 * 32 * G::PITCH;                               // 32 keys of K and of V
  static constexpr int NW = ONE ? 1 : 4;
  // fp32 has one stage: K of the next tile is loaded behind the scores and lands under the products with V, and V likewise
  static constexpr bool HALVES = sizeof(T) == 4;
  static constexpr int RING = HALVES ? STAGE : 2 * STAGE;
  static constexpr int OPITCH = DP + 4;                                          // floats of a row in the exchange
  static constexpr int XCHG = ONE ? 0 : NW * 32 * (OPITCH + 2) * 4;
  static constexpr int LDS = NW * RING > XCHG ? NW * RING : XCHG;
};
template <typename T, int DP, bool ONE>
__global__ __launch_bounds__(256) void window_attn_few_kernel(const WaArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using G = Geo<T, DP>;
  using F = Few<T, DP, ONE>;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Item item = xcd_item(blockIdx.x, a.B * a.Hkv, a.ntiles * a.nsplit);
  const int split = item.at % a.nsplit, tile = item.at / a.nsplit, bh = item.bh, bht = bh * a.ntiles + tile, hk = bh % a.Hkv, b = bh / a.Hkv;
  const Seq s = seq_of(a, b);
  const int R = a.Tq * a.G, r0 = tile * 32, rend = min(r0 + 32, s.ql * a.G);
  const int r = r0 + (lane & 31), i = r / a.G, g = r - i * a.G;
  const bool row_ok = r < s.ql * a.G;
  const T* kb = (const T*)a.k + b * a.k_bs + hk * a.k_hs;
  const T* vb = (const T*)a.v + b * a.v_bs + hk * a.v_hs;
  const uint32_t ks = a.k_ts * G::ES, vs = a.v_ts * G::ES;
  const int dbytes = a.D * G::ES;
  f32x16 o[G::ND];
#pragma unroll
  for (int d = 0; d < G::ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float c = a.scale * kLog2e, slack = softmax_slack(c);
  if (r0 < rend) {
    Frags16<Planes<T>::N, DP> qf;
    load_frags16<T, DP>(qf, (const T*)a.q + b * a.q_bs + (long)i * a.q_ts + (long)(hk * a.G + g) * a.q_hs, row_ok, a.D, lane);
    const int p = i + s.shift, p0 = r0 / a.G + s.shift, p1 = (rend - 1) / a.G + s.shift;
    const Tiles t = tiles_of(a, s, p0, p1, 32);
    const int n = t.na + t.nb, per = (n + a.nsplit - 1) / a.nsplit;
    const int first = split * per + wave, last = min(n, (split + 1) * per);
    const uint32_t ring = lds + wave * F::RING;
    constexpr int LOADS = 32 * G::PITCH / 1024;                 // of K or V of a tile
    auto stage_k = [&](int it, int buf) {
      const int j0 = tile_start(t, it, 32);
      stage_rows<T, DP, 32, 1>(ring + buf * F::STAGE, (const char*)(kb + (long)j0 * a.k_ts), ks, s.kl - j0, dbytes, 0, lane);
    };
    auto stage_v = [&](int it, int buf) {
      const int j0 = tile_start(t, it, 32);
      stage_rows<T, DP, 32, 1>(ring + buf * F::STAGE + F::STAGE / 2, (const char*)(vb + (long)j0 * a.v_ts), vs, s.kl - j0, dbytes, 0, lane);
    };
    if (first < last) stage_k(first, 0), stage_v(first, 0);
    arrived16(qf);             // from here on only direct loads are counted
    int buf = 0;
    for (int it = first; it < last; it += F::NW, buf ^= !F::HALVES) {
      const bool more = it + F::NW < last;
      if constexpr (F::HALVES) {
        wait_vm<LOADS>();                                       // K is there
      } else if (more) {
        stage_k(it + F::NW, buf ^ 1), stage_v(it + F::NW, buf ^ 1);
        wait_vm<2 * LOADS>();
      } else {
        wait_vm<0>();
      }
      const int j0 = tile_start(t, it, 32);
      const uint32_t kt = ring + buf * F::STAGE, vt = kt + F::STAGE / 2;
      const int cls = seen_class(a, s, j0, p0, p1);
      f32x16 acc;
      if (cls) few_scores<T, DP>(acc, kt, qf, lane);
      if constexpr (F::HALVES) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // K has been read
        if (more) {
          stage_k(it + F::NW, 0);
          wait_vm<LOADS>();                                     // V is there
        } else {
          wait_vm<0>();
        }
      }
      if (cls) {
        float sc[1][16];
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[0][e] = acc[e];
        if (cls == 1) mask_scores(sc[0], a, s, j0, p, lane);
        float mc = softmax_max<G::ND>(sc[0], m, l, o, c, slack);
        softmax_huge<1>(sc, m, mc);
        mc += a.down;
        softmax_exp<0, 16>(sc[0], l, mc, c);
        cols_times<DP>(o, vt, 0, sc[0], lane, T());
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this stage (fp32: V) has been read before the ring comes round to it
      if (F::HALVES && more) stage_v(it + F::NW, 0);
    }
    l = half_sum(l);
  }
  if constexpr (ONE) {
    const float inv = row_ok && l != 0.f ? 1.0f / l : 0.f;
    bool bad = false;
    if (r < R) {
      const int h4 = 4 * (lane >> 5);
#pragma unroll
      for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            v[x] = inv != 0.f ? o[d][4 * e + x] * inv : (l != l ? l : 0.f);
            bad |= v[x] != v[x];
          }
          if (32 * d + 8 * e + h4 < a.D) store_out<T>(a, b, i, hk * a.G + g, 32 * d + 8 * e + h4, v);
        }
      if (a.lse && lane < 32) a.lse[((long)b * a.Hkv * a.G + hk * a.G + g) * a.Tq + i] = row_ok && l != 0.f ? log_sum(a, m, l) : -INFINITY;
    }
    uint64_t again = __ballot(bad && row_ok && l == l);
    again = (again | (again >> 32)) & 0xffffffffull;
    while (again) {
      const int n = __builtin_ctzll(again);
      again &= again - 1;
      row_again<T>(a, s, b, hk, r0 + n, lane);
    }
    return;
  }
  // the waves' shares are joined in LDS, in wave order
  __syncthreads();
  float* xo = reinterpret_cast<float*>(smem);                                   // [NW][32][OPITCH]
  float* xm = xo + F::NW * 32 * F::OPITCH;                                      // [NW][32] m, then l
  float* xl = xm + F::NW * 32;
  {
    const int n = lane & 31, h4 = 4 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < G::ND; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x4*>(xo + (wave * 32 + n) * F::OPITCH + 32 * d + 8 * e + h4) =
            (f32x4){o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
    if (lane < 32) xm[wave * 32 + n] = m, xl[wave * 32 + n] = l;
  }
  __syncthreads();
  constexpr int NT = F::NW * 64, D4 = DP / 4, RPP = NT / D4;                      // rows of one pass of the workgroup
  for (int n0 = 0; n0 < 32; n0 += RPP) {
    const int n = n0 + threadIdx.x / D4, d = 4 * (threadIdx.x % D4);
    if (n >= 32) continue;
    float mm = xm[n];
#pragma unroll
    for (int w = 1; w < F::NW; ++w) mm = fmaxf(mm, xm[w * 32 + n]);
    float ll = 0.f;
    f32x4 oo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < F::NW; ++w) {
      const float mw = xm[w * 32 + n];
      const float f = mw == mm ? 1.f : __builtin_amdgcn_exp2f((mw - mm) * c);
      if (xl[w * 32 + n] == 0.f) continue;                                       // a share that saw nothing
      ll += f * xl[w * 32 + n];
      const f32x4 ow = *reinterpret_cast<const f32x4*>(xo + (w * 32 + n) * F::OPITCH + d);
#pragma unroll
      for (int x = 0; x < 4; ++x) oo[x] = fmaf(f, ow[x], oo[x]);
    }
    if (a.nsplit > 1) {
      if (r0 + n < R) {
        float* part = a.ws + ((long)bht * a.nsplit + split) * 32 * (DP + 2);
        *reinterpret_cast<f32x4*>(part + n * DP + d) = oo;
        if (d == 0) part[32 * DP + n] = mm, part[32 * DP + 32 + n] = ll;
      }
      continue;
    }
    const int rr = r0 + n, ii = rr / a.G, gg = rr - ii * a.G;
    bool bad = false;
    const bool ok = rr < s.ql * a.G;
    if (rr < R) {
      const float inv = ok && ll != 0.f ? 1.0f / ll : 0.f;
      float v[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        v[x] = inv != 0.f ? oo[x] * inv : (ll != ll ? ll : 0.f);
        bad |= v[x] != v[x];
      }
      if (d < a.D) store_out<T>(a, b, ii, hk * a.G + gg, d, v);
      if (a.lse && d == 0) a.lse[((long)b * a.Hkv * a.G + hk * a.G + gg) * a.Tq + ii] = ok && ll != 0.f ? log_sum(a, mm, ll) : -INFINITY;
    }
    uint64_t again = __ballot(bad && ok && ll == ll);
    while (again) {                                                              // D4 (8 .. 32) lanes hold a row
      const int f = __builtin_ctzll(again), row_lane = f - f % D4;
      again &= ~(((1ull << D4) - 1) << row_lane);
      row_again<T>(a, s, b, hk, __builtin_amdgcn_readlane(rr, f), lane);
    }
  }
#endif
}

// Joins the key splits of one row: 256 threads = 4 channels each x groups that take the splits in turn, then the groups in order.
template <typename T, int DP>
__global__ __launch_bounds__(256) void window_attn_join_kernel(const WaArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int D4 = DP / 4, NG = 256 / D4;
  __shared__ f32x4 xo[NG][D4];
  __shared__ float xm[NG], xl[NG];
  const int R = a.Tq * a.G;
  const int rr = blockIdx.x % R, bh = blockIdx.x / R, hk = bh % a.Hkv, b = bh / a.Hkv;
  const int tile = rr >> 5, n = rr & 31;
  const int grp = threadIdx.x / D4, dv = threadIdx.x % D4;
  const Seq s = seq_of(a, b);
  const float c = a.scale * kLog2e;
  constexpr long PART = 32 * (DP + 2);
  const float* base = a.ws + ((long)(bh * a.ntiles + tile) * a.nsplit) * PART;
  // every load of the row is on its way before the first is used: at most 64 splits, 64 / NG of them to a group
  constexpr int PER = 64 / NG;
  f32x4 ow[PER];
  float mw[PER], lw[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int sp = grp + k * NG;
    const float* part = base + min(sp, a.nsplit - 1) * PART;
    mw[k] = part[32 * DP + n];
    lw[k] = sp < a.nsplit ? part[32 * DP + 32 + n] : 0.f;
    ow[k] = *reinterpret_cast<const f32x4*>(part + n * DP + 4 * dv);
  }
  float mm = -INFINITY, ll = 0.f;
  f32x4 oo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < PER; ++k) mm = lw[k] == 0.f ? mm : fmaxf(mm, mw[k]);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (lw[k] == 0.f) continue;                                                  // a share that saw nothing
    const float f = mw[k] == mm ? 1.f : __builtin_amdgcn_exp2f((mw[k] - mm) * c);
    ll = fmaf(f, lw[k], ll);
#pragma unroll
    for (int x = 0; x < 4; ++x) oo[x] = fmaf(f, ow[k][x], oo[x]);
  }
  xo[grp][dv] = oo;
  if (dv == 0) xm[grp] = mm, xl[grp] = ll;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  float M = xm[0];
  for (int k = 1; k < NG; ++k) M = fmaxf(M, xm[k]);
  float L = 0.f;
  f32x4 O = {0.f, 0.f, 0.f, 0.f};
  const int x4 = threadIdx.x % D4;
  for (int k = 0; k < NG; ++k) {
    if (xl[k] == 0.f) continue;
    const float f = xm[k] == M ? 1.f : __builtin_amdgcn_exp2f((xm[k] - M) * c);
    L += f * xl[k];
#pragma unroll
    for (int x = 0; x < 4; ++x) O[x] = fmaf(f, xo[k][x4][x], O[x]);
  }
  const int i = rr / a.G, g = rr - i * a.G;
  const bool ok = i < s.ql;
  const float inv = ok && L != 0.f ? 1.0f / L : 0.f;
  float v[4];
  bool bad = false;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    v[x] = inv != 0.f ? O[x] * inv : (L != L ? L : 0.f);
    bad |= v[x] != v[x];
  }
  if ((int)threadIdx.x < D4 && 4 * (int)threadIdx.x < a.D) store_out<T>(a, b, i, hk * a.G + g, 4 * threadIdx.x, v);
  if (a.lse && threadIdx.x == 0) a.lse[((long)b * a.Hkv * a.G + hk * a.G + g) * a.Tq + i] = ok && L != 0.f ? log_sum(a, M, L) : -INFINITY;
  if (__ballot(bad && ok && L == L)) row_again<T>(a, s, b, hk, rr, threadIdx.x);
#endif
}

// ---- backward ----------------------------------------------------------------------------------------------------------------------
// With P = exp(scale q k^T - lse), delta = sum_d dO O, dP = dO V^T, dS = P (dP - delta):
//   dV = P^T dO,   dQ = scale dS K,   dK = scale dS^T Q.
// The exponent s c - lse2 (c = scale log2 e, lse2 = lse log2 e) is off by what lse was rounded by, at most 6 2^-24 |lse2|: up to |lse2| = kBuilt that is less than
// the scores' own sums are off (fp32: 3e-5 of P) or a fraction of P's rounding (bf16: 5e-4).  Beyond, P would neither sum to 1 nor stay finite (one key that a row
// sees alone: P = 1.02 at a score of 1e5, 9 at 1e7): dQ's waves take the maximum m and the sum l of such rows again from the scores as they see them, and
// P = 2^((s - m) c - log2 l) then.  The forward kernels, dQ and dK / dV have the same bits of s: all add the same products in the same order.  The way there costs
// rows that do not need it up to 3 % (dK / dV, bf16: 40.7 -> 42.0 us at 8192 tokens, 8 heads of 64 channels, window 257; 227 -> 234 at dQ's size below), rows
// that do one more walk over their keys, straight from memory (backward pass with every row far: 390 -> 470 us, fp32 at the sizes below; 8 / 1 heads of 128, 4096
// tokens, causal, bf16: 290 -> 550).
// Two kernels take S and dP again, each in the orientation that leaves its sums in one wave's registers, so nothing is added by atomics
// and the order of every sum is fixed: dQ walks the keys of 128 rows (like the forward pass), dK / dV walk the rows that see 32 keys a
// wave.  The sinks are seen by every later row: their rows beyond the window are cut into shares that run as workgroups of their own.
// dQ, bf16, 2 x 4096 tokens, 16 / 4 heads of 128 channels, window 1024: 118 us, 766 TFLOP/s; fp32, 16 x 625 tokens and fewer, 8 heads of 128,
// window 129: 155 us, where one wave has a SIMD to itself (422 registers: the planes of Q and dO alone are 192) and nothing covers its vector work.

template <typename T>
constexpr float kBuilt = sizeof(T) == 4 ? 128.f : 2048.f;
// Numbers of 32 rows: exponents' offsets [32], delta [32], what is taken off the scores first [32] (0, or a far row's maximum), and 1 if any of these is not 0
constexpr int kStat = 100;

// Maximum and sum of exponentials of a wave's 32 rows (planes qf, lane n and n + 32: row n at position p; all of them at [p0, p1]), from scores in the bits of
// rows16, straight from memory
template <typename T, int DP>
__device__ __forceinline__ void rows_max_sum(const WaArgs& a, const Seq& s, const T* kb, int p, int p0, int p1, const Frags16<Planes<T>::N, DP>& qf, float c, int lane,
                                             float& m, float& l) {
  constexpr int N = Planes<T>::N;
  const Tiles t = tiles_of(a, s, p0, p1, 32);
  m = -INFINITY, l = 0.f;
  for (int it = 0; it < t.na + t.nb; ++it) {
    const int j0 = tile_start(t, it, 32), j = j0 + (lane & 31);
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
    for (int x = 0; x < G16<DP>::NC; ++x) {
      bf16x8 k[N], q[N];
      load_piece16<T>(k, kb + (long)j * a.k_ts, x, j < s.kl, a.D, lane);
#pragma unroll
      for (int n = 0; n < N; ++n) q[n] = qf[n][x];
      mma_planes<N>(acc, k, q);
    }
    float sc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = acc[e];
    mask_scores(sc, a, s, j0, p, lane);
    float top = sc[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, sc[e]);
    top = fmaxf(half_max(top), m);
    if (top == -INFINITY) continue;
    l *= __builtin_amdgcn_exp2f((m - top) * c);
    m = top;
#pragma unroll
    for (int e = 0; e < 16; ++e) l += __builtin_amdgcn_exp2f((sc[e] - m) * c);
  }
  l = half_sum(l);
}

// The gradient of one query row, over the keys it sees alone (see row_again), 32 at a time, with weights that sum to 1 whatever the scores
template <typename T>
__device__ __forceinline__ void dq_again(const WaArgs& a, const Seq& s, int b, int hk, int r, float delta, int lane) {
  fresh(lane);
  const int i = r / a.G, g = r - i * a.G;
  const long hq = (long)(hk * a.G + g);
  const T* q = (const T*)a.q + b * a.q_bs + i * a.q_ts + hq * a.q_hs;
  const T* dO = (const T*)a.dout + b * a.do_bs + i * a.do_ts + hq * a.do_hs;
  const T* k = (const T*)a.k + b * a.k_bs + hk * a.k_hs;
  const T* v = (const T*)a.v + b * a.v_bs + hk * a.v_hs;
  T* dq = (T*)a.dq + b * a.dq_bs + i * a.dq_ts + hq * a.dq_hs;
  const int p = i + s.shift, hi = min(p + a.right, s.kl - 1), lo = max(p - a.left, 0);
  const float c = a.scale * kLog2e;
  const Tiles t = tiles_of(a, s, p, p, 32);
  const int d0 = lane, d1 = lane + 64;
  const bool on0 = no_number<T>(dq + min(d0, a.D - 1), d0 < a.D), on1 = no_number<T>(dq + min(d1, a.D - 1), d1 < a.D);
  float m = -INFINITY, l = 0.f, r0 = 0.f, r1 = 0.f;
  for (int it = 0; it < t.na + t.nb; ++it) {
    const int j0 = tile_start(t, it, 32), j = j0 + (lane & 31);
    const bool seen = j <= hi && (j >= lo || j < a.sinks);
    const float sc = row_times<T, true>(q, k + (long)j * a.k_ts, j < s.kl, a.D, lane);
    const float top = fmaxf(wave_max(seen ? sc : -INFINITY), m);
    if (top == -INFINITY) continue;
    const float dp = row_times<T>(dO, v + (long)j * a.v_ts, j < s.kl, a.D, lane);
    float ds = seen ? __builtin_amdgcn_exp2f((sc - top) * c) : 0.f;
    const float was = l * __builtin_amdgcn_exp2f((m - top) * c);
    l = was + 0.5f * wave_sum(ds);                                         // (both lane halves hold the keys)
    m = top, ds = seen ? ds / l * (dp - delta) : 0.f, r0 *= was / l, r1 *= was / l;
    const uint32_t mask = (uint32_t)__ballot(seen);
#pragma unroll 4
    for (int n = 0; n < 32; ++n) {
      const T* kr = k + (long)(j0 + n) * a.k_ts;
      const bool in = mask >> n & 1;
      const float w = __shfl(ds, n, 64), k0 = in && on0 ? Elem<T>::ld(kr + d0) : 0.f, k1 = in && on1 ? Elem<T>::ld(kr + d1) : 0.f;
      r0 = fmaf(w, k0, r0);
      r1 = fmaf(w, k1, r1);
    }
    if (__all((!on0 || r0 != r0) && (!on1 || r1 != r1))) break;
  }
  if (on0) dq[d0] = (T)(r0 * a.scale);
  if (on1) dq[d1] = (T)(r1 * a.scale);
}

template <typename T, int DP, int OCC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(OCC))) void window_attn_dq_kernel(const WaArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using W = Walk<T, DP>;
  constexpr int ND = DP / 32, N = W::N;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Item item = xcd_item(blockIdx.x, a.B * a.Hkv, a.ntiles * a.nkey);
  const int tile = item.at / a.nkey, share = item.at % a.nkey, bh = item.bh, hk = bh % a.Hkv, b = bh / a.Hkv;
  const Seq s = seq_of(a, b);
  const int R = a.Tq * a.G, r0 = tile * 128, rw = r0 + wave * 32;
  const int rend = min(r0 + 128, s.ql * a.G);
  const int r = rw + (lane & 31), i = r / a.G, g = r - i * a.G;
  const long hq = (long)(hk * a.G + g);
  const bool row_ok = r < s.ql * a.G;
  f32x16 dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[d][e] = 0.f;
  Frags16<N, DP> qf, df;
  float delta = 0.f, lse2 = INFINITY, off_s = 0.f;                          // (off_s, lse2: see kStat)
  bool far = false;                                                        // of any row of the wave
  const int p = i + s.shift;
  const int wp0 = rw / a.G + s.shift, wp1 = (min(rw + 32, rend) - 1) / a.G + s.shift;
  const float c = a.scale * kLog2e;
  // the rows' own data, behind the first tile's loads; a row that sees nothing has lse = -inf: +inf makes its probabilities 0
  auto rows_ready = [&] {
    load_frags16<T, DP>(qf, (const T*)a.q + b * a.q_bs + (long)i * a.q_ts + hq * a.q_hs, row_ok, a.D, lane);
    const T* orow = (const T*)a.out + b * a.o_bs + (long)i * a.o_ts + hq * a.o_hs;
    const T* drow = (const T*)a.dout + b * a.do_bs + (long)i * a.do_ts + hq * a.do_hs;
    const float lse = row_ok ? a.lse[((long)b * a.Hkv * a.G + hq) * a.Tq + i] : -INFINITY;
    if constexpr (N == 1) {
      Frags16<1, DP> of, lf;
      load_frags16<T, DP>(df, drow, row_ok, a.D, lane);
      load_frags16<T, DP>(of, orow, row_ok, a.D, lane);
      load_frags16<T, DP>(lf, a.out_lo + (((long)b * a.Tq + i) * (a.Hkv * a.G) + hq) * a.D, row_ok && a.out_lo, a.D, lane);
#pragma unroll
      for (int x = 0; x < G16<DP>::NC; ++x) {
        float ov[8], dv[8], lv[8];
        Elem<__bf16>::unpack(__builtin_bit_cast(u32x4, of[0][x]), ov);
        Elem<__bf16>::unpack(__builtin_bit_cast(u32x4, df[0][x]), dv);
        Elem<__bf16>::unpack(__builtin_bit_cast(u32x4, lf[0][x]), lv);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf(lv[e], dv[e], delta);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf(ov[e], dv[e], delta);
      }
    } else {
#pragma unroll
      for (int x = 0; x < G16<DP>::NC; ++x) {
        const int d = 16 * x + 8 * (lane >> 5);
        const bool in = row_ok && d < a.D;
        float dv[8];
        u32x4 w[2], o[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          w[k] = in ? *reinterpret_cast<const u32x4*>(drow + d + 4 * k) : (u32x4){0u, 0u, 0u, 0u};
          o[k] = in ? *reinterpret_cast<const u32x4*>(orow + d + 4 * k) : (u32x4){0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) dv[e] = __uint_as_float(w[e >> 2][e & 3]), delta = fmaf(__uint_as_float(o[e >> 2][e & 3]), dv[e], delta);
        bf16x8 p[N];
        split8<N>(dv, p);
#pragma unroll
        for (int n = 0; n < N; ++n) df[n][x] = p[n];
      }
    }
    delta = half_sum(delta);
    if (lse == -INFINITY) delta = 0.f;
    else lse2 = lse * kLog2e;
    arrived16(qf);
    arrived16(df);
    const bool mine = lse > -INFINITY && __builtin_fabsf(lse2) > kBuilt<T>;
    if (__ballot(mine)) {
      far = true;
      float m, l;
      rows_max_sum<T, DP>(a, s, (const T*)a.k + b * a.k_bs + hk * a.k_hs, p, wp0, wp1, qf, c, lane, m, l);
      if (mine) off_s = l == 0.f ? 0.f : m, lse2 = l == 0.f ? INFINITY : __builtin_amdgcn_logf(l);
    }
  };
  if (r0 < rend) {
    const LaneOff<DP> off(lds, lane);
    const bool wave_ok = rw < rend;
    const Tiles t = tiles_of(a, s, r0 / a.G + s.shift, (rend - 1) / a.G + s.shift, W::BN);
    auto one = [&](int j0, auto at) {
      constexpr uint32_t A = decltype(at)::value;
      const int cls = wave_ok ? seen_class(a, s, j0, wp0, wp1) : 0;
      if (!cls) return;
      f32x16 acc, dp;
      float sc[16];
      constexpr int NC = G16<DP>::NC;
      rows16<N, DP, A, W::PLANE>(acc, off, qf);
      if (__builtin_expect(far, 0)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] -= off_s;
      }
      rows16<N, DP, A + W::TILE, W::PLANE>(dp, off, df, [&](int k) {
#pragma unroll
        for (int e = k * 16 / NC; e < (k + 1) * 16 / NC; ++e) sc[e] = __builtin_amdgcn_exp2f(fmaf(acc[e], c, -lse2));
      });
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] *= dp[e] - delta;
      if (cls == 1) {
        asm volatile("");
        const int base = j0 + 4 * (lane >> 5);
        const int hi = min(p + a.right, s.kl - 1) - base, lo = p - a.left - base, sk = a.sinks - base;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int x = 8 * (e >> 2) + (e & 3);
          if (!(x <= hi && (x >= lo || x < sk))) sc[e] = 0.f;
        }
      }
      bf16x8 db[2][N];
      pack16<N>(db, sc);
      cols16<N, DP, A, W::PLANE>(dq, off, db);
    };
    const int n = t.na + t.nb, per = (n + a.nkey - 1) / a.nkey;
    walk_keys<T, DP>(a, s, t, share * per, min(n, (share + 1) * per), (const T*)a.k + b * a.k_bs + hk * a.k_hs, (const T*)a.v + b * a.v_bs + hk * a.v_hs, lds, wave, lane, rows_ready,
                     [&](int j0, auto st) {
      constexpr uint32_t S0 = decltype(st)::value;
      one(j0, std::integral_constant<uint32_t, S0>());
      if constexpr (W::BN == 64) one(j0 + 32, std::integral_constant<uint32_t, S0 + 32 * G16<DP>::PITCH>());
    });
  }
  if (share == 0) {                                                        // (both lane halves hold the row's numbers)
    float* stat = a.stat + ((long)bh * a.ntiles32 + tile * 4 + wave) * kStat;
    stat[lane] = lane < 32 ? lse2 : delta;
    if (lane < 32) stat[64 + lane] = off_s;
    if (lane == 0) stat[96] = far ? 1.f : 0.f;
  }
  if (a.nkey > 1) {
    if (r < R) {
      float* part = a.near + (((long)bh * a.nkey + share) * R + r) * DP + 4 * (lane >> 5);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<f32x4*>(part + 32 * d + 8 * e) = (f32x4){dq[d][4 * e], dq[d][4 * e + 1], dq[d][4 * e + 2], dq[d][4 * e + 3]};
    }
    return;
  }
  bool bad = false;
  if (r < R) {
    T* qrow = (T*)a.dq + b * a.dq_bs + (long)i * a.dq_ts + hq * a.dq_hs;
    const int h4 = 4 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          v[x] = row_ok ? dq[d][4 * e + x] * a.scale : 0.f;
          bad |= v[x] != v[x];
        }
        if (32 * d + 8 * e + h4 < a.D) store4<T>(qrow + 32 * d + 8 * e + h4, v);
      }
  }
  uint64_t again = __ballot(bad && lse2 == lse2 && delta == delta);
  again = (again | (again >> 32)) & 0xffffffffull;
  while (again) {
    const int n = __builtin_ctzll(again);
    again &= again - 1;
    dq_again<T>(a, s, b, hk, rw + n, __shfl(delta, n, 64), lane);
  }
#endif
}

// The shares of dQ (nkey > 1), in order: one wave a row
template <typename T, int DP>
__global__ __launch_bounds__(256) void window_attn_dq_join_kernel(const WaArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = a.Tq * a.G, per = (R + 3) / 4;
  const int r = 4 * (int)(blockIdx.x % per) + wave, bh = blockIdx.x / per, hk = bh % a.Hkv, b = bh / a.Hkv;
  if (r >= R) return;
  const Seq s = seq_of(a, b);
  const int i = r / a.G, g = r - i * a.G;
  float sum[2] = {0.f, 0.f};
  const float* part = a.near + ((long)bh * a.nkey * R + r) * DP + lane;
#pragma unroll 4
  for (int n = 0; n < a.nkey; ++n)
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (64 * x + lane < DP) sum[x] += part[(long)n * R * DP + 64 * x];
  T* row = (T*)a.dq + b * a.dq_bs + (long)i * a.dq_ts + (long)(hk * a.G + g) * a.dq_hs;
  bool bad = false;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float v = i < s.ql ? sum[x] * a.scale : 0.f;
    if (64 * x + lane < a.D) {
      row[64 * x + lane] = (T)v;
      bad |= v != v;
    }
  }
  const float* stat = a.stat + ((long)bh * a.ntiles32 + (r >> 5)) * kStat + (r & 31);
  const float lse2 = stat[0], delta = stat[32];
  if (__ballot(bad) && lse2 == lse2 && delta == delta) dq_again<T>(a, s, b, hk, r, delta, lane);
#endif
}

// One thread's part of staging ROWS packed rows (query i, head g of the group) of q or dout: row r lies at (r / G) * ts + (r % G) * hs
template <typename T, int DP, int ROWS, int NW>
struct PackedStager;
template <int DP, int ROWS, int NW>
struct PackedStager<__bf16, DP, ROWS, NW> {
  using G = G16<DP>;
  static constexpr int TOTAL = ROWS * G::PITCH / 1024;
  __device__ __forceinline__ void load(uint32_t lds, const __bf16* base, long ts, long hs, int gs, int r0, int rend, int D, int wave, int lane) {
    const int i0 = r0 / gs;
    const u32x4 srd = make_srd(base + i0 * ts);
    const uint32_t tsb = ts * 2, hsb = hs * 2;
#pragma unroll
    for (int n = 0; n < (TOTAL + NW - 1) / NW; ++n) {
      const int it = wave + n * NW;
      if (TOTAL % NW == 0 || it < TOTAL) {
        const int row = it * (1024 / G::PITCH) + lane / G::CH, chunk = (lane % G::CH) ^ swz<__bf16, DP>(row);
        const int i = (r0 + row) / gs, g = r0 + row - i * gs;
        const bool ok = r0 + row < rend && chunk * 8 < D;
        dma16(lds + it * 1024, ok ? (uint32_t)(i - i0) * tsb + (uint32_t)g * hsb + chunk * 16 : kOutside, srd);
      }
    }
  }
};
template <int DP, int ROWS, int NW>
struct PackedStager<float, DP, ROWS, NW> {
  using G = G16<DP>;
  static constexpr int ITEMS = ROWS * G::CH, NT = NW * 64, PER = (ITEMS + NT - 1) / NT;
  static constexpr uint32_t PLANE = ROWS * G::PITCH;
  u32x4 held[PER][2];
  __device__ __forceinline__ void load(uint32_t, const float* base, long ts, long hs, int gs, int r0, int rend, int D, int, int) {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int item = threadIdx.x + NT * n, row = item / G::CH, chunk = item % G::CH;
      const int i = (r0 + row) / gs, g = r0 + row - i * gs;
      const bool ok = r0 + row < rend && chunk * 8 < D && item < ITEMS;
      const float* p = base + i * ts + g * hs + chunk * 8;
      held[n][0] = ok ? *reinterpret_cast<const u32x4*>(p) : (u32x4){0u, 0u, 0u, 0u};
      held[n][1] = ok ? *reinterpret_cast<const u32x4*>(p + 4) : (u32x4){0u, 0u, 0u, 0u};
    }
  }
  __device__ __forceinline__ void put(uint32_t lds) const {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int item = threadIdx.x + NT * n, row = item / G::CH, chunk = item % G::CH;
      if (ITEMS % NT == 0 || item < ITEMS) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(held[n][0][i]), x[4 + i] = __uint_as_float(held[n][1][i]);
        bf16x8 p[3];
        split8<3>(x, p);
        const uint32_t at = lds + row * G::PITCH + ((chunk ^ swz<__bf16, DP>(row)) << 4);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<lds_u32x4_t*>(at + k * PLANE) = __builtin_bit_cast(u32x4, p[k]);
      }
    }
  }
};

// The gradients of one key (and value) row over the query rows that see it alone (see row_again), 32 at a time, with scores in the bits of dQ's
template <typename T>
__device__ __forceinline__ void dkv_again(const WaArgs& a, const Seq& s, int b, int hk, int j, int lane, bool want_dk, bool want_dv) {
  fresh(lane);
  const T* k = (const T*)a.k + b * a.k_bs + j * a.k_ts + hk * a.k_hs;
  const T* v = (const T*)a.v + b * a.v_bs + j * a.v_ts + hk * a.v_hs;
  const int d0 = lane, d1 = lane + 64;
  T* dk = (T*)a.dk + b * a.dk_bs + j * a.dk_ts + hk * a.dk_hs;
  T* dv = (T*)a.dv + b * a.dv_bs + j * a.dv_ts + hk * a.dv_hs;
  const int e0 = min(d0, a.D - 1), e1 = min(d1, a.D - 1);
  const bool k0 = want_dk && no_number<T>(dk + e0, d0 < a.D), k1 = want_dk && no_number<T>(dk + e1, d1 < a.D);
  const bool v0 = want_dv && no_number<T>(dv + e0, d0 < a.D), v1 = want_dv && no_number<T>(dv + e1, d1 < a.D);
  const float c = a.scale * kLog2e;
  const int ilo = max(0, j - a.right - s.shift), ihi = j < a.sinks ? s.ql - 1 : min(s.ql - 1, j + a.left - s.shift);
  const int rlo = ilo * a.G, rhi = (ihi + 1) * a.G;
  float dk0 = 0.f, dk1 = 0.f, dv0 = 0.f, dv1 = 0.f;
  for (int r0 = rlo & ~31; r0 < rhi; r0 += 32) {
    const int r = r0 + (lane & 31), i = r / a.G;
    const bool in = r >= rlo && r < rhi;
    const long hq = (long)hk * a.G + (r - i * a.G);
    const float* stat = a.stat + ((long)(b * a.Hkv + hk) * a.ntiles32 + (r0 >> 5)) * kStat + (lane & 31);
    const float sc = row_times<T>(k, (const T*)a.q + b * a.q_bs + i * a.q_ts + hq * a.q_hs, in, a.D, lane);
    const float dp = row_times<T>(v, (const T*)a.dout + b * a.do_bs + i * a.do_ts + hq * a.do_hs, in, a.D, lane);
    const float p = in ? __builtin_amdgcn_exp2f(fmaf(sc - stat[64], c, -stat[0])) : 0.f, ds = in ? p * (dp - stat[32]) : 0.f;
    const uint32_t mask = (uint32_t)__ballot(in);
#pragma unroll 4
    for (int n = 0; n < 32; ++n) {
      if (!(mask >> n & 1)) continue;
      const int at = (r0 + n) / a.G;
      const long hn = (long)hk * a.G + (r0 + n - at * a.G);
      const T* q = (const T*)a.q + b * a.q_bs + at * a.q_ts + hn * a.q_hs;
      const T* dO = (const T*)a.dout + b * a.do_bs + at * a.do_ts + hn * a.do_hs;
      const float pn = __shfl(p, n, 64), dn = __shfl(ds, n, 64);
      dv0 = fmaf(pn, v0 ? Elem<T>::ld(dO + d0) : 0.f, dv0);
      dv1 = fmaf(pn, v1 ? Elem<T>::ld(dO + d1) : 0.f, dv1);
      dk0 = fmaf(dn, k0 ? Elem<T>::ld(q + d0) : 0.f, dk0);
      dk1 = fmaf(dn, k1 ? Elem<T>::ld(q + d1) : 0.f, dk1);
    }
    if (__all((!k0 || dk0 != dk0) && (!k1 || dk1 != dk1) && (!v0 || dv0 != dv0) && (!v1 || dv1 != dv1))) break;
  }
  if (k0) dk[d0] = (T)(dk0 * a.scale);
  if (k1) dk[d1] = (T)(dk1 * a.scale);
  if (v0) dv[d0] = (T)dv0;
  if (v1) dv[d1] = (T)dv1;
}

// What the dK / dV kernel walks over the rows with: RS rows a stage (q, dout and their statistics), two stages for bf16
template <typename T, int DP>
struct RowWalk {
  static constexpr int N = Planes<T>::N, RS = N == 1 ? 64 : 32, NSTAGE = N == 1 ? 2 : 1;
  static constexpr uint32_t PLANE = RS * G16<DP>::PITCH, TILE = N * PLANE, STAT = 2 * TILE, STAGE = 2 * TILE + 1024;
  // At 128 channels two waves share 32 keys, one for dV and one for dK: each has one accumulator, so two waves fit a SIMD where one with both
  // had it alone, for a quarter more matrix instructions (both take S).  bf16, 2 x 4096 tokens, 16 / 4 heads, window 1024: 241 -> 223 us.
  // fp32 holds its V planes in LDS, 24 KB a wave: 16 x 625 tokens and fewer, 8 heads, window 129: 298 -> 235 us.  At 64 channels too, 12 KB a wave,
  // where 57 registers were spilled and none is now: 2048 tokens, 8 / 1 heads, causal: 122 -> 82 us.
  static constexpr bool TWO = DP == 128, VLDS = DP >= 64 && N == 3;
  static constexpr int NW = TWO ? 8 : 4;
  // fp32: the dV wave, which has registers and time left, stages for its pair (the dK wave spilled what it held for it:
  // 239 -> 229 us)
  static constexpr int STAGERS = VLDS ? 4 : NW;
  static constexpr uint32_t VF = NSTAGE * STAGE, LDS = VF + (VLDS ? 4 * N * G16<DP>::NC * 1024 : 0);
};
// Fragments a lane parks in LDS: piece (n, c) at base + (c N + n) 1024 + 16 lane
template <int N, int DP>
__device__ __forceinline__ void park(uint32_t base, const Frags16<N, DP>& f, int lane) {
#pragma unroll
  for (int c = 0; c < G16<DP>::NC; ++c)
#pragma unroll
    for (int n = 0; n < N; ++n) *reinterpret_cast<lds_u32x4_t*>(base + (c * N + n) * 1024 + 16 * lane) = __builtin_bit_cast(u32x4, f[n][c]);
}
// rows16 whose right fragments are parked at `at` (the lane's address)
template <int N, int DP, uint32_t IMM, uint32_t PLANE, typename F = Nothing>
__device__ __forceinline__ void rows16_parked(f32x16& acc, const LaneOff<DP>& off, uint32_t at, F&& between = F()) {
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
#pragma unroll
  for (int c = 0; c < G16<DP>::NC; ++c) {
    bf16x8 a[N], b[N];
#pragma unroll
    for (int n = 0; n < N; ++n) a[n] = __builtin_bit_cast(bf16x8, lds_ld16(off.row[c] + IMM + n * PLANE)), b[n] = __builtin_bit_cast(bf16x8, lds_ld16(at + (c * N + n) * 1024));
    mma_planes<N>(acc, a, b);
    between(c);
  }
}
enum { kBoth = 0, kOnlyDv = 1, kOnlyDk = 2 };
// One step: the 32 staged rows at A (statistics at ST) against this wave's 32 keys.  Element e of S is row 8 (e / 4) + 4 h + e % 4, column the
// lane's key; [rlo, rhi] are the packed rows (of the whole sequence) that see the lane's key, checked when `part`.
template <typename T, int DP, uint32_t A, uint32_t ST, int ROLE>
__device__ __forceinline__ void dkv_step(f32x16 (&dk)[DP / 32], f32x16 (&dv)[DP / 32], const LaneOff<DP>& off, uint32_t stat,
                                         const Frags16<Planes<T>::N, DP>& kf, const Frags16<Planes<T>::N, DP>& vf, uint32_t vat, float c, bool moved, bool part, int r0,
                                         int rlo, int rhi, int lane) {
  using W = RowWalk<T, DP>;
  constexpr int NC = G16<DP>::NC, STEPS = DP / 16;
  f32x16 acc, dp;
  float p[16], ds[16];
  u32x4 l4[4], d4[4];
  auto hide = [&](float (&x)[16]) {
    asm volatile("");
    const int base = r0 + 4 * (lane >> 5);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int row = base + 8 * (e >> 2) + (e & 3);
      if (row < rlo || row > rhi) x[e] = 0.f;
    }
  };
  rows16<W::N, DP, A, W::PLANE, true>(acc, off, kf, [&](int k) {
#pragma unroll
    for (int e = k * 4 / NC; e < (k + 1) * 4 / NC; ++e) l4[e] = lds_ld16(stat + ST + 32 * e);
  });
  if (__builtin_expect(moved, 0)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const u32x4 m4 = lds_ld16(stat + ST + 256 + 32 * e);
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[4 * e + x] -= __uint_as_float(m4[x]);
    }
  }
  // the exponentials stand between the products for dP, the score gradients between those for dV
  auto exps = [&](int k) {
#pragma unroll
    for (int e = k * 16 / NC; e < (k + 1) * 16 / NC; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(acc[e], c, -__uint_as_float(l4[e >> 2][e & 3])));
    if constexpr (ROLE != kOnlyDv)
#pragma unroll
      for (int e = k * 4 / NC; e < (k + 1) * 4 / NC; ++e) d4[e] = lds_ld16(stat + ST + 128 + 32 * e);
  };
  if constexpr (ROLE == kOnlyDv) {
#pragma unroll
    for (int k = 0; k < NC; ++k) exps(k);
  } else if constexpr (W::VLDS) {
    rows16_parked<W::N, DP, A + W::TILE, W::PLANE>(dp, off, vat, exps);
  } else {
    rows16<W::N, DP, A + W::TILE, W::PLANE>(dp, off, vf, exps);
  }
  auto grads = [&](int e) { ds[e] = p[e] * (dp[e] - __uint_as_float(d4[e >> 2][e & 3])); };
  bf16x8 pb[2][W::N];
  if constexpr (ROLE != kOnlyDk) {
    if (part) hide(p);
    pack16<W::N>(pb, p);
    cols16<W::N, DP, A + W::TILE, W::PLANE>(dv, off, pb, [&](int k) {
      if constexpr (ROLE == kBoth)
#pragma unroll
        for (int e = k * 16 / STEPS; e < (k + 1) * 16 / STEPS; ++e) grads(e);
    });
  }
  if constexpr (ROLE != kOnlyDv) {
    if constexpr (ROLE == kOnlyDk)
#pragma unroll
      for (int e = 0; e < 16; ++e) grads(e);
    if (part) hide(ds);   // (an unseen row's dP may be infinite: 0 times it is not 0)
    pack16<W::N>(pb, ds);
    cols16<W::N, DP, A, W::PLANE>(dk, off, pb);
  }
}

// dK / dV.  Workgroups from nsink on: 128 keys, 32 keys a wave (or pair of waves), the rows inside the keys' windows.  The first nsink
// workgroups: the rows beyond the window of 32 KB keys that are sinks, a share of them each; the waves are KB key blocks x row blocks of a
// stage, and every wave leaves its fp32 sums.  Sinks among the 128 keys leave theirs as the first shares.  Where the keys are too few to fill the chip
// (grouped heads, small batches), the rows of 128 keys are cut into nrow shares too.
// Bound by the LDS reads of its tiles (each of the four products reads one) and the waits at its barriers, at two waves a SIMD: matrix units busy
// 38 % of the time, LDS 25 %.  bf16, 2 x 4096 tokens, 16 / 4 heads of 128 channels, window 1024: 234 us, 515 TFLOP/s of what is seen; 8192 tokens, 8
// heads of 64, window 257: 42 us, 420 TFLOP/s.
template <typename T, int DP, int OCC>
__global__ __launch_bounds__((RowWalk<T, DP>::NW * 64)) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void window_attn_dkv_kernel(const WaArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using W = RowWalk<T, DP>;
  constexpr int ND = DP / 32, N = W::N, NB = W::RS / 32, KB = 4 / NB;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kw = wave & 3;   // (waves kw and kw + 4: the same keys)
  const int nst = (a.sink_rows / 32 + KB - 1) / KB;                      // sink tiles of a (batch, key head)
  const int nsink = a.B * a.Hkv * nst * a.nsplit;
  const bool far = (int)blockIdx.x < nsink;
  int bh, jw, split = 0;                                                  // (near: of nrow shares of the rows)
  if (far) {
    const Item item = xcd_item(blockIdx.x, a.B * a.Hkv, nst * a.nsplit);
    split = item.at % a.nsplit;
    bh = item.bh;
    jw = (item.at / a.nsplit) * KB * 32 + (kw % KB) * 32;
  } else {
    const Item item = xcd_item(blockIdx.x - nsink, a.B * a.Hkv, a.ntiles * a.nrow);
    split = item.at % a.nrow;
    bh = item.bh;
    jw = (item.at / a.nrow) * 128 + kw * 32;
  }
  const int hk = bh % a.Hkv, b = bh / a.Hkv;
  const Seq s = seq_of(a, b);
  const int j = jw + (lane & 31);
  const int kend = far ? min(s.kl, a.sinks) : s.kl;                       // keys of this pass
  const bool key_ok = j < kend;
  const int h4 = 4 * (lane >> 5);
  // Queries [lo(first), hi(last)] see a key of [first, last]: inside the window from first - right on up to last + left, beyond it from
  // first + left + 1 on; clamped to [0, q_len], the end exclusive
  auto lo = [&](int key) { return max(0, min(s.ql, far ? key + a.left - s.shift + 1 : key - a.right - s.shift)); };
  auto hi = [&](int key) { return far ? s.ql : max(0, min(s.ql, key + a.left - s.shift + 1)); };
  const int block_first = far ? jw - (kw % KB) * 32 : jw - kw * 32, block_last = min(block_first + (far ? KB * 32 : 128), kend) - 1;
  const int wave_last = min(jw + 31, kend - 1);

  auto work = [&](auto role) {
    constexpr int ROLE = decltype(role)::value;
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) dk[d][e] = 0.f, dv[d][e] = 0.f;
    if (block_first <= block_last) {
      int t0 = lo(block_first) * a.G / W::RS, t1 = (hi(block_last) * a.G + W::RS - 1) / W::RS;
      const int shares = far ? a.nsplit : a.nrow, per = (max(0, t1 - t0) + shares - 1) / shares;
      t0 += split * per;
      t1 = min(t1, t0 + per);
      const T* qb = (const T*)a.q + b * a.q_bs + (long)hk * a.G * a.q_hs;
      const T* db = (const T*)a.dout + b * a.do_bs + (long)hk * a.G * a.do_hs;
      const float* stat = a.stat + (long)bh * a.ntiles32 * kStat;
      const int rend = s.ql * a.G;
      constexpr bool STAGES = !(W::VLDS && ROLE == kOnlyDk);
      PackedStager<T, DP, W::RS, W::STAGERS> sq, sd;
      auto load = [&](int t, uint32_t at) {
        if constexpr (!STAGES) return;
        sq.load(at, qb, a.q_ts, a.q_hs, a.G, t * W::RS, rend, a.D, wave, lane);
        sd.load(at + W::TILE, db, a.do_ts, a.do_hs, a.G, t * W::RS, rend, a.D, wave, lane);
      };
      auto load_stat = [&](int t, uint32_t at) {
        if (wave == 0) dma16(at + W::STAT, lane < W::RS / 32 * (kStat / 4) ? lane * 16u : kOutside, make_srd(stat + (long)t * (W::RS / 32 * kStat)));
      };
      if (t0 < t1) {
        load(t0, lds);
        load_stat(t0, lds);
      }
      bool moved = false;                                                  // scores of any of these rows, see kStat
      for (int x = t0 * NB + lane; x < t1 * NB; x += 64) moved |= stat[(long)x * kStat + 96] != 0.f;
      moved = __ballot(moved) != 0;
      Frags16<N, DP> kf, vf;
      const uint32_t vat = lds + W::VF + kw * (N * G16<DP>::NC * 1024) + 16 * lane;
      load_frags16<T, DP>(kf, (const T*)a.k + b * a.k_bs + (long)j * a.k_ts + hk * a.k_hs, key_ok, a.D, lane);
      if constexpr (ROLE != kOnlyDv) {
        load_frags16<T, DP>(vf, (const T*)a.v + b * a.v_bs + (long)j * a.v_ts + hk * a.v_hs, key_ok, a.D, lane);
        if constexpr (W::VLDS) park<N, DP>(vat - 16 * lane, vf, lane);
        else arrived16(vf);
      }
      arrived16(kf);
      const float c = a.scale * kLog2e;
      const bool wave_ok = jw <= wave_last;
      const int wr0 = lo(jw) * a.G, wr1 = wave_ok ? hi(wave_last) * a.G : 0;             // rows some key of this wave is seen by
      const int fr0 = lo(jw + 31) * a.G, fr1 = jw + 31 < kend ? hi(jw) * a.G : 0;          // rows all of its keys are seen by
      const int rlo = key_ok ? lo(j) * a.G : 1, rhi = key_ok ? hi(j) * a.G - 1 : 0;        // this lane's key
      const LaneOff<DP> off(lds, lane);
      const uint32_t stat_off = lds + W::STAT + 16 * (lane >> 5);
      auto step = [&](int t, auto st) {
        constexpr uint32_t S0 = decltype(st)::value;
        auto sub = [&](auto k) {
          constexpr int B32 = decltype(k)::value;
          const int r0 = t * W::RS + 32 * B32;
          if ((far && NB > 1 && kw / KB != B32) || r0 >= wr1 || r0 + 32 <= wr0) return;
          dkv_step<T, DP, S0 + B32 * 32 * G16<DP>::PITCH, S0 + B32 * kStat * 4, ROLE>(dk, dv, off, stat_off, kf, vf, vat, c, moved, r0 < fr0 || r0 + 32 > fr1, r0, rlo, rhi, lane);
        };
        sub(std::integral_constant<int, 0>());
        if constexpr (NB == 2) sub(std::integral_constant<int, 1>());
      };
      if constexpr (N == 1) {
        for (int t = t0; t < t1; t += 2) {
          wait_vm<0>();
          wg_barrier();
          if (t + 1 < t1) load(t + 1, lds + W::STAGE), load_stat(t + 1, lds + W::STAGE);
          step(t, std::integral_constant<uint32_t, 0>());
          if (t + 1 >= t1) break;
          wait_vm<0>();
          wg_barrier();
          if (t + 2 < t1) load(t + 2, lds), load_stat(t + 2, lds);
          step(t + 1, std::integral_constant<uint32_t, W::STAGE>());
        }
      } else {
        for (int t = t0; t < t1; ++t) {
          if (t > t0) {
            wg_barrier();                       // the tile before has been read
            load_stat(t, lds);
          }
          if constexpr (STAGES) {
            sq.put(lds);
            sd.put(lds + W::TILE);
          }
          wait_vm<0>();
          if (t + 1 < t1) load(t + 1, lds);
          wg_barrier();
          step(t, std::integral_constant<uint32_t, 0>());
        }
      }
    }
    bool bad_k = false, bad_v = false;
    const bool sink = far || j < a.sinks;
    if (sink || a.nrow > 1) {
      if (sink ? j < a.sink_rows : j < a.Tk) {
        float* part = sink ? a.part + (((long)bh * a.nparts + (far ? a.nrow + split * NB + kw / KB : split)) * a.sink_rows + j) * 2 * DP
                           : a.near + (((long)bh * a.nrow + split) * a.Tk + j) * 2 * DP;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = 32 * d + 8 * e + h4;
            if constexpr (ROLE != kOnlyDv) *reinterpret_cast<f32x4*>(part + at) = (f32x4){dk[d][4 * e], dk[d][4 * e + 1], dk[d][4 * e + 2], dk[d][4 * e + 3]};
            if constexpr (ROLE != kOnlyDk) *reinterpret_cast<f32x4*>(part + DP + at) = (f32x4){dv[d][4 * e], dv[d][4 * e + 1], dv[d][4 * e + 2], dv[d][4 * e + 3]};
          }
      }
    } else if (j < a.Tk) {
      T* krow = (T*)a.dk + b * a.dk_bs + (long)j * a.dk_ts + hk * a.dk_hs;
      T* vrow = (T*)a.dv + b * a.dv_bs + (long)j * a.dv_ts + hk * a.dv_hs;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x[4], y[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            x[z] = key_ok ? dk[d][4 * e + z] * a.scale : 0.f;
            y[z] = key_ok ? dv[d][4 * e + z] : 0.f;
            bad_k |= x[z] != x[z];
            bad_v |= y[z] != y[z];
          }
          const int at = 32 * d + 8 * e + h4;
          if (ROLE != kOnlyDv && at < a.D) store4<T>(krow + at, x);
          if (ROLE != kOnlyDk && at < a.D) store4<T>(vrow + at, y);
        }
    }
    const uint64_t mk = ROLE == kOnlyDv ? 0 : __ballot(bad_k), mv = ROLE == kOnlyDk ? 0 : __ballot(bad_v);
    uint64_t again = mk | mv;
    again = (again | (again >> 32)) & 0xffffffffull;
    while (again) {
      const int n = __builtin_ctzll(again);
      again &= again - 1;
      dkv_again<T>(a, s, b, hk, jw + n, lane, (mk >> n | mk >> (n + 32)) & 1, (mv >> n | mv >> (n + 32)) & 1);
    }
  };
  if constexpr (W::TWO) {
    if (wave < 4) work(std::integral_constant<int, kOnlyDv>());
    else work(std::integral_constant<int, kOnlyDk>());
  } else {
    work(std::integral_constant<int, kBoth>());
  }
#endif
}

// The shares, in order: one workgroup a sink, its 4 waves take the shares in turn; then (nrow > 1) one wave a key
template <typename T, int DP>
__global__ __launch_bounds__(256) void window_attn_dkv_join_kernel(const WaArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int PER = 2 * DP / 64;
  __shared__ float share[4][2 * DP];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nk = min(a.sinks, a.Tk), per = nk + (a.nrow > 1 ? (a.Tk - nk + 3) / 4 : 0);
  const int at0 = blockIdx.x % per, bh = blockIdx.x / per, hk = bh % a.Hkv, b = bh / a.Hkv;
  const Seq s = seq_of(a, b);
  const bool sink = at0 < nk;
  const int j = sink ? at0 : nk + 4 * (at0 - nk) + wave;
  float sum[PER];
#pragma unroll
  for (int x = 0; x < PER; ++x) sum[x] = 0.f;
  if (sink) {
    const float* part = a.part + ((long)bh * a.nparts * a.sink_rows + j) * 2 * DP + lane;
#pragma unroll 4
    for (int n = wave; n < a.nparts; n += 4)
#pragma unroll
      for (int x = 0; x < PER; ++x) sum[x] += part[(long)n * a.sink_rows * 2 * DP + 64 * x];
#pragma unroll
    for (int x = 0; x < PER; ++x) share[wave][64 * x + lane] = sum[x];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      const int at = 64 * x + lane;
      sum[x] = (share[0][at] + share[1][at]) + (share[2][at] + share[3][at]);
    }
  } else {
    if (j >= a.Tk) return;
    const float* part = a.near + ((long)bh * a.nrow * a.Tk + j) * 2 * DP + lane;
#pragma unroll 4
    for (int n = 0; n < a.nrow; ++n)
#pragma unroll
      for (int x = 0; x < PER; ++x) sum[x] += part[(long)n * a.Tk * 2 * DP + 64 * x];
  }
  bool bad = false;
#pragma unroll
  for (int x = 0; x < PER; ++x) {
    const int at = 64 * x + lane, d = at % DP;
    const bool isk = at < DP;
    const float v = j < s.kl ? (isk ? sum[x] * a.scale : sum[x]) : 0.f;
    T* row = isk ? (T*)a.dk + b * a.dk_bs + (long)j * a.dk_ts + hk * a.dk_hs : (T*)a.dv + b * a.dv_bs + (long)j * a.dv_ts + hk * a.dv_hs;
    if (d < a.D) {
      row[d] = (T)v;
      bad |= v != v;
    }
  }
  if (__ballot(bad)) dkv_again<T>(a, s, b, hk, j, lane, true, true);
#endif
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
int compute_units() {
  static int n_dev[kTdxMaxDevices] = {};
  int& n = n_dev[tdx_device_slot()];
  if (n == 0) {
    int dev = 0, v = 0;
    n = hipGetDevice(&dev) == hipSuccess && hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0 ? v : 256;
  }
  return n;
}

bool strides_ok(long bs, long ts, long hs, int es) { return bs >= 0 && ts >= 0 && hs >= 0 && ((bs | ts | hs) * es) % 16 == 0; }
bool pointer_ok(const void* p) { return p && ((uintptr_t)p & 15) == 0; }

// Checks and translates the part of the descriptor that both directions read; returns a status code.
int translate(const tdx_window_attn_desc* d, WaArgs& a, const char* fn) {
  TDX_CHECK_ARG(d, "%s: null descriptor", fn);
  TDX_CHECK_ARG(d->dtype == TDX_F32 || d->dtype == TDX_BF16, "%s: bad dtype %d", fn, d->dtype);
  TDX_CHECK_ARG(d->B >= 0 && d->Tq >= 0 && d->Tk >= 0 && d->Hq >= 1 && d->Hkv >= 1 && d->Hq % d->Hkv == 0, "%s: bad shape B=%d Tq=%d Tk=%d Hq=%d Hkv=%d", fn,
                d->B, d->Tq, d->Tk, d->Hq, d->Hkv);
  TDX_CHECK_ARG(d->Tq < (1 << 28) && d->Tk < (1 << 28) && (int64_t)d->Tq * (d->Hq / d->Hkv) < (1 << 30), "%s: Tq=%d Tk=%d are too long", fn, d->Tq, d->Tk);
  TDX_CHECK_ARG(d->D >= 8 && d->D <= 128 && d->D % 8 == 0, "%s: D=%d (a multiple of 8, at most 128)", fn, d->D);
  TDX_CHECK_ARG(std::isfinite(d->scale) && d->scale > 0.f && std::isfinite(d->scale * kLog2e), "%s: scale=%g (finite, also times log2 e, > 0)", fn, (double)d->scale);
  TDX_CHECK_ARG(d->sinks >= 0, "%s: sinks=%d", fn, d->sinks);
  const int es = d->dtype == TDX_F32 ? 4 : 2;
  a = WaArgs{};
  a.q = d->q, a.k = d->k, a.v = d->v, a.out = d->out, a.lse = d->lse;
  a.q_bs = d->q_bs, a.q_ts = d->q_ts, a.q_hs = d->q_hs, a.k_bs = d->k_bs, a.k_ts = d->k_ts, a.k_hs = d->k_hs;
  a.v_bs = d->v_bs, a.v_ts = d->v_ts, a.v_hs = d->v_hs, a.o_bs = d->out_bs, a.o_ts = d->out_ts, a.o_hs = d->out_hs;
  a.B = d->B, a.Tq = d->Tq, a.Tk = d->Tk, a.Hkv = d->Hkv, a.G = d->Hq / d->Hkv, a.D = d->D, a.scale = d->scale;
  a.q_lens = d->q_lens, a.k_lens = d->k_lens;
  a.down = (float)(8 + std::bit_width((uint32_t)d->Tk)), a.up = std::ldexp(1.f, (int)a.down);
  a.out_lo = d->dtype == TDX_BF16 ? (__bf16*)d->out_lo : nullptr;
  TDX_CHECK_ARG(((uintptr_t)a.out_lo & 15) == 0, "%s: misaligned out_lo", fn);
  // a limit beyond every length is none; sinks that hold every key too
  a.left = d->left < 0 || d->left >= d->Tk || d->sinks >= d->Tk ? kFar : d->left;
  a.right = d->right < 0 || (int64_t)d->right >= (int64_t)d->Tk + d->Tq ? kFar : d->right;
  a.sinks = a.left == kFar ? 0 : d->sinks;
  if (d->B == 0 || d->Tq == 0) return TDX_OK;
  TDX_CHECK_ARG(pointer_ok(d->q) && pointer_ok(d->out) && (d->Tk == 0 || (pointer_ok(d->k) && pointer_ok(d->v))), "%s: null or misaligned pointer", fn);
  TDX_CHECK_ARG(strides_ok(d->q_bs, d->q_ts, d->q_hs, es) && strides_ok(d->k_bs, d->k_ts, d->k_hs, es) && strides_ok(d->v_bs, d->v_ts, d->v_hs, es) &&
                    strides_ok(d->out_bs, d->out_ts, d->out_hs, es), "%s: strides must be multiples of 16 bytes and not negative", fn);
  TDX_CHECK_ARG(d->k_ts * es < (1 << 24) && d->v_ts * es < (1 << 24), "%s: the token strides of k and v must be below 16 MiB", fn);
  TDX_CHECK_ARG((65 * d->q_ts + a.G * d->q_hs) * es < (1ll << 31), "%s: the strides of q are too large", fn);
  TDX_CHECK_ARG(((uintptr_t)d->q_lens & 3) == 0 && ((uintptr_t)d->k_lens & 3) == 0, "%s: misaligned lengths", fn);
  return TDX_OK;
}

// Which forward kernel: the few-row kernel for a token or so, and while the many-row kernel (128 rows a workgroup) would leave 3 of 8 compute units
// idle, 5 of 8 for bf16 at 128 channels.  Measured, us, many-row / few-row: 252 workgroups (2 x 2000 tokens, 8 / 2 heads, window 512) bf16 17 / 27 at 64
// channels, 23 / 63 at 128, fp32 42 / 62 and 67 / 141; 192 (3000, 8 heads, window 257) 16 / 21, 19 / 41, 35 / 43, 53 / 79; 128 (2048, 8 / 1 heads, causal)
// 32 / 25, 43 / 54, 127 / 81, 204 / 172; 64 (1000, 8 heads, window 257) 16 / 11, 19 / 15, 34 / 16, 52 / 27.
struct Plan {
  bool few, one;
  int ntiles, nsplit;
  int64_t threads;                    // of the largest launch
};
constexpr int64_t kMostThreads = 0xffffffffLL;   // a launch counts its threads in 32 bits
constexpr int kMostSplits = 64;       // (the join kernel holds a row's shares in registers)
int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
template <typename T>
int few_per_unit(int dp) {              // workgroups of the few-row kernel that fit a compute unit: 160 KB of LDS, 2 waves a SIMD at least below 128 channels
  const int lds = dp == 32 ? Few<T, 32, false>::LDS : dp == 64 ? Few<T, 64, false>::LDS : Few<T, 128, false>::LDS;
  return std::max(1, std::min(160 * 1024 / lds, dp == 128 ? 1 : 2));
}
int few_per_unit(int es, int dp) { return es == 4 ? few_per_unit<float>(dp) : few_per_unit<__bf16>(dp); }
Plan plan_forward(const WaArgs& a, int es) {
  Plan p{};
  const long rows = (long)a.Tq * a.G, bh = (long)a.B * a.Hkv;
  p.few = rows <= 32 || bh * ((rows + 127) / 128) < compute_units() * (es == 2 && padded(a.D) == 128 ? 3 : 5) / 8;
  p.ntiles = (int)((rows + (p.few ? 31 : 127)) / (p.few ? 32 : 128));
  p.nsplit = 1;
  if (p.few) {
    // key tiles a row tile sees at most
    const long span = a.left == kFar ? a.Tk : std::min<long>(a.Tk, (long)a.left + 32 / a.G + 1 + (a.right == kFar ? a.Tk : a.right) + a.sinks);
    const long tiles = (span + 31) / 32, wgs = bh * p.ntiles;
    p.one = tiles <= 2;
    // Splits of the keys: the rounds of workgroups over the chip, of so many tiles a wave and two tiles' time to begin with, then the join (one
    // workgroup a row), in tiles' times.  Measured, fp32, 8 heads of 128 channels, one token: 300 keys 36 -> 16 us with 5 splits, 4096 keys 33 -> 17
    // with 32 and 27 with 64; bf16, 16 x 8 heads, 512 keys: 13 with 2, 18 with 4; 1000 tokens, 8 heads, window 257: 11 alone, 21 with a join.
    const int fit = compute_units() * few_per_unit(es, padded(a.D)), most = (int)std::min({(long)kMostSplits, tiles, 2 * fit / wgs});
    const double join = (2.5 + bh * rows / 1700.) * (es == 4 ? 0.5 : 1);   // (an fp32 tile takes twice as long)
    double best = 0;
    for (int n = 1; n <= most && !p.one; ++n) {
      const double cost = (double)(((int)wgs * n + fit - 1) / fit) * (((int)tiles + 4 * n - 1) / (4 * n) + 2) + (n > 1 ? join : 0);
      if (n == 1 || cost < best) best = cost, p.nsplit = n;
    }
  }
  p.threads = bh * std::max<int64_t>((int64_t)p.ntiles * p.nsplit * (p.one ? 64 : 256), p.nsplit > 1 ? rows * 256 : 0);
  return p;
}

template <typename K>
int reserve_lds(K kernel, size_t bytes, bool& done) {
  if (!done) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess)
      TDX_FAIL(TDX_ERR_HIP, "tdx_window_attention: cannot reserve LDS");
    done = true;
  }
  return TDX_OK;
}
#define WA_LAUNCH(kernel, grid, threads, lds, st, args)                        \
  do {                                                                         \
    static bool done_dev[kTdxMaxDevices] = {};                                 \
    const int rc__ = reserve_lds(&kernel, lds, done_dev[tdx_device_slot()]);   \
    if (rc__) return rc__;                                                     \
    hipLaunchKernelGGL((kernel), dim3((unsigned)(grid)), dim3(threads), lds, st, args); \
  } while (0)

template <typename T, int DP>
int launch_forward(WaArgs& a, const Plan& p, hipStream_t st) {
  const long bh = (long)a.B * a.Hkv;
  a.ntiles = p.ntiles, a.nsplit = p.nsplit;
  if (p.few) {
    if (p.one) WA_LAUNCH((window_attn_few_kernel<T, DP, true>), bh * p.ntiles, 64, (Few<T, DP, true>::LDS), st, a);
    else WA_LAUNCH((window_attn_few_kernel<T, DP, false>), bh * p.ntiles * p.nsplit, (Few<T, DP, false>::NW * 64), (Few<T, DP, false>::LDS), st, a);
    TDX_CHECK_LAUNCH("window_attn_few_kernel");
    if (p.nsplit > 1) {
      hipLaunchKernelGGL((window_attn_join_kernel<T, DP>), dim3((unsigned)(bh * a.Tq * a.G)), dim3(256), 0, st, a);
      TDX_CHECK_LAUNCH("window_attn_join_kernel");
    }
    return TDX_OK;
  }
  WA_LAUNCH((window_attn_kernel<T, DP>), bh * p.ntiles, 256, (Walk<T, DP>::LDS), st, a);
  TDX_CHECK_LAUNCH("window_attn_kernel");
  return TDX_OK;
}
template <typename T>
int launch_forward_d(WaArgs& a, const Plan& p, hipStream_t st) {
  switch (padded(a.D)) {
    case 32: return launch_forward<T, 32>(a, p, st);
    case 64: return launch_forward<T, 64>(a, p, st);
    default: return launch_forward<T, 128>(a, p, st);
  }
}

// Backward: bytes of the row statistics, of the sinks' shares and of all keys'
struct BwdPlan {
  int sink_rows, nsplit, nparts, nrow, nkey;
  int64_t stat_bytes, part_bytes, near_bytes, threads;
  int64_t bytes() const { return stat_bytes + part_bytes + near_bytes; }
};
// Into how many shares `wgs` workgroups of `stages` stages are cut: the rounds over the chip, of so many stages and two stages' time to begin with,
// then the join, in stages' times (2 us, fp32 4; the join 4 us and its `bytes` a share twice at 4 TB/s).  A compute unit counts for two workgroups
// below 128 channels, for one there (dQ with two beside each other: 110 -> 97 us, and 13 to join).
int shares(int64_t wgs, int64_t stages, int64_t dp, int64_t bytes, int es) {
  const int64_t chip = (int64_t)compute_units() * (dp == 128 ? 1 : 2);
  double best = 0;
  int best_n = 1;
  const int most = (int)std::min({(int64_t)64, stages, 2 * chip / std::max<int64_t>(wgs, 1)});   // (two rounds: more shares only add to the join)
  for (int n = 1; n <= most; ++n) {
    const double join = n > 1 ? (2 + (double)(n * bytes) * 2 / 8e6) * (es == 4 ? 0.5 : 1) : 0;
    const double cost = (double)(((int)wgs * n + (int)chip - 1) / (int)chip) * (((int)stages + n - 1) / n + 2) + join;
    if (n == 1 || cost < best) best = cost, best_n = n;
  }
  return best_n;
}
BwdPlan plan_backward(const WaArgs& a, int es) {
  BwdPlan p{};
  const int64_t rows = (int64_t)a.Tq * a.G, bh = (int64_t)a.B * a.Hkv, dp = padded(a.D);
  p.stat_bytes = bh * ((rows + 127) / 128) * 4 * kStat * 4;
  const int64_t keys = ((int64_t)a.Tk + 127) / 128, tiles = (rows + 127) / 128;
  // dK / dV, bf16, 4096 tokens, 8 / 1 heads of 128 channels, causal (32 workgroups without shares): 1112 -> 173 us and 7 to join; 4 x 955, 16 / 4 heads
  // of 64 (128 workgroups): 148 -> 51 and 8; fp32, 2048, 8 / 1 heads of 64, causal (16 workgroups): 2029 -> 82 and 7.  dQ of the last (128
  // workgroups): 149 -> 65 and 7.
  const int64_t seen = a.left == kFar || a.right == kFar ? a.Tq : std::min<int64_t>(a.Tq, (int64_t)a.left + a.right + 128);
  p.nrow = shares(bh * keys, (seen * a.G + (es == 4 ? 31 : 63)) / (es == 4 ? 32 : 64), dp, bh * a.Tk * dp * 2 * 4, es);
  const int64_t span = a.left == kFar || a.right == kFar ? a.Tk : std::min<int64_t>(a.Tk, (int64_t)a.left + a.right + 128 / a.G + a.sinks);
  p.nkey = shares(bh * tiles, (span + (es == 4 ? 31 : 63)) / (es == 4 ? 32 : 64), dp, bh * rows * dp * 4, es);
  // one after the other, the two need the same memory
  p.near_bytes = std::max(p.nrow > 1 ? bh * p.nrow * a.Tk * 2 * dp * 4 : 0, p.nkey > 1 ? bh * p.nkey * rows * dp * 4 : 0);
  int64_t sink_wgs = 0;
  if (a.sinks > 0) {
    const int nb = es == 4 ? 1 : 2, kb = 4 / nb;                        // row and key blocks of a workgroup (RowWalk)
    p.sink_rows = (a.sinks + 31) / 32 * 32;
    const int64_t wgs = bh * ((p.sink_rows / 32 + kb - 1) / kb);
    // one workgroup a compute unit, 8 stages each at least
    p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>((compute_units() + wgs - 1) / wgs, rows / (nb * 32 * 8)));
    p.nparts = p.nrow + p.nsplit * nb;
    p.part_bytes = bh * p.nparts * p.sink_rows * 2 * dp * 4;
    sink_wgs = wgs * p.nsplit;
  }
  p.threads = std::max({bh * tiles * p.nkey * 256, p.nkey > 1 ? bh * ((rows + 3) / 4) * 256 : 0, (sink_wgs + bh * keys * p.nrow) * (dp == 128 ? 512 : 256), bh * (std::min(a.sinks, a.Tk) + (p.nrow > 1 ? (a.Tk + 3) / 4 : 0)) * 256});
  return p;
}

template <typename T, int DP>
int launch_backward(WaArgs& a, const BwdPlan& p, hipStream_t st) {
  const long bh = (long)a.B * a.Hkv;
  constexpr int OCC = 2, OCC_Q = sizeof(T) == 4 ? (DP == 128 ? 1 : DP == 64 ? 2 : 3) : (DP == 128 ? 2 : DP == 64 ? 3 : 4), KB = 4 / (RowWalk<T, DP>::RS / 32);
  const long rt = ((long)a.Tq * a.G + 127) / 128;
  a.ntiles = (int)rt, a.ntiles32 = (int)rt * 4, a.nsplit = p.nsplit, a.nparts = p.nparts, a.sink_rows = p.sink_rows, a.nrow = p.nrow, a.nkey = p.nkey;
  WA_LAUNCH((window_attn_dq_kernel<T, DP, OCC_Q>), bh * rt * a.nkey, 256, (Walk<T, DP>::LDS), st, a);
  TDX_CHECK_LAUNCH("window_attn_dq_kernel");
  if (a.nkey > 1) {
    hipLaunchKernelGGL((window_attn_dq_join_kernel<T, DP>), dim3((unsigned)(bh * (((long)a.Tq * a.G + 3) / 4))), dim3(256), 0, st, a);
    TDX_CHECK_LAUNCH("window_attn_dq_join_kernel");
  }
  if (a.Tk == 0) return TDX_OK;
  a.ntiles = (a.Tk + 127) / 128;
  const long sink_wgs = bh * ((p.sink_rows / 32 + KB - 1) / KB) * p.nsplit;
  WA_LAUNCH((window_attn_dkv_kernel<T, DP, OCC>), sink_wgs + bh * a.ntiles * a.nrow, (RowWalk<T, DP>::NW * 64), (RowWalk<T, DP>::LDS), st, a);
  TDX_CHECK_LAUNCH("window_attn_dkv_kernel");
  if (p.sink_rows || p.nrow > 1) {
    const int nk = std::min(a.sinks, a.Tk);
    hipLaunchKernelGGL((window_attn_dkv_join_kernel<T, DP>), dim3((unsigned)(bh * (nk + (p.nrow > 1 ? (a.Tk - nk + 3) / 4 : 0)))), dim3(256), 0, st, a);
    TDX_CHECK_LAUNCH("window_attn_dkv_join_kernel");
  }
  return TDX_OK;
}
template <typename T>
int launch_backward_d(WaArgs& a, const BwdPlan& p, hipStream_t st) {
  switch (padded(a.D)) {
    case 32: return launch_backward<T, 32>(a, p, st);
    case 64: return launch_backward<T, 64>(a, p, st);
    default: return launch_backward<T, 128>(a, p, st);
  }
}

}  // namespace

extern "C" int64_t tdx_window_attention_ws_bytes(const tdx_window_attn_desc* d) {
  WaArgs a;
  if (translate(d, a, "tdx_window_attention_ws_bytes") != TDX_OK || a.B == 0 || a.Tq == 0) return 0;
  const Plan p = plan_forward(a, d->dtype == TDX_F32 ? 4 : 2);
  return p.nsplit > 1 ? (int64_t)a.B * a.Hkv * p.ntiles * p.nsplit * 32 * (padded(a.D) + 2) * 4 : 0;
}

extern "C" int tdx_window_attention(const tdx_window_attn_desc* d, void* stream) {
  WaArgs a;
  if (const int rc = translate(d, a, "tdx_window_attention")) return rc;
  if (a.B == 0 || a.Tq == 0) return TDX_OK;
  const Plan p = plan_forward(a, d->dtype == TDX_F32 ? 4 : 2);
  const int64_t need = p.nsplit > 1 ? (int64_t)a.B * a.Hkv * p.ntiles * p.nsplit * 32 * (padded(a.D) + 2) * 4 : 0;
  TDX_CHECK_ARG(need == 0 || (pointer_ok(d->ws) && d->ws_bytes >= need), "tdx_window_attention: workspace of %lld bytes needed, got %lld", (long long)need, (long long)d->ws_bytes);
  TDX_CHECK_ARG((long)a.B * a.Hkv * a.Tq * a.G < 0x7fffffffL && p.threads <= kMostThreads, "tdx_window_attention: too many rows");
  a.ws = (float*)d->ws;
  return d->dtype == TDX_F32 ? launch_forward_d<float>(a, p, (hipStream_t)stream) : launch_forward_d<__bf16>(a, p, (hipStream_t)stream);
}

extern "C" int64_t tdx_window_attention_bwd_ws_bytes(const tdx_window_attn_desc* d) {
  WaArgs a;
  if (translate(d, a, "tdx_window_attention_bwd_ws_bytes") != TDX_OK || a.B == 0 || a.Tq == 0) return 0;
  const BwdPlan p = plan_backward(a, d->dtype == TDX_F32 ? 4 : 2);
  return p.bytes();
}

extern "C" int tdx_window_attention_bwd(const tdx_window_attn_desc* d, void* stream) {
  WaArgs a;
  if (const int rc = translate(d, a, "tdx_window_attention_bwd")) return rc;
  if (a.B == 0 || a.Tq == 0) TDX_CHECK_ARG(a.B == 0 || a.Tk == 0, "tdx_window_attention_bwd: no query rows (the gradients of k and v are zero: fill them)");
  if (a.B == 0 || a.Tq == 0) return TDX_OK;
  const int es = d->dtype == TDX_F32 ? 4 : 2;
  TDX_CHECK_ARG(d->lse && pointer_ok(d->dout) && pointer_ok(d->dq) && (a.Tk == 0 || (pointer_ok(d->dk) && pointer_ok(d->dv))),
                "tdx_window_attention_bwd: null or misaligned pointer");
  TDX_CHECK_ARG(strides_ok(d->dout_bs, d->dout_ts, d->dout_hs, es) && strides_ok(d->dq_bs, d->dq_ts, d->dq_hs, es) && strides_ok(d->dk_bs, d->dk_ts, d->dk_hs, es) &&
                    strides_ok(d->dv_bs, d->dv_ts, d->dv_hs, es), "tdx_window_attention_bwd: strides must be multiples of 16 bytes and not negative");
  TDX_CHECK_ARG((65 * d->dout_ts + a.G * d->dout_hs) * es < (1ll << 31), "tdx_window_attention_bwd: the strides of dout are too large");
  const BwdPlan p = plan_backward(a, es);
  TDX_CHECK_ARG(pointer_ok(d->ws) && d->ws_bytes >= p.bytes(), "tdx_window_attention_bwd: workspace of %lld bytes needed, got %lld",
                (long long)p.bytes(), (long long)d->ws_bytes);
  TDX_CHECK_ARG((long)a.B * a.Hkv * std::max<long>((long)a.Tq * a.G, a.Tk) < 0x7fffffffL && p.threads <= kMostThreads, "tdx_window_attention_bwd: too many rows");
  a.dout = d->dout, a.dq = d->dq, a.dk = d->dk, a.dv = d->dv;
  a.do_bs = d->dout_bs, a.do_ts = d->dout_ts, a.do_hs = d->dout_hs, a.dq_bs = d->dq_bs, a.dq_ts = d->dq_ts, a.dq_hs = d->dq_hs;
  a.dk_bs = d->dk_bs, a.dk_ts = d->dk_ts, a.dk_hs = d->dk_hs, a.dv_bs = d->dv_bs, a.dv_ts = d->dv_ts, a.dv_hs = d->dv_hs;
  a.stat = (float*)d->ws, a.part = (float*)((char*)d->ws + p.stat_bytes), a.near = a.part + p.part_bytes / 4;
  return d->dtype == TDX_F32 ? launch_backward_d<float>(a, p, (hipStream_t)stream) : launch_backward_d<__bf16>(a, p, (hipStream_t)stream);
}
