// C[m, n] = epilogue(sum_k X(m, k) W(n, k)): the matrix product of the token blocks on the CDNA4 matrix pipe.
//
// A workgroup owns a BM x BN tile.  K is walked in steps of 128 bytes per row (64 elements of 16 bits, 32 of 32 bits); a step's
// two operand tiles are moved by LDS-DMA (buffer_load_dwordx4 ... lds: 16 bytes per lane, no registers in between) into a ring of 2
// to 4 LDS stages while earlier ones are multiplied.  Both memory orders of an operand are read as they lie:
//   K adjacent  LDS rows of 128 bytes, one per m (n); a lane's fragment is one ds_read_b128
//   K strided   LDS rows of BM (BN) elements, one per k; fragments by the transposing ds_read_b64_tr_b16 (16 bit) or
//               ds_read_b32 (32 bit)
// with the 16-byte pieces of a row permuted by the row index (the lanes of the DMA fetch permuted addresses: LDS-DMA writes lane
// after lane), so that the fragment reads of a wave spread over all banks.  Rows past M or N repeat the last one (not stored),
// pieces past K are out of the buffer descriptor's range and arrive as zeros; the piece that
// an adjacent K, or the last of strided k rows, ends in comes through registers.
//
// The product is taken as W X^T per wave (MFMA rows = n, columns = m): a lane then holds 4 adjacent n of one m.  Results pass
// through LDS once more (32 rows of f32 per wave) so that every lane stores 8 adjacent columns, with bias, activation,
// dropout words (two Philox calls for 8 columns), residual and the one rounding on the way.
#include <type_traits>

#include "token_common.h"

using namespace token;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

struct TileArgs {
  const char* x; const char* w;
  int64_t ld_x, ld_w;            // bytes
  int64_t M, N;
  int64_t K;
  int nk;                        // K steps
  int ntm, ntn, nsplit;
  float* part; int64_t ld_part;  // nsplit > 1: slab s of raw sums at part + s * M * ld_part
  Epilogue e;
};

// The matrix instructions by type and size MF (32 x 32 or 16 x 16 results, 16 or 4 per lane): one takes 16 bytes per lane of either
// operand, row lane % MF, bytes 16 (lane / MF) .. of a group of 1024 / MF bytes along k (32-bit types: four instructions, j)
template <typename T, int MF> struct Mma;
#define MMA(T, MF, RES, CALL)                                                     \
  template <> struct Mma<T, MF> {                                                 \
    typedef T v8 __attribute__((ext_vector_type(8)));                             \
    typedef RES acc;                                                              \
    static __device__ __forceinline__ acc mma1(u32x4 a, u32x4 b, int, acc c) {    \
      return CALL(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0); \
    }                                                                             \
  }
MMA(bf16, 32, f32x16, __builtin_amdgcn_mfma_f32_32x32x16_bf16);
MMA(f16, 32, f32x16, __builtin_amdgcn_mfma_f32_32x32x16_f16);
MMA(bf16, 16, f32x4, __builtin_amdgcn_mfma_f32_16x16x32_bf16);
MMA(f16, 16, f32x4, __builtin_amdgcn_mfma_f32_16x16x32_f16);
#undef MMA
template <> struct Mma<float, 32> {
  typedef f32x16 acc;
  static __device__ __forceinline__ acc mma1(u32x4 a, u32x4 b, int j, acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
  }
};
template <> struct Mma<float, 16> {
  typedef f32x4 acc;
  static __device__ __forceinline__ acc mma1(u32x4 a, u32x4 b, int j, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
  }
};

// 16 bytes per lane from buffer `srd` + voff into LDS at `lds` (wave-uniform) + lane * 16.  The wait for the data is the caller's
// (barrier_all): no register is written, so the compiler has nothing to track.  Nor does it keep the distances in front of the fetch, as it
// sees none in this block: 1 wait state after m0 is here, and of the 5 between a vector instruction that writes a scalar register and the
// vector memory instruction that uses it none is needed, for open() makes the descriptor by scalar instructions.  (Waits instead, in this
// block or after open(): 512 x 4096 x 1024 bf16 17.7 -> 18.2 or 18.6 us.)  The tests count both in the built library.
__device__ __forceinline__ void dma16(uint32_t lds, uint32_t voff, i32x4 srd) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(srd) : "memory");      // m0 is reserved: the compiler sets it before any use of its own
#endif
}
// everything this wave has in flight has landed, then all waves of the workgroup have got here
__device__ __forceinline__ void barrier_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// the same, with the N latest fetches of this wave still on their way
template <int N> __device__ __forceinline__ void barrier_but() {
  static_assert(N >= 0 && N < 64, "the counter has 6 bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(lds_char*)p; }

constexpr uint32_t kOutside = 0x80000000u;      // = num_records: a lane with this offset reads zeros

// One operand's tile of R rows (m or n) per K step: how it is fetched and how its fragments are read.  A lane fetches 16 bytes at a
// time, from addresses that are multiples of 4.
template <typename T, int R, bool S, int NT, int MF>
struct Side {
  static constexpr int E = sizeof(T), KS = 128 / E, PASSES = R * 128 / (NT * 16);      // KS: k per step
  static constexpr int ROWB = S ? R * E : 128;                                        // bytes of an LDS row
  static_assert(R * 128 % (NT * 16) == 0 && NT % 128 == 0 && (S || R % MF == 0), "tile / threads");

  // Where 16-byte piece `chunk` of row `row` lies in LDS, and back.  64 banks of 4 bytes serve 256 bytes a cycle; the lanes of one
  // cycle read  adjacent: 16 rows at one chunk | strided, 16 bit: 4 k rows x 2 neighbouring pairs of chunks | strided, 32 bit: 2 (4) k
  // rows, 4 apart, x 8 (4) chunks.  These keys put them on different banks (a row of 128 bytes gives the first bit by itself).
  static __device__ __forceinline__ int key(int row) {
    if constexpr (!S) return (row >> 1) & 7;
    else if constexpr (E == 4) return MF == 32 ? ((row >> 2) & 1) << 3 : ((row >> 2) & 3) << 2;
    else return ROWB == 128 ? ((row >> 1) & 1) << 2 : (row & 3) << 1;
  }
  static constexpr bool FOLD = S && E == 2 && ROWB > 128;      // the pair's lowest bit also goes into bit 3
  static __device__ __forceinline__ int slot_of(int chunk, int row) { return chunk ^ key(row) ^ (FOLD ? (chunk & 2) << 2 : 0); }
  static __device__ __forceinline__ int chunk_of(int slot, int row) {
    const int c = slot ^ key(row);
    return FOLD ? c ^ (c & 2) << 2 : c;
  }

  const char* base;
  int64_t step;
  i32x4 srd;
  uint32_t voff[PASSES];    // buffer offset of this lane's piece in each pass
  int kpos;                 // and where along k the first one lies: adjacent, in bytes; strided, in rows

  int cut;                  // strided: bit i: the piece of pass i is the one that the k rows end in

  static constexpr int STEP = NT * 16 / ROWB;      // LDS rows from pass to pass
  static_assert(NT * 16 % ROWB == 0, "a pass takes whole rows");
  // the same for pass i: the keys of rows STEP apart are the same, or differ in one bit
  __device__ __forceinline__ int kpos_of(int i) const {
    if constexpr (S) return kpos + i * STEP;
    else return kpos ^ ((key(STEP) * i & 7) << 4);
  }
  __device__ __forceinline__ void init(const char* p, int64_t ld_, int64_t r0, int64_t rows, int kstep0) {
    const uint32_t ld = (uint32_t)ld_;
    int inner;                // strided: bytes of a k row from r0 on;  adjacent: the last row of the tile that exists
    if constexpr (!S) {
      base = p + r0 * ld_ + (int64_t)kstep0 * 128;
      step = 128;
      inner = rows - 1 - r0 < R ? (int)(rows - 1 - r0) : R;
    } else {
      base = p + r0 * E + (int64_t)kstep0 * KS * ld_;
      step = (int64_t)KS * ld_;
      inner = (rows - r0) * E < R * E ? (int)(rows - r0) * E : R * E;
    }
    // in scalar registers from here on: each step's descriptor is made by scalar instructions (dma16)
    base = (const char*)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)((uint64_t)base >> 32)) << 32) |
                         (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint64_t)base));
    const int at = threadIdx.x * 16, row0 = at / ROWB, slot = at % ROWB >> 4;
    kpos = S ? row0 : chunk_of(slot, row0) * 16;
    cut = 0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int row = row0 + i * STEP, b = chunk_of(slot, row) * 16;
      if constexpr (!S) voff[i] = (uint32_t)(row < inner ? row : inner) * ld + b;
      else {
        voff[i] = b < inner ? row * ld + b : kOutside;
        if (b < inner && b + 16 > inner) cut |= 1 << i;
      }
    }
  }
  // the next step's tile: open, then one piece after the other into LDS at `lds`; left: what of K there is from the step's start on, in
  // bytes (adjacent) or rows (strided), 0 or less: nothing.  A piece that is not whole is left out; not so a strided one, whose
  // other end lies in the next k row and falls to columns that are not stored -- but there is none after the last row.
  __device__ __forceinline__ void open() {
    const uint64_t b = (uint64_t)base;
    srd[0] = (int)(uint32_t)b;
    srd[1] = (int)(uint32_t)(b >> 32) & 0xffff;
    srd[2] = (int)kOutside;
    srd[3] = 0x00027000;
    base += step;
  }
  __device__ __forceinline__ void piece(int i, uint32_t lds, int left) {
    bool in;
    if constexpr (S) in = kpos_of(i) < left - (cut >> i & 1);
    else in = kpos_of(i) + 16 <= left;
    dma16(lds + i * NT * 16, in ? voff[i] : kOutside, srd);
  }
  // fragment of the MF rows from r on, k group kk, for Mma<T, MF>
  static __device__ __forceinline__ u32x4 frag(const char* tile, int r, int kk) {
    const int lane = threadIdx.x & 63, rl = lane % MF, kl = lane / MF;
    u32x4 v = {};
    if constexpr (!S) {
      v = *(const u32x4*)(tile + (r + rl) * ROWB + (slot_of(kk * (64 / MF) + kl, rl) << 4));
    } else if constexpr (E == 2) {
#if defined(__HIP_DEVICE_COMPILE__)
      // 16 lanes hand in 4 k rows x 16 elements and get 4 k of one element each
      const int i = lane & 15, half = MF == 32 ? (lane >> 4) & 1 : 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int krow = kk * (512 / MF) + kl * 8 + h * 4 + (i >> 2), chunk = (r >> 3) + half * 2 + ((i & 3) >> 1);
        const char* p = tile + krow * ROWB + (slot_of(chunk, krow) << 4) + (i & 1) * 8;
        const s16x4 q = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
        const unsigned long long u = __builtin_bit_cast(unsigned long long, q);
        v[2 * h] = (unsigned)u;
        v[2 * h + 1] = (unsigned)(u >> 32);
      }
#endif
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int krow = kk * (256 / MF) + kl * 4 + j, c = r + rl;
        v[j] = *(const uint32_t*)(tile + krow * ROWB + (slot_of(c >> 2, krow) << 4) + (c & 3) * 4);
      }
    }
    return v;
  }
};

// Bound by the matrix pipe where K and the tiles are many.  8192 x 16384 x 4096 bf16, gelu, pre: 988 us = 1110 TFLOP/s, where a library
// product alone takes 833; both run into the power limit there (on zeros this one reaches 1430).  Tiles by cost (kTile below): 2 x 4
// results of 32 x 32 a wave read 6 fragments for 8 products, 1 x 2 read 3 for 2.  128 bytes of K a step: 64-byte steps in a deeper ring
// were slower throughout, a 256 x 256 tile as 4 waves of 4 x 4 too.  Two waves per
// SIMD are asked for so that the sums stay in ordinary registers: as accumulation registers they cost a move each at the end.
// 8192 x 2048 x 8192 (bf16) with X adjacent and W strided: 225 us, both strided: 229 (1220, 1200 TFLOP/s; library 208).
// 2048 x 2048 x 8192 with residual and dropout: 79 us = 875 TFLOP/s, 256 workgroups of 128 x 128, one each: its start and end lie
// bare.  f32 1537 x 777 x 1001: 34 us + join 6, one wave of tiles with the pipe at half its rate.
template <typename T, int MF, int TM, int TN, int WM, int WN, int NS, bool XS, bool WS>
__global__ __launch_bounds__(WM * WN * 64, 2) void token_tile_kernel(const TileArgs a) {
  constexpr int NT = WM * WN * 64, BM = WM * TM * MF, BN = WN * TN * MF, STAGE = (BM + BN) * 128;
  constexpr int PITCH = TN * MF + 4;
  typedef Side<T, BM, XS, NT, MF> X;
  typedef Side<T, BN, WS, NT, MF> W;
  typedef Mma<T, MF> I;
  extern __shared__ __attribute__((aligned(16))) char smem[];

  // Blocks go to the 8 XCDs in turn; each XCD gets a contiguous run of tiles, walked in bands of 8 tile rows: the ~32 tiles that
  // are in flight on it form a patch whose operand rows its L2 holds
  const int tiles = a.ntm * a.ntn, nb = tiles * a.nsplit;
  const int xcd = blockIdx.x & 7, q = nb >> 3, rem = nb & 7;
  const int t = xcd * q + (xcd < rem ? xcd : rem) + (blockIdx.x >> 3);
  const int z = t / tiles, tile = t - z * tiles;
  const int band = tile / (8 * a.ntn), in = tile - band * 8 * a.ntn, bm = a.ntm - band * 8 < 8 ? a.ntm - band * 8 : 8;
  const int64_t m0 = (int64_t)(band * 8 + in % bm) * BM, n0 = (int64_t)(in / bm) * BN;
  const int k0 = (int)((int64_t)a.nk * z / a.nsplit), k1 = (int)((int64_t)a.nk * (z + 1) / a.nsplit);

  X sx;
  W sw;
  sx.init(a.x, a.ld_x, m0, a.M, k0);
  sw.init(a.w, a.ld_w, n0, a.N, k0);
  const uint32_t l0 = __builtin_amdgcn_readfirstlane(lds_addr(smem) + (threadIdx.x & ~63u) * 16);      // this wave's lanes in each pass
  const int64_t k_end = (int64_t)k1 * X::KS < a.K ? (int64_t)k1 * X::KS : a.K;
  int64_t k_left = k_end - (int64_t)k0 * X::KS;
  // one of the PX + PW pieces of the next step's tiles
  constexpr int PX = X::PASSES, PW = W::PASSES;
  auto open = [&]() { sx.open(); sw.open(); };
  auto piece = [&](int i, int stage) {
    const int left = k_left < 65536 ? (int)k_left : 65536;
    if (i < PX) sx.piece(i, l0 + stage * STAGE, XS ? left : left * (int)sizeof(T));
    else sw.piece(i - PX, l0 + stage * STAGE + BM * 128, WS ? left : left * (int)sizeof(T));
  };
  const int wave = threadIdx.x >> 6, wm = (wave % WM) * TM * MF, wn = (wave / WM) * TN * MF;
  // NJ instructions per pair of fragments, each over all pairs before the next: an instruction that adds to what the last one left
  // waits for it.  A single pair has two sums in turn.
  constexpr int NM = TM * TN, NJ = sizeof(T) == 4 ? 4 : 1, ND = NM == 1 && NJ > 1 ? 2 : 1;
  typename I::acc acc[TM][TN][ND] = {};
  u32x4 fx[2][TM], fw[2][TN];
  auto read = [&](int set, int stage, int kk, int f) {      // fragment f of the TM + TN
    const char* s = smem + stage * STAGE;
    if (f < TM) fx[set][f] = X::frag(s, wm + f * MF, kk);
    else fw[set][f - TM] = W::frag(s + BM * 128, wn + (f - TM) * MF, kk);
  };
  // one k group of a step: the products of the fragments in `set`, between them one by one the reads of the next ones and the fetches
  // f0 .. f1 into stage fstage.  The compiler would sink the reads to their use; the order is kept.
  auto group = [&](int set, int rstage, int rkk, int f0, int f1, int fstage) {
    constexpr int NF = TM + TN, RP = (NF + NM * NJ - 1) / (NM * NJ);
#pragma unroll
    for (int q = 0; q < NM * NJ; ++q) {
#pragma unroll
      for (int f = q * RP; f < (q + 1) * RP; ++f)
        if (f < NF) read(set ^ 1, rstage, rkk, f);
#pragma unroll
      for (int f = f0; f < f1; ++f)
        if ((f - f0) * NM * NJ / (f1 - f0) == q) piece(f, fstage);
      const int i = q % NM % TM, j = q % NM / TM;
      acc[i][j][q / NM % ND] = I::mma1(fw[set][j], fx[set][i], q / NM, acc[i][j][q / NM % ND]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // NS stages in a ring, NG k groups a step.  The last group of a step is multiplied after the barrier that ends it: its fragments are
  // in registers, the reads of the next stage's first group, which only now may start, pass under those products, and so do the
  // fetches of the step NS further on, into the stage that has just been read.  With two stages they are made at once, for
  // they have less than a step to arrive; with more they are spread over the next NG groups.  The barrier waits for the next
  // stage's fetches alone; those of the NS - 2 stages after it stay on their way.  What is read or fetched past the last step is
  // not used (fetches out of range leave zeros).
  constexpr int P = PX + PW, NG = MF / 8, Q = NS == 2 ? P : (P + NG - 1) / NG;      // fetches in a group
  constexpr auto upto = [](int g) { return g * Q < P ? g * Q : P; };
  // What the fetches leave out comes element by element through registers, before the last step's fragments are read.  K adjacent: the
  // piece that each row ends in, a row per lane, zeros past K.  K strided: the piece that the last k row of the range ends in.
  static_assert(NT >= BM + BN, "a row per lane");
  constexpr int V = 16 / (int)sizeof(T);
  const int row = threadIdx.x, odd = (int)(a.K % V);
  const bool ends = !(XS && WS) && odd != 0 && k1 == a.nk;
  const bool cut_x = XS && a.M - m0 < BM && (a.M - m0) % V != 0, cut_w = WS && a.N - n0 < BN && (a.N - n0) % V != 0;
  const bool ragged = ends || cut_x || cut_w;
  u32x4 tail = {0, 0, 0, 0};
  char* tail_to = nullptr;
  if (ragged) {
    const T* from = nullptr;
    int count = 0;
    const bool in_x = row < BM;
    const int r = in_x ? row : row - BM;
    if (in_x ? XS : WS) {
      if (r == 0 && (in_x ? cut_x : cut_w)) {
        const int64_t left = in_x ? a.M - m0 : a.N - n0, first = left / V * V;
        count = (int)(left - first);
        from = (const T*)((in_x ? a.x : a.w) + (k_end - 1) * (in_x ? a.ld_x : a.ld_w)) + (in_x ? m0 : n0) + first;
        const int krow = (int)((k_end - 1) % X::KS), chunk = (int)(first / V);
        if constexpr (XS) { if (in_x) tail_to = smem + krow * X::ROWB + (X::slot_of(chunk, krow) << 4); }
        if constexpr (WS) { if (!in_x) tail_to = smem + BM * 128 + krow * W::ROWB + (W::slot_of(chunk, krow) << 4); }
      }
    } else if (ends && row < BM + BN) {
      count = odd;
      const int64_t at = in_x ? (m0 + r < a.M ? m0 + r : a.M - 1) * a.ld_x : (n0 + r < a.N ? n0 + r : a.N - 1) * a.ld_w;
      from = (const T*)((in_x ? a.x : a.w) + at) + (a.K - odd);
      const int chunk = (int)((a.K - odd) * (int64_t)sizeof(T) % 128) >> 4;
      if constexpr (!XS) { if (in_x) tail_to = smem + r * 128 + (X::slot_of(chunk, r) << 4); }
      if constexpr (!WS) { if (!in_x) tail_to = smem + BM * 128 + r * 128 + (W::slot_of(chunk, r) << 4); }
    }
    if (count > 0) {
      T v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = j < count ? from[j] : (T)0.f;
      __builtin_memcpy(&tail, v, 16);
    }
  }
  auto add_tail = [&](int stage) {
    if (tail_to) *(u32x4*)(tail_to + stage * STAGE) = tail;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  if (k1 > k0) {
#pragma unroll 1
    for (int st = 0; st < NS - 1; ++st) {
      open();
#pragma unroll
      for (int f = 0; f < P; ++f) piece(f, st);
      k_left -= X::KS;
    }
    open();
#pragma unroll
    for (int f = 0; f < Q; ++f) piece(f, NS - 1);
    barrier_but<(NS - 2) * P + Q>();
    if (ragged && k1 - k0 == 1) add_tail(0);
#pragma unroll
    for (int f = 0; f < TM + TN; ++f) read(0, 0, 0, f);
    int stage = 0, prev = NS - 1;
#pragma unroll 1
    for (int k = k0; k < k1; ++k) {
      const int next = stage + 1 == NS ? 0 : stage + 1;
#pragma unroll
      for (int g = 0; g < NG - 1; ++g) group(g & 1, stage, g + 1, upto(g + 1), upto(g + 2), prev);
      barrier_but<(NS - 2) * P>();
      if (ragged && k == k1 - 2) add_tail(next);
      k_left -= X::KS;
      open();
      group((NG - 1) & 1, next, 0, 0, upto(1), stage);
      prev = stage;
      stage = next;
    }
    barrier_all();
  }

  if constexpr (ND == 2) acc[0][0][0] += acc[0][0][ND - 1];

  // this wave's results, MF rows at a time, through LDS to lanes of neighbouring columns
  float* sh = (float*)smem + wave * (MF * PITCH);
  const int lane = threadIdx.x & 63;
  uint64_t seed = 0, offset = 0;
  if (a.e.drop.on) drop_key(a.e.drop, seed, offset);
  constexpr int COLS = TN * MF, LPR = COLS / 8, RPP = 64 / LPR;      // lanes per row of 8-column pieces, rows per pass
  static_assert(MF % RPP == 0 && MF * COLS % 512 == 0, "whole passes");
  // the largest tile is for results of 16 M elements and more, which would only push operands out of L2: 990 -> 975 us for
  // 8192 x 4096 x 16384 with pre
  constexpr bool ONCE = BM * BN == 65536;
  const int64_t np = n0 + wn + (lane % LPR) * 8;
  float b8[8] = {};
  if (a.e.vec && np < a.N) bias8<T>(a.e, np, b8);
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int c = 0; c < MF * MF / 256; ++c)
        *(f32x4*)(sh + (lane % MF) * PITCH + j * MF + c * 8 + (lane / MF) * 4) =
            f32x4{acc[i][j][0][c * 4], acc[i][j][0][c * 4 + 1], acc[i][j][0][c * 4 + 2], acc[i][j][0][c * 4 + 3]};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // the rows below are other lanes' writes of this wave
    const int64_t mi = m0 + wm + i * MF;
    if (a.nsplit > 1) {
      float* to = a.part + ((int64_t)z * a.M + mi) * a.ld_part + np;
#pragma unroll 1
      for (int r = lane / LPR; r < MF; r += RPP) {
        float v[8];
        load8(sh + r * PITCH + (lane % LPR) * 8, v);
        if (mi + r < a.M && np < a.N) store8(to + r * a.ld_part, v);
      }
    } else if (a.e.vec) {
      Raw8<T> res = {}, next = {};      // the next row's residual is on its way while this row is worked on
      int r = lane / LPR;
      if (mi + r < a.M && np < a.N) res = residual8<T>(a.e, mi + r, np);
#pragma unroll 1
      for (; r < MF; r += RPP) {
        if (r + RPP < MF && mi + r + RPP < a.M && np < a.N) next = residual8<T>(a.e, mi + r + RPP, np);
        float v[8];
        load8(sh + r * PITCH + (lane % LPR) * 8, v);
        if (mi + r < a.M && np < a.N) epilogue8<T, ONCE>(a.e, seed, offset, mi + r, np, v, b8, res);
        res = next;
      }
    } else {
#pragma unroll 1
      for (int r0 = 0; r0 < MF * COLS / 64; r0 += 8) {
        int64_t m[8], n[8];
        float u[8];
        unsigned live = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int at = (r0 + q) * 64 + lane;
          m[q] = mi + at / COLS;
          n[q] = n0 + wn + at % COLS;
          if (m[q] < a.M && n[q] < a.N) live |= 1u << q;
          u[q] = sh[at / COLS * PITCH + at % COLS];
        }
        epilogue1<T, 8>(a.e, seed, offset, m, n, live, u);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ---- few rows of X (tokens of as many sequences): the weight's rows are read once, straight into fragments ------------------
// A workgroup of 8 waves owns 16 columns n, or 8 as long as that is one round of workgroups over the CUs, up to N = 2048 (1 x 8192 x 2048
// bf16: 9.3 us, with 16 columns 12.0; 16 rows 14.5 against 16.9).  Past it a second round costs more than the CUs that 16 columns leave
// idle: N = 2056, 16 columns 12.5 us, 8 columns 16.1; 16 rows 19.6 against 26.1; N = 4088 17.3 against 20.2.  The waves share out K in pieces of 128 bytes per row of w, so that a wave reads whole
// lines; MFMA rows = the 16 columns, MFMA columns = 16 rows of X (MB of them).  Any order of k inside a piece serves, as both
// operands take the same: lane (r, q) takes bytes q * 16 .. of each 64.  The waves' sums meet in LDS.
// Bound by the weight's bytes and, when small, by latency: one row of 4096 x 4096 bf16 (34 MB) 8.2 us = 4.1 TB/s, 12 rows of
// 10240 x 2560 f16 (52 MB) 15 us = 3.5 TB/s.  Up to 4 pieces in flight a wave, as the registers
// allow (2 or 6: 8.9 us), through the caches (past them: 9.0, 12 rows 20.6).
struct FewArgs {
  const char* x; const char* w;
  int64_t ld_x, ld_w;            // bytes
  int64_t M, N;
  int kb;                        // bytes of a row
  Epilogue e;
};

// How rows lie: every 16-byte piece aligned and whole | starts at multiples of 4 bytes | at any element (16-bit types).  Pieces
// that start inside a word are put together from the five words that hold them: one row of 4096 x 4096, stride 4097, 13.9 us, against 17.1
// with loads that straddle words (8.3 for stride 4098, 7.9 for 4096).
enum { kPieces, kWords, kElements };
// a whole piece
template <int ROWS>
__device__ __forceinline__ u32x4 row_piece(const char* p) {
  typedef u32x4 __attribute__((aligned(4))) words;
  if constexpr (ROWS == kPieces) return *(const u32x4*)p;
  if constexpr (ROWS == kWords) return *(const words*)p;
  const uint32_t odd = (uint32_t)(uintptr_t)p & 2;
  p -= odd;
  u32x4 v = *(const words*)p;
  const uint32_t last = *(const uint32_t*)(p + (odd ? 16 : 12));      // no word that holds nothing of the row is touched
#pragma unroll
  for (int j = 0; j < 3; ++j) v[j] = __builtin_amdgcn_alignbyte(v[j + 1], v[j], odd);
  v[3] = __builtin_amdgcn_alignbyte(last, v[3], odd);
  return v;
}
// the piece that a row ends in: n bytes, zeros behind.  No branches: the loads leave together.
template <typename T>
__device__ __forceinline__ u32x4 row_end(const char* p, int n) {
  constexpr int E = sizeof(T);
  typedef typename std::conditional<E == 4, uint32_t, uint16_t>::type U;
  u32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 16 / E; ++j) {
    const uint32_t u = *(const U*)(p + (E * j < n ? E * j : 0));
    v[j * E / 4] |= E * j < n ? u << (E * j % 4 * 8) : 0u;
  }
  return v;
}

template <typename T, int MB, int ROWS, int COLS>
__global__ __launch_bounds__(512, 1) void token_few_kernel(const FewArgs a) {
  __shared__ __attribute__((aligned(16))) float sh[8][MB * 16][20];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * COLS;
  const char* xrow[MB];
  const char* wrow = a.w + (n0 + r < a.N ? n0 + r : a.N - 1) * a.ld_w;
#pragma unroll
  for (int i = 0; i < MB; ++i) xrow[i] = a.x + (i * 16 + r < a.M ? i * 16 + r : a.M - 1) * a.ld_x;
  // what the last lines need besides the sums is fetched under them
  const int mo = threadIdx.x >> 1;
  const int64_t no = n0 + (threadIdx.x & 1) * 8;
  float b8[8] = {};
  Raw8<T> res = {};
  if (a.e.vec && mo < a.M && (threadIdx.x & 1) * 8 < COLS && no < a.N) {
    bias8<T>(a.e, no, b8);
    res = residual8<T>(a.e, mo, no);
  }
  f32x4 acc[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int U = MB == 1 ? 4 : MB == 2 || ROWS != kElements ? 2 : 1;      // pieces in flight
  const int whole = ROWS == kPieces ? a.kb : a.kb & ~15;
  // where rows end inside a piece, the last wave, which has the least to do, takes it by itself
  const bool ends = ROWS != kPieces && wave == 7 && whole < a.kb;
  u32x4 ew = {0, 0, 0, 0}, ex[MB] = {};
  if constexpr (ROWS != kPieces) {
    if (ends && q == 0) {
      ew = row_end<T>(wrow + whole, a.kb - whole);
#pragma unroll
      for (int i = 0; i < MB; ++i) ex[i] = row_end<T>(xrow[i] + whole, a.kb - whole);
    }
  }
  for (int b0 = wave * 128; b0 < whole; b0 += 1024 * U) {
    u32x4 fw[U][2], fx[U][2][MB];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int b = b0 + u * 1024 + h * 64 + q * 16;
        fw[u][h] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < MB; ++i) fx[u][h][i] = u32x4{0, 0, 0, 0};
        if (b < whole) {
          if (r < COLS) fw[u][h] = row_piece<ROWS>(wrow + b);      // 8 columns: the other lanes fetch nothing
#pragma unroll
          for (int i = 0; i < MB; ++i) fx[u][h][i] = row_piece<ROWS>(xrow[i] + b);
        }
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < (sizeof(T) == 4 ? 4 : 1); ++j)
#pragma unroll
          for (int i = 0; i < MB; ++i) acc[i] = Mma<T, 16>::mma1(fw[u][h], fx[u][h][i], j, acc[i]);
  }
  if constexpr (ROWS != kPieces) {
    if (ends) {
#pragma unroll
      for (int j = 0; j < (sizeof(T) == 4 ? 4 : 1); ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i) acc[i] = Mma<T, 16>::mma1(ew, ex[i], j, acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) *(f32x4*)&sh[wave][i * 16 + r][q * 4] = acc[i];
  __syncthreads();
  uint64_t seed = 0, offset = 0;
  if (a.e.drop.on) drop_key(a.e.drop, seed, offset);
  if (a.e.vec) {
    const int m = threadIdx.x >> 1, c = (threadIdx.x & 1) * 8;
    if (m >= a.M || c >= COLS || n0 + c >= a.N) return;
    float v[8], u[8];
    load8(&sh[0][m][c], v);
#pragma unroll
    for (int s = 1; s < 8; ++s) {
      load8(&sh[s][m][c], u);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += u[j];
    }
    epilogue8<T>(a.e, seed, offset, m, n0 + c, v, b8, res);
  } else {
    for (int i = threadIdx.x; i < MB * 256; i += 512) {
      const int64_t m = i >> 4, n = n0 + (i & 15);
      if (m >= a.M || (i & 15) >= COLS || n >= a.N) continue;
      float v = sh[0][m][i & 15];
#pragma unroll
      for (int s = 1; s < 8; ++s) v += sh[s][m][i & 15];
      epilogue1<T, 1>(a.e, seed, offset, &m, &n, 1, &v);
    }
  }
}

// out = epilogue(sum of the slabs, in their order): 8 columns per lane, or one where the rows' pieces are not whole.  Bound by the
// slabs' way in from L2: 2 of 1537 x 777 with residual (15 MB) 5.5 us.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void token_join_kernel(const float* __restrict__ part, int nsplit, int64_t M, int64_t ld_part, const Epilogue e) {
  uint64_t seed = 0, offset = 0;
  if (e.drop.on) drop_key(e.drop, seed, offset);
  const int64_t per = VEC ? ld_part / 8 : e.cols, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= M * per) return;
  const int64_t m = i / per, n = (i - m * per) * (VEC ? 8 : 1);
  const float* p = part + m * ld_part + n;
  if constexpr (VEC) {
    float v[8], u[8];
    float b[8];
    bias8<T>(e, n, b);
    const Raw8<T> res = residual8<T>(e, m, n);
    load8(p, v);
    for (int s = 1; s < nsplit; ++s) {
      load8(p + s * M * ld_part, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += u[j];
    }
    epilogue8<T>(e, seed, offset, m, n, v, b, res);
  } else {
    float v = *p;
    for (int s = 1; s < nsplit; ++s) v += p[s * M * ld_part];
    epilogue1<T, 1>(e, seed, offset, &m, &n, 1, &v);
  }
}

// dst [rows][cols_pad] = src [rows][cols], zeros behind: an operand that the tiles cannot fetch as it lies.
// Bound by latency at the sizes it is met at: 160 x 7376 bf16, odd rows, 2.9 us
template <typename U>
__global__ __launch_bounds__(256) void token_pack_kernel(const U* __restrict__ src, int64_t ld, U* __restrict__ dst, int64_t rows, int cols, int cols_pad) {
  constexpr int V = 16 / sizeof(U);
  typedef U v16 __attribute__((ext_vector_type(V)));
  const int per = cols_pad / V;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * V;
    v16 v;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = c + j < cols ? src[r * ld + c + j] : (U)0;
    *(v16*)(dst + r * cols_pad + c) = v;
  }
}

#define LAUNCHED() do { if (hipGetLastError() != hipSuccess) return SGA_ERR_HIP; } while (0)

// How a product is run
struct Plan {
  int few;                   // 16-row blocks of token_few_kernel, 0: tiles
  int tile;                  // index into the tile table; -1: too many tiles for a launch
  int nsplit;
  bool pack_x, pack_w;
  int64_t ldp_x, ldp_w;      // elements, packed
  int64_t x_off, w_off, part_off, bytes, ld_part;
};

// whether an operand has to be copied first: its rows do not all start at multiples of 4 bytes, or a tile's rows span more than the 2 GiB
// that an offset of the buffer descriptor does, or the k rows lie so close that the 16 bytes a row ends in may reach past the last one
bool needs_pack(const Operand& o, int64_t rows, int E) {
  if ((o.strided ? 128 / E : 256) * o.ld * E >= (1ll << 31) - 65536) return true;
  if (o.strided && o.ld * E < 16 && rows * E % 16) return true;
  return (((uint64_t)(uintptr_t)o.p | (uint64_t)(o.ld * E)) & 3) != 0;
}

// The tiles and what they cost, measured over 20 shapes from 32 x 4096 x 4096 to 8192 x 16384 x 4096 (128 to 8192 workgroups, K splits 1
// to 8; the plan found is within 6 % of the fastest there): ns of a K step of a workgroup with 1 and with 2 of them on its CU (as
// many as the LDS holds), 16- and 32-bit types, and of the rest of a tile's life.
struct Tile {
  int m, n, per_cu;
  double step[2][2], once;
  constexpr int lanes() const { return m * n > 8192 ? 512 : 256; }      // of a workgroup (run_tile_of)
};
constexpr int64_t kMaxLanes = 0xffffffff;      // of a launch: the grid is counted in lanes, in 32 bits, and one past that starts over at 0
constexpr int kTiles = 5;
const Tile kTile[kTiles] = {{256, 256, 1, {{1600, 0}, {7350, 0}}, 9000},
                            {256, 128, 1, {{930, 0}, {3800, 0}}, 5000},
                            {128, 128, 1, {{560, 0}, {1960, 0}}, 3500},
                            {96, 64, 2, {{300, 470}, {880, 1500}}, 3000},
                            {64, 64, 2, {{270, 410}, {620, 1090}}, 2500}};
constexpr int kCUs = 256;

Plan make_plan(const Product& p) {
  const int E = (int)dtype_bytes(p.dtype), V = 16 / E;
  Plan o = {};
  // token_few_kernel reads X again for every 8 or 16 columns, the tiles in whole tile rows: at 16 rows and 4096 x 4096 weights (bf16) 11.0 us
  // against 14.7, at 32 rows 13.9 against 12.7; up to 64 rows where there is little to read at all (1024 x 1024: 7.0 against 8.3) and
  // rows are short (48 rows, 160 x 7376, odd rows: 66 us, as its 10 workgroups go along K alone; the tiles, which split K, 16)
  if (!p.x.strided && !p.w.strided && (p.M <= 16 || (p.M <= 64 && p.K * E <= 4096 && p.M * p.N * p.K <= 1 << 26))) {
    o.few = p.M <= 16 ? 1 : p.M <= 32 ? 2 : 4;
    return o;
  }
  o.pack_x = needs_pack(p.x, p.M, E);
  o.pack_w = needs_pack(p.w, p.N, E);
  if (o.pack_x) { o.ldp_x = round_up(p.x.strided ? p.M : p.K, V); o.x_off = o.bytes; o.bytes += round_up((p.x.strided ? p.K : p.M) * o.ldp_x * E, 256); }
  if (o.pack_w) { o.ldp_w = round_up(p.w.strided ? p.N : p.K, V); o.w_off = o.bytes; o.bytes += round_up((p.w.strided ? p.K : p.N) * o.ldp_w * E, 256); }
  const int64_t nk = ceil_div(p.K, 128 / E);
  // rows off the 16-byte grid cost a lone workgroup a fifth more per step (two on a CU cover it for each other); results that leave
  // element by element, 4 us more at the end of a tile, which the join's many small workgroups do not feel
  const bool off = (((uint64_t)(uintptr_t)p.x.p | (uint64_t)(p.x.ld * E) | (uint64_t)(uintptr_t)p.w.p | (uint64_t)(p.w.ld * E)) & 15) != 0;
  double best = 1e300;
  o.tile = -1;
  o.nsplit = 1;
  for (int t = 0; t < kTiles; ++t) {
    if (kTile[t].m == 96 && p.x.strided) continue;      // the keys of a k row need a power of two
    const int64_t tiles = ceil_div(p.M, kTile[t].m) * ceil_div(p.N, kTile[t].n);
    const Tile& c = kTile[t];
    const double* step = c.step[E == 4];
    for (int s = 1; s == 1 || (s <= 16 && s <= nk); ++s) {
      if (tiles * s * c.lanes() > kMaxLanes) continue;
      const int64_t at_once = (int64_t)kCUs * c.per_cu, rest = tiles * s % at_once;
      const double steps = (double)ceil_div(nk, s);
      double cost = (double)(tiles * s / at_once) * (steps * step[c.per_cu - 1] + c.once);
      if (rest) cost += steps * step[rest > kCUs] * (off && rest <= kCUs ? 1.2 : 1.0) + c.once;
      if (s == 1 && !p.e.vec) cost += 4000.0;
      if (s > 1) cost += 3000.0 + (double)p.M * p.N * (s * 8.0 + E) / 4000.0;      // a launch, the slabs' way out and back at 4 TB/s
      if (cost < best) { best = cost; o.tile = t; o.nsplit = s; }
    }
  }
  if (o.nsplit > 1) { o.ld_part = round_up(p.N, 8); o.part_off = o.bytes; o.bytes += round_up(o.nsplit * p.M * o.ld_part * 4, 256); }
  return o;
}

template <typename T, int MF, int TM, int TN, int WM, int WN, int NS, bool XS, bool WS>
int run_tile(const TileArgs& a, hipStream_t st) {
  constexpr int BM = WM * TM * MF, BN = WN * TN * MF, MAIN = NS * (BM + BN) * 128, EPI = WM * WN * MF * (TN * MF + 4) * 4;
  static_assert(WM * WN * 64 == Tile{BM, BN}.lanes(), "the plan counts on it");
  constexpr int LDS = MAIN > EPI ? MAIN : EPI;
  const void* f = reinterpret_cast<const void*>(&token_tile_kernel<T, MF, TM, TN, WM, WN, NS, XS, WS>);
  if (LDS > 65536 && hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return SGA_ERR_HIP;
  hipLaunchKernelGGL((token_tile_kernel<T, MF, TM, TN, WM, WN, NS, XS, WS>), dim3((unsigned)(a.ntm * a.ntn * a.nsplit)), dim3(WM * WN * 64), LDS, st, a);
  LAUNCHED();
  return SGA_OK;
}
template <typename T, bool XS, bool WS>
int run_tile_of(int tile, const TileArgs& a, hipStream_t st) {
  switch (tile) {
    case 0: return run_tile<T, 32, 2, 4, 4, 2, 2, XS, WS>(a, st);
    case 1: return run_tile<T, 32, 2, 2, 4, 2, 3, XS, WS>(a, st);
    case 2: return run_tile<T, 32, 1, 2, 4, 2, 4, XS, WS>(a, st);
    case 3:
      if constexpr (!XS) return run_tile<T, 16, 3, 2, 2, 2, 4, XS, WS>(a, st);
      return SGA_ERR_UNSUPPORTED;      // 96 rows of a strided X: make_plan takes another tile
    default: return run_tile<T, 32, 1, 1, 2, 2, 4, XS, WS>(a, st);
  }
}
template <typename T>
int run_order(int tile, bool xs, bool ws, const TileArgs& a, hipStream_t st) {
  if (!xs && !ws) return run_tile_of<T, false, false>(tile, a, st);
  if (!xs) return run_tile_of<T, false, true>(tile, a, st);
  return run_tile_of<T, true, true>(tile, a, st);
}

template <typename T, int MB>
int run_few(const Product& p, hipStream_t st) {
  const int64_t E = sizeof(T);
  const FewArgs a = {(const char*)p.x.p, (const char*)p.w.p, p.x.ld * E, p.w.ld * E, p.M, p.N, (int)(p.K * E), p.e};
  const uint64_t rows = (uintptr_t)a.x | (uintptr_t)a.w | (uint64_t)a.ld_x | (uint64_t)a.ld_w;
  auto launch = [&](auto columns) {
    constexpr int COLS = decltype(columns)::value;
    const dim3 grid((unsigned)ceil_div(p.N, COLS));
    if (!((rows | (uint64_t)a.kb) & 15)) hipLaunchKernelGGL((token_few_kernel<T, MB, kPieces, COLS>), grid, dim3(512), 0, st, a);
    else if (sizeof(T) == 4 || !(rows & 3)) hipLaunchKernelGGL((token_few_kernel<T, MB, kWords, COLS>), grid, dim3(512), 0, st, a);
    else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((token_few_kernel<T, MB, kElements, COLS>), grid, dim3(512), 0, st, a);
  };
  if (p.N <= 8 * kCUs) launch(std::integral_constant<int, 8>());
  else launch(std::integral_constant<int, 16>());
  LAUNCHED();
  return SGA_OK;
}

template <typename T>
int run(const Product& p, char* ws, hipStream_t st) {
  const Plan o = make_plan(p);
  if (o.tile < 0) return SGA_ERR_UNSUPPORTED;
  if (o.few) return o.few == 1 ? run_few<T, 1>(p, st) : o.few == 2 ? run_few<T, 2>(p, st) : run_few<T, 4>(p, st);
  TileArgs a = {};
  typedef typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type U;
  auto side = [&](const Operand& op, int64_t rows, bool pack, int64_t ldp, int64_t off, const char*& q, int64_t& ld) -> int {
    q = (const char*)op.p;
    ld = op.ld * (int64_t)sizeof(T);
    if (!pack) return SGA_OK;
    const int64_t outer = op.strided ? p.K : rows, inner = op.strided ? rows : p.K;
    const int64_t blocks = ceil_div(outer * ldp / (16 / (int)sizeof(U)), 256);
    hipLaunchKernelGGL((token_pack_kernel<U>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, st, (const U*)op.p, op.ld, (U*)(ws + off),
                       outer, (int)inner, (int)ldp);
    LAUNCHED();
    q = ws + off;
    ld = ldp * (int64_t)sizeof(T);
    return SGA_OK;
  };
  int s = side(p.x, p.M, o.pack_x, o.ldp_x, o.x_off, a.x, a.ld_x);
  if (s == SGA_OK) s = side(p.w, p.N, o.pack_w, o.ldp_w, o.w_off, a.w, a.ld_w);
  if (s != SGA_OK) return s;
  a.M = p.M; a.N = p.N; a.K = p.K;
  a.nk = (int)ceil_div(p.K, 128 / (int)sizeof(T));
  a.ntm = (int)ceil_div(p.M, kTile[o.tile].m);
  a.ntn = (int)ceil_div(p.N, kTile[o.tile].n);
  a.nsplit = o.nsplit;
  a.part = o.nsplit > 1 ? (float*)(ws + o.part_off) : nullptr;
  a.ld_part = o.ld_part;
  a.e = p.e;
  s = run_order<T>(o.tile, p.x.strided, p.w.strided, a, st);
  if (s != SGA_OK || o.nsplit == 1) return s;
  if (p.e.vec)
    hipLaunchKernelGGL((token_join_kernel<T, true>), dim3((unsigned)ceil_div(p.M * (o.ld_part / 8), 256)), dim3(256), 0, st, a.part, o.nsplit, p.M, o.ld_part, p.e);
  else
    hipLaunchKernelGGL((token_join_kernel<T, false>), dim3((unsigned)ceil_div(p.M * p.N, 256)), dim3(256), 0, st, a.part, o.nsplit, p.M, o.ld_part, p.e);
  LAUNCHED();
  return SGA_OK;
}

}  // namespace

namespace token {

int64_t product_workspace(const Product& p) { return make_plan(p).bytes; }

int launch_product(const Product& p, char* ws, hipStream_t st) {
  return p.dtype == SGA_DTYPE_F32 ? run<float>(p, ws, st) : p.dtype == SGA_DTYPE_BF16 ? run<bf16>(p, ws, st) : run<f16>(p, ws, st);
}

}  // namespace token
