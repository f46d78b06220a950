// lm_gemm.hpp -- the matrix products of the linear cross entropy: one tile loop, three epilogues.
//
//   out[row][col] = sum_k R[row][k] C[col][k]
//
// Both operands are 16-bit floats in memory.  An operand is K-contiguous (KC: its rows run along k) or
// K-strided (KS: its rows run along row / col, one row for each k); a KS tile is transposed on its
// way out of LDS by ds_read_b64_tr_b16, so that no operand is ever transposed in HBM:
//   logits  z  = X W^T    R = X [t][h]  KC    C = W [v][h]  KC
//   grad    dX = g W      R = g [t][v]  KC    C = W [v][h]  KS
//   grad    dW = g^T X    R = g [t][v]  KS    C = X [t][h]  KS
// The C operand is the MFMA's A matrix: a lane then holds 4 consecutive output columns, and the
// softmax over columns reduces inside a lane.
//
// An operand of fp32 precision is two fp16 limbs of its values times a power of two that brings the
// largest under 2^15: x 2^s = hi + 2^-11 lo.  fp16 holds 11 bits down to 2^-14 and steps of 2^-24 below; the low
// limb is stored 2^11 up, so that it keeps its bits where hi has few left: x is off by 2^-22 of itself, or by
// 2^-50 of the largest where that is more (with lo as it is: 2^-39).  A product of two of them is a list of
// segments, hi lo + lo hi, then the accumulators times 2^-11, then hi hi (lo lo is below 2^-22), which the loop
// walks through as if k were three times as long, and a power of two undoes the scales.  bf16 operands are
// one segment of bf16.  Accumulation is fp32 in the MFMA.
//
// Tiles go to LDS by buffer_load_dwordx4 ... lds, NBUF - 1 to NBUF steps of 64 k ahead; rows and columns
// past the end get an offset past the descriptor's range, which loads zeros.  16-byte chunks are
// placed so that the reads of a wave spread over all banks: KC chunk c of row r at c ^ (r/2 % 8),
// KS 64-byte slot s of row k at s ^ (k%4 + 4 (k/8 % 2)).

// Rates (8192 x 4096 x 128256): logits with their softmax 1250-1340 TFLOP/s, dX 1280-1320, dW 1240, where the
// library's plain product of the size reaches 1250-1433 on the same cards.  All of them are bound by
// power: the matrix cores are busy 73 % of the cycles here and 84 % there, at 1.6 and 1.4 GHz.  A tile is 256 x 256
// by 8 waves of 64 x 128: 128 accumulators a lane leave room for two sets of fragments at two waves a SIMD,
// and a step's reads (192 KiB) and loads (64 KiB) take LDS less time than the MFMAs take.  4 waves of
// 128 x 128 read a third less and were 8 % slower on dX: alone on its SIMD, a wave cannot hide the barrier.

constexpr int kBK = 64;
constexpr int kMaxSeg = 3;
constexpr uint32_t kOob = 0x80000000u;  // == num_records: loads zeros

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

struct GemmArgs {
  const uint16_t* r[kMaxSeg];
  const uint16_t* c[kMaxSeg];
  int nseg;
  int64_t ldr, ldc;      // elements
  int cols;              // valid output columns (C rows when KC, C columns when KS)
  int k;                 // static k extent (k_dev: tokens)
  const int* n_valid;    // device: the number of tokens that take part
  int k_dev;             // k extent is *n_valid, else *n_valid bounds the rows
  int rows;              // valid output rows (k_dev) or allocated rows
  int row_tiles, col_tiles, splits;
  // epilogues
  const int* tgt;        // per compact token: column of its target within the shard, -1: none
  const float* lse;      // per compact token
  const float* gl;       // per compact token: upstream gradient
  const int* scale;      // device: the exponent of the power of two that undoes the operands' scales, NULL: 0
  int col0;              // first shard column of this piece
  float2* part;          // stats: [part][token] (c, sum of 2^(x log2(e) - c))
  float* tlogit;         // stats: per compact token
  int64_t ldpart;
  uint16_t* gb[2];       // g in bf16 and what that lacks in another, each or both NULL
  float* delta;          // per compact token: what the target's g lacks
  uint16_t* gh[2];       // g 2^(13 - e) in two fp16 limbs, 2^e the power of two below |gl|, or NULL: off by
                         // 2^-22 of itself or 2^-49 of |gl|
  int64_t ldg;
  float* slab;           // dX: [split][token][ldslab]
  int64_t ldslab, slab_stride;
  int add;               // dX: add to the slab; dW: accumulate
  void* out;             // dW
  int64_t ldo;
  int out_bf16, out_vec;
};

enum { EPI_STATS = 0, EPI_GRAD = 1, EPI_SLAB = 2, EPI_OUT = 3 };

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}

// lane l's 16 bytes at base + voff land at LDS byte lds + 16 l.  Completion is counted by hand
// (wait_barrier), which is why this is asm and not the builtin: with the builtin hipcc waits for
// all of them before any LDS read.
// The wait states cover a descriptor or m0 that the instruction before has written, also from a vector
// register (5), which hipcc does not look for in front of asm.
// ONCE: what is loaded is not loaded again by another block (non-temporal).
template <bool ONCE>
__device__ __forceinline__ void load_lds16(const i32x4& rsrc, uint32_t voff, uint32_t lds) {
  if constexpr (ONCE)
    asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen nt lds" : : "v"(voff), "s"(rsrc), "{m0}"(lds) : "memory");
  else
    asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(voff), "s"(rsrc), "{m0}"(lds) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}
__device__ __forceinline__ i32x4 make_rsrc(const void* p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(a));
  r[1] = __builtin_amdgcn_readfirstlane(static_cast<int>((a >> 32) & 0xFFFF));
  r[2] = __builtin_amdgcn_readfirstlane(static_cast<int>(bytes));
  r[3] = 0x00020000;
  return r;
}

// One operand's tile: BN rows (KC) or columns (KS) by 64 k, loaded by NW waves in units of 1 KiB.
// KTAIL: the operand ends with k in memory; the other operand is zero there, but 0 x NaN is not.
template <int BN, bool KS, int NW, bool KTAIL, bool ONCE>
struct Tile {
  static constexpr int kBytes = BN * kBK * 2;
  static constexpr int kUnits = kBytes / 1024;
  static constexpr int kPerWave = kUnits / NW;
  static constexpr int kRowBytes = KS ? BN * 2 : 128;
  static constexpr int kUnitRows = 1024 / kRowBytes;
  static_assert(kUnits % NW == 0, "every wave issues the same number of loads");
  uint32_t voff[kPerWave];
  int kk[kPerWave];  // KC with KTAIL: k of the lane's chunk within the tile
  uint32_t ldb;      // bytes of a row in memory
  i32x4 rsrc;
  int kleft;

  // first: first row (KC) / column (KS) of the tile; limit: rows / columns that exist
  __device__ __forceinline__ void init(int wave, int lane, int first, int limit, int64_t ld) {
    ldb = static_cast<uint32_t>(ld * 2);
#pragma unroll
    for (int u = 0; u < kPerWave; ++u) {
      const int unit = wave * kPerWave + u;
      const int byte = lane * 16;
      const int row = unit * kUnitRows + byte / kRowBytes;
      const int pos = (byte % kRowBytes) / 16;
      if constexpr (KS) {
        const int f = ((row & 3) | (((row >> 3) & 1) << 2)) & (BN / 32 - 1);
        const int chunk = pos ^ (f << 2);
        voff[u] = first + chunk * 8 < limit ? row * ldb + chunk * 16 : kOob;
      } else {
        const int chunk = pos ^ ((row >> 1) & 7);
        kk[u] = chunk * 8;
        voff[u] = first + row < limit ? row * ldb + chunk * 16 : kOob;
      }
    }
  }
  // A step: base is the tile's first byte there; k_left: k that exist from it on (0: past the end,
  // everything loads zeros).  A KS tile ends with its descriptor's range, a KC tile lane by lane.
  __device__ __forceinline__ void step(const void* base, int k_left) {
    kleft = k_left;
    const uint32_t range = KS && k_left < kBK ? k_left * ldb : k_left > 0 ? kOob : 0u;
    rsrc = make_rsrc(base, range);
  }
  template <int U>
  __device__ __forceinline__ void issue(int wave, uint32_t lds) const {
    uint32_t v = voff[U];
    if constexpr (!KS && KTAIL) v = kk[U] < kleft ? v : kOob;
    load_lds16<ONCE>(rsrc, v, lds + (wave * kPerWave + U) * 1024);
  }
};

// The MFMA operand of 32 rows (KC) / columns (KS) from `base` on, k = 16 ks + 8 (lane / 32) .. + 8.
template <int BN, bool KS>
struct Frag {
  uint32_t off[4];      // KC: by ks
  uint32_t kpart;       // KS
  int f;
  __device__ __forceinline__ void init(int lane) {
    if constexpr (KS) {
      const int k = (lane >> 5) * 8 + ((lane & 15) >> 2);
      f = ((k & 3) | (((k >> 3) & 1) << 2)) & (BN / 32 - 1);
      kpart = static_cast<uint32_t>(k * BN * 2 + (((lane >> 4) & 1) * 16 + 4 * (lane & 3)) * 2);
    } else {
      const int row = lane & 31;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) off[ks] = row * 128 + (((2 * ks + (lane >> 5)) ^ ((row >> 1) & 7)) * 16);
    }
  }
  __device__ __forceinline__ bf16x8 read(const char* tile, int block32, int ks) const {
    if constexpr (KS) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const uint32_t a = kpart + static_cast<uint32_t>(((block32 ^ f) & (BN / 32 - 1)) * 64) + ks * (16 * BN * 2);
      lds_s16x4* p = (lds_s16x4*)(tile + a);
      lds_s16x4* q = (lds_s16x4*)(tile + a + 4 * BN * 2);
      union {
        s16x4 h[2];
        bf16x8 v;
      } u;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(q);
      return u.v;
    } else {
      return *reinterpret_cast<const bf16x8*>(tile + block32 * 4096 + off[ks]);
    }
  }
};

// Tiles in an order that lets the blocks that run together share operands: blocks go round-robin
// to the 8 XCDs, so each XCD gets a contiguous range of tiles, walked in columns of 4 row tiles (measured
// on 32 x 501 tiles of 256 x 256: 1241 TFLOP/s against 1224 in columns of 8 and 1174 of 16).
__device__ __forceinline__ void tile_of(int id, int row_tiles, int col_tiles, int* rt, int* ct) {
  const int n = row_tiles * col_tiles, xcd = id & 7, local = id >> 3;
  const int per = n >> 3, extra = n & 7;
  const int t = xcd * per + (xcd < extra ? xcd : extra) + local;
  const int group = 4 * col_tiles, g = t / group, r0 = g * 4;
  const int gr = row_tiles - r0 < 4 ? row_tiles - r0 : 4;
  const int in = t - g * group;
  *rt = r0 + in % gr;
  *ct = in / gr;
}

constexpr float kLowUp = 2048.0f;  // what the low limb of an operand is stored times
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

// compile-time loop: f(integral_constant 0), ..., f(N - 1)
template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<N, I + 1>(f);
  }
}

template <bool F16>
__device__ __forceinline__ f32x16 mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// e with 2^e <= |x| < 2^(e + 1) (0 for 0, infinities and NaN)
__device__ __forceinline__ int exp_below(float x) {
  const float v = fabsf(x);
  if (!(v > 0.0f && v <= 3.402823466e38f)) return 0;
  int e;
  frexpf(v, &e);
  return e - 1;
}
constexpr int kGradExp = 13;  // |p - [v = y]| < 1 and the mantissa of gl below 2: under 2^14

// The loop over steps of 64 k is software-pipelined by hand.  A step is four phases of 16 k; in each,
// a wave's MFMAs run on fragments in registers while it reads the next phase's from LDS.  The barrier
// stands before the last phase: there every wave has its last fragments of this step's tile, so the
// tile's buffer is free for the step NBUF on, whose loads are issued in between the phase's MFMAs, and
// the next step's tile has arrived (vmcnt), whose first fragments the phase reads.
//
// ONCE: one tile of rows, so that every part of C is read by one block.
template <int BR, int BC, int WR, int WC, bool RKS, bool CKS, bool F16, int EPI, int NBUF, bool ONCE>
__global__ void __launch_bounds__(64 * (BR / WR) * (BC / WC)) gemm_kernel(const GemmArgs a) {
  constexpr int NWR = BR / WR, NWC = BC / WC, NW = NWR * NWC;
  constexpr int TR = WR / 32, TC = WC / 32;
  using RT = Tile<BR, RKS, NW, false, false>;
  using CT = Tile<BC, CKS, NW, true, ONCE>;
  constexpr int kStage = RT::kBytes + CT::kBytes;
  constexpr int kLoads = RT::kPerWave + CT::kPerWave;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave % NWR, wc = wave / NWR;
  int rt, ct;
  tile_of(blockIdx.x, a.row_tiles, a.col_tiles, &rt, &ct);
  const int row0 = rt * BR, c0 = ct * BC;
  const int n_valid = *a.n_valid;
  // the whole block leaves, before any load; rows of g up to a step of k are read as k by dW: zeros
  if (!a.k_dev && row0 >= (EPI == EPI_GRAD ? (n_valid + kBK - 1) / kBK * kBK : n_valid)) return;
  const int k_all = a.k_dev ? (n_valid + kBK - 1) / kBK * kBK : a.k;  // g and X are zero up to there
  const int ksteps = (k_all + kBK - 1) / kBK;
  // this split's steps of k
  const int k_lo = static_cast<int>(static_cast<int64_t>(ksteps) * blockIdx.y / a.splits);
  const int k_hi = static_cast<int>(static_cast<int64_t>(ksteps) * (blockIdx.y + 1) / a.splits);
  const int per_seg = k_hi - k_lo, steps = per_seg * a.nseg;

  RT rtile;
  CT ctile;
  rtile.init(wave, lane, row0, 0x7FFFFFFF, a.ldr);
  ctile.init(wave, lane, c0, a.cols, a.ldc);
  Frag<BR, RKS> rf;
  Frag<BC, CKS> cf;
  rf.init(lane);
  cf.init(lane);
  f32x16 acc[TC][TR];
#pragma unroll
  for (int i = 0; i < TC; ++i)
#pragma unroll
    for (int j = 0; j < TR; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  static_assert(NW * 32 * WC * 4 <= NBUF * kStage, "the epilogue's rows fit");
  const uint32_t lds0 = lds_addr(lds);
  // The next step's addresses, kept in scalar registers and made while MFMAs run; past the end a step
  // loads zeros, so that the counts of the waits hold.
  const int64_t rstep = RKS ? a.ldr * (2 * kBK) : 2 * kBK, cstep = CKS ? a.ldc * (2 * kBK) : 2 * kBK;
  const int64_t rfirst = RKS ? k_lo * rstep + row0 * 2 : row0 * a.ldr * 2 + k_lo * rstep;
  const int64_t cfirst = CKS ? k_lo * cstep + c0 * 2 : c0 * a.ldc * 2 + k_lo * cstep;
  const char* rp = reinterpret_cast<const char*>(a.r[0]) + rfirst;
  const char* cp = reinterpret_cast<const char*>(a.c[0]) + cfirst;
  int seg = 0, left = per_seg, k_left = k_all - k_lo * kBK;  // steps and k of this segment
  uint32_t slot = 0, into = lds0;
  auto next_step = [&]() {
    rtile.step(rp, left > 0 ? kBK : 0);
    ctile.step(cp, left > 0 ? k_left : 0);
    into = lds0 + slot;
    slot = slot + kStage == NBUF * kStage ? 0 : slot + kStage;
    rp += rstep;
    cp += cstep;
    k_left -= kBK;
    if (--left == 0 && ++seg < a.nseg) {
      rp = reinterpret_cast<const char*>(a.r[seg]) + rfirst;
      cp = reinterpret_cast<const char*>(a.c[seg]) + cfirst;
      left = per_seg;
      k_left = k_all - k_lo * kBK;
    }
  };
  auto issue = [&](auto u) {
    constexpr int U = decltype(u)::value;
    if constexpr (U < RT::kPerWave) rtile.template issue<U>(wave, into);
    else ctile.template issue<U - RT::kPerWave>(wave, into + RT::kBytes);
  };
  bf16x8 cv[2][TC], rv[2][TR];
  auto read = [&](int set, auto q, const char* stage, int ks) {
    constexpr int Q = decltype(q)::value;
    if constexpr (Q < TC) cv[set][Q] = cf.read(stage + RT::kBytes, wc * TC + Q, ks);
    else rv[set][Q - TC] = rf.read(stage, wr * TR + Q - TC, ks);
  };
  if (steps > 0) {
    each<NBUF>([&](auto) {
      next_step();
      each<kLoads>(issue);
    });
    wait_barrier<kLoads*(NBUF - 1)>();
    each<TC + TR>([&](auto q) { read(0, q, lds, 0); });
  }
  uint32_t at = 0;
  const int last_segment = steps - per_seg;
  for (int step = 0; step < steps; ++step) {
    if constexpr (F16) {
      if (step == last_segment && step > 0) {  // the segments before had one low limb each
#pragma unroll
        for (int i = 0; i < TC; ++i)
#pragma unroll
          for (int j = 0; j < TR; ++j) acc[i][j] *= 1.0f / kLowUp;
      }
    }
    const char* now = lds + at;
    at = at + kStage == NBUF * kStage ? 0 : at + kStage;
    const char* then = lds + at;
    each<4>([&](auto phase) {
      constexpr int P = decltype(phase)::value, set = P & 1;
      if constexpr (P == 1) next_step();
      if constexpr (P == 3) wait_barrier<kLoads*(NBUF - 2)>();
      __builtin_amdgcn_sched_barrier(0);
      each<TC * TR>([&](auto m) {
        constexpr int M = decltype(m)::value, i = M / TR, j = M % TR;
        constexpr int NM = TC * TR, NR = TC + TR;
        constexpr int per = (NR + NM - 1) / NM;  // reads after each MFMA until there are none left
        acc[i][j] = mfma<F16>(cv[set][i], rv[set][j], acc[i][j]);
        each<per>([&](auto r) {
          constexpr int Q = M * per + decltype(r)::value;
          if constexpr (Q < NR) read(set ^ 1, std::integral_constant<int, Q>{}, P == 3 ? then : now, (P + 1) & 3);
        });
        if constexpr (P == 3) {
          constexpr int lo = M * kLoads / NM, hi = (M + 1) * kLoads / NM;
          each<hi - lo>([&](auto u) { issue(std::integral_constant<int, lo + decltype(u)::value>{}); });
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    });
  }
  // no load into LDS outlives the loop, and no wave still reads a tile: the epilogue takes the memory
  wait_barrier<0>();

  // lane: row row0 + wr WR + 32 j + lane % 32, columns cw + 32 i + 8 (e / 4) + 4 (lane / 32) + e % 4
  const int hi = lane >> 5, hi4 = hi * 4;
  const int cw = c0 + wc * WC;
  const bool whole = c0 + BC <= a.cols;  // no column of the tile is past the end
  const int scale_exp = a.scale ? *a.scale : 0;
  // of logits, where an exponent past fp32's would make a NaN of 0: what such a logit is does not matter
  const float scale = ldexpf(1.0f, scale_exp < -126 ? -126 : scale_exp > 126 ? 126 : scale_exp);
  const float l2e = kLog2e * scale;      // exact: scale is a power of two
  if constexpr (EPI == EPI_STATS) {
    // Exponentials to base 2: x log2(e) - c is one fma, and c (the rounded maximum) one exact number in
    // both the terms and the result, so that its rounding does not matter.
#pragma unroll
    for (int j = 0; j < TR; ++j) {
      const int row = row0 + wr * WR + 32 * j + (lane & 31);
      const int tgt = row < n_valid ? a.tgt[row] - a.col0 - cw : -1;  // column within the wave's
      if (!whole) {
#pragma unroll
        for (int i = 0; i < TC; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (cw + 32 * i + 8 * (e >> 2) + hi4 + (e & 3) >= a.cols) acc[i][j][e] = -INFINITY;
      }
      if (__any(tgt >= 0 && tgt < WC)) {
#pragma unroll
        for (int i = 0; i < TC; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (32 * i + 8 * (e >> 2) + hi4 + (e & 3) == tgt) a.tlogit[row] = acc[i][j][e] * scale;
      }
      float m = acc[0][j][0];
#pragma unroll
      for (int i = 0; i < TC; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float c = m == -INFINITY ? 0.0f : m * l2e;
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < TC; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e & 3] += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], l2e, -c));
      float sum = (s[0] + s[1]) + (s[2] + s[3]);
      sum += __shfl_xor(sum, 32, 64);
      if (lane < 32 && row < n_valid)
        a.part[(static_cast<int64_t>(a.col0 / BC + ct) * NWC + wc) * a.ldpart + row] =
            make_float2(m == -INFINITY ? m : c, sum);
    }
    return;
  }
  // The others store matrices: 32 rows at a time go through the wave's own LDS, so that a store
  // instruction writes whole cache lines.  Chunk c (4 columns) of row r lies at c ^ r.
  constexpr int CH = WC / 4, kRowsAt = 64 / CH;
  float* mine = reinterpret_cast<float*>(lds) + wave * (32 * WC);
#pragma unroll
  for (int j = 0; j < TR; ++j) {
    const int rowb = row0 + wr * WR + 32 * j, row = rowb + (lane & 31);
    const int r = lane & 31;
    bool live = true;
    int tgt = -1;
    float l2 = 0.0f, l2lo = 0.0f, gl = 0.0f, gm = 0.0f;
    bool here = false;  // some token's target is among the wave's columns
    if constexpr (EPI == EPI_GRAD) {
      live = row < n_valid;
      if (live) {
        tgt = a.tgt[row] - a.col0 - cw;
        gl = a.gl[row];
        gm = ldexpf(gl, kGradExp - exp_below(gl));  // exponents add: 2^13 / 2^e is past fp32 for gl below 2^-114
        const float lse = a.lse[row];
        l2 = lse * kLog2e;  // and what it lacks, so that p is not off by the rounding of a large lse
        l2lo = fmaf(lse, kLog2e, -l2);
      }
      here = __any(tgt >= 0 && tgt < WC);
    }
#pragma unroll
    for (int i = 0; i < TC; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = cw + 32 * i + 8 * q + hi4;
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = acc[i][j][4 * q + e];
          if constexpr (EPI == EPI_GRAD) x = __builtin_amdgcn_exp2f(fmaf(x, l2e, -l2) - l2lo);
          v[e] = x;
        }
        if constexpr (EPI == EPI_GRAD) {
          if (here) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] -= col - cw + e == tgt ? 1.0f : 0.0f;
          }
          if (!live) v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          if (!whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = col + e < a.cols ? v[e] : 0.0f;
          }
        }
        *reinterpret_cast<f32x4*>(mine + r * WC + ((8 * i + 2 * q + hi) ^ (r & (CH - 1))) * 4) = v;
      }
    asm volatile("" ::: "memory");  // LDS operations of a wave are done in order
#pragma unroll
    for (int t = 0; t < 32 / kRowsAt; ++t) {
      const int rr = t * kRowsAt + lane / CH, c = lane % CH;
      const int orow = rowb + rr, col = cw + 4 * c;
      f32x4 v = *reinterpret_cast<const f32x4*>(mine + rr * WC + (c ^ (rr & (CH - 1))) * 4);
      if constexpr (EPI == EPI_GRAD) {
        const int64_t to = static_cast<int64_t>(orow) * a.ldg + col;
        const float glr = __shfl(gl, rr, 64);  // lane rr has row rr's
        if (a.gb[0]) {
          f32x4 u = v * glr;
          u32x2 w;
          w[0] = pack_bf16(u[0], u[1]);
          w[1] = pack_bf16(u[2], u[3]);
          *reinterpret_cast<u32x2*>(a.gb[0] + to) = w;
          if (here || a.gb[1]) {
            u[0] -= __uint_as_float(w[0] << 16);
            u[1] -= __uint_as_float(w[0] & 0xFFFF0000u);
            u[2] -= __uint_as_float(w[1] << 16);
            u[3] -= __uint_as_float(w[1] & 0xFFFF0000u);
          }
          if (a.gb[1]) {
            w[0] = pack_bf16(u[0], u[1]);
            w[1] = pack_bf16(u[2], u[3]);
            *reinterpret_cast<u32x2*>(a.gb[1] + to) = w;
          }
          if (here) {
            const int at = __shfl(tgt, rr, 64) - 4 * c;
            if (orow < n_valid && at >= 0 && at < 4) a.delta[orow] = at == 0 ? u[0] : at == 1 ? u[1] : at == 2 ? u[2] : u[3];
          }
        }
        if (a.gh[0]) {
          v *= __shfl(gm, rr, 64);
          u32x2 w;
          w[0] = pack_f16(v[0], v[1]);
          w[1] = pack_f16(v[2], v[3]);
          *reinterpret_cast<u32x2*>(a.gh[0] + to) = w;
          w[0] = pack_f16((v[0] - f16_lo(w[0])) * kLowUp, (v[1] - f16_hi(w[0])) * kLowUp);
          w[1] = pack_f16((v[2] - f16_lo(w[1])) * kLowUp, (v[3] - f16_hi(w[1])) * kLowUp);
          *reinterpret_cast<u32x2*>(a.gh[1] + to) = w;
        }
      } else if constexpr (EPI == EPI_SLAB) {
        if (orow < n_valid && col < a.ldslab) {
          f32x4* o = reinterpret_cast<f32x4*>(a.slab + blockIdx.y * a.slab_stride + static_cast<int64_t>(orow) * a.ldslab + col);
          if (a.add) v += *o;
          *o = v;
        }
      } else if (orow < a.rows && col < a.cols) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], scale_exp);
        const int64_t at = static_cast<int64_t>(orow) * a.ldo + col;
        if (a.out_bf16) {
          uint16_t* o = static_cast<uint16_t*>(a.out) + at;
          if (a.out_vec) {  // cols % 4 == 0: all four exist
            u32x2 w;
            if (a.add) {
              w = *reinterpret_cast<const u32x2*>(o);
              v[0] += __uint_as_float(w[0] << 16);
              v[1] += __uint_as_float(w[0] & 0xFFFF0000u);
              v[2] += __uint_as_float(w[1] << 16);
              v[3] += __uint_as_float(w[1] & 0xFFFF0000u);
            }
            w[0] = pack_bf16(v[0], v[1]);
            w[1] = pack_bf16(v[2], v[3]);
            *reinterpret_cast<u32x2*>(o) = w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < a.cols) o[e] = f32_to_bf16(a.add ? bf16_to_f32(o[e]) + v[e] : v[e]);
          }
        } else {
          float* o = static_cast<float*>(a.out) + at;
          if (a.out_vec) {
            f32x4 w = v;
            if (a.add) w += *reinterpret_cast<const f32x4*>(o);
            *reinterpret_cast<f32x4*>(o) = w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < a.cols) o[e] = a.add ? o[e] + v[e] : v[e];
          }
        }
      }
    }
    asm volatile("" ::: "memory");
  }
}
