// lm_gemm.hpp -- the matrix products of the linear cross entropy: one tile loop, three epilogues.
//
//   out[row][col] = sum_k R[row][k] C[col][k]
//
// Both operands are bf16 in memory.  An operand is K-contiguous (KC: its rows run along k) or
// K-strided (KS: its rows run along row / col, one row for each k); a KS tile is transposed on its
// way out of LDS by ds_read_b64_tr_b16, so that no operand is ever transposed in HBM:
//   logits  z  = X W^T    R = X [t][h]  KC    C = W [v][h]  KC
//   grad    dX = g W      R = g [t][v]  KC    C = W [v][h]  KS
//   grad    dW = g^T X    R = g [t][v]  KS    C = X [t][h]  KS
// The C operand is the MFMA's A matrix: a lane then holds 4 consecutive output columns, and the
// softmax over columns reduces inside a lane.
//
// fp32 operands are sums of bf16 limbs (x = x1 + x2 + x3, each the bf16 nearest to what is left, 8
// bits each); a product of them is a list of segments, the limb pairs that matter, which the loop
// walks through as if k were that much longer.  Accumulation is fp32 in the MFMA.
//
// Tiles go to LDS by buffer_load_dwordx4 ... lds, NBUF - 1 steps of 64 k ahead; rows and columns
// past the end get an offset past the descriptor's range, which loads zeros.  16-byte chunks are
// placed so that the reads of a wave spread over all banks: KC chunk c of row r at c ^ (r/2 % 8),
// KS 64-byte slot s of row k at s ^ (k%4 + 4 (k/8 % 2)).

constexpr int kBK = 64;
constexpr int kMaxSeg = 6;
constexpr uint32_t kOob = 0x80000000u;  // == num_records: loads zeros

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
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
  int col0;              // first shard column of this piece
  float2* part;          // stats: [part][token] (max, sum)
  float* tlogit;         // stats: per compact token
  int64_t ldpart;
  uint16_t* g[3];        // limbs of g
  int nlimb;
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
__device__ __forceinline__ void load_lds16(const i32x4& rsrc, uint32_t voff, uint32_t lds) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(voff), "s"(rsrc), "s"(lds)
      : "memory");
}
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}
__device__ __forceinline__ i32x4 make_rsrc(const void* p) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(a));
  r[1] = __builtin_amdgcn_readfirstlane(static_cast<int>((a >> 32) & 0xFFFF));
  r[2] = static_cast<int>(kOob);
  r[3] = 0x00020000;
  return r;
}

// One operand's tile: BN rows (KC) or columns (KS) by 64 k, loaded by NW waves.
template <int BN, bool KS, int NW>
struct Tile {
  static constexpr int kBytes = BN * kBK * 2;
  static constexpr int kUnits = kBytes / 1024;  // wave loads
  static constexpr int kPerWave = kUnits / NW;
  static constexpr int kRowBytes = KS ? BN * 2 : 128;
  static constexpr int kUnitRows = 1024 / kRowBytes;
  static_assert(kUnits % NW == 0, "every wave issues the same number of loads");
  uint32_t voff[kPerWave];
  int kk[kPerWave];  // k of the lane's chunk within the tile

  // first: first row (KC) / column (KS) of the tile; limit: rows / columns that exist
  __device__ __forceinline__ void init(int wave, int lane, int first, int limit, int64_t ld) {
#pragma unroll
    for (int u = 0; u < kPerWave; ++u) {
      const int unit = wave * kPerWave + u;
      const int byte = lane * 16;
      const int row = unit * kUnitRows + byte / kRowBytes;
      const int pos = (byte % kRowBytes) / 16;
      if constexpr (KS) {
        const int f = ((row & 3) | (((row >> 3) & 1) << 2)) & (BN / 32 - 1);
        const int chunk = pos ^ (f << 2);
        kk[u] = row;
        voff[u] = first + chunk * 8 < limit ? static_cast<uint32_t>(row * ld * 2 + chunk * 16) : kOob;
      } else {
        const int chunk = pos ^ ((row >> 1) & 7);
        kk[u] = chunk * 8;
        voff[u] = first + row < limit ? static_cast<uint32_t>(row * ld * 2 + chunk * 16) : kOob;
      }
    }
  }
  // kleft: k that exist from this step on
  __device__ __forceinline__ void issue(const void* base, int wave, uint32_t lds, int kleft) const {
    const i32x4 rsrc = make_rsrc(base);
#pragma unroll
    for (int u = 0; u < kPerWave; ++u) {
      uint32_t v = voff[u];
      if (kleft < kBK) v = kk[u] < kleft ? v : kOob;
      load_lds16(rsrc, v, lds + (wave * kPerWave + u) * 1024);
    }
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
// to the 8 XCDs, so each XCD gets a contiguous range of tiles, walked in columns of 8 row tiles.
__device__ __forceinline__ void tile_of(int id, int row_tiles, int col_tiles, int* rt, int* ct) {
  const int n = row_tiles * col_tiles, xcd = id & 7, local = id >> 3;
  const int per = n >> 3, extra = n & 7;
  const int t = xcd * per + (xcd < extra ? xcd : extra) + local;
  const int group = 8 * col_tiles, g = t / group, r0 = g * 8;
  const int gr = row_tiles - r0 < 8 ? row_tiles - r0 : 8;
  const int in = t - g * group;
  *rt = r0 + in % gr;
  *ct = in / gr;
}

constexpr float kLog2e = 1.44269504088896341f;

template <int BR, int BC, int WR, int WC, bool RKS, bool CKS, int EPI, int NBUF>
__global__ void __launch_bounds__(64 * (BR / WR) * (BC / WC)) gemm_kernel(const GemmArgs a) {
  constexpr int NWR = BR / WR, NWC = BC / WC, NW = NWR * NWC;
  constexpr int TR = WR / 32, TC = WC / 32;
  using RT = Tile<BR, RKS, NW>;
  using CT = Tile<BC, CKS, NW>;
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

  const uint32_t lds0 = lds_addr(lds);
  int seg = 0, ks_at = k_lo;
  auto issue = [&](int step) {
    const uint32_t at = lds0 + static_cast<uint32_t>(step % NBUF) * kStage;
    const bool real = step < steps;  // past the end: zeros, so that the counts of the waits hold
    const int64_t k0 = static_cast<int64_t>(ks_at) * kBK;
    const uint16_t* rp = a.r[seg] + (RKS ? k0 * a.ldr + row0 : static_cast<int64_t>(row0) * a.ldr + k0);
    const uint16_t* cp = a.c[seg] + (CKS ? k0 * a.ldc + c0 : static_cast<int64_t>(c0) * a.ldc + k0);
    rtile.issue(rp, wave, at, real ? kBK : 0);
    ctile.issue(cp, wave, at + RT::kBytes, real ? k_all - static_cast<int>(k0) : 0);
    if (real && ++ks_at == k_hi && seg + 1 < a.nseg) {
      ks_at = k_lo;
      ++seg;
    }
  };
  if (steps > 0) {
#pragma unroll
    for (int s = 0; s < NBUF - 1; ++s) issue(s);
  }
  for (int step = 0; step < steps; ++step) {
    wait_barrier<kLoads*(NBUF - 2)>();  // this step's tile is there; all have read the one before
    issue(step + NBUF - 1);
    const char* rb = lds + (step % NBUF) * kStage;
    const char* cb = rb + RT::kBytes;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      bf16x8 cv[TC], rv[TR];
#pragma unroll
      for (int i = 0; i < TC; ++i) cv[i] = cf.read(cb, wc * TC + i, ks);
#pragma unroll
      for (int j = 0; j < TR; ++j) rv[j] = rf.read(rb, wr * TR + j, ks);
#pragma unroll
      for (int i = 0; i < TC; ++i)
#pragma unroll
        for (int j = 0; j < TR; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cv[i], rv[j], acc[i][j], 0, 0, 0);
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // no load into LDS outlives the loop

  // lane: row row0 + wr WR + 32 j + lane % 32, columns c0 + wc WC + 32 i + 8 (e / 4) + 4 (lane / 32) + e % 4
  const int hi4 = (lane >> 5) * 4;
  const int cw = c0 + wc * WC;
#pragma unroll
  for (int j = 0; j < TR; ++j) {
    const int row = row0 + wr * WR + 32 * j + (lane & 31);
    if constexpr (EPI == EPI_STATS) {
      const int tgt = row < n_valid ? a.tgt[row] : -1;
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < TC; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int col = cw + 32 * i + 8 * (e >> 2) + hi4 + (e & 3);
          if (col < a.cols) {
            m = fmaxf(m, acc[i][j][e]);
            if (col + a.col0 == tgt) a.tlogit[row] = acc[i][j][e];
          }
        }
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float mb = (m == -INFINITY ? 0.0f : m);
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < TC; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int col = cw + 32 * i + 8 * (e >> 2) + hi4 + (e & 3);
          if (col < a.cols) s += __builtin_amdgcn_exp2f((acc[i][j][e] - mb) * kLog2e);
        }
      s += __shfl_xor(s, 32, 64);
      if (lane < 32 && row < n_valid)
        a.part[(static_cast<int64_t>(a.col0 / BC + ct) * NWC + wc) * a.ldpart + row] = make_float2(m, s);
    } else if constexpr (EPI == EPI_GRAD) {
      const bool live = row < n_valid;
      const int tgt = live ? a.tgt[row] : -1;
      const float lse = live ? a.lse[row] : 0.0f, gl = live ? a.gl[row] : 0.0f;
#pragma unroll
      for (int i = 0; i < TC; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = cw + 32 * i + 8 * q + hi4;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float p = __builtin_amdgcn_exp2f((acc[i][j][4 * q + e] - lse) * kLog2e);
            if (col + e + a.col0 == tgt) p -= 1.0f;
            v[e] = live && col + e < a.cols ? p * gl : 0.0f;
          }
          for (int n = 0; n < a.nlimb; ++n) {
            u32x2 w;
            w[0] = pack_bf16(v[0], v[1]);
            w[1] = pack_bf16(v[2], v[3]);
            *reinterpret_cast<u32x2*>(a.g[n] + static_cast<int64_t>(row) * a.ldg + col) = w;
            v[0] -= __uint_as_float(w[0] << 16);
            v[1] -= __uint_as_float(w[0] & 0xFFFF0000u);
            v[2] -= __uint_as_float(w[1] << 16);
            v[3] -= __uint_as_float(w[1] & 0xFFFF0000u);
          }
        }
    } else if constexpr (EPI == EPI_SLAB) {
      if (row < n_valid) {
        float* o = a.slab + blockIdx.y * a.slab_stride + static_cast<int64_t>(row) * a.ldslab;
#pragma unroll
        for (int i = 0; i < TC; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int col = cw + 32 * i + 8 * q + hi4;
            if (col < a.ldslab) {
              f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
              if (a.add) v += *reinterpret_cast<const f32x4*>(o + col);
              *reinterpret_cast<f32x4*>(o + col) = v;
            }
          }
      }
    } else {
      if (row < a.rows) {
#pragma unroll
        for (int i = 0; i < TC; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int col = cw + 32 * i + 8 * q + hi4;
            float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            if (a.out_bf16) {
              uint16_t* o = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(row) * a.ldo + col;
              if (a.out_vec && col < a.cols) {  // cols % 4 == 0: all four exist
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
              float* o = static_cast<float*>(a.out) + static_cast<int64_t>(row) * a.ldo + col;
              if (a.out_vec && col < a.cols) {
                f32x4 w = {v[0], v[1], v[2], v[3]};
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
    }
  }
}
