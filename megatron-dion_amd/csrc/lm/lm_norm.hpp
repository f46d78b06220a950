// lm_norm.hpp -- residual RMS norm with dropout, 8-bit output, and its backward pass.
//
// One pass over the data: a row is held in registers (NV vectors of 8 elements for each of the
// LPR threads that share it) between its sum of squares and its scaling, so the forward reads x
// and the residual and writes h and y once, and the backward reads gy, h and grad_h and writes the
// gradients once.  Rows of up to 1024 elements go to a wave each (no barrier), longer ones to a
// block.  Rows may start and end anywhere: wide accesses need no alignment here, and only a row's last
// vector goes element by element.  Bound by memory: 8192 x 4096 bf16 with residual and dropout 54 us forward
// (4.9 TB/s), 63 us backward (5.3 TB/s; its partial weight gradients 7 us more), with 8-bit output 44 us.
// Four blocks for each CU in the backward: two (96 us) leave too few loads in flight.

struct NormArgs {
  const void *x, *residual, *weight, *gy, *gh;
  const void* h_in;
  void *h, *y, *gx, *gr, *gw;
  float *scale, *rstd_out, *part;
  const float* rstd;
  int64_t rows;
  int cols, w_bf16, gw_bf16, accumulate, sblock, sblocks;
  float eps;
  int64_t ldx, ldr, ldh, ldy, ldgy, ldgh, ldgx, ldgr;
  DropArgs drop;
  int dropping;
};

template <bool RAGGED>
__device__ __forceinline__ void load_weight(const NormArgs& a, int c, float* w) {
  if (a.w_bf16) load8<RAGGED>(static_cast<const bf16*>(a.weight), c, a.cols, w);
  else load8<RAGGED>(static_cast<const float*>(a.weight), c, a.cols, w);
}

// sum over the LPR threads that share a row; `red`: LPR / 64 floats of LDS (LPR > 64)
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (LPR > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // the last use of red is over
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < LPR / 64; ++i) v += red[i];
  }
  return v;
}

__device__ __forceinline__ float e4m3_clamp(float v) {  // NaN stays NaN
  return v > 448.0f ? 448.0f : v < -448.0f ? -448.0f : v;
}

__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(v), 0.0f, 0, false) & 0xFF);
}
// round_e4m3(v / s) from column c of a row on.  The quotient is fp32's: a product with 1 / s alone has a rounding
// more, which takes values next to the middle of two codes to the other one.  The product and one correction by
// its exact remainder are right for ordinary scales (8192 x 4096 in blocks of 128 columns: 49.0 us, 50.5 with a
// division for each element); below 2^-90 the remainder may not be held, and an infinite scale has none.
template <bool RAGGED>
__device__ __forceinline__ void store8_e4m3(uint8_t* row, int c, int cols, const float* v, float s) {
  float q[8];
  if (s >= 8.07793567e-28f && s <= 3.402823466e38f) {
    const float inv = 1.0f / s;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float p = v[k] * inv;
      q[k] = e4m3_clamp(fmaf(fmaf(-p, s, v[k]), inv, p));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = e4m3_clamp(v[k] / s);
  }
  if (!RAGGED || c + 8 <= cols) {
    u32x2 o;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * k], q[4 * k + 1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * k + 2], q[4 * k + 3], w, true);
      o[k] = static_cast<uint32_t>(w);
    }
    *reinterpret_cast<u32x2_any*>(row + c) = o;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < cols) row[c + k] = to_e4m3(q[k]);
  }
}

// The 8-bit output's scales: blocks of columns that neighbouring lanes hold, or any blocks (through LDS).
enum { Q8_NONE = 0, Q8_LANES = 1, Q8_ANY = 2 };

// threads of a block: 4 rows of 64 threads, or one row of LPR
template <int LPR>
constexpr int norm_threads() { return LPR > 64 ? LPR : 256; }

template <typename T, int LPR, int NV, int Q8, bool RAGGED>
__global__ void __launch_bounds__(norm_threads<LPR>()) norm_fwd_kernel(const NormArgs a) {
  constexpr int RPB = LPR > 64 ? 1 : 4;
  __shared__ float red[16];
  extern __shared__ uint32_t amax[];  // Q8_ANY: sblocks words for each row of the block
  const int t = LPR > 64 ? threadIdx.x : (threadIdx.x & 63);
  const int sub = LPR > 64 ? 0 : (threadIdx.x >> 6);
  const int64_t row = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * RPB + sub;
  const bool live = row < a.rows;  // whole waves: RPB == 4 has a row for each wave
  float v[NV][8];
  if constexpr (Q8 == Q8_ANY) {
    for (int i = t; i < a.sblocks; i += LPR) amax[sub * a.sblocks + i] = 0u;
    __syncthreads();
  }
  float ss = 0.0f;
  if (live) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* r = static_cast<const T*>(a.residual) + row * a.ldr;
    T* h = static_cast<T*>(a.h) + row * a.ldh;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + t) * 8;
      if (c < a.cols) load8<RAGGED>(x, c, a.cols, v[i]);
    }
    float q[NV][8];
    if (a.residual) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * LPR + t) * 8;
        if (c < a.cols) load8<RAGGED>(r, c, a.cols, q[i]);
      }
    }
    if (a.dropping) {
      const Key key = philox_key(a.drop);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * LPR + t) * 8;
        if (c < a.cols) drop8<RAGGED>(v[i], static_cast<uint64_t>(row) * a.cols + c, key, a.drop);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + t) * 8;
      if (c < a.cols) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (a.residual) v[i][k] = __fadd_rn(v[i][k], q[i][k]);
          v[i][k] = to_f32(from_f32<T>(v[i][k]));  // the norm is of h as it is stored
          ss = fmaf(v[i][k], v[i][k], ss);
        }
        if (a.h) store8<RAGGED>(h, c, a.cols, v[i]);
      }
    }
  }
  ss = row_sum<LPR>(ss, red);
  const float rstd = 1.0f / sqrtf(ss / static_cast<float>(a.cols) + a.eps);
  if (live && t == 0) a.rstd_out[row] = rstd;
  if (live) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + t) * 8;
      if (c < a.cols) {
        float w[8];
        load_weight<RAGGED>(a, c, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = v[i][k] * rstd * w[k];
        if constexpr (Q8 == Q8_NONE) store8<RAGGED>(static_cast<T*>(a.y) + row * a.ldy, c, a.cols, v[i]);
      }
    }
  }
  if constexpr (Q8 == Q8_LANES) {
    // a scale's columns are those of 2^n neighbouring lanes of a wave (sblock = 8 .. 512)
    const int span = a.sblock >> 3, shift = 31 - __clz(a.sblock);
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * LPR + t) * 8;
        float m = 0.0f;
        if (c < a.cols) {
#pragma unroll
          for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(v[i][k]));  // passes over NaN
        }
        for (int o = 1; o < span; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        const float s = fmaxf(m / 448.0f, 1.17549435e-38f);
        if (c < a.cols) {
          if ((t & (span - 1)) == 0) a.scale[row * a.sblocks + (c >> shift)] = s;
          store8_e4m3<RAGGED>(static_cast<uint8_t*>(a.y) + row * a.ldy, c, a.cols, v[i], s);
        }
      }
    }
  }
  if constexpr (Q8 == Q8_ANY) {
    // |y| as bits is ordered like an integer; a maximum does not depend on the order it is taken in
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * LPR + t) * 8;
        if (c < a.cols) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float y = fabsf(v[i][k]);
            if ((!RAGGED || c + k < a.cols) && y == y) atomicMax(&amax[sub * a.sblocks + (c + k) / a.sblock], __float_as_uint(y));
          }
        }
      }
    }
    __syncthreads();
    if (live) {
      for (int i = t; i < a.sblocks; i += LPR)
        a.scale[row * a.sblocks + i] = fmaxf(__uint_as_float(amax[sub * a.sblocks + i]) / 448.0f, 1.17549435e-38f);
      uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.ldy;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * LPR + t) * 8;
        if (c < a.cols) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (!RAGGED || c + k < a.cols) {
              const float s = fmaxf(__uint_as_float(amax[sub * a.sblocks + (c + k) / a.sblock]) / 448.0f, 1.17549435e-38f);
              y[c + k] = to_e4m3(v[i][k] / s);
            }
        }
      }
    }
  }
}

// Weight-gradient partials: each block (or wave, LPR == 64) sums its rows in registers.
template <typename T, int LPR, int NV, bool RAGGED>
__global__ void __launch_bounds__(norm_threads<LPR>()) norm_bwd_kernel(const NormArgs a) {
  constexpr int RPB = LPR > 64 ? 1 : 4;
  __shared__ float red[16];
  const int t = LPR > 64 ? threadIdx.x : (threadIdx.x & 63);
  const int64_t first = LPR > 64 ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t step = static_cast<int64_t>(gridDim.x) * RPB;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LPR + t) * 8;
#pragma unroll
    for (int k = 0; k < 8; ++k) w[i][k] = dw[i][k] = 0.0f;
    if (c < a.cols) load_weight<RAGGED>(a, c, w[i]);
  }
  Key key = {0, 0, 0, 0};
  if (a.dropping) key = philox_key(a.drop);
  for (int64_t row = first; row < a.rows; row += step) {
    const float rstd = a.rstd[row];
    float u[NV][8], g[NV][8], q[NV][8], dot = 0.0f;  // u = h rstd, g = gy then w gy
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + t) * 8;
      if (c < a.cols) {
        load8<RAGGED>(static_cast<const T*>(a.h_in) + row * a.ldh, c, a.cols, u[i]);
        load8<RAGGED>(static_cast<const T*>(a.gy) + row * a.ldgy, c, a.cols, g[i]);
        if (a.gh) load8<RAGGED>(static_cast<const T*>(a.gh) + row * a.ldgh, c, a.cols, q[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + t) * 8;
      if (c < a.cols) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          u[i][k] *= rstd;
          dw[i][k] = fmaf(g[i][k], u[i][k], dw[i][k]);
          g[i][k] *= w[i][k];
          dot = fmaf(g[i][k], u[i][k], dot);
        }
      }
    }
    if (a.gx || a.gr) {
      const float mean = row_sum<LPR>(dot, red) / static_cast<float>(a.cols);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * LPR + t) * 8;
        if (c < a.cols) {
          float d[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) d[k] = rstd * (g[i][k] - u[i][k] * mean);
          if (a.gh) {
#pragma unroll
            for (int k = 0; k < 8; ++k) d[k] += q[i][k];
          }
          if (a.gr) store8<RAGGED>(static_cast<T*>(a.gr) + row * a.ldgr, c, a.cols, d);
          if (a.gx) {
            if (a.dropping) drop8<RAGGED>(d, static_cast<uint64_t>(row) * a.cols + c, key, a.drop);
            store8<RAGGED>(static_cast<T*>(a.gx) + row * a.ldgx, c, a.cols, d);
          }
        }
      }
    }
  }
  if (a.part) {
    float* p = a.part + first * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + t) * 8;
      if (c < a.cols) store8<RAGGED>(p, c, a.cols, dw[i]);
    }
  }
}

// grad_weight = the sum of the partials in a fixed order: 16 columns a block, 64 threads a column,
// four partials in flight a thread
__global__ void __launch_bounds__(1024) norm_dw_kernel(const NormArgs a, int parts) {
  __shared__ float red[64][17];
  const int x = threadIdx.x & 15, k = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
  float s = 0.0f;
  if (c < a.cols) {
    const float* p = a.part + c;
    int i = k;
    for (; i + 192 < parts; i += 256)
      s += (p[static_cast<int64_t>(i) * a.cols] + p[static_cast<int64_t>(i + 64) * a.cols]) +
           (p[static_cast<int64_t>(i + 128) * a.cols] + p[static_cast<int64_t>(i + 192) * a.cols]);
    for (; i < parts; i += 64) s += p[static_cast<int64_t>(i) * a.cols];
  }
  red[k][x] = s;
#pragma unroll
  for (int half = 32; half > 0; half >>= 1) {
    __syncthreads();
    if (k < half) red[k][x] += red[k + half][x];
  }
  if (k == 0 && c < a.cols) {
    s = red[0][x];
    if (a.gw_bf16) {
      uint16_t* o = static_cast<uint16_t*>(a.gw) + c;
      *o = f32_to_bf16(a.accumulate ? bf16_to_f32(*o) + s : s);
    } else {
      float* o = static_cast<float*>(a.gw) + c;
      *o = a.accumulate ? *o + s : s;
    }
  }
}

namespace rms {

constexpr int kMaxCols = 16384;

// Blocks of the backward kernel, each of which leaves one partial row of grad_weight (four, where a
// row is a wave's): four for each CU.
long bwd_blocks(int64_t rows, bool wave_rows) {
  const long want = wave_rows ? ceil_div(rows, 4) : rows;
  return want < 1024 ? (want < 1 ? 1 : want) : 1024;
}
bool wave_rows(int cols) { return cols <= 1024; }

size_t ws_bytes(const DionNormDesc* d) {
  const bool w = wave_rows(d->cols);
  return sizeof(float) * static_cast<size_t>(bwd_blocks(d->rows, w)) * (w ? 4 : 1) * d->cols;
}

// The threads of a row: a wave for up to 1024 columns, else as many as hold it in two vectors each.
// f(LPR, NV)
template <typename F>
void with_row(int cols, F&& f) {
  using std::integral_constant;
  if (cols <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (cols <= 1024) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (cols <= 2048) f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (cols <= 4096) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (cols <= 8192) f(integral_constant<int, 512>{}, integral_constant<int, 2>{});
  else f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
}

template <typename T, int Q8>
int forward(const NormArgs& a, hipStream_t st) {
  with_row(a.cols, [&](auto lpr, auto nv) {
    constexpr int LPR = decltype(lpr)::value, NV = decltype(nv)::value, RPB = LPR > 64 ? 1 : 4;
    const size_t lds = Q8 == Q8_ANY ? sizeof(uint32_t) * RPB * a.sblocks : 0;
    // a grid's axis has to stay below 2^32 threads: 2^21 blocks of up to 1024, then rows of them
    const long blocks = ceil_div(a.rows, RPB), bx = blocks < (1 << 21) ? blocks : 1 << 21;
    const dim3 grid(bx, ceil_div(blocks, bx)), block(norm_threads<LPR>());
    if (a.cols % 8) hipLaunchKernelGGL((norm_fwd_kernel<T, LPR, NV, Q8, true>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((norm_fwd_kernel<T, LPR, NV, Q8, false>), grid, block, lds, st, a);
  });
  return check_launch("rms_norm_add");
}

template <typename T>
int backward(const NormArgs& a, hipStream_t st) {
  const bool wr = wave_rows(a.cols);
  const long blocks = bwd_blocks(a.rows, wr);
  with_row(a.cols, [&](auto lpr, auto nv) {
    constexpr int LPR = decltype(lpr)::value, NV = decltype(nv)::value;
    const dim3 grid(blocks), block(norm_threads<LPR>());
    if (a.cols % 8) hipLaunchKernelGGL((norm_bwd_kernel<T, LPR, NV, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((norm_bwd_kernel<T, LPR, NV, false>), grid, block, 0, st, a);
  });
  int rc = check_launch("rms_norm_add_backward");
  if (rc != DION_OK || a.gw == nullptr) return rc;
  hipLaunchKernelGGL(norm_dw_kernel, dim3(ceil_div(a.cols, 16)), dim3(1024), 0, st, a,
                     static_cast<int>(blocks * (wr ? 4 : 1)));
  return check_launch("rms_norm_add_backward(weight)");
}

}  // namespace rms
