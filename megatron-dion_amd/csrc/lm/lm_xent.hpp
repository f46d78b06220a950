// lm_xent.hpp -- the linear cross entropy: tokens that take part, limbs, the pieces of the vocabulary.
//
// What it reads, writes and computes (T tokens that take part, H, V words): T H + V H elements, three
// products of 2 T H V operations for loss and gradients, and a fourth because the logits are not kept.
// 8192 x 4096 x 128256 in bf16: 6.7 ms forward, 27.7 with the gradients (1.25 PFLOP/s, bound by power, see
// lm_gemm.hpp); one token x 4096 x 32000: 59 us, bound by reading W (4.4 TB/s).
//
// forward   select, pack X [, pack W] -> logits tiles, each leaving (maximum, sum of exp) of its columns
//           for each token -> join them: lse, loss
// backward  select, pack X -> for each piece of the vocabulary: [pack W], logits again, g = the
//           gradient of the logits to the workspace, dX += g W, dW = g^T X -> round dX
//
// Only tokens with a target (and, backward, a gradient) take part: select numbers them, pack X
// gathers their rows, and every product runs over that many.  What a hidden state without a target
// holds is never read.
//
// Precision: bf16 inputs are multiplied as they are.  g is one bf16 (2^-8) where it makes bf16 results,
// whose own rounding is as large (for dW of up to 256 tokens, where few roundings do not average out, two
// bf16, 2^-16 over bf16's whole range.  One fp16 limb, 2^-11, is 0 below p = 4e-12; gradients of 8 / 256
// tokens x 4096 x 32000 take 263 / 377 us with it, 268 / 418 with two bf16), and two fp16 limbs where the result is
// fp32: grad_weight into an fp32 main_grad (4096 tokens x 768 x 50257: 1.87 ms a pass, 2.34 with three
// bf16 limbs; two bf16 limbs left 2.6e-6 of the 2-norm, twice what an fp32 product is off), and everything
// for fp32 inputs, which are two fp16 limbs themselves.  The power of two that brings such an operand
// into fp16's range comes from its largest finite value; g's is known, |p - [v = y]| <= 1 times the
// mantissa of the token's gl, whose power of two goes into X (for dW) or is put back at the end (for dX).
// Two limbs of g are off by 2^-22 of it or by 2^-49 of |gl|, whichever is more: a word's row keeps fp32's
// bits down to p = 1e-8 and has 9 left at 1e-12; below 1e-15 it is 0.  bf16 hidden states times that power of
// two are one limb: off by 2^-39 of the largest of these products.

namespace xent {

struct Tokens {  // compact arrays, by the number a token has among those that take part
  int* count;    // [1]
  int* pos;      // [tokens]: number of a token, -1: takes no part
  int* index;    // [tokens_p]: token of a number
  int* tgt;      // [tokens_p]
  float* lse;    // [tokens_p] (backward)
  float* gl;     // [tokens_p] (backward)
  float* tlogit; // [tokens_p] (forward)
  float* delta;  // [tokens_p] (backward, bf16 inputs): what the target's g lost when it was rounded
  float* amax;   // [3][kAmaxBlocks]: largest |X|, |W| of a block's share, and of |X| 2^e the exponent + kExpBias
  int* scale;    // [4]: kScaleZ ...
};
constexpr int kAmaxBlocks = 512;
// exponents of what undoes the scales of z = X W^T, dX = g W (without the token's 2^e), dW = g^T X
enum { kScaleZ = 0, kScaleDx = 1, kScaleDw = 2 };

struct SelectArgs {
  const int64_t* target;
  const float *lse, *gl;  // backward
  int tokens;
  int64_t ignore, start, vocab, total;
  Tokens out;
};

// Numbers the tokens that take part, in order; the whole block (1024 threads) takes part, 4 tokens a
// thread at a time.  f(t, n): token t (this thread's) has the number n, -1: none.  Returns how many there are.
template <typename F>
__device__ __forceinline__ int select(const SelectArgs& a, F&& f) {
  __shared__ int wsum[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0;
  for (int t0 = 0; t0 < a.tokens; t0 += 4096) {
    const int t = t0 + 4 * static_cast<int>(threadIdx.x);
    bool in[4];
    int mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      in[k] = t + k < a.tokens && a.target[t + k] != a.ignore && (!a.gl || !(a.gl[t + k] == 0.0f));  // NaN takes part
      mine += in[k];
    }
    int upto = mine;  // of the wave's lanes up to this one
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int below = __shfl_up(upto, o, 64);
      if (lane >= o) upto += below;
    }
    if (lane == 63) wsum[wave] = upto;
    __syncthreads();
    int before = base + upto - mine, all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += wsum[w];
      all += wsum[w];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (t + k < a.tokens) f(t + k, in[k] ? before : -1);
      before += in[k];
    }
    base += all;
    __syncthreads();
  }
  return base;
}

// What the products need to know of token t, whose number is n.
__device__ __forceinline__ void put_token(const SelectArgs& a, int t, int n) {
  a.out.pos[t] = n;
  if (n < 0) return;
  const int64_t y = a.target[t];
  const bool known = y >= 0 && y < a.total;  // a target that is no word: loss and gradient say so
  a.out.index[n] = t;
  a.out.tgt[n] = known && y >= a.start && y < a.start + a.vocab ? static_cast<int>(y - a.start) : -1;
  if (a.gl) {
    a.out.gl[n] = known ? a.gl[t] : NAN;
    a.out.delta[n] = 0.0f;
    a.out.lse[n] = a.lse[t];
  } else {
    a.out.tlogit[n] = known ? 0.0f : NAN;
  }
}

struct PackArgs {
  const void* src;
  int64_t ld;
  const int* index;    // NULL: rows as they are
  const int* count;    // with index: rows that exist
  int rows, cols;      // source extents
  int rows_p, cols_p;  // packed extents, zeros outside the source
  uint16_t* dst;       // limbs one after the other
  int nlimb;
  int f16;             // fp16 limbs of the values times a power of two, else one bf16
  int amax;            // f16: which row of Tokens::amax
  const float* gl;     // not NULL: times the power of two below |gl| of the row's token, too
};

// Scales are held as exponents and applied by ldexp: with fp32's whole range in the inputs, 2^s, 2^-s and
// 2^(s + e) are past it.  s that brings m under 2^15, from m and from its exponent.
constexpr int kExpBias = 1024;
__device__ __forceinline__ int scale_of(float m) { return m > 0.0f ? 14 - exp_below(m) : 0; }
__device__ __forceinline__ int scale_of_exp(float biased) {
  return biased > 0.0f ? 14 - (static_cast<int>(biased) - kExpBias) : 0;
}

// the largest of a row of Tokens::amax; the whole block takes part
__device__ __forceinline__ float block_amax(const float* p, int n) {
  __shared__ float red[16];
  float m = 0.0f;
  for (int i = threadIdx.x; i < n; i += blockDim.x) m = fmaxf(m, p[i]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = red[0];
  for (int i = 1; i < static_cast<int>(blockDim.x >> 6); ++i) m = fmaxf(m, red[i]);
  return m;
}

struct AmaxArgs {
  const void *x, *w;
  int64_t ldx, ldw;
  int tokens, vocab, hidden;
  int want_x, want_w, want_xg;
  const int64_t* target;
  const float* gl;
  int64_t ignore;
  float* out;  // Tokens::amax
};

template <typename T>
__device__ __forceinline__ float amax8(const T* p, int c, int cols) {
  float v[8], m = 0.0f;
  load8(p, c, cols, v);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float y = fabsf(v[k]);
    m = fmaxf(m, y <= 3.402823466e38f ? y : 0.0f);  // the largest finite one
  }
  return m;
}

// Each block's share of the largest |X| (tokens that take part), |W|, and the exponent of |X| 2^e.
template <typename T>
__global__ void __launch_bounds__(256) amax_kernel(const AmaxArgs a) {
  __shared__ float red[4];
  const int per = (a.hidden + 7) / 8;
  float mx = 0.0f, mg = 0.0f, mw = 0.0f;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * 256;
  if (a.want_x || a.want_xg)
    for (int64_t i = first; i < static_cast<int64_t>(a.tokens) * per; i += step) {
      const int t = static_cast<int>(i / per), c = static_cast<int>(i - static_cast<int64_t>(t) * per) * 8;
      if (a.target[t] == a.ignore || (a.gl && a.gl[t] == 0.0f)) continue;
      const float m = amax8(static_cast<const T*>(a.x) + t * a.ldx, c, a.hidden);
      mx = fmaxf(mx, m);
      if (a.want_xg && m > 0.0f) mg = fmaxf(mg, static_cast<float>(exp_below(m) + exp_below(a.gl[t]) + kExpBias));
    }
  if (a.want_w)
    for (int64_t i = first; i < static_cast<int64_t>(a.vocab) * per; i += step) {
      const int t = static_cast<int>(i / per), c = static_cast<int>(i - static_cast<int64_t>(t) * per) * 8;
      mw = fmaxf(mw, amax8(static_cast<const T*>(a.w) + t * a.ldw, c, a.hidden));
    }
  float v[3] = {mx, mw, mg};
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v[k] = fmaxf(v[k], __shfl_xor(v[k], o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v[k];
    __syncthreads();
    if (threadIdx.x == 0) a.out[k * kAmaxBlocks + blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  }
}

// 8 columns of a row of src, `i`: which; f16: times 2^s
template <typename T>
__device__ __forceinline__ void pack8(const PackArgs& a, int64_t i, int rows, const int* index, int s2) {
  const int per = a.cols_p / 8;
  const int row = static_cast<int>(i / per), c = static_cast<int>(i - static_cast<int64_t>(row) * per) * 8;
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 0.0f;
  if (row < rows) {
    const T* s = static_cast<const T*>(a.src) + static_cast<int64_t>(index ? index[row] : row) * a.ld;
    if (c < a.cols) load8(s, c, a.cols, v);
  }
  uint16_t* o = a.dst + static_cast<int64_t>(row) * a.cols_p + c;
  u32x4 q;
  if (a.f16) {
    if (a.gl && row < rows) s2 += exp_below(a.gl[index[row]]);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = ldexpf(v[k], s2);
    for (int l = 0; l < a.nlimb; ++l) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        q[k] = pack_f16(v[2 * k], v[2 * k + 1]);
        v[2 * k] = (v[2 * k] - f16_lo(q[k])) * kLowUp;
        v[2 * k + 1] = (v[2 * k + 1] - f16_hi(q[k])) * kLowUp;
      }
      *reinterpret_cast<u32x4*>(o) = q;
      o += static_cast<int64_t>(a.rows_p) * a.cols_p;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = pack_bf16(v[2 * k], v[2 * k + 1]);
    *reinterpret_cast<u32x4*>(o) = q;
  }
}

// What undoes the scales 2^sx, 2^sw, 2^sg (one thread).
__device__ __forceinline__ void put_scales(int* scale, int sx, int sw, int sg) {
  scale[kScaleZ] = -sx - sw;
  scale[kScaleDx] = -kGradExp - sw;
  scale[kScaleDw] = -kGradExp - sg;
}

__global__ void __launch_bounds__(1024) select_kernel(const SelectArgs a, int amax_blocks) {
  const int n = select(a, [&](int t, int k) { put_token(a, t, k); });
  if (threadIdx.x == 0) *a.out.count = n;
  if (amax_blocks) {
    const float mx = block_amax(a.out.amax, amax_blocks), mw = block_amax(a.out.amax + kAmaxBlocks, amax_blocks),
                mg = block_amax(a.out.amax + 2 * kAmaxBlocks, amax_blocks);
    if (threadIdx.x == 0) put_scales(a.out.scale, scale_of(mx), scale_of(mw), scale_of_exp(mg));
  }
}

template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const PackArgs a, const float* amax, int amax_blocks) {
  const int rows = a.index ? *a.count : a.rows;
  int s2 = 0;
  if (a.f16) {
    const float m = block_amax(amax + a.amax * kAmaxBlocks, amax_blocks);
    s2 = a.amax == 2 ? scale_of_exp(m) : scale_of(m);
  }
  const int64_t n = static_cast<int64_t>(a.rows_p) * (a.cols_p / 8);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    pack8<T>(a, i, rows, a.index, s2);
}

// select and the packs in one launch, for few tokens: each of the first `tok_blocks` blocks numbers the
// tokens for itself (a round of 4096) and gathers a share of their rows, and the first one writes the
// numbers down; the others pack the weight (513 x 1000 x 5003 in fp32: forward 51.1 us, backward 100.7;
// 54.2 and 108.9 where every block numbered the tokens first).  x: hidden states for z, xg: for dW (fp16), w: the
// weight's first piece (0 rows: none).
constexpr int kFewTokens = 2048;

template <typename T>
__global__ void __launch_bounds__(1024) prepare_kernel(const SelectArgs a, const PackArgs x, const PackArgs xg,
                                                       const PackArgs w, int amax_blocks, int tok_blocks) {
  __shared__ int index[kFewTokens];
  if (static_cast<int>(blockIdx.x) >= tok_blocks) {
    const int s2 = w.f16 ? scale_of(block_amax(a.out.amax + kAmaxBlocks, amax_blocks)) : 0;
    const int64_t n = static_cast<int64_t>(w.rows_p) * (w.cols_p / 8), step = static_cast<int64_t>(gridDim.x - tok_blocks) * 1024;
    for (int64_t i = static_cast<int64_t>(blockIdx.x - tok_blocks) * 1024 + threadIdx.x; i < n; i += step)
      pack8<T>(w, i, w.rows, nullptr, s2);
    return;
  }
  const int count = select(a, [&](int t, int n) {
    if (n >= 0) index[n] = t;
    if (blockIdx.x == 0) put_token(a, t, n);
  });
  int s2[3] = {0, 0, 0};
  if (amax_blocks) {
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (k == 2 ? xg.rows_p > 0 : x.f16 != 0) {
        const float m = block_amax(a.out.amax + k * kAmaxBlocks, amax_blocks);
        s2[k] = k == 2 ? scale_of_exp(m) : scale_of(m);
      }
    if (blockIdx.x == 0 && threadIdx.x == 0) put_scales(a.out.scale, s2[0], s2[1], s2[2]);
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.out.count = count;
  const int64_t nx = static_cast<int64_t>(x.rows_p) * (x.cols_p / 8), ng = static_cast<int64_t>(xg.rows_p) * (xg.cols_p / 8);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 1024 + threadIdx.x; i < nx + ng;
       i += static_cast<int64_t>(tok_blocks) * 1024) {
    if (i < nx) pack8<T>(x, i, count, index, s2[0]);
    else pack8<T>(xg, i - nx, count, index, s2[2]);
  }
}

// (c, sum of 2^(x log2(e) - c)) of two sets of logits; an empty set (c = -inf) has the sum 0 (or NaN)
__device__ __forceinline__ float2 join2(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x), mb = m == -INFINITY ? 0.0f : m;
  return make_float2(m, a.y * __builtin_amdgcn_exp2f(a.x - mb) + b.y * __builtin_amdgcn_exp2f(b.x - mb));
}

// Joins the tiles' (c, sum): TB tokens a block, 256 / TB threads a token, four parts in flight a thread.
template <int TB>
__global__ void __launch_bounds__(256) join_kernel(const float2* part, int parts, int64_t ldpart, int tokens, Tokens o,
                                                   float* loss, float* lse, float* tlogit) {
  constexpr int NT = 256 / TB;
  __shared__ float2 red[NT][TB];
  const int t = blockIdx.x * TB + threadIdx.x % TB, k = threadIdx.x / TB;
  const int n = t < tokens ? o.pos[t] : -1;
  float2 v = make_float2(-INFINITY, 0.0f);
  if (n >= 0) {
    const float2* p = part + n;
    int i = k;
    for (; i + 3 * NT < parts; i += 4 * NT) {
      const float2 a = p[i * ldpart], b = p[(i + NT) * ldpart], c = p[(i + 2 * NT) * ldpart], d = p[(i + 3 * NT) * ldpart];
      v = join2(v, join2(join2(a, b), join2(c, d)));
    }
    for (; i < parts; i += NT) v = join2(v, p[i * ldpart]);
  }
  red[k][threadIdx.x % TB] = v;
#pragma unroll
  for (int half = NT / 2; half > 0; half >>= 1) {
    __syncthreads();
    if (k < half) red[k][threadIdx.x % TB] = join2(red[k][threadIdx.x % TB], red[k + half][threadIdx.x % TB]);
  }
  if (k == 0 && t < tokens) {
    const float m = red[0][threadIdx.x].x, s = red[0][threadIdx.x].y;
    const float l = n < 0 ? 0.0f : fmaf(m, kLn2, logf(s)), z = n < 0 ? 0.0f : o.tlogit[n];
    lse[t] = l;
    if (tlogit) tlogit[t] = z;
    if (loss) loss[t] = l - z;
  }
}

// grad_hidden = the sum of the splits' slabs, rounded; zeros where a token takes no part.  A row of dX is
// mostly its target's, whose g is near -gl: what that one number lost as a bf16 (up to 2^-8 of the row) is
// put back in fp32, from one row of W.
template <typename T>
__global__ void __launch_bounds__(256) round_kernel(const float* slab, int splits, int64_t stride, int64_t ldslab,
                                                    int tokens, int cols, const int* scale, const Tokens tok,
                                                    const T* w, int64_t ldw, T* out, int64_t ldo) {
  const int per = (cols + 7) / 8;
  const int64_t n = static_cast<int64_t>(tokens) * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int t = static_cast<int>(i / per), c = static_cast<int>(i - static_cast<int64_t>(t) * per) * 8;
    const int p = tok.pos[t];
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (p >= 0) {
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {  // four in flight
        float q[8];
        load_vec<8>(slab + s * stride + static_cast<int64_t>(p) * ldslab + c, q);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += q[k];
      }
      if (scale) {
        const int e2 = *scale + exp_below(tok.gl[p]);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = ldexpf(v[k], e2);
      }
      const float lost = w ? tok.delta[p] : 0.0f;
      if (lost != 0.0f) {
        float q[8];
        load8(w + static_cast<int64_t>(tok.tgt[p]) * ldw, c, cols, q);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = fmaf(lost, q[k], v[k]);
      }
    }
    store8(out + static_cast<int64_t>(t) * ldo, c, cols, v);
  }
}

// ------------------------------------------------------------------------------- plan
struct Plan {
  int f32;             // fp32 inputs
  int wide;            // backward: grad_weight in fp32 precision, from two fp16 limbs of g
  int limbs_in;        // of X and W
  int g_bf16;          // backward: bf16 of g (bf16 inputs): one, or two for dW of few tokens
  int g_arrays;        // backward: 16-bit arrays of g: the bf16, then the fp16 limbs
  int logits, dx;      // tiles of the products (kTiles); dW's goes by the piece
  int tokens_p, hidden_p;
  bool pack_w;
  int piece;      // vocabulary rows of a piece (multiple of 256)
  int pieces;
  int splits;     // dX: parts of a piece's k
  int parts;      // forward: (c, sum) pairs of a token
  int amax_blocks;
  // workspace offsets
  size_t tok, xp, xg, wp, part, g, slab, total;
};

constexpr size_t kPieceBytes = size_t(1) << 30;  // g of one piece, unless the caller says less

// W can be read where it lies: bf16 in 16-byte chunks that end with the row
bool w_direct(const DionXentDesc* d) {
  return d->dtype == DION_DTYPE_BF16 && d->hidden % 8 == 0 && d->ld_weight % 8 == 0 && !d->pack_weight;
}

// The tiles there are: rows x columns, and the columns of a wave (the logits leave one (max, sum) for
// each of them).
struct TileShape {
  int br, bc, wc;
};
constexpr TileShape kTiles[4] = {{64, 64, 32}, {64, 128, 64}, {128, 128, 64}, {256, 256, 128}};

// The largest tile, up to `most`, that makes `parts` x `rows` x `cols` into enough blocks for 256 CUs.  The
// tokens bound `most` for dX and dW, but not for the logits: under more than 32640 words a few tokens take
// tiles of 128 rows, from 48897 on of 256, most of them zeros: the logits' last line has what that
// costs.  Measured (us, tile 256 / 128 / 64x128 / 64; blocks of the first):
//   logits   8192 tokens x 32000 words, h 4096: 907 (2000 blocks) / 1074 / 1470 / 1767 at 4096 tokens;
//            122 (250) / 148 / 188 / 222 at 512;  106 (125) / 78 / 102 / 114 at 256;
//            91 / 60 / 55 / 68 at 128;  89 / 58 / 49 / 54 at 1
//   fp32, 154 of 513 tokens x 5003 words, h 1000: 135 / 78 / 68 / 71
//   dX       (splits of k make up for few tiles) 1759 / 2010 / 2720 / 3865 at 4096 tokens, 177 / 180 / 204 / 236
//            at 256, 164 / 132 / 144 / 146 at 128 (with their logits)
//   dW       324 / 330 / 388 / 417 at 512 tokens, 253 / 234 / 271 / 289 at 256, 65 / 45 / 38 / 35 where it
//            has 16 / 64 / 128 / 256 blocks (2000 words, h 512; all with their logits)
int pick_tile(long rows, long cols, long parts, int most) {
  const long blocks[4] = {0, 128, 256, 192};
  for (int t = most; t > 0; --t)
    if (ceil_div(rows, kTiles[t].br) * ceil_div(cols, kTiles[t].bc) * parts >= blocks[t]) return t;
  return 0;
}

Plan make_plan(const DionXentDesc* d, int op) {
  Plan p;
  memset(&p, 0, sizeof(p));
  p.f32 = d->dtype == DION_DTYPE_F32;
  p.wide = op == DION_XENT_BACKWARD && (p.f32 || d->gw_dtype == DION_DTYPE_F32);
  p.limbs_in = p.f32 ? 2 : 1;
  p.g_bf16 = p.f32 ? 0 : !p.wide && d->tokens <= 256 ? 2 : 1;
  p.g_arrays = p.g_bf16 + (p.wide ? 2 : 0);
  p.logits = pick_tile(d->tokens, d->vocab, 1, 3);
  p.dx = pick_tile(d->tokens, d->hidden, ceil_div(d->vocab, 256), d->tokens >= 256 ? 3 : d->tokens > 64 ? 2 : 1);
  const int br = kTiles[p.logits].br > kTiles[p.dx].br ? kTiles[p.logits].br : kTiles[p.dx].br;
  p.tokens_p = static_cast<int>(round_up(d->tokens, br));
  p.hidden_p = static_cast<int>(round_up(d->hidden, kBK));
  p.pack_w = p.f32 || !w_direct(d);
  const long vocab_p = round_up(d->vocab, 256);
  long piece = vocab_p;
  if (op == DION_XENT_BACKWARD) {
    const size_t most = d->piece_bytes > 0 ? static_cast<size_t>(d->piece_bytes) : kPieceBytes;
    piece = static_cast<long>(most / (static_cast<size_t>(p.g_arrays) * p.tokens_p * 2)) / 256 * 256;
    if (p.pack_w && piece > 32768) piece = 32768;
  } else {
    // a grid's axis has to stay below 2^32 threads: 2^22 tiles at most, of 256 x 256 by 512
    piece = (1L << 38) / p.tokens_p / 256 * 256;
    if (p.pack_w && piece > 32768) piece = 32768;
  }
  if (piece < 256) piece = 256;
  if (piece > vocab_p) piece = vocab_p;
  // whole rounds of dW's 256 x 256 tiles over 256 CUs, where a piece has one
  const long in_round = 256 / ceil_div(d->hidden, 256) * 256;
  if (op == DION_XENT_BACKWARD && in_round > 0 && piece > in_round && piece < vocab_p) piece = piece / in_round * in_round;
  p.piece = static_cast<int>(piece);
  p.pieces = static_cast<int>(ceil_div(d->vocab, p.piece));
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  const size_t tp = static_cast<size_t>(p.tokens_p);
  p.tok = take(512 + 3 * kAmaxBlocks * sizeof(float) + 7 * tp * 4);
  p.xp = take(static_cast<size_t>(p.limbs_in) * tp * p.hidden_p * 2);
  if (p.wide) p.xg = take(static_cast<size_t>(p.limbs_in) * tp * p.hidden_p * 2);
  if (p.f32 || p.wide) {
    const long units = (d->tokens + (p.f32 ? d->vocab : 0)) * ceil_div(d->hidden, 8);
    p.amax_blocks = static_cast<int>(units > kAmaxBlocks * 1024L ? kAmaxBlocks : ceil_div(units, 1024));
  }
  if (p.pack_w) p.wp = take(static_cast<size_t>(p.limbs_in) * p.piece * p.hidden_p * 2);
  if (op == DION_XENT_FORWARD) {
    p.parts = p.pieces * (p.piece / kTiles[p.logits].wc);
    p.part = take(static_cast<size_t>(p.parts) * tp * sizeof(float2));
  } else {
    const TileShape t = kTiles[p.dx];
    const long tiles = ceil_div(d->tokens, t.br) * ceil_div(d->hidden, t.bc);
    const long want = (t.br == 256 ? 256 : t.br == 128 ? 512 : 1024) / tiles;  // as many blocks as fit at once
    const long most = p.piece / 256;
    p.splits = static_cast<int>(want < 1 ? 1 : want > most ? most : want);
    p.g = take(static_cast<size_t>(p.g_arrays) * tp * p.piece * 2);
    p.slab = take(static_cast<size_t>(p.splits) * tp * p.hidden_p * 4);
  }
  p.total = at;
  return p;
}

// limb pairs (i, j) of a product, the small ones first
void segments(GemmArgs* a, const uint16_t* r, size_t rstride, int rlimbs, const uint16_t* c, size_t cstride, int climbs) {
  a->nseg = 0;
  const int most = rlimbs > climbs ? rlimbs : climbs;
  for (int sum = most - 1; sum >= 0; --sum)
    for (int i = 0; i <= sum; ++i)
      if (i < rlimbs && sum - i < climbs) {
        a->r[a->nseg] = r + static_cast<size_t>(i) * rstride;
        a->c[a->nseg] = c + static_cast<size_t>(sum - i) * cstride;
        ++a->nseg;
      }
}

template <int BR, int BC, int WR, int WC, bool RKS, bool CKS, bool F16, int EPI, int NBUF, bool ONCE = false>
int launch_tile(GemmArgs a, long rows, long cols, hipStream_t st, const char* what) {
  a.row_tiles = static_cast<int>(ceil_div(rows, BR));
  a.col_tiles = static_cast<int>(ceil_div(cols, BC));
  constexpr int threads = 64 * (BR / WR) * (BC / WC);
  constexpr size_t lds = static_cast<size_t>(NBUF) * (BR + BC) * kBK * 2;
  auto* kernel = gemm_kernel<BR, BC, WR, WC, RKS, CKS, F16, EPI, NBUF, ONCE>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    if (e != hipSuccess) return fail(DION_E_LAUNCH, "hipFuncSetAttribute(%zu): %s", lds, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kernel, dim3(a.row_tiles * a.col_tiles, a.splits), dim3(threads), lds, st, a);
  return check_launch(what);
}

template <bool RKS, bool CKS, bool F16, int EPI>
int launch_as(int tile, const GemmArgs& a, long rows, long cols, hipStream_t st, const char* what) {
  switch (tile) {
    case 3: return launch_tile<256, 256, 64, 128, RKS, CKS, F16, EPI, 2>(a, rows, cols, st, what);
    case 2: return launch_tile<128, 128, 64, 64, RKS, CKS, F16, EPI, 2>(a, rows, cols, st, what);
    case 1:
      // The loss of up to 64 tokens alone: W passes by once, non-temporal.  One token under 32000 words of
      // 4096: 60.2 us against 64.5 where a gigabyte of other weights has been read since, 63.7 against 48.1
      // where the last-level cache still holds W.  The tokens alone choose it: a weight that the cache holds
      // from one call to the next pays, and so do limbs in the workspace, which the call has just written (fp32
      // reads the high one twice).  The backward pass reads W twice and keeps it.
      if constexpr (EPI == EPI_STATS)
        if (rows <= 64) return launch_tile<64, 128, 32, 64, RKS, CKS, F16, EPI, 3, true>(a, rows, cols, st, what);
      return launch_tile<64, 128, 32, 64, RKS, CKS, F16, EPI, 3>(a, rows, cols, st, what);
    default: return launch_tile<64, 64, 32, 32, RKS, CKS, F16, EPI, 3>(a, rows, cols, st, what);
  }
}
template <bool RKS, bool CKS, int EPI>
int launch(bool f16, int tile, const GemmArgs& a, long rows, long cols, hipStream_t st, const char* what) {
  return f16 ? launch_as<RKS, CKS, true, EPI>(tile, a, rows, cols, st, what)
             : launch_as<RKS, CKS, false, EPI>(tile, a, rows, cols, st, what);
}

Tokens tokens_at(char* ws, const Plan& p) {
  Tokens t;
  char* b = ws + p.tok;
  const size_t n = static_cast<size_t>(p.tokens_p);
  t.count = reinterpret_cast<int*>(b);
  t.scale = reinterpret_cast<int*>(b + 256);
  t.amax = reinterpret_cast<float*>(b + 512);
  t.pos = reinterpret_cast<int*>(t.amax + 3 * kAmaxBlocks);
  t.index = t.pos + n;
  t.tgt = t.index + n;
  t.lse = reinterpret_cast<float*>(t.tgt + n);
  t.gl = t.lse + n;
  t.tlogit = t.gl + n;
  t.delta = t.tlogit + n;
  return t;
}

PackArgs pack_args(const void* src, int64_t ld, const int* index, const int* count, int rows, int cols, int rows_p,
                   int cols_p, uint16_t* dst, int nlimb, bool f16, int amax, const float* gl) {
  PackArgs a;
  memset(&a, 0, sizeof(a));
  a.src = src;
  a.ld = ld;
  a.index = index;
  a.count = count;
  a.rows = rows;
  a.cols = cols;
  a.rows_p = rows_p;
  a.cols_p = cols_p;
  a.dst = dst;
  a.nlimb = nlimb;
  a.f16 = f16;
  a.amax = amax;
  a.gl = gl;
  return a;
}

int pack(const PackArgs& a, const Tokens& tok, const Plan& p, hipStream_t st, const char* what) {
  const long blocks = ceil_div(static_cast<long>(a.rows_p) * (a.cols_p / 8), 256);
  const dim3 grid(blocks < 8192 ? blocks : 8192);
  if (p.f32) hipLaunchKernelGGL(pack_kernel<float>, grid, dim3(256), 0, st, a, tok.amax, p.amax_blocks);
  else hipLaunchKernelGGL(pack_kernel<bf16>, grid, dim3(256), 0, st, a, tok.amax, p.amax_blocks);
  return check_launch(what);
}

// The limbs of the weight's rows v0 .. v0 + n in the workspace.
PackArgs weight_args(const DionXentDesc* d, const Plan& p, const void* weight, int v0, int n, char* ws) {
  const char* src = static_cast<const char*>(weight) +
                    static_cast<int64_t>(v0) * d->ld_weight * (d->dtype == DION_DTYPE_F32 ? 4 : 2);
  return pack_args(src, d->ld_weight, nullptr, nullptr, n, d->hidden, p.piece, p.hidden_p,
                   reinterpret_cast<uint16_t*>(ws + p.wp), p.limbs_in, p.f32, 1, nullptr);
}

// Numbers the tokens, gathers their hidden states, and packs the weight's first piece where it has to be.
int prepare(const DionXentDesc* d, const Plan& p, const void* hidden, const void* weight, const int64_t* target,
            const float* lse, const float* gl, const Tokens& tok, char* ws, hipStream_t st) {
  SelectArgs a;
  memset(&a, 0, sizeof(a));
  a.target = target;
  a.lse = lse;
  a.gl = gl;
  a.tokens = static_cast<int>(d->tokens);
  a.ignore = d->ignore_index;
  a.start = d->vocab_start;
  a.vocab = d->vocab;
  a.total = d->vocab_total;
  a.out = tok;
  if (p.amax_blocks) {
    AmaxArgs m;
    memset(&m, 0, sizeof(m));
    m.x = hidden;
    m.w = weight;
    m.ldx = d->ld_hidden;
    m.ldw = d->ld_weight;
    m.tokens = a.tokens;
    m.vocab = d->vocab;
    m.hidden = d->hidden;
    m.want_x = m.want_w = p.f32;
    m.want_xg = p.wide;
    m.target = target;
    m.gl = gl;
    m.ignore = d->ignore_index;
    m.out = tok.amax;
    if (p.f32) hipLaunchKernelGGL(amax_kernel<float>, dim3(p.amax_blocks), dim3(256), 0, st, m);
    else hipLaunchKernelGGL(amax_kernel<bf16>, dim3(p.amax_blocks), dim3(256), 0, st, m);
    const int rc = check_launch("xent(amax)");
    if (rc != DION_OK) return rc;
  }
  const PackArgs x = pack_args(hidden, d->ld_hidden, tok.index, tok.count, p.tokens_p, d->hidden, p.tokens_p,
                               p.hidden_p, reinterpret_cast<uint16_t*>(ws + p.xp), p.limbs_in, p.f32, 0, nullptr);
  PackArgs xg, w;
  memset(&xg, 0, sizeof(xg));
  memset(&w, 0, sizeof(w));
  xg.cols_p = w.cols_p = 8;
  if (p.wide) {
    xg = x;
    xg.dst = reinterpret_cast<uint16_t*>(ws + p.xg);
    xg.f16 = 1;
    xg.amax = 2;
    xg.gl = gl;
  }
  if (p.pack_w) w = weight_args(d, p, weight, 0, d->vocab < p.piece ? d->vocab : p.piece, ws);
  if (d->tokens <= kFewTokens) {
    const long xb = ceil_div(static_cast<long>(x.rows_p + xg.rows_p) * (x.cols_p / 8), 1024);
    const long wb = ceil_div(static_cast<long>(w.rows_p) * (w.cols_p / 8), 1024);
    const int tb = static_cast<int>(xb < 512 ? xb : 512);  // as many as run at once: each numbers the tokens first
    const dim3 grid(tb + (wb < 2048 ? wb : 2048));
    if (p.f32) hipLaunchKernelGGL(prepare_kernel<float>, grid, dim3(1024), 0, st, a, x, xg, w, p.amax_blocks, tb);
    else hipLaunchKernelGGL(prepare_kernel<bf16>, grid, dim3(1024), 0, st, a, x, xg, w, p.amax_blocks, tb);
    return check_launch("xent(prepare)");
  }
  hipLaunchKernelGGL(select_kernel, dim3(1), dim3(1024), 0, st, a, p.amax_blocks);
  int rc = check_launch("xent(select)");
  if (rc == DION_OK) rc = pack(x, tok, p, st, "xent(pack hidden)");
  if (rc == DION_OK && p.wide) rc = pack(xg, tok, p, st, "xent(pack hidden for dW)");
  if (rc == DION_OK && p.pack_w) rc = pack(w, tok, p, st, "xent(pack weight)");
  return rc;
}

// The W operand of a piece that starts at row v0: where it lies, or its limbs in the workspace (the
// first piece's are there already).
int piece_w(const DionXentDesc* d, const Plan& p, const void* weight, int v0, int n, const Tokens& tok, char* ws,
            const uint16_t** w, int64_t* ld, size_t* stride, hipStream_t st) {
  if (!p.pack_w) {
    *w = static_cast<const uint16_t*>(weight) + static_cast<int64_t>(v0) * d->ld_weight;
    *ld = d->ld_weight;
    *stride = 0;
    return DION_OK;
  }
  *w = reinterpret_cast<uint16_t*>(ws + p.wp);
  *ld = p.hidden_p;
  *stride = static_cast<size_t>(p.piece) * p.hidden_p;
  return v0 == 0 ? DION_OK : pack(weight_args(d, p, weight, v0, n, ws), tok, p, st, "xent(pack weight)");
}

void logits_args(GemmArgs* a, const DionXentDesc* d, const Plan& p, const uint16_t* x, const uint16_t* w, int64_t ldw,
                 size_t wstride, int v0, int n, const Tokens& tok) {
  memset(a, 0, sizeof(*a));
  segments(a, x, static_cast<size_t>(p.tokens_p) * p.hidden_p, p.limbs_in, w, wstride, p.limbs_in);
  a->ldr = p.hidden_p;
  a->ldc = ldw;
  a->cols = n;
  a->k = p.pack_w ? p.hidden_p : d->hidden;
  a->n_valid = tok.count;
  a->rows = p.tokens_p;
  a->splits = 1;
  a->tgt = tok.tgt;
  a->col0 = v0;
  a->scale = p.f32 ? tok.scale + kScaleZ : nullptr;
}

int forward(const DionXentDesc* d, const void* hidden, const void* weight, const int64_t* target, float* loss,
            float* lse, float* tlogit, char* ws, hipStream_t st) {
  const Plan p = make_plan(d, DION_XENT_FORWARD);
  const Tokens tok = tokens_at(ws, p);
  uint16_t* x = reinterpret_cast<uint16_t*>(ws + p.xp);
  int rc = prepare(d, p, hidden, weight, target, nullptr, nullptr, tok, ws, st);
  if (rc != DION_OK) return rc;
  float2* part = reinterpret_cast<float2*>(ws + p.part);
  for (int v0 = 0; v0 < d->vocab; v0 += p.piece) {
    const int n = d->vocab - v0 < p.piece ? d->vocab - v0 : p.piece;
    const uint16_t* w;
    int64_t ldw;
    size_t stride;
    rc = piece_w(d, p, weight, v0, n, tok, ws, &w, &ldw, &stride, st);
    if (rc != DION_OK) return rc;
    GemmArgs a;
    logits_args(&a, d, p, x, w, ldw, stride, v0, n, tok);
    a.part = part;
    a.ldpart = p.tokens_p;
    a.tlogit = tok.tlogit;
    rc = launch<false, false, EPI_STATS>(p.f32, p.logits, a, d->tokens, n, st, "xent(logits)");
    if (rc != DION_OK) return rc;
  }
  // tiles that exist, the last piece's ragged one among them
  const int parts = static_cast<int>(ceil_div(d->vocab, kTiles[p.logits].bc)) * (kTiles[p.logits].bc / kTiles[p.logits].wc);
  // neighbouring tokens share cache lines, but few tokens need all the threads
#define DION_JOIN(TB)                                                                                      \
  hipLaunchKernelGGL(join_kernel<TB>, dim3(ceil_div(d->tokens, TB)), dim3(256), 0, st, part, parts,        \
                     static_cast<int64_t>(p.tokens_p), static_cast<int>(d->tokens), tok, loss, lse, tlogit)
  if (d->tokens >= 4096) DION_JOIN(16);
  else if (d->tokens >= 512) DION_JOIN(8);
  else DION_JOIN(1);
#undef DION_JOIN
  return check_launch("xent(join)");
}

int backward(const DionXentDesc* d, const void* hidden, const void* weight, const int64_t* target, const float* lse,
             const float* grad_loss, void* grad_hidden, void* grad_weight, char* ws, hipStream_t st) {
  const Plan p = make_plan(d, DION_XENT_BACKWARD);
  const Tokens tok = tokens_at(ws, p);
  uint16_t* x = reinterpret_cast<uint16_t*>(ws + p.xp);
  uint16_t* g = reinterpret_cast<uint16_t*>(ws + p.g);
  float* slab = reinterpret_cast<float*>(ws + p.slab);
  const size_t gstride = static_cast<size_t>(p.tokens_p) * p.piece, xstride = static_cast<size_t>(p.tokens_p) * p.hidden_p;
  int rc = prepare(d, p, hidden, weight, target, lse, grad_loss, tok, ws, st);
  if (rc != DION_OK) return rc;
  const int gw_size = d->gw_dtype == DION_DTYPE_F32 ? 4 : 2;
  for (int v0 = 0; v0 < d->vocab; v0 += p.piece) {
    const int n = d->vocab - v0 < p.piece ? d->vocab - v0 : p.piece;
    const uint16_t* w;
    int64_t ldw;
    size_t stride;
    rc = piece_w(d, p, weight, v0, n, tok, ws, &w, &ldw, &stride, st);
    if (rc != DION_OK) return rc;
    GemmArgs a;
    logits_args(&a, d, p, x, w, ldw, stride, v0, n, tok);
    a.lse = tok.lse;
    a.gl = tok.gl;
    uint16_t* limbs = g + p.g_bf16 * gstride;  // fp16
    for (int l = 0; l < p.g_bf16; ++l) a.gb[l] = g + l * gstride;
    if (p.g_bf16) a.delta = tok.delta;
    for (int l = 0; p.wide && l < 2; ++l) a.gh[l] = limbs + l * gstride;
    a.ldg = p.piece;
    rc = launch<false, false, EPI_GRAD>(p.f32, p.logits, a, p.tokens_p, n, st, "xent(logit gradients)");
    if (rc != DION_OK) return rc;
    if (grad_hidden) {
      memset(&a, 0, sizeof(a));
      segments(&a, g, gstride, p.limbs_in, w, stride, p.limbs_in);
      a.ldr = p.piece;
      a.ldc = ldw;
      a.cols = p.pack_w ? p.hidden_p : d->hidden;
      a.k = n;
      a.n_valid = tok.count;
      a.rows = p.tokens_p;
      a.splits = p.splits;
      a.slab = slab;
      a.ldslab = p.hidden_p;
      a.slab_stride = static_cast<int64_t>(p.tokens_p) * p.hidden_p;
      a.add = v0 > 0;
      rc = launch<false, true, EPI_SLAB>(p.f32, p.dx, a, d->tokens, d->hidden, st, "xent(grad hidden)");
      if (rc != DION_OK) return rc;
    }
    if (grad_weight) {
      memset(&a, 0, sizeof(a));
      if (p.wide) segments(&a, limbs, gstride, 2, reinterpret_cast<uint16_t*>(ws + p.xg), xstride, p.limbs_in);
      else segments(&a, g, gstride, p.g_bf16, x, xstride, 1);
      a.scale = p.wide ? tok.scale + kScaleDw : nullptr;
      a.ldr = p.piece;
      a.ldc = p.hidden_p;
      a.cols = d->hidden;
      a.n_valid = tok.count;
      a.k_dev = 1;
      a.rows = n;
      a.splits = 1;
      a.add = d->accumulate;
      a.out = static_cast<char*>(grad_weight) + static_cast<int64_t>(v0) * d->ld_grad_weight * gw_size;
      a.ldo = d->ld_grad_weight;
      a.out_bf16 = gw_size == 2;
      a.out_vec = d->hidden % 4 == 0 && d->ld_grad_weight % 4 == 0 && aligned16(grad_weight);
      // tiles stay inside the piece of g (a multiple of 256 words): what lies past n there makes rows
      // that are not stored
      const int tile = pick_tile(n, d->hidden, 1, d->tokens >= 512 ? 3 : 2);
      rc = launch<true, true, EPI_OUT>(p.wide, tile, a, n, d->hidden, st, "xent(grad weight)");
      if (rc != DION_OK) return rc;
    }
  }
  if (grad_hidden) {
    const long blocks = ceil_div(d->tokens * ceil_div(d->hidden, 8), 256);
    const dim3 grid(blocks < 8192 ? blocks : 8192);
    const int64_t sstride = static_cast<int64_t>(p.tokens_p) * p.hidden_p;
    if (p.f32)
      hipLaunchKernelGGL(round_kernel<float>, grid, dim3(256), 0, st, slab, p.splits, sstride,
                         static_cast<int64_t>(p.hidden_p), static_cast<int>(d->tokens), d->hidden,
                         tok.scale + kScaleDx, tok, static_cast<const float*>(nullptr), int64_t(0),
                         static_cast<float*>(grad_hidden), d->ld_grad_hidden);
    else
      hipLaunchKernelGGL(round_kernel<bf16>, grid, dim3(256), 0, st, slab, p.splits, sstride,
                         static_cast<int64_t>(p.hidden_p), static_cast<int>(d->tokens), d->hidden,
                         static_cast<const int*>(nullptr), tok, static_cast<const bf16*>(weight), d->ld_weight,
                         static_cast<bf16*>(grad_hidden), d->ld_grad_hidden);
    rc = check_launch("xent(round grad hidden)");
  }
  return rc;
}

}  // namespace xent
