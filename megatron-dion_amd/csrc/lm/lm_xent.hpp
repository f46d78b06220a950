// lm_xent.hpp -- the linear cross entropy: tokens that take part, limbs, the pieces of the vocabulary.
//
// forward   select -> pack X -> [pack W] logits tiles, each leaving (max, sum of exp) of its columns
//           for each token -> join them: lse, loss
// backward  select -> pack X -> for each piece of the vocabulary: [pack W], logits again, g = the
//           gradient of the logits to the workspace, dX += g W, dW = g^T X -> round dX
//
// Only tokens with a target (and, backward, a gradient) take part: select numbers them, pack X
// gathers their rows, and every product runs over that many.  What a hidden state without a target
// holds is never read.
//
// g is rounded to bf16 limbs for the matrix cores: one limb (2^-8) where all outputs are bf16, whose
// own rounding is as large; three (2^-24) for dW where grad_weight is fp32 (two, 2^-16, measured 2.6e-6 of
// its 2-norm, twice what an fp32 product is off) and for fp32 inputs, which are split into three limbs
// themselves (24 bits, the products kept down to 2^-24).

namespace xent {

struct Tokens {  // compact arrays, by the number a token has among those that take part
  int* count;    // [1]
  int* pos;      // [tokens]: number of a token, -1: takes no part
  int* index;    // [tokens_p]: token of a number
  int* tgt;      // [tokens_p]
  float* lse;    // [tokens_p] (backward)
  float* gl;     // [tokens_p] (backward)
  float* tlogit; // [tokens_p] (forward)
};

// One block: numbers the tokens that take part, in order.
__global__ void __launch_bounds__(1024) select_kernel(const int64_t* target, const float* lse, const float* gl,
                                                      int tokens, int64_t ignore, int64_t start, int64_t vocab,
                                                      int64_t total, Tokens o) {
  __shared__ int wsum[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0;
  for (int t0 = 0; t0 < tokens; t0 += 1024) {
    const int t = t0 + threadIdx.x;
    int64_t y = 0;
    float g = 0.0f;
    bool in = false;
    if (t < tokens) {
      y = target[t];
      in = y != ignore;
      if (gl) {
        g = gl[t];
        in = in && !(g == 0.0f);  // NaN takes part
      }
    }
    const uint64_t mask = __ballot(in);
    if (lane == 0) wsum[wave] = __popcll(mask);
    __syncthreads();
    int before = base, all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += wsum[w];
      all += wsum[w];
    }
    if (in) {
      const int n = before + __popcll(mask & ((1ull << lane) - 1));
      const bool known = y >= 0 && y < total;
      o.index[n] = t;
      o.tgt[n] = known && y >= start && y < start + vocab ? static_cast<int>(y - start) : -1;
      if (gl) {
        o.gl[n] = known ? g : NAN;  // a target that is no word: the gradient says so
        o.lse[n] = lse[t];
      } else {
        o.tlogit[n] = known ? 0.0f : NAN;
      }
    }
    if (t < tokens) o.pos[t] = in ? before + __popcll(mask & ((1ull << lane) - 1)) : -1;
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *o.count = base;
}

struct PackArgs {
  const void* src;
  int64_t ld;
  const int* index;    // NULL: rows as they are
  const int* count;    // with index: rows that exist
  int rows, cols;      // source extents
  int rows_p, cols_p;  // packed extents, zeros outside the source
  uint16_t* dst[3];
  int nlimb, vec;
};

// rows of src as bf16 limbs, 8 columns a thread
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const PackArgs a) {
  const int rows = a.index ? *a.count : a.rows;
  const int per = a.cols_p / 8;
  const int64_t n = static_cast<int64_t>(a.rows_p) * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int row = static_cast<int>(i / per), c = static_cast<int>(i - static_cast<int64_t>(row) * per) * 8;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.0f;
    if (row < rows) {
      const T* s = static_cast<const T*>(a.src) + static_cast<int64_t>(a.index ? a.index[row] : row) * a.ld + c;
      if (a.vec && c + 8 <= a.cols) {
        load_vec<8>(s, v);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c + k < a.cols) v[k] = to_f32(s[k]);
      }
    }
    for (int l = 0; l < a.nlimb; ++l) {
      u32x4 q;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        q[k] = pack_bf16(v[2 * k], v[2 * k + 1]);
        v[2 * k] -= __uint_as_float(q[k] << 16);
        v[2 * k + 1] -= __uint_as_float(q[k] & 0xFFFF0000u);
      }
      *reinterpret_cast<u32x4*>(a.dst[l] + static_cast<int64_t>(row) * a.cols_p + c) = q;
    }
  }
}

// Joins the tiles' (max, sum): 32 tokens a block, 8 threads a token.
__global__ void __launch_bounds__(256) join_kernel(const float2* part, int parts, int64_t ldpart, int tokens, Tokens o,
                                                   float* loss, float* lse, float* tlogit) {
  __shared__ float2 red[8][32];
  const int t = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
  const int n = t < tokens ? o.pos[t] : -1;
  float m = -INFINITY, s = 0.0f;
  if (n >= 0) {
    for (int i = k; i < parts; i += 8) {
      const float2 p = part[static_cast<int64_t>(i) * ldpart + n];
      const float mn = fmaxf(m, p.x), mb = mn == -INFINITY ? 0.0f : mn;
      s = s * __builtin_amdgcn_exp2f((m - mb) * kLog2e) + p.y * __builtin_amdgcn_exp2f((p.x - mb) * kLog2e);
      m = mn;
    }
  }
  red[k][threadIdx.x & 31] = make_float2(m, s);
  __syncthreads();
  if (k == 0 && t < tokens) {
    for (int i = 1; i < 8; ++i) {
      const float2 p = red[i][threadIdx.x & 31];
      const float mn = fmaxf(m, p.x), mb = mn == -INFINITY ? 0.0f : mn;
      s = s * __builtin_amdgcn_exp2f((m - mb) * kLog2e) + p.y * __builtin_amdgcn_exp2f((p.x - mb) * kLog2e);
      m = mn;
    }
    const float l = n < 0 ? 0.0f : m + logf(s), z = n < 0 ? 0.0f : o.tlogit[n];
    lse[t] = l;
    if (tlogit) tlogit[t] = z;
    if (loss) loss[t] = l - z;
  }
}

// grad_hidden = the sum of the splits' slabs, rounded; zeros where a token takes no part
template <typename T>
__global__ void __launch_bounds__(256) round_kernel(const float* slab, int splits, int64_t stride, int64_t ldslab,
                                                    const int* pos, int tokens, int cols, T* out, int64_t ldo) {
  const int per = static_cast<int>((cols + 3) / 4);
  const int64_t n = static_cast<int64_t>(tokens) * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int t = static_cast<int>(i / per), c = static_cast<int>(i - static_cast<int64_t>(t) * per) * 4;
    const int p = pos[t];
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p >= 0)
      for (int s = 0; s < splits; ++s)
        v += *reinterpret_cast<const f32x4*>(slab + s * stride + static_cast<int64_t>(p) * ldslab + c);
    T* o = out + static_cast<int64_t>(t) * ldo + c;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c + k < cols) o[k] = from_f32<T>(v[k]);
  }
}

// ------------------------------------------------------------------------------- plan
struct Plan {
  int limbs_in;   // of X and W
  int limbs_g;
  int br;         // tile rows of the logits and dX products: 32, 128 or 256
  int bc;         // tile columns: 128 or 256
  int tokens_p, hidden_p;
  bool pack_w;
  int piece;      // vocabulary rows of a piece (multiple of 256)
  int pieces;
  int splits;     // dX: parts of a piece's k
  int parts;      // forward: (max, sum) pairs of a token
  // workspace offsets
  size_t tok, xp, wp, part, g, slab, total;
};

constexpr size_t kPieceBytes = size_t(1) << 30;  // g of one piece, unless the caller says less

// W can be read where it lies: bf16 in 16-byte chunks that end with the row
bool w_direct(const DionXentDesc* d) {
  return d->dtype == DION_DTYPE_BF16 && d->hidden % 8 == 0 && d->ld_weight % 8 == 0 && !d->pack_weight;
}

Plan make_plan(const DionXentDesc* d, int op) {
  Plan p;
  memset(&p, 0, sizeof(p));
  const bool f32 = d->dtype == DION_DTYPE_F32;
  p.limbs_in = f32 ? 3 : 1;
  p.limbs_g = f32 || d->gw_dtype == DION_DTYPE_F32 ? 3 : 1;
  p.br = d->tokens <= 32 ? 32 : d->tokens <= 128 ? 128 : 256;
  p.bc = p.br == 256 ? 256 : 128;
  p.tokens_p = static_cast<int>(round_up(d->tokens, p.br < 64 ? 64 : p.br));
  p.hidden_p = static_cast<int>(round_up(d->hidden, kBK));
  p.pack_w = f32 || !w_direct(d);
  const long vocab_p = round_up(d->vocab, 256);
  long piece = vocab_p;
  if (op == DION_XENT_BACKWARD) {
    const size_t most = d->piece_bytes > 0 ? static_cast<size_t>(d->piece_bytes) : kPieceBytes;
    piece = static_cast<long>(most / (static_cast<size_t>(p.limbs_g) * p.tokens_p * 2)) / 256 * 256;
    if (p.pack_w && piece > 32768) piece = 32768;
  } else if (p.pack_w) {
    piece = 32768;
  }
  if (piece < 256) piece = 256;
  if (piece > vocab_p) piece = vocab_p;
  p.pieces = static_cast<int>(ceil_div(d->vocab, piece));
  p.piece = static_cast<int>(round_up(ceil_div(d->vocab, p.pieces), 256));  // pieces of like size
  p.pieces = static_cast<int>(ceil_div(d->vocab, p.piece));
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  const size_t tp = static_cast<size_t>(p.tokens_p);
  p.tok = take(256 + 6 * tp * 4);
  p.xp = take(static_cast<size_t>(p.limbs_in) * tp * p.hidden_p * 2);
  if (p.pack_w) p.wp = take(static_cast<size_t>(p.limbs_in) * p.piece * p.hidden_p * 2);
  if (op == DION_XENT_FORWARD) {
    const int per = p.bc / (p.br == 256 ? 128 : p.br == 128 ? 64 : 32);
    p.parts = static_cast<int>(p.pieces * (p.piece / p.bc)) * per;
    p.part = take(static_cast<size_t>(p.parts) * tp * sizeof(float2));
  } else {
    const long tiles = static_cast<long>(p.tokens_p / p.br > 0 ? p.tokens_p / p.br : 1) * ceil_div(d->hidden, p.bc);
    const long want = (p.br == 256 ? 256 : 1024) / (tiles < 1 ? 1 : tiles);  // one or four blocks a CU
    const long most = p.piece / 256;
    p.splits = static_cast<int>(want < 1 ? 1 : want > most ? most : want);
    p.g = take(static_cast<size_t>(p.limbs_g) * tp * p.piece * 2);
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

template <int BR, int BC, int WR, int WC, bool RKS, bool CKS, int EPI, int NBUF>
int launch_tile(GemmArgs a, long rows, long cols, hipStream_t st, const char* what) {
  a.row_tiles = static_cast<int>(ceil_div(rows, BR));
  a.col_tiles = static_cast<int>(ceil_div(cols, BC));
  constexpr int threads = 64 * (BR / WR) * (BC / WC);
  constexpr size_t lds = static_cast<size_t>(NBUF) * (BR + BC) * kBK * 2;
  auto* kernel = gemm_kernel<BR, BC, WR, WC, RKS, CKS, EPI, NBUF>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    if (e != hipSuccess) return fail(DION_E_LAUNCH, "hipFuncSetAttribute(%zu): %s", lds, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kernel, dim3(a.row_tiles * a.col_tiles, a.splits), dim3(threads), lds, st, a);
  return check_launch(what);
}

template <bool RKS, bool CKS, int EPI>
int launch(int br, const GemmArgs& a, long rows, long cols, hipStream_t st, const char* what) {
  if (br == 256) return launch_tile<256, 256, 64, 128, RKS, CKS, EPI, 2>(a, rows, cols, st, what);
  if (br == 128) return launch_tile<128, 128, 64, 64, RKS, CKS, EPI, 2>(a, rows, cols, st, what);
  if constexpr (!RKS) return launch_tile<32, 128, 32, 32, RKS, CKS, EPI, 3>(a, rows, cols, st, what);
  return fail(DION_E_INVALID, "%s: no tile", what);
}

Tokens tokens_at(char* ws, const Plan& p) {
  Tokens t;
  char* b = ws + p.tok;
  const size_t n = static_cast<size_t>(p.tokens_p);
  t.count = reinterpret_cast<int*>(b);
  t.pos = reinterpret_cast<int*>(b + 256);
  t.index = t.pos + n;
  t.tgt = t.index + n;
  t.lse = reinterpret_cast<float*>(t.tgt + n);
  t.gl = t.lse + n;
  t.tlogit = t.gl + n;
  return t;
}

int pack(const void* src, int dtype, int64_t ld, const int* index, const int* count, int rows, int cols, int rows_p,
         int cols_p, uint16_t* dst, int nlimb, hipStream_t st, const char* what) {
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
  for (int l = 0; l < nlimb; ++l) a.dst[l] = dst + static_cast<size_t>(l) * rows_p * cols_p;
  a.nlimb = nlimb;
  a.vec = aligned16(src) && ld % 8 == 0;
  const long blocks = ceil_div(static_cast<long>(rows_p) * (cols_p / 8), 256);
  const dim3 grid(blocks < 8192 ? blocks : 8192);
  if (dtype == DION_DTYPE_F32) hipLaunchKernelGGL(pack_kernel<float>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(pack_kernel<bf16>, grid, dim3(256), 0, st, a);
  return check_launch(what);
}

// The W operand of a piece that starts at row v0: where it lies, or its limbs in the workspace.
int piece_w(const DionXentDesc* d, const Plan& p, const void* weight, int v0, int n, char* ws, const uint16_t** w,
            int64_t* ld, size_t* stride, hipStream_t st) {
  if (!p.pack_w) {
    *w = static_cast<const uint16_t*>(weight) + static_cast<int64_t>(v0) * d->ld_weight;
    *ld = d->ld_weight;
    *stride = 0;
    return DION_OK;
  }
  uint16_t* dst = reinterpret_cast<uint16_t*>(ws + p.wp);
  const int esz = d->dtype == DION_DTYPE_F32 ? 4 : 2;
  const char* src = static_cast<const char*>(weight) + static_cast<int64_t>(v0) * d->ld_weight * esz;
  *w = dst;
  *ld = p.hidden_p;
  *stride = static_cast<size_t>(p.piece) * p.hidden_p;
  return pack(src, d->dtype, d->ld_weight, nullptr, nullptr, n, d->hidden, p.piece, p.hidden_p, dst, p.limbs_in, st,
              "xent(pack weight)");
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
}

int forward(const DionXentDesc* d, const void* hidden, const void* weight, const int64_t* target, float* loss,
            float* lse, float* tlogit, char* ws, hipStream_t st) {
  const Plan p = make_plan(d, DION_XENT_FORWARD);
  const Tokens tok = tokens_at(ws, p);
  uint16_t* x = reinterpret_cast<uint16_t*>(ws + p.xp);
  hipLaunchKernelGGL(select_kernel, dim3(1), dim3(1024), 0, st, target, nullptr, nullptr, static_cast<int>(d->tokens),
                     d->ignore_index, d->vocab_start, static_cast<int64_t>(d->vocab), d->vocab_total, tok);
  int rc = check_launch("xent(select)");
  if (rc != DION_OK) return rc;
  rc = pack(hidden, d->dtype, d->ld_hidden, tok.index, tok.count, p.tokens_p, d->hidden, p.tokens_p, p.hidden_p, x,
            p.limbs_in, st, "xent(pack hidden)");
  if (rc != DION_OK) return rc;
  float2* part = reinterpret_cast<float2*>(ws + p.part);
  for (int v0 = 0; v0 < d->vocab; v0 += p.piece) {
    const int n = d->vocab - v0 < p.piece ? d->vocab - v0 : p.piece;
    const uint16_t* w;
    int64_t ldw;
    size_t stride;
    rc = piece_w(d, p, weight, v0, n, ws, &w, &ldw, &stride, st);
    if (rc != DION_OK) return rc;
    GemmArgs a;
    logits_args(&a, d, p, x, w, ldw, stride, v0, n, tok);
    a.part = part;
    a.ldpart = p.tokens_p;
    a.tlogit = tok.tlogit;
    rc = launch<false, false, EPI_STATS>(p.br, a, d->tokens, n, st, "xent(logits)");
    if (rc != DION_OK) return rc;
  }
  // tiles that exist, the last piece's ragged one among them
  const int per = p.bc / (p.br == 256 ? 128 : p.br == 128 ? 64 : 32);
  const int parts = static_cast<int>(ceil_div(d->vocab, p.bc)) * per;
  hipLaunchKernelGGL(join_kernel, dim3(ceil_div(d->tokens, 32)), dim3(256), 0, st, part, parts,
                     static_cast<int64_t>(p.tokens_p), static_cast<int>(d->tokens), tok, loss, lse, tlogit);
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
  hipLaunchKernelGGL(select_kernel, dim3(1), dim3(1024), 0, st, target, lse, grad_loss, static_cast<int>(d->tokens),
                     d->ignore_index, d->vocab_start, static_cast<int64_t>(d->vocab), d->vocab_total, tok);
  int rc = check_launch("xent(select)");
  if (rc != DION_OK) return rc;
  rc = pack(hidden, d->dtype, d->ld_hidden, tok.index, tok.count, p.tokens_p, d->hidden, p.tokens_p, p.hidden_p, x,
            p.limbs_in, st, "xent(pack hidden)");
  if (rc != DION_OK) return rc;
  const int gw_size = d->gw_dtype == DION_DTYPE_F32 ? 4 : 2;
  for (int v0 = 0; v0 < d->vocab; v0 += p.piece) {
    const int n = d->vocab - v0 < p.piece ? d->vocab - v0 : p.piece;
    const uint16_t* w;
    int64_t ldw;
    size_t stride;
    rc = piece_w(d, p, weight, v0, n, ws, &w, &ldw, &stride, st);
    if (rc != DION_OK) return rc;
    GemmArgs a;
    logits_args(&a, d, p, x, w, ldw, stride, v0, n, tok);
    a.lse = tok.lse;
    a.gl = tok.gl;
    for (int l = 0; l < p.limbs_g; ++l) a.g[l] = g + l * gstride;
    a.nlimb = p.limbs_g;
    a.ldg = p.piece;
    rc = launch<false, false, EPI_GRAD>(p.br, a, p.tokens_p, n, st, "xent(logit gradients)");
    if (rc != DION_OK) return rc;
    if (grad_hidden) {
      memset(&a, 0, sizeof(a));
      segments(&a, g, gstride, d->dtype == DION_DTYPE_F32 ? 3 : 1, w, stride, p.limbs_in);
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
      rc = launch<false, true, EPI_SLAB>(p.br, a, d->tokens, d->hidden, st, "xent(grad hidden)");
      if (rc != DION_OK) return rc;
    }
    if (grad_weight) {
      memset(&a, 0, sizeof(a));
      segments(&a, g, gstride, p.limbs_g, x, xstride, p.limbs_in);
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
      // a piece of g is made of whole tiles, so its rows past n hold zeros; 256-row tiles stay inside it
      rc = launch<true, true, EPI_OUT>(p.br == 256 ? 256 : 128, a, n, d->hidden, st, "xent(grad weight)");
      if (rc != DION_OK) return rc;
    }
  }
  if (grad_hidden) {
    const long blocks = ceil_div(d->tokens * ceil_div(d->hidden, 4), 256);
    const dim3 grid(blocks < 8192 ? blocks : 8192);
    const int64_t sstride = static_cast<int64_t>(p.tokens_p) * p.hidden_p;
    if (d->dtype == DION_DTYPE_F32)
      hipLaunchKernelGGL(round_kernel<float>, grid, dim3(256), 0, st, slab, p.splits, sstride,
                         static_cast<int64_t>(p.hidden_p), tok.pos, static_cast<int>(d->tokens), d->hidden,
                         static_cast<float*>(grad_hidden), d->ld_grad_hidden);
    else
      hipLaunchKernelGGL(round_kernel<bf16>, grid, dim3(256), 0, st, slab, p.splits, sstride,
                         static_cast<int64_t>(p.hidden_p), tok.pos, static_cast<int>(d->tokens), d->hidden,
                         static_cast<bf16*>(grad_hidden), d->ld_grad_hidden);
    rc = check_launch("xent(round grad hidden)");
  }
  return rc;
}

}  // namespace xent
