// lm_dropout.hpp -- out = residual + D(x), the mask made again from the counter wherever it is needed.
//
// Bytes per bf16 element: 2 read (4 with a residual), 2 written; 10 Philox rounds make the words of
// 4 elements (20 32x32->64-bit products and 40 exclusive ors, about 25 VALU cycles per element of
// a lane), which is near what the streams leave: the generator has to overlap the loads.  Measured on
// 8192 x 14336 bf16: 104-108 us (4.4-4.5 TB/s; a copy of 4 GiB reaches 4.77).  4 elements share a counter
// because Philox makes 4 words; 32 bits for each keep p exact to 2^-32.

struct DropoutArgs {
  const void *x, *residual;
  void* out;
  int64_t ldx, ldr, ldo;
  int64_t rows, cols;  // cols: elements of a row (vector kernel: one row of rows * cols if contiguous)
  DropArgs drop;
};

// 16-byte accesses at any alignment; grid y: rows; the ragged end of a row (cols % VEC) goes element by element
template <typename T, int VEC, bool RES>
__global__ void __launch_bounds__(256) dropout_vec_kernel(const DropoutArgs a) {
  const Key key = philox_key(a.drop);
  const int64_t nvec = a.cols / VEC;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* r = static_cast<const T*>(a.residual) + row * a.ldr;
    T* o = static_cast<T*>(a.out) + row * a.ldo;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i <= nvec;
         i += static_cast<int64_t>(gridDim.x) * 256) {
      if (i < nvec) {
        float v[VEC], q[VEC];
        load_vec<VEC>(x + i * VEC, v);
        if constexpr (RES) load_vec<VEC>(r + i * VEC, q);
        drop_groups<VEC>(v, static_cast<uint64_t>(row) * a.cols + i * VEC, key, a.drop);
        if constexpr (RES) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[k] = __fadd_rn(v[k], q[k]);
        }
        store_vec<VEC>(o + i * VEC, v);
      } else {
        for (int64_t c = nvec * VEC; c < a.cols; ++c) {
          float v = to_f32(x[c]);
          drop_one(&v, static_cast<uint64_t>(row) * a.cols + c, key, a.drop);
          if constexpr (RES) v = __fadd_rn(v, to_f32(r[c]));
          o[c] = from_f32<T>(v);
        }
      }
    }
  }
}

// rows that start within a group: a thread makes the words of 4 consecutive elements and walks over row ends
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_any_kernel(const DropoutArgs a) {
  const Key key = philox_key(a.drop);
  const int64_t n = a.rows * a.cols, groups = (n + 3) / 4;
  for (int64_t g = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; g < groups;
       g += static_cast<int64_t>(gridDim.x) * 256) {
    uint32_t w[4];
    philox4(key, static_cast<uint64_t>(g), w);
    int64_t row = 4 * g / a.cols, col = 4 * g - row * a.cols;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (4 * g + k < n) {
        float v = drop1(to_f32(static_cast<const T*>(a.x)[row * a.ldx + col]), w[k], a.drop);
        if constexpr (RES) v = __fadd_rn(v, to_f32(static_cast<const T*>(a.residual)[row * a.ldr + col]));
        static_cast<T*>(a.out)[row * a.ldo + col] = from_f32<T>(v);
        if (++col == a.cols) {
          col = 0;
          ++row;
        }
      }
    }
  }
}

namespace dropout {

template <typename T, bool RES>
int launch(DropoutArgs a, hipStream_t st) {
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  if (a.ldx == a.cols && a.ldo == a.cols && (!RES || a.ldr == a.cols)) {  // one long row
    a.cols *= a.rows;
    a.rows = 1;
    a.ldx = a.ldr = a.ldo = a.cols;
  }
  const bool vec = a.rows == 1 || a.cols % 4 == 0;  // every row starts with a group of 4 elements
  constexpr long kBlocks = 256 * 16;  // 16 blocks of 256 threads for each of 256 CUs, then a loop
  if (vec) {
    const long bx = ceil_div(a.cols / VEC + 1, 256), by = a.rows < 32768 ? a.rows : 32768;
    const long most = kBlocks / by > 1 ? kBlocks / by : 1;
    hipLaunchKernelGGL((dropout_vec_kernel<T, VEC, RES>), dim3(bx < most ? bx : most, by), dim3(256), 0, st, a);
  } else {
    const long b = ceil_div(ceil_div(a.rows * a.cols, 4), 256);
    hipLaunchKernelGGL((dropout_any_kernel<T, RES>), dim3(b < kBlocks ? b : kBlocks), dim3(256), 0, st, a);
  }
  return check_launch("dropout_add");
}

}  // namespace dropout
