// Dropout with a mask that is formed from counters (layers.hpp) and never
// stored: one pass that reads x and writes y.  The generator costs two
// 32x32-bit products a round for four elements; the pass is bound by memory
// for fp32 and close to the balance of the two for 16-bit types.
#include "layers.hpp"

namespace ppo {
namespace {

// A thread takes 16 bytes of a row (four columns in 32 bits, eight in 16), so
// that a wave's store is one run of whole lines; it goes past the L2, which y
// rarely fits (bf16 16384 x 8192 106 -> 90 us, fp32 8192 x 8192 94 -> 83, small
// ones as before).  A workgroup is kX threads along the columns by 256 / kX
// rows, so narrow rows fill it too.  Rows that start off 16 bytes keep their
// chunks: shifted words in, an unaligned store out (16384 x 8191 115 us; 290
// element by element).
template <class T, bool kVec>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, T* y, int64_t rows, int64_t cols,
                                                      const Dropout d, int tx_bits) {
  constexpr int kN = 16 / sizeof(T);
  const int tx = threadIdx.x & ((1 << tx_bits) - 1), ty = threadIdx.x >> tx_bits;
  const int64_t c = (((int64_t)blockIdx.x << tx_bits) + tx) * kN;
  if (c >= cols) return;
  const uint64_t seed = d.mode == 1 ? dropout_seed(d) : 0;
  const int64_t step = (int64_t)gridDim.y * (256 >> tx_bits);
  for (int64_t r = (int64_t)blockIdx.y * (256 >> tx_bits) + ty; r < rows; r += step) {
    const T* xr = x + r * cols + c;
    T* yr = y + r * cols + c;
    const uint64_t id = d.rows ? (uint64_t)d.rows[r] : (uint64_t)r;
    const int count = (int)min((int64_t)kN, cols - c);
    struct __attribute__((aligned(16))) Chunk { T v[kN]; } in;
    if (kVec) {
      in = *reinterpret_cast<const Chunk*>(xr);
    } else if (count == kN) {
      in = __builtin_bit_cast(Chunk, load16_shifted(reinterpret_cast<const char*>(xr)));
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) in.v[i] = i < count ? xr[i] : from_f32<T>(0.0f);
    }
    float v[kN / 4][4];
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i / 4][i % 4] = to_f32(in.v[i]);
#pragma unroll
    for (int q = 0; q < kN / 4; ++q) drop4(d, seed, id, (uint32_t)(c >> 2) + q, v[q]);
#pragma unroll
    for (int i = 0; i < kN; ++i) in.v[i] = from_f32<T>(v[i / 4][i % 4]);
    if (kVec) {
      __builtin_nontemporal_store(__builtin_bit_cast(v4f, in), reinterpret_cast<v4f*>(yr));
    } else if (count == kN) {
      *reinterpret_cast<v4i_any*>(yr) = __builtin_bit_cast(v4i, in);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (i < count) yr[i] = in.v[i];
    }
  }
}

}  // namespace
}  // namespace ppo

extern "C" int ppo_layer_dropout(const void* x, void* y, int dtype, int64_t rows, int64_t cols,
                                 const ppo_dropout* drop, void* stream_ptr) {
  using namespace ppo;
  if (!dtype_ok(dtype) || rows < 0 || cols < 0 || !drop || !(drop->p >= 0.0 && drop->p <= 1.0))
    return PPO_ERR_INVALID_ARG;
  if (rows == 0 || cols == 0) return PPO_OK;
  if (!x || !y) return PPO_ERR_INVALID_ARG;
  // (columns / 4 is a 32-bit counter; rows are only indexed)
  if (cols > ((int64_t)1 << 33) || rows > ((int64_t)1 << 46) / cols) return PPO_ERR_TOO_LARGE;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  const Dropout d = make_dropout(drop->p, drop->seed, drop->seed_at, drop->row_ids);
  const int64_t chunk = dtype == PPO_DTYPE_F32 ? 4 : 8, groups = div_up(cols, chunk);
  int bits = 0;
  while (bits < 8 && ((int64_t)1 << bits) < groups) ++bits;
  const int64_t bx = div_up(groups, (int64_t)1 << bits), by = div_up(rows, 256 >> bits);
  const dim3 grid((unsigned)bx, (unsigned)(by < 65535 ? by : 65535));
  return with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    const bool vec = cols % chunk == 0 && aligned16(x) && aligned16(y);
    if (vec)
      hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(256), 0, stream, (const T*)x, (T*)y,
                         rows, cols, d, bits);
    else
      hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(256), 0, stream, (const T*)x,
                         (T*)y, rows, cols, d, bits);
    return last_launch_status();
  });
}
