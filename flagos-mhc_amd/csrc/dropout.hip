// Dropout whose mask is a function of the element's index, never stored.
//
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", SC 2011): key = the 64-bit seed, counter = (index of the
// element's group of 8, the 64-bit offset).  The 128 bits of a group are 16
// bits for each of its elements, element 2j the low and 2j + 1 the high half
// of word j.  An element is kept where its 16 bits are at least threshold =
// round(p * 65536), so the probability of dropping is a multiple of 2^-16,
// and kept elements are multiplied by 65536 / (65536 - threshold): the
// expectation is exact for the probability in use.  16 bits an element
// instead of 32 halve the generator's work (10 rounds of two 32x32 products
// a group), which at 32 bits would exceed the time of reading and writing
// bf16 rows.  65536 x 7168 bf16: 358 us, 5.2 TB/s, bound by HBM; blocks in runs
// of one XCD (400 us interleaved over all eight).
#include "common.hpp"
#include "mhc_launch.hpp"

namespace mhc {
namespace {

struct DropArgs {
  const void* x;
  void* y;
  int64_t n;
  uint32_t threshold;
  float scale;
  uint64_t seed, offset;
  const uint64_t* state;  // device: (seed, offset) in their place, or null
};

__device__ __forceinline__ void philox10(uint64_t group, uint64_t seed, uint64_t offset, uint32_t (&c)[4]) {
  c[0] = (uint32_t)group;
  c[1] = (uint32_t)(group >> 32);
  c[2] = (uint32_t)offset;
  c[3] = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c[0] * 0xD2511F53u, p1 = (uint64_t)c[2] * 0xCD9E8D57u;
    c[0] = (uint32_t)(p1 >> 32) ^ c[1] ^ k0;
    c[1] = (uint32_t)p1;
    c[2] = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
    c[3] = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

__device__ __forceinline__ bool kept(const uint32_t (&c)[4], int j, uint32_t threshold) {
  return ((c[j >> 1] >> (16 * (j & 1))) & 0xffffu) >= threshold;
}

template <typename S>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a) {
  constexpr int VEC = Store<S>::VEC;
  const S* x = static_cast<const S*>(a.x);
  S* y = static_cast<S*>(a.y);
  uint64_t seed = a.seed, offset = a.offset;
  if (a.state) {
    seed = a.state[0];
    offset = a.state[1];
  }
  const int64_t full = a.n / 8, step = (int64_t)gridDim.x * 256;
  const int64_t first = xcd_contig(blockIdx.x, gridDim.x) * 256 + threadIdx.x;
  for (int64_t g = first; g < full; g += step) {
    u32x4 v[8 / VEC];
#pragma unroll
    for (int i = 0; i < 8 / VEC; ++i) v[i] = ld16nt_u(x + g * 8 + i * VEC);
    uint32_t c[4];
    philox10((uint64_t)g, seed, offset, c);
#pragma unroll
    for (int i = 0; i < 8 / VEC; ++i) {
      float f[VEC];
      Store<S>::unpack(v[i], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = kept(c, i * VEC + j, a.threshold) ? f[j] * a.scale : 0.f;
      st16nt_u(y + g * 8 + i * VEC, Store<S>::pack(f));
    }
  }
  if (first == 0 && a.n % 8) {  // the last, shorter group
    uint32_t c[4];
    philox10((uint64_t)full, seed, offset, c);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t i = full * 8 + j;
      if (i < a.n) store_elem<S>(y, i, kept(c, j, a.threshold) ? load_elem<S>(x, i) * a.scale : 0.f);
    }
  }
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" int mhc_dropout(const void* x, void* y, int64_t n, int32_t dtype, double p, uint64_t seed,
                           uint64_t offset, const uint64_t* state, void* stream) {
  clear_error();
  if (n < 0 || !(p >= 0.0 && p <= 1.0)) return set_error(MHC_ERR_INVALID, "dropout: n=%lld p=%g", (long long)n, p);
  if (dtype != MHC_DTYPE_F32 && dtype != MHC_DTYPE_BF16 && dtype != MHC_DTYPE_F16)
    return set_error(MHC_ERR_UNSUPPORTED, "dropout: dtype %d not supported", dtype);
  if (n == 0) return MHC_OK;
  if (!x || !y) return set_error(MHC_ERR_INVALID, "dropout: null pointer");
  const uint32_t thr = (uint32_t)(p * 65536.0 + 0.5);
  // threshold 65536: nothing is kept and the factor is not used
  const float scale = thr < 65536u ? (float)(65536.0 / (double)(65536u - thr)) : 0.f;
  const DropArgs a = {x, y, n, thr, scale, seed, offset, state};
  int64_t blocks = (n / 8 + 255) / 256;
  const int64_t most = (int64_t)device_cu_count() * 16;
  blocks = blocks < 1 ? 1 : (blocks > most ? most : blocks);
  const dim3 g((unsigned)blocks), b(256);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MHC_DTYPE_F32)
    hipLaunchKernelGGL(dropout_kernel<float>, g, b, 0, st, a);
  else if (dtype == MHC_DTYPE_BF16)
    hipLaunchKernelGGL(dropout_kernel<bf16_t>, g, b, 0, st, a);
  else
    hipLaunchKernelGGL(dropout_kernel<f16_t>, g, b, 0, st, a);
  return check_launch("dropout");
}
