// Dropout whose mask is recomputed instead of stored: y = keep ? x / (1 - p) : 0, keep from tsg_philox.h.  The backward is
// the same call on the gradient.  A dropped element is 0 whatever x holds there (a select, not a product).
//
// Bound: one read and one write of the tensor (HBM), against ten Philox rounds for four elements (20 32 x 32 -> 64 bit
// products, quarter rate).  40306 x 1280 f32: 74 us, 5.5 TB/s (a large device copy: 5.1); 16384 x 4096 bf16: 54 us, 5.0 TB/s; one
// pass over 251 x 306 is 3 us, all launch.
#include "tsg_philox.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

// Eight elements (two blocks) per thread: 16-byte accesses for the 16-bit types, two of them for f32.
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, T* __restrict__ y, long n, TsgRng r, int aligned) {
  const long i0 = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i0 >= n) return;
  const unsigned step = tsg_rng_step(r);
  const bool whole = aligned && i0 + 8 <= n;
  T v[8];
  if (whole) {
#pragma unroll
    for (int b = 0; b < (int)sizeof(T) * 8; b += 16)
      *reinterpret_cast<uint4*>(reinterpret_cast<char*>(v) + b) = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(x + i0) + b);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = i0 + e < n ? x[i0 + e] : (T)0.0f;
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint4 w = tsg_philox((unsigned long long)(i0 >> 2) + half, r.site, step, r.k0, r.k1);
    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool keep = u[e] >= r.threshold && !r.all;
      v[4 * half + e] = keep ? (T)((float)v[4 * half + e] * r.scale) : (T)0.0f;
    }
  }
  if (whole) {
#pragma unroll
    for (int b = 0; b < (int)sizeof(T) * 8; b += 16)
      *reinterpret_cast<uint4*>(reinterpret_cast<char*>(y + i0) + b) = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(v) + b);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i0 + e < n) y[i0 + e] = v[e];
  }
}

}  // namespace

extern "C" int tsg_dropout(const tsg_dropout_desc* d, void* stream) {
  if (!d || d->n < 0 || !(d->p >= 0.0 && d->p <= 1.0)) return TSG_E_INVALID;
  if (d->dtype != TSG_F32 && d->dtype != TSG_BF16 && d->dtype != TSG_F16) return TSG_E_INVALID;
  if (d->n == 0) return 0;
  if (!d->x || !d->y) return TSG_E_INVALID;
  const long blocks = (long)((d->n + 2047) / 2048);
  if (blocks > 0x7fffffffL) return TSG_E_LIMIT;
  const TsgRng r = tsg_make_rng(d->p, d->seed, d->site, d->step, d->step_dev);
  const int aligned = ((uintptr_t)d->x | (uintptr_t)d->y) % 16 == 0;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)blocks), block(256);
  if (d->dtype == TSG_F32)
    hipLaunchKernelGGL(dropout_kernel<float>, grid, block, 0, s, (const float*)d->x, (float*)d->y, (long)d->n, r, aligned);
  else if (d->dtype == TSG_BF16)
    hipLaunchKernelGGL(dropout_kernel<__bf16>, grid, block, 0, s, (const __bf16*)d->x, (__bf16*)d->y, (long)d->n, r, aligned);
  else
    hipLaunchKernelGGL(dropout_kernel<_Float16>, grid, block, 0, s, (const _Float16*)d->x, (_Float16*)d->y, (long)d->n, r, aligned);
  TSG_LAUNCH_CHECK();
  return 0;
}
