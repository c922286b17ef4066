// Softmax cross entropy over a large vocabulary from the states themselves: z_tv = h_t . w_v + b_v, loss_t = log sum_v
// exp(z_tv) - z_t,target, without the [rows][vocabulary] logits ever being kept.
//
// forward   products of 128 vocabulary rows x 128 states; their epilogue leaves (maximum, sum of exp) per state and
//           128 vocabulary rows, and the target's logit; a small kernel joins them.
// backward  the vocabulary is taken in pieces.  Per piece the products are computed once more, their epilogue turns them into
//           dz_tv = g_t (softmax_tv - [v == target_t]) in 16 bits, and two further products read that:
//           dW = dz^T h (whole for the piece) and dh += dz W (summed over the pieces in f32).  db comes from dz before
//           its rounding.  8 T V K operations instead of the 6 of a form that keeps the logits.
// Operands that run down a tile's rows (dz and h in dW, W in dh) are read through the transposing LDS loads, so nothing is
// ever stored a second time in another order.
//
// Types.  bf16 / f16 states and weights go to the matrix cores as they are.  f32 ones are carried as two f16 numbers,
// x 2^e = hi + lo with e from the tensor's largest magnitude (hi, lo: 22 bits together; an element 2^-18 below the
// largest still has them all), and a product is three passes, hi hi + hi lo + lo hi, summed in f32: the dropped term is
// 2^-22 relative, next to f32's own 2^-24 per addition, at a third of the f16 rate (833 TFLOP/s) against 157 of the f32
// matrix cores.  dz is rounded to the operand type (bf16: 2^-9 relative); for f16 and f32 it is scaled by 2^15 over the largest
// |g| first, so that probabilities down to 1e-9 stay above f16's subnormals; for f32 it is hi + lo as well.
// All sums, maxima and logarithms are f32.  Nothing depends on the order of workgroups: no floating-point atomics.
#include "tsg_mma.h"

namespace {

#ifndef V_TK
#define V_TK 64
#endif
constexpr int TM = 128, TN = 128, TK = V_TK;  // tile of a workgroup: four waves of 64 x 64

// 2^(15 - e) for 2^(e-1) <= v < 2^e: brings the largest magnitude into [2^14, 2^15)
__device__ __forceinline__ float scale_of(unsigned bits) {
  const float v = __uint_as_float(bits);
  if (!(v > 0.0f) || !(v < INFINITY)) return 1.0f;
  int e;
  frexpf(v, &e);
  int s = 15 - e;
  s = s > 126 ? 126 : (s < -126 ? -126 : s);
  return ldexpf(1.0f, s);
}

struct XentArgs {
  const char *h, *w;            // operands of the products (f32: their planes in the workspace)
  long h_row, w_row;            // bytes
  long h_plane, w_plane;        // bytes from hi to lo; 0 for 16-bit types
  const char* bias;             // in the caller's type, or null
  int bias_f32;
  const long* target;
  long ignore;
  int rows, hidden, vocab;
  int v0, vc;                   // this piece of the vocabulary
  const float* scales;          // f32: what h and w were multiplied by
  unsigned* gmax;               // backward: bits of the largest |g|
  float2* part;                 // forward: [vocab tiles][rows]
  float* zt;                    // forward: [rows] the target's logit
  float2* stat;                 // [rows] maximum, log2 of the sum
  float* g;                     // backward: [rows] gradient of the row's loss, 0 for rows left out
  unsigned long long* used;     // backward: bit t % 64 of word t / 64: g_t != 0
  char* dz;                     // [rows][ldz] 16-bit; f32: lo plane dz_plane further on
  long ldz, dz_plane;           // elements, bytes
  float* db_part;               // [row tiles][vc]
  float* dh_part;               // [splits][rows][hidden]
  int splits, split_len, first;
  char* dw;
  long dw_row;
};

struct Operand {
  const char* p;   // element (0, 0) of the workgroup's stretch
  long row, plane;
  int rows, cols;  // extent from there, in the order of memory (cols a multiple of 8)
  const unsigned long long* used;  // MASKED products: the memory rows (64 a word) that count
};

// acc[m][n] += A B over k in [0, K): AC / BC: the operand's memory rows are k.  passes: 1, or 3 with two planes each.
// MASKED: B's memory rows are read as zeros where its `used` bit is clear.
template <typename D, bool AC, bool BC, bool MASKED = false>
__device__ __forceinline__ void product(tsg_f32x16 (&acc)[2][2], char* lds, const Operand& a, const Operand& b, int K, int passes, int wave, int lane) {
  constexpr int TILE = TM * TK * 2;
  const int per = (K + TK - 1) / TK, steps = per * passes;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  // a wave's 64 rows or columns: rows lie 128 bytes apart, columns 2
  const unsigned a0 = tsg_lds_addr(lds) + (AC ? TsgLane<D, TM / 8>::col_in_order(lane) ^ (wm * 2) : TsgLane<D, TK / 8>::row(lane) + wm * TK * 2);
  const unsigned b0 = tsg_lds_addr(lds) + TILE + (BC ? TsgLane<D, TN / 8>::col_in_order(lane) ^ (wn * 2) : TsgLane<D, TK / 8>::row(lane) + wn * TK * 2);
  TsgLoader<AC ? TK : TM, (AC ? TM : TK) / 8, 4> al;
  TsgLoader<BC ? TK : TN, (BC ? TN : TK) / 8, 4> bl;
  // a tile whose memory rows are k is as wide as the operand is; one whose columns are k ends where k ends (its last step: below)
  al.init(a.row, AC ? a.cols / 8 : TK / 8, tsg_lds_addr(lds), wave, lane);
  bl.init(b.row, BC ? b.cols / 8 : TK / 8, tsg_lds_addr(lds) + TILE, wave, lane);
  auto fetch = [&](int pass, int k0, int buf) {
    const char* ap = a.p + (pass == 2 ? a.plane : 0);
    const char* bp = b.p + (pass == 1 ? b.plane : 0);
    if (!AC || !BC) {
      if (K - k0 < TK && K % TK) {  // the last, narrower step
        if (!AC) al.init(a.row, (a.cols - k0) / 8, tsg_lds_addr(lds), wave, lane);
        if (!BC) bl.init(b.row, (b.cols - k0) / 8, tsg_lds_addr(lds) + TILE, wave, lane);
      }
    }
    if (AC) al.load(ap + (long)k0 * a.row, a.rows - k0, a.cols * 2, buf * 2 * TILE);
    else al.load(ap + k0 * 2, a.rows, min(a.cols - k0, TK) * 2, buf * 2 * TILE);
    if (BC && MASKED) bl.load(bp + (long)k0 * b.row, b.rows - k0, b.cols * 2, buf * 2 * TILE, b.used[k0 / 64] >> (k0 % 64));
    else if (BC) bl.load(bp + (long)k0 * b.row, b.rows - k0, b.cols * 2, buf * 2 * TILE);
    else bl.load(bp + k0 * 2, b.rows, min(b.cols - k0, TK) * 2, buf * 2 * TILE);
    if (!AC || !BC) {
      if (K - k0 < TK && K % TK) {
        if (!AC) al.init(a.row, TK / 8, tsg_lds_addr(lds), wave, lane);
        if (!BC) bl.init(b.row, TK / 8, tsg_lds_addr(lds) + TILE, wave, lane);
      }
    }
  };
  int pass = 0, k0 = 0;
  if (steps) fetch(0, 0, 0);
  for (int step = 0, buf = 0; step < steps; ++step, buf ^= 1) {
    tsg_dma_wait();
    __syncthreads();
    if (step + 1 < steps) {
      k0 += TK;
      if (k0 >= K) k0 = 0, ++pass;
      fetch(pass, k0, buf ^ 1);
    }
    const unsigned at = tsg_opaque(a0) + buf * 2 * TILE, bt = tsg_opaque(b0) + buf * 2 * TILE;
#pragma unroll
    for (int s = 0; s < TK / 16; ++s) {
      tsg_u4 fa[2], fb[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        fa[x] = AC ? tsg_col_frag<TM / 8>(at, x, 16 * s * TM * 2) : tsg_row_frag<D>(at, s, 32 * x * TK * 2);
        fb[x] = BC ? tsg_col_frag<TN / 8>(bt, x, 16 * s * TN * 2) : tsg_row_frag<D>(bt, s, 32 * x * TK * 2);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) tsg_mma<D>(fa[x], fb[y], acc[x][y]);
    }
  }
  __syncthreads();  // the epilogue may use the tiles' memory
}

__device__ __forceinline__ void zero_acc(tsg_f32x16 (&acc)[2][2]) {
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[x][y][i] = 0.0f;
}

// Tile order: workgroup b runs on XCD b % 8; every XCD gets its own stretch of the tiles, walked in bands of eight column
// tiles, so that the 64 or so workgroups of an XCD share rows and columns in its L2.
__device__ __forceinline__ void tile_of(int b, int total, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int q = total / 8, r = total % 8, x = b % 8;
  const int id = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + b / 8;
  const int band = id / (8 * tiles_m), left = tiles_n - band * 8, wide = left < 8 ? left : 8, in = id - band * 8 * tiles_m;
  tm = in / wide;
  tn = band * 8 + in % wide;
}

// The two products over h and w have the vocabulary down the accumulator's rows and the states across its columns, so that a
// lane's 32 registers of a state are reduced without leaving the lane.
template <typename D> __device__ __forceinline__ void logits(const XentArgs& a, tsg_f32x16 (&acc)[2][2], char* lds, int m0, int n0, int wave, int lane, bool split) {
  zero_acc(acc);
  const Operand A = {a.w + (long)m0 * a.w_row, a.w_row, a.w_plane, a.vocab - m0, a.hidden, nullptr};
  const Operand B = {a.h + (long)n0 * a.h_row, a.h_row, a.h_plane, a.rows - n0, a.hidden, nullptr};
  product<D, false, false>(acc, lds, A, B, a.hidden, split ? 3 : 1, wave, lane);
  const int h = lane >> 5, wm = (wave >> 1) * 64;
  const float by = split ? 1.0f / (a.scales[0] * a.scales[1]) : 1.0f;
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int v = m0 + wm + 32 * x + (i & 3) + 8 * (i >> 2) + 4 * h;
      float b = 0.0f;
      if (a.bias && v < a.vocab) b = a.bias_f32 ? reinterpret_cast<const float*>(a.bias)[v] : (float)reinterpret_cast<const typename D::type*>(a.bias)[v];
#pragma unroll
      for (int y = 0; y < 2; ++y) acc[x][y][i] = v < a.vocab ? (split ? acc[x][y][i] * by : acc[x][y][i]) + b : -INFINITY;
    }
}

template <typename D>
__global__ __launch_bounds__(256, 2) void xent_stat_kernel(XentArgs a, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[4 * TM * TK * 2];
  __shared__ float2 join[2][TN];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
  tsg_f32x16 z[2][2];
  logits<D>(a, z, lds, tm * TM, tn * TN, wave, lane, a.h_plane != 0);
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const int n = wn + 32 * y + (lane & 31), t = tn * TN + n;
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, z[x][y][i]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float off = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    const long at = (t < a.rows ? a.target[t] : -1) - (tm * TM + wm + 4 * h);
    float zt = 0.0f;
    bool mine = false;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (at == 32 * x + (i & 3) + 8 * (i >> 2)) zt = z[x][y][i], mine = true;
        sum += __builtin_amdgcn_exp2f((z[x][y][i] - off) * 1.44269504088896340736f);
      }
    sum += __shfl_xor(sum, 32, 64);
    if (mine && t < a.rows && a.target[t] < a.vocab) a.zt[t] = zt;
    if (h == 0) join[wave >> 1][n] = make_float2(top, sum);
  }
  __syncthreads();
  const int n = threadIdx.x, t = tn * TN + n;
  if (n < TN && t < a.rows) {
    const float2 p = join[0][n], q = join[1][n];
    const float top = fmaxf(p.x, q.x), off = top == -INFINITY ? 0.0f : top;
    a.part[(long)tm * a.rows + t] = make_float2(top, p.y * __builtin_amdgcn_exp2f((p.x - off) * 1.44269504088896340736f) +
                                                         q.y * __builtin_amdgcn_exp2f((q.x - off) * 1.44269504088896340736f));
  }
}

// 32 states per workgroup, eight stretches of the vocabulary tiles
__global__ __launch_bounds__(256) void xent_join_kernel(XentArgs a, int tiles_m, float* loss) {
  __shared__ float2 join[8][32];
  const int n = threadIdx.x & 31, part = threadIdx.x >> 5, t = blockIdx.x * 32 + n;
  float top = -INFINITY, sum = 0.0f;
  if (t < a.rows)
    for (int m = part; m < tiles_m; m += 8) {
      const float2 p = a.part[(long)m * a.rows + t];
      const float to = fmaxf(top, p.x), off = to == -INFINITY ? 0.0f : to;
      sum = sum * __builtin_amdgcn_exp2f((top - off) * 1.44269504088896340736f) + p.y * __builtin_amdgcn_exp2f((p.x - off) * 1.44269504088896340736f);
      top = to;
    }
  join[part][n] = make_float2(top, sum);
  __syncthreads();
  if (part || t >= a.rows) return;
  top = -INFINITY;
  for (int p = 0; p < 8; ++p) top = fmaxf(top, join[p][n].x);
  const float off = top == -INFINITY ? 0.0f : top;
  sum = 0.0f;
  for (int p = 0; p < 8; ++p) sum += join[p][n].y * __builtin_amdgcn_exp2f((join[p][n].x - off) * 1.44269504088896340736f);
  const float l2 = __builtin_amdgcn_logf(sum);
  a.stat[t] = make_float2(off, l2);
  const long tg = a.target[t];
  float l = 0.0f;
  if (tg != a.ignore) l = tg >= 0 && tg < a.vocab ? (off - a.zt[t]) + l2 * 0.693147180559945309417f : NAN;
  loss[t] = l;
}

// sum or mean of the rows' losses, and the number of rows counted; one workgroup, f64 partial sums
__global__ __launch_bounds__(1024) void xent_reduce_kernel(XentArgs a, const float* loss, float* out, int mean) {
  __shared__ double s[16];
  __shared__ int c[16];
  double sum = 0.0;
  int n = 0;
  for (int t = threadIdx.x; t < a.rows; t += 1024) {
    if (out) sum += (double)loss[t];
    n += a.target[t] != a.ignore;
  }
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64), n += __shfl_xor(n, o, 64);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = sum, c[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) sum += s[w], n += c[w];
  if (out) *out = (float)(mean ? sum / (double)n : sum);
}

// g_t and the largest |g_t|, one workgroup.  reduction 0: d_loss per row; 1: one gradient for the sum; 2: for the mean
__global__ __launch_bounds__(1024) void xent_grad_kernel(XentArgs a, const float* d_loss, int reduction) {
  __shared__ float top[16];
  __shared__ int c[16];
  int n = 0;
  for (int t = threadIdx.x; t < a.rows; t += 1024) n += a.target[t] != a.ignore;
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if ((threadIdx.x & 63) == 0) c[threadIdx.x >> 6] = n;
  __syncthreads();
  n = 0;
  for (int w = 0; w < 16; ++w) n += c[w];
  float m = 0.0f;
  for (int t = threadIdx.x; t < (a.rows + 63) / 64 * 64; t += 1024) {  // whole waves: 64 rows a word of `used`
    const bool in = t < a.rows;
    const long tg = in ? a.target[t] : a.ignore;
    float g = !in ? 0.0f : reduction == 0 ? d_loss[t] : (reduction == 1 ? *d_loss : *d_loss / (float)n);
    if (tg == a.ignore) g = 0.0f;
    else if (tg < 0 || tg >= a.vocab) g = NAN;  // no such entry: the loss of this row was NaN
    if (in) a.g[t] = g;
    const unsigned long long used = __ballot(g != 0.0f);
    if ((threadIdx.x & 63) == 0) a.used[t >> 6] = used;
    m = fmaxf(m, fabsf(g));
  }
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) m = fmaxf(m, top[w]);
  *a.gmax = __float_as_uint(m);
}

template <typename D, bool SPLIT>
__global__ __launch_bounds__(256, 2) void xent_dz_kernel(XentArgs a, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[SPLIT || TK == 64 ? 4 * TM * 64 * 2 + 2 * 16 * TM : TN * (TM * 2 + 16)];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
  constexpr bool split = SPLIT;
  const int m0 = a.v0 + tm * TM;
  tsg_f32x16 z[2][2];
  logits<D>(a, z, lds, m0, tn * TN, wave, lane, split);
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  // rows of 128 entries, 16 bytes of padding: [128 states][272 bytes], hi and (f32) lo
  constexpr int ROW = TM * 2 + 16, PLANE = TN * ROW;
  const float gs = __is_same(D, TsgBf16) ? 1.0f : scale_of(*a.gmax);
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const int n = wn + 32 * y + (lane & 31), t = tn * TN + n;
    const bool in = t < a.rows;
    const float2 st = in ? a.stat[t] : make_float2(0.0f, INFINITY);
    const float g = in ? a.g[t] * gs : 0.0f;
    const long at = (in ? a.target[t] : -1) - (m0 + wm + 4 * h);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float d[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z[x][y][4 * q + r] - st.x, 1.44269504088896340736f, -st.y));
          d[r] = g == 0.0f ? 0.0f : (at == 32 * x + 8 * q + r ? p - 1.0f : p) * g;  // a row left out adds nothing, whatever it holds
          z[x][y][4 * q + r] = d[r];
        }
        char* to = lds + n * ROW + (wm + 32 * x + 8 * q + 4 * h) * 2;
        uint2 hi;
        hi.x = tsg_pack2<D>(d[0], d[1]);
        hi.y = tsg_pack2<D>(d[2], d[3]);
        *reinterpret_cast<uint2*>(to) = hi;
        if (split) {
          typedef typename D::type T;
          uint2 lo;
          lo.x = tsg_pack2<D>(d[0] - (float)(T)d[0], d[1] - (float)(T)d[1]);
          lo.y = tsg_pack2<D>(d[2] - (float)(T)d[2], d[3] - (float)(T)d[3]);
          *reinterpret_cast<uint2*>(to + PLANE) = lo;
        }
      }
  }
  float sums[32];
  if (a.db_part) {
    // sums over the states: 32 registers x 32 lanes -> one register per lane, halving both in every step
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[16 * x + i] = z[x][0][i] + z[x][1][i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < o; ++i) {
        const float keep = up ? sums[i + o] : sums[i], send = up ? sums[i] : sums[i + o];
        sums[i] = keep + __shfl_xor(send, o, 64);
      }
    }
  }
  __syncthreads();
  for (int p = 0; p < (split ? 2 : 1); ++p)
#pragma unroll
    for (int k = 0; k < TN * 16 / 256; ++k) {
      const int id = k * 256 + threadIdx.x, n = id >> 4, c = id & 15, t = tn * TN + n;
      if (t < a.rows)
        *reinterpret_cast<tsg_u4*>(a.dz + p * a.dz_plane + ((long)t * a.ldz + tm * TM + c * 8) * 2) =
            *reinterpret_cast<const tsg_u4*>(lds + p * PLANE + n * ROW + c * 16);
    }
  if (a.db_part) {
    __syncthreads();
    float* join = reinterpret_cast<float*>(lds);  // [2 column waves][128]
    const int r = lane & 31;  // the step that looked at bit o of the lane kept the registers with bit o set like it
    const int i = r & 15, x = r >> 4;
    join[(wave & 1) * TM + wm + 32 * x + (i & 3) + 8 * (i >> 2) + 4 * h] = sums[0];
    __syncthreads();
    const int v = tm * TM + threadIdx.x;
    if (threadIdx.x < TM && v < a.vc) a.db_part[(long)tn * a.vc + v] = join[threadIdx.x] + join[TM + threadIdx.x];
  }
}

// dW of the piece: rows v, columns k', summed over the states
template <typename D, typename OUT>
__global__ __launch_bounds__(256, 2) void xent_dw_kernel(XentArgs a, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[4 * TM * TK * 2];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
  const bool split = a.h_plane != 0;
  tsg_f32x16 acc[2][2];
  zero_acc(acc);
  const Operand A = {a.dz + (long)tm * TM * 2, a.ldz * 2, a.dz_plane, a.rows, (int)a.ldz - tm * TM, nullptr};
  const Operand B = {a.h + (long)tn * TN * 2, a.h_row, a.h_plane, a.rows, a.hidden - tn * TN, a.used};
  product<D, true, true, true>(acc, lds, A, B, a.rows, split ? 3 : 1, wave, lane);
  float by = __is_same(D, TsgBf16) ? 1.0f : 1.0f / scale_of(*a.gmax);
  if (split) by /= a.scales[0];
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int v = a.v0 + tm * TM + wm + 32 * x + (i & 3) + 8 * (i >> 2) + 4 * h, k = tn * TN + wn + 32 * y + (lane & 31);
        if (v < a.vocab && k < a.hidden) reinterpret_cast<OUT*>(a.dw + (long)v * a.dw_row)[k] = (OUT)(acc[x][y][i] * by);
      }
}

// dh: rows t, columns k', summed over a stretch of the piece; the stretches' sums are added up over the pieces
template <typename D>
__global__ __launch_bounds__(256, 2) void xent_dh_kernel(XentArgs a, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[4 * TM * TK * 2];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
  const int split_id = blockIdx.x / (tiles_m * tiles_n);
  int tm, tn;
  tile_of(blockIdx.x % (tiles_m * tiles_n), tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
  const bool split = a.h_plane != 0;
  const int c0 = split_id * a.split_len, len = min(a.split_len, a.vc - c0);
  tsg_f32x16 acc[2][2];
  zero_acc(acc);
  if (len > 0) {
    // ldz covers the piece up to a multiple of 128 with zeros, W ends at its last row: the shorter one decides
    const Operand A = {a.dz + ((long)tm * TM * a.ldz + c0) * 2, a.ldz * 2, a.dz_plane, a.rows - tm * TM, (len + 7) / 8 * 8, nullptr};
    const Operand B = {a.w + (long)(a.v0 + c0) * a.w_row + (long)tn * TN * 2, a.w_row, a.w_plane, len, a.hidden - tn * TN, nullptr};
    product<D, false, true>(acc, lds, A, B, len, split ? 3 : 1, wave, lane);
  }
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  float* out = a.dh_part + (long)split_id * a.rows * a.hidden;
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = tm * TM + wm + 32 * x + (i & 3) + 8 * (i >> 2) + 4 * h, k = tn * TN + wn + 32 * y + (lane & 31);
        if (t < a.rows && k < a.hidden) {
          float* p = out + (long)t * a.hidden + k;
          *p = a.first ? acc[x][y][i] : *p + acc[x][y][i];
        }
      }
}

template <typename OUT>
__global__ __launch_bounds__(256) void xent_dh_out_kernel(XentArgs a, OUT* dh, long dh_row, int scaled) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x, n = (long)a.rows * a.hidden;
  if (i >= n) return;
  float s = 0.0f;
  for (int p = 0; p < a.splits; ++p) s += a.dh_part[p * n + i];
  if (scaled) s /= scale_of(*a.gmax);
  if (a.h_plane) s /= a.scales[1];
  dh[(i / a.hidden) * dh_row + i % a.hidden] = (OUT)s;
}

template <typename OUT> __global__ __launch_bounds__(256) void xent_db_out_kernel(XentArgs a, OUT* db, int tiles_n, int scaled) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= a.vc) return;
  float s = 0.0f;
  for (int t = 0; t < tiles_n; ++t) s += a.db_part[(long)t * a.vc + v];
  if (scaled) s /= scale_of(*a.gmax);
  db[a.v0 + v] = (OUT)s;
}

// ---- f32 operands: largest magnitudes, then the two planes
__device__ __forceinline__ float4 row4(const float* x, long row, long i, int chunks) {
  return *reinterpret_cast<const float4*>(x + (i / chunks) * row + (i % chunks) * 4);
}
struct Planes {
  const float *h, *w;
  long h_row, n_h, w_row, n_w;
  int chunks, hb, wb;  // blocks [0, hb): h, hb + [0, wb): w
  float* amax;         // [hb + wb] a maximum per block
  const long* target;
  long ignore;
  char *hp, *wp;
  long h_plane, w_plane;
  float* scales;       // [2] the two scales, for the products and for the backward
};
__device__ __forceinline__ float block_max(float m, float* shared) {
  m = tsg_wave_max(m);
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = m;
  __syncthreads();
  return fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3]));
}
// rows of h that are left out may hold anything: they have no say
__global__ __launch_bounds__(256) void xent_amax_kernel(Planes a) {
  __shared__ float join[4];
  const bool first = (int)blockIdx.x < a.hb;
  const float* x = first ? a.h : a.w;
  const long row = first ? a.h_row : a.w_row, n = (first ? a.n_h : a.n_w) * a.chunks;
  const long b = first ? blockIdx.x : blockIdx.x - a.hb, nb = first ? a.hb : a.wb;
  float m = 0.0f;
  for (long i = b * 256 + threadIdx.x; i < n; i += nb * 256) {
    if (first && a.target[i / a.chunks] == a.ignore) continue;
    const float4 v = row4(x, row, i, a.chunks);
    m = fmaxf(m, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
  }
  m = block_max(m, join);
  if (threadIdx.x == 0) a.amax[blockIdx.x] = m;
}
// forward: the scales from the blocks' maxima (every block joins them itself); backward (amax null): as the forward left them
__global__ __launch_bounds__(256) void xent_planes_kernel(Planes a) {
  __shared__ float join[4];
  const bool first = (int)blockIdx.x < a.hb;
  const float* x = first ? a.h : a.w;
  const long row = first ? a.h_row : a.w_row, n = (first ? a.n_h : a.n_w) * a.chunks;
  const long b = first ? blockIdx.x : blockIdx.x - a.hb, nb = first ? a.hb : a.wb;
  char* out = first ? a.hp : a.wp;
  const long plane = first ? a.h_plane : a.w_plane;
  float by;
  if (a.amax) {
    const float* from = a.amax + (first ? 0 : a.hb);
    float m = 0.0f;
    for (int i = threadIdx.x; i < nb; i += 256) m = fmaxf(m, from[i]);
    by = scale_of(__float_as_uint(block_max(m, join)));
    if (b == 0 && threadIdx.x == 0) a.scales[first ? 0 : 1] = by;
  } else {
    by = a.scales[first ? 0 : 1];
  }
  for (long i = b * 256 + threadIdx.x; i < n; i += nb * 256) {
    const float4 v = row4(x, row, i, a.chunks);
    const float s[4] = {v.x * by, v.y * by, v.z * by, v.w * by};
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = s[e] - (float)(_Float16)s[e];
    uint2 hi, lo;
    hi.x = tsg_pack2<TsgF16>(s[0], s[1]), hi.y = tsg_pack2<TsgF16>(s[2], s[3]);
    lo.x = tsg_pack2<TsgF16>(r[0], r[1]), lo.y = tsg_pack2<TsgF16>(r[2], r[3]);
    *reinterpret_cast<uint2*>(out + i * 8) = hi;
    *reinterpret_cast<uint2*>(out + plane + i * 8) = lo;
  }
}

// ------------------------------------------------------------------------------------------------------ host side
struct Layout {
  size_t gmax, amax, planes, h_plane, w_plane, part, zt, g, used, dz, dz_plane, db, dh, total;
  int vc, splits, split_len;
};
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// dz of a piece takes at most `budget` bytes (but 128 vocabulary rows at least): large pieces fill the chip, small ones keep
// the workspace small.
constexpr int PLANE_BLOCKS = 512;
constexpr size_t DZ_BUDGET = (size_t)1 << 30;

Layout layout_of(const tsg_xent_desc* d, bool backward) {
  Layout l = {};
  const size_t T = (size_t)d->n_rows, V = (size_t)d->n_vocab, K = (size_t)d->hidden;
  const bool f32 = d->dtype == TSG_F32;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t p = at;
    at += up256(n);
    return p;
  };
  l.gmax = take(4);
  if (f32) {
    l.amax = take(2 * PLANE_BLOCKS * 4);
    l.h_plane = up256(T * K * 2), l.w_plane = up256(V * K * 2);
    l.planes = take(2 * (l.h_plane + l.w_plane));
  }
  if (!backward) {
    l.part = take((size_t)tsg_cdiv(V, TM) * T * 8);
    l.zt = take(T * 4);
  } else {
    const size_t each = f32 ? 4 : 2;
    size_t vc = DZ_BUDGET / (T * each) / TM * TM;
    if (vc < TM) vc = TM;
    const size_t all = (V + TM - 1) / TM * TM;
    if (vc > all) vc = all;
    if (vc > ((size_t)1 << 22)) vc = (size_t)1 << 22;  // 128 rows of dz stay below 2^31 bytes
    const size_t pieces = (all + vc - 1) / vc;  // even pieces
    vc = ((all + pieces - 1) / pieces + TM - 1) / TM * TM;
    l.vc = (int)vc;
    l.dz_plane = f32 ? up256(T * vc * 2) : 0;
    l.dz = take(f32 ? 2 * l.dz_plane : T * vc * 2);
    l.g = take(T * 4);
    l.used = take((T + 63) / 64 * 8);
    l.db = d->bias ? take((size_t)tsg_cdiv(T, TN) * vc * 4) : 0;
    const size_t tiles = (size_t)tsg_cdiv(T, TM) * tsg_cdiv(K, TN);
    size_t s = (512 + tiles - 1) / tiles;  // two workgroups a CU
    if (s > vc / TM) s = vc / TM;
    if (s < 1) s = 1;
    l.split_len = (int)(((vc + s - 1) / s + TK - 1) / TK * TK);
    l.splits = (int)((vc + l.split_len - 1) / l.split_len);
    l.dh = take((size_t)l.splits * T * K * 4);
  }
  l.total = at;
  return l;
}

int check_xent(const tsg_xent_desc* d, bool backward) {
  if (!d) return TSG_E_INVALID;
  if (d->dtype != TSG_F32 && d->dtype != TSG_BF16 && d->dtype != TSG_F16) return TSG_E_INVALID;
  if (d->n_rows < 0 || d->n_vocab <= 0 || d->hidden <= 0 || d->reduction < 0 || d->reduction > 2) return TSG_E_INVALID;
  if (d->n_rows > 0x7fffff00L || d->n_vocab > 0x7fffff00L) return TSG_E_LIMIT;
  if ((int64_t)tsg_cdiv(d->n_rows, TN) * tsg_cdiv(d->n_vocab, TM) > 0x7fffffffL) return TSG_E_LIMIT;
  if (d->n_rows * (int64_t)d->hidden > ((int64_t)1 << 38)) return TSG_E_LIMIT;
  if (d->hidden % 8) return TSG_E_INVALID;
  const int epc = d->dtype == TSG_F32 ? 4 : 8;
  if (!d->h || !d->w || !d->target || !d->stats || (uintptr_t)d->h % 16 || (uintptr_t)d->w % 16 || (uintptr_t)d->stats % 8) return TSG_E_INVALID;
  if (d->h_row < d->hidden || d->w_row < d->hidden || d->h_row % epc || d->w_row % epc) return TSG_E_INVALID;
  if (d->h_row * 4 >= (1 << 23) || d->w_row * 4 >= (1 << 23)) return TSG_E_LIMIT;  // offsets inside a tile are 32-bit
  if (!backward && !d->row_loss) return TSG_E_INVALID;
  if (!backward && d->reduction && !d->loss) return TSG_E_INVALID;
  if (d->dtype == TSG_F32 && !d->scales) return TSG_E_INVALID;
  if (backward && (!d->d_loss || !d->dh || !d->dw || (d->bias && !d->dbias))) return TSG_E_INVALID;
  if (backward && (d->dh_row < d->hidden || d->dw_row < d->hidden)) return TSG_E_INVALID;
  return 0;
}

XentArgs args_of(const tsg_xent_desc* d, const Layout& l) {
  XentArgs a = {};
  char* ws = (char*)d->workspace;
  const bool f32 = d->dtype == TSG_F32;
  a.gmax = (unsigned*)(ws + l.gmax);
  a.scales = d->scales;
  if (f32) {
    a.h = ws + l.planes, a.h_plane = (long)l.h_plane, a.h_row = d->hidden * 2L;
    a.w = ws + l.planes + 2 * l.h_plane, a.w_plane = (long)l.w_plane, a.w_row = d->hidden * 2L;
  } else {
    a.h = (const char*)d->h, a.w = (const char*)d->w, a.h_row = d->h_row * 2, a.w_row = d->w_row * 2;
  }
  a.bias = (const char*)d->bias, a.bias_f32 = f32;
  a.target = (const long*)d->target, a.ignore = d->ignore_index;
  a.rows = (int)d->n_rows, a.hidden = d->hidden, a.vocab = (int)d->n_vocab;
  a.stat = (float2*)d->stats;
  a.v0 = 0, a.vc = a.vocab;
  return a;
}

void make_planes(const tsg_xent_desc* d, const XentArgs& a, const Layout& l, bool backward, hipStream_t s) {
  Planes p;
  p.h = (const float*)d->h, p.w = (const float*)d->w, p.h_row = d->h_row, p.w_row = d->w_row, p.n_h = d->n_rows, p.n_w = d->n_vocab;
  p.chunks = d->hidden / 4;
  auto blocks = [&](int64_t n) {
    const int64_t b = (n * p.chunks + 1023) / 1024;
    return (int)(b > PLANE_BLOCKS ? PLANE_BLOCKS : b);
  };
  p.hb = blocks(p.n_h), p.wb = blocks(p.n_w);
  p.amax = backward ? nullptr : (float*)((char*)d->workspace + l.amax);
  p.target = (const long*)d->target, p.ignore = d->ignore_index;
  p.hp = (char*)a.h, p.wp = (char*)a.w, p.h_plane = a.h_plane, p.w_plane = a.w_plane;
  p.scales = d->scales;
  const dim3 grid((unsigned)(p.hb + p.wb));
  if (!backward) hipLaunchKernelGGL(xent_amax_kernel, grid, dim3(256), 0, s, p);
  hipLaunchKernelGGL(xent_planes_kernel, grid, dim3(256), 0, s, p);
}

template <typename D> void launch_stat(const XentArgs& a, int tm, int tn, hipStream_t s) {
  hipLaunchKernelGGL(xent_stat_kernel<D>, dim3((unsigned)(tm * tn)), dim3(256), 0, s, a, tm, tn);
}

template <typename D, typename OUT> void backward_piece(XentArgs a, const tsg_xent_desc* d, const Layout& l, hipStream_t s) {
  const int tv = tsg_cdiv(a.vc, TM), tt = tsg_cdiv(a.rows, TN), tk = tsg_cdiv(a.hidden, TN);
  const int scaled = !__is_same(D, TsgBf16);
  hipLaunchKernelGGL((xent_dz_kernel<D, __is_same(OUT, float)>), dim3((unsigned)(tv * tt)), dim3(256), 0, s, a, tv, tt);
  hipLaunchKernelGGL((xent_dw_kernel<D, OUT>), dim3((unsigned)(tv * tk)), dim3(256), 0, s, a, tv, tk);
  hipLaunchKernelGGL(xent_dh_kernel<D>, dim3((unsigned)(tt * tk * l.splits)), dim3(256), 0, s, a, tt, tk);
  if (d->bias) hipLaunchKernelGGL(xent_db_out_kernel<OUT>, dim3(tsg_cdiv(a.vc, 256)), dim3(256), 0, s, a, (OUT*)d->dbias, tt, scaled);
  if (a.v0 + a.vc >= a.vocab)
    hipLaunchKernelGGL(xent_dh_out_kernel<OUT>, dim3((unsigned)(((long)a.rows * a.hidden + 255) / 256)), dim3(256), 0, s, a, (OUT*)d->dh, (long)d->dh_row, scaled);
}

}  // namespace

extern "C" int tsg_xent_workspace(const tsg_xent_desc* d, size_t* forward_bytes_host, size_t* backward_bytes_host) {
  if (!d || !forward_bytes_host || !backward_bytes_host || d->n_rows < 0 || d->n_vocab <= 0 || d->hidden <= 0) return TSG_E_INVALID;
  *forward_bytes_host = d->n_rows ? layout_of(d, false).total : 0;
  *backward_bytes_host = d->n_rows ? layout_of(d, true).total : 0;
  return 0;
}

extern "C" int tsg_xent_forward(const tsg_xent_desc* d, void* stream) {
  const int rc = check_xent(d, false);
  if (rc) return rc;
  if (d->n_rows == 0) return TSG_E_INVALID;
  const Layout l = layout_of(d, false);
  if (!d->workspace || (uintptr_t)d->workspace % 256 || d->workspace_bytes < l.total) return TSG_E_TOO_SMALL;
  hipStream_t s = (hipStream_t)stream;
  XentArgs a = args_of(d, l);
  a.part = (float2*)((char*)d->workspace + l.part);
  a.zt = (float*)((char*)d->workspace + l.zt);
  if (d->dtype == TSG_F32) make_planes(d, a, l, false, s);
  const int tm = tsg_cdiv(a.vocab, TM), tn = tsg_cdiv(a.rows, TN);
  if (d->dtype == TSG_BF16) launch_stat<TsgBf16>(a, tm, tn, s);
  else launch_stat<TsgF16>(a, tm, tn, s);
  hipLaunchKernelGGL(xent_join_kernel, dim3(tsg_cdiv(a.rows, 32)), dim3(256), 0, s, a, tm, d->row_loss);
  if (d->reduction) hipLaunchKernelGGL(xent_reduce_kernel, dim3(1), dim3(1024), 0, s, a, (const float*)d->row_loss, d->loss, d->reduction == 2);
  TSG_LAUNCH_CHECK();
  return 0;
}

extern "C" int tsg_xent_backward(const tsg_xent_desc* d, void* stream) {
  const int rc = check_xent(d, true);
  if (rc) return rc;
  if (d->n_rows == 0) return TSG_E_INVALID;
  const Layout l = layout_of(d, true);
  if (!d->workspace || (uintptr_t)d->workspace % 256 || d->workspace_bytes < l.total) return TSG_E_TOO_SMALL;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)d->workspace;
  XentArgs a = args_of(d, l);
  a.g = (float*)(ws + l.g);
  a.used = (unsigned long long*)(ws + l.used);
  a.dz = ws + l.dz, a.dz_plane = (long)l.dz_plane;
  a.db_part = d->bias ? (float*)(ws + l.db) : nullptr;
  a.dh_part = (float*)(ws + l.dh);
  a.splits = l.splits, a.split_len = l.split_len;
  a.dw = (char*)d->dw, a.dw_row = d->dw_row * (d->dtype == TSG_F32 ? 4 : 2);
  a.ldz = l.vc;
  if (d->dtype == TSG_F32) make_planes(d, a, l, true, s);
  hipLaunchKernelGGL(xent_grad_kernel, dim3(1), dim3(1024), 0, s, a, d->d_loss, d->reduction);
  for (int64_t v0 = 0; v0 < d->n_vocab; v0 += l.vc) {
    a.v0 = (int)v0;
    a.vc = (int)(d->n_vocab - v0 < l.vc ? d->n_vocab - v0 : l.vc);
    a.first = v0 == 0;
    if (d->dtype == TSG_BF16) backward_piece<TsgBf16, __bf16>(a, d, l, s);
    else if (d->dtype == TSG_F16) backward_piece<TsgF16, _Float16>(a, d, l, s);
    else backward_piece<TsgF16, float>(a, d, l, s);
    TSG_LAUNCH_CHECK();
  }
  return 0;
}
