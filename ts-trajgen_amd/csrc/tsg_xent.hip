// Softmax cross entropy over a large vocabulary from the states themselves: z_tv = h_t . w_v + b_v, loss_t = log sum_v
// exp(z_tv) - z_t,target, without the [rows][vocabulary] logits ever being kept.
//
// forward   products in tiles of 256, 128 or 64 vocabulary rows by as many states (shape_of); their epilogue leaves (maximum, sum of
//           exp) per state and tile, and the target's logit; a small kernel joins them.
// backward  the vocabulary is taken in pieces (DZ_LEAST, DZ_MOST).  Per piece the products are computed once more, their epilogue turns them into
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
// matrix cores.  dz is rounded to the operand type (bf16: 2^-9 relative); it is brought to 2^15 for a
// whole probability first, so that those down to 1e-9 stay above f16's subnormals; for f32 it is hi + lo as well.  Errors of dh and dW
// against 64 bits, 16-bit types, 100 drawn shapes: at most 1.32 times those of 32-bit sums rounded once (1.47 for a pair of rows).
// 16384 states x 50021 entries x 1024 wide, bf16 (1.68 TFLOP a product; five pieces): statistics 1.65-1.74 ms (970-1020 TFLOP/s), dz 1.91 ms (880),
// dW 1.62 ms (1040), dh 1.42 ms (1180); a large bf16 matrix product of the library: 1129.  8192 x 40307 x 256, f32 (four pieces): 0.61, 0.88, 0.60
// and 0.53 ms, the f32 rate of the library's product (153 TFLOP/s) would take 1.10 ms each.  The first two pay for their epilogues, which nothing
// runs under: a 256 x 256 tile is one workgroup a CU, whose waves leave the products together (5000 x 40307 x 512, f16: matrix cores 27 % of
// the time, vector units 36 %, both 1 %).
// All sums, maxima and logarithms are f32.  Nothing depends on the order of workgroups: no floating-point atomics.
#include "tsg_mma.h"

namespace {

constexpr int TK = 64;  // k of one step
// A workgroup's tile: WM x WN waves of XM x XN products of 32 x 32
template <int XM_, int XN_, int WM_, int WN_> struct Tile {
  static constexpr int XM = XM_, XN = XN_, WM = WM_, WN = WN_, WAVES = WM * WN, TM = 32 * XM * WM, TN = 32 * XN * WN;
  static constexpr int A = TM * TK * 2, STAGE = (TM + TN) * TK * 2;  // bytes of one step's tiles
};
// 256 x 256 reads half as much per product from the L2 as 128 x 128 (which the L2's rate bounds at about 900 TFLOP/s), but needs two
// rounds of tiles for the 256 CUs; 64 x 64 is for the products of a few rows, where the chip would otherwise stand empty.
typedef Tile<4, 2, 2, 4> Big;
typedef Tile<2, 2, 2, 2> Mid;
typedef Tile<1, 1, 2, 2> Few;

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

// dz of a row is held as (softmax - onehot) q 2^15 with q in (1/2, 1] and g = q 2^-k largest |g|, k the row's own.  A row whose g is small
// beside the others' would lose its probabilities below f16's smallest number in units that all rows share (f32, g of 1e-7 of the largest:
// dh off by 1.4e-3).  k comes back where dh is written; for dW the states are multiplied by 2^-k instead (xent_fold_kernel).  Under 'sum' and
// 'mean', where all g are alike, q = 1 and k = 0: the target's entry is -2^15 but for its own probability, no constant rounding of g goes into
// every row of the gradients, and the states are read as they are.
struct DzUnit {  // what one of dz stands for, m 2^e; apart, so that neither end of f32 is passed on the way
  float m;
  int e;
  __device__ __forceinline__ float of(float sum, int k = 0) const { return ldexpf(sum * m, e - k); }
};
// other: what the second operand of the sum was multiplied by, a power of two, or null
__device__ __forceinline__ DzUnit dz_unit(unsigned gmax, const float* other = nullptr) {
  DzUnit u = {1.0f, 0};
  int e = 1;
  if (gmax) u.m = frexpf(__uint_as_float(gmax), &u.e);
  if (other) frexpf(*other, &e);  // 2^(e - 1)
  u.e -= 15 + e - 1;
  return u;
}
// what a magnitude says to a common scale: one that is not finite spoils its own row, not the others' precision
__device__ __forceinline__ float weight_of(float v) { return fabsf(v) < INFINITY ? fabsf(v) : 0.0f; }

struct XentArgs {
  const char *h, *w;            // operands of the products (f32: their planes in the workspace)
  long h_row, w_row;            // bytes
  long h_plane, w_plane;        // bytes from hi to lo; 0 for 16-bit types
  const char* bias;             // in the caller's type, or null
  const long* target;
  long ignore;
  int rows, hidden, vocab;
  int v0, vc;                   // this piece of the vocabulary
  const float* scales;          // f32: what h and w were multiplied by
  unsigned* gmax;               // backward: bits of the largest |g|
  float2* part;                 // forward: [vocab tiles][rows]
  float* zt;                    // forward: [rows] the target's logit
  float2* stat;                 // [rows] maximum, log2 of the sum
  float* g;                     // backward: [rows] q 2^15 with the sign of g, 0 for rows left out
  int* shift;                   // backward: [rows] k
  const char* hd;               // the states as dW reads them: h, or h 2^-k times *hd_by
  long hd_row, hd_plane;
  const float* hd_by;           // or null: 1
  unsigned long long* used;     // backward: bit t % 64 of word t / 64: g_t != 0
  char* dz;                     // [rows][ldz] 16-bit; f32: lo plane dz_plane further on
  long ldz, dz_plane;           // elements, bytes
  float* db_part;               // [row tiles][vc]
  float* dh_part;               // [splits][rows][hidden]
  int splits, split_len, first;
  float* dw_part;               // [dw_splits][vc][hidden], or null: whole sums go to dw
  int dw_len;                   // rows of a stretch
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
template <typename T> using Acc = tsg_f32x16[T::XM][T::XN];
template <typename D, typename T, bool AC, bool BC, bool MASKED = false>
__device__ __forceinline__ void product(Acc<T>& acc, char* lds, const Operand& a, const Operand& b, int K, int passes, int wave, int lane) {
  const int per = (K + TK - 1) / TK, steps = per * passes;
  const int wm = wave / T::WN * 32 * T::XM, wn = wave % T::WN * 32 * T::XN;
  // a wave's rows or columns: rows lie 128 bytes apart, columns 2
  const unsigned a0 = tsg_lds_addr(lds) + (AC ? TsgLane<D, T::TM / 8>::col_in_order(lane) ^ (wm * 2) : TsgLane<D, TK / 8>::row(lane) + wm * TK * 2);
  const unsigned b0 = tsg_lds_addr(lds) + T::A + (BC ? TsgLane<D, T::TN / 8>::col_in_order(lane) ^ (wn * 2) : TsgLane<D, TK / 8>::row(lane) + wn * TK * 2);
  TsgLoader<AC ? TK : T::TM, (AC ? T::TM : TK) / 8, T::WAVES> al;
  TsgLoader<BC ? TK : T::TN, (BC ? T::TN : TK) / 8, T::WAVES> bl;
  // a tile whose memory rows are k is as wide as the operand is; one whose columns are k ends where k ends (its last step: below)
  const unsigned at0 = tsg_lds_addr(lds), bt0 = tsg_lds_addr(lds) + T::A;
  al.init(a.row, AC ? a.cols / 8 : TK / 8, at0, wave, lane);
  bl.init(b.row, BC ? b.cols / 8 : TK / 8, bt0, wave, lane);
  unsigned long long used = MASKED ? b.used[0] : 0ull;
  auto fetch = [&](int pass, int k0, int buf) {
    const char* ap = a.p + (pass == 2 ? a.plane : 0);
    const char* bp = b.p + (pass == 1 ? b.plane : 0);
    const bool narrow = (!AC || !BC) && K - k0 < TK;  // the last step of a K that is no multiple of 64
    if (narrow) {
      if (!AC) al.init(a.row, (a.cols - k0) / 8, at0, wave, lane);
      if (!BC) bl.init(b.row, (b.cols - k0) / 8, bt0, wave, lane);
    }
    if (AC) al.load(ap + (long)k0 * a.row, a.rows - k0, a.cols * 2, buf * T::STAGE);
    else al.load(ap + k0 * 2, a.rows, min(a.cols - k0, TK) * 2, buf * T::STAGE);
    if (BC && MASKED) bl.load(bp + (long)k0 * b.row, b.rows - k0, b.cols * 2, buf * T::STAGE, used);
    else if (BC) bl.load(bp + (long)k0 * b.row, b.rows - k0, b.cols * 2, buf * T::STAGE);
    else bl.load(bp + k0 * 2, b.rows, min(b.cols - k0, TK) * 2, buf * T::STAGE);
    if (narrow) {
      if (!AC) al.init(a.row, TK / 8, at0, wave, lane);
      if (!BC) bl.init(b.row, TK / 8, bt0, wave, lane);
    }
  };
  int pass = 0, k0 = 0;
  if (steps) {
    fetch(0, 0, 0);
    if (MASKED) used = b.used[(TK < K ? TK : 0) / 64];
  }
  for (int step = 0, buf = 0; step < steps; ++step, buf ^= 1) {
    tsg_dma_wait();
    __syncthreads();
    if (step + 1 < steps) {
      k0 += TK;
      if (k0 >= K) k0 = 0, ++pass;
      fetch(pass, k0, buf ^ 1);
      if (MASKED) used = b.used[(k0 + TK < K ? k0 + TK : 0) / 64];  // for the step after: a scalar load under this one's products
    }
    const unsigned at = tsg_opaque(a0) + buf * T::STAGE, bt = tsg_opaque(b0) + buf * T::STAGE;
#pragma unroll
    for (int s = 0; s < TK / 16; ++s) {
      tsg_u4 fa[T::XM], fb[T::XN];
#pragma unroll
      for (int x = 0; x < T::XM; ++x) fa[x] = AC ? tsg_col_frag<T::TM / 8>(at, x, 16 * s * T::TM * 2) : tsg_row_frag<D>(at, s, 32 * x * TK * 2);
#pragma unroll
      for (int y = 0; y < T::XN; ++y) fb[y] = BC ? tsg_col_frag<T::TN / 8>(bt, y, 16 * s * T::TN * 2) : tsg_row_frag<D>(bt, s, 32 * y * TK * 2);
#pragma unroll
      for (int x = 0; x < T::XM; ++x)
#pragma unroll
        for (int y = 0; y < T::XN; ++y) tsg_mma<D>(fa[x], fb[y], acc[x][y]);
    }
    constexpr int READS = T::XM * (AC ? 2 : 1) + T::XN * (BC ? 2 : 1), PRODUCTS = T::XM * T::XN;  // of 16 k
    tsg_interleave<READS * TK / 16, PRODUCTS * TK / 16, READS, (READS + PRODUCTS - 1) / PRODUCTS>();
  }
  __syncthreads();  // the epilogue may use the tiles' memory
}

template <typename T> __device__ __forceinline__ void zero_acc(Acc<T>& acc) {
#pragma unroll
  for (int x = 0; x < T::XM; ++x)
#pragma unroll
    for (int y = 0; y < T::XN; ++y)
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
// lane's registers of a state are reduced without leaving the lane.
template <typename D, typename T, bool SPLIT> __device__ __forceinline__ void logits(const XentArgs& a, Acc<T>& acc, char* lds, int m0, int n0, int wave, int lane) {
  zero_acc<T>(acc);
  const Operand A = {a.w + (long)m0 * a.w_row, a.w_row, a.w_plane, a.vocab - m0, a.hidden, nullptr};
  const Operand B = {a.h + (long)n0 * a.h_row, a.h_row, a.h_plane, a.rows - n0, a.hidden, nullptr};
  product<D, T, false, false>(acc, lds, A, B, a.hidden, SPLIT ? 3 : 1, wave, lane);
  const int h = lane >> 5, wm = wave / T::WN * 32 * T::XM;
  const float by = SPLIT ? 1.0f / (a.scales[0] * a.scales[1]) : 1.0f;
#pragma unroll
  for (int x = 0; x < T::XM; ++x)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int v = m0 + wm + 32 * x + (i & 3) + 8 * (i >> 2) + 4 * h;
      float b = 0.0f;
      if (a.bias && v < a.vocab) b = SPLIT ? reinterpret_cast<const float*>(a.bias)[v] : (float)reinterpret_cast<const typename D::type*>(a.bias)[v];
#pragma unroll
      for (int y = 0; y < T::XN; ++y) acc[x][y][i] = v < a.vocab ? (SPLIT ? acc[x][y][i] * by : acc[x][y][i]) + b : -INFINITY;
      if (i == 15) __builtin_amdgcn_sched_barrier(0);  // or the biases of all 32 XM rows are fetched at once, into registers that are not there
    }
}

// orders LDS alone: __syncthreads would wait for the stores to memory as well
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;

template <typename D, typename T, bool SPLIT>
__global__ __launch_bounds__(64 * T::WAVES, 2) void xent_stat_kernel(XentArgs a, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[2 * T::STAGE];
  __shared__ float2 join[T::WM][T::TN];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
  Acc<T> z;
  logits<D, T, SPLIT>(a, z, lds, tm * T::TM, tn * T::TN, wave, lane);
  const int wm = wave / T::WN * 32 * T::XM, wn = wave % T::WN * 32 * T::XN;
#pragma unroll
  for (int y = 0; y < T::XN; ++y) {
    const int n = wn + 32 * y + (lane & 31), t = tn * T::TN + n;
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < T::XM; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, z[x][y][i]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float off = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    const long target = t < a.rows ? a.target[t] : -1;
    const int at = target >= 0 && target < a.vocab ? (int)target - (tm * T::TM + wm + 4 * h) : -1;
    float zt = 0.0f;
    bool mine = false;
#pragma unroll
    for (int x = 0; x < T::XM; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (at == 32 * x + (i & 3) + 8 * (i >> 2)) zt = z[x][y][i], mine = true;
        sum += __builtin_amdgcn_exp2f((z[x][y][i] - off) * LOG2E);
      }
    sum += __shfl_xor(sum, 32, 64);
    if (mine) a.zt[t] = zt;
    if (h == 0) join[wave / T::WN][n] = make_float2(top, sum);
  }
  __syncthreads();
  for (int n = threadIdx.x; n < T::TN; n += 64 * T::WAVES) {
    const int t = tn * T::TN + n;
    if (t >= a.rows) break;
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < T::WM; ++w) top = fmaxf(top, join[w][n].x);
    const float off = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < T::WM; ++w) sum += join[w][n].y * __builtin_amdgcn_exp2f((join[w][n].x - off) * LOG2E);
    a.part[(long)tm * a.rows + t] = make_float2(top, sum);
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
      sum = sum * __builtin_amdgcn_exp2f((top - off) * LOG2E) + p.y * __builtin_amdgcn_exp2f((p.x - off) * LOG2E);
      top = to;
    }
  join[part][n] = make_float2(top, sum);
  __syncthreads();
  if (part || t >= a.rows) return;
  top = -INFINITY;
  for (int p = 0; p < 8; ++p) top = fmaxf(top, join[p][n].x);
  const float off = top == -INFINITY ? 0.0f : top;
  sum = 0.0f;
  for (int p = 0; p < 8; ++p) sum += join[p][n].y * __builtin_amdgcn_exp2f((join[p][n].x - off) * LOG2E);
  const float l2 = __builtin_amdgcn_logf(sum);
  a.stat[t] = make_float2(off, l2);
  const long tg = a.target[t];
  float l = 0.0f;
  if (tg != a.ignore) l = tg >= 0 && tg < a.vocab ? (off - a.zt[t]) + l2 * LN2 : NAN;
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

// q_t, k_t and the largest |g_t|, one workgroup.  reduction 0: d_loss per row; 1: one gradient for the sum; 2: for the mean
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
    m = fmaxf(m, weight_of(g));
  }
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();
  for (int w = 0; w < 16; ++w) m = fmaxf(m, top[w]);
  if (threadIdx.x == 0) *a.gmax = __float_as_uint(m);
  int em;
  const float mm = frexpf(m, &em);
  for (int t = threadIdx.x; t < a.rows; t += 1024) {  // its own rows again
    const float g = a.g[t];
    float q = g;
    int k = 0;
    if (g != 0.0f && fabsf(g) < INFINITY) {
      int e;
      q = frexpf(g, &e) / mm;
      if (fabsf(q) > 1.0f) q *= 0.5f, ++e;
      k = em - e;
    }
    a.g[t] = q * 0x1p15f;
    a.shift[t] = k;
  }
}

template <typename D, typename T, bool SPLIT>
__global__ __launch_bounds__(64 * T::WAVES, 2) void xent_dz_kernel(XentArgs a, int tiles_m, int tiles_n) {
  constexpr int ROW = T::TM * 2 + 16;  // a state's dz of the tile in LDS, 16 bytes of padding
  __shared__ __attribute__((aligned(1024))) char lds[T::TN * ROW > 2 * T::STAGE ? T::TN * ROW : 2 * T::STAGE];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
  const int m0 = a.v0 + tm * T::TM;
  Acc<T> z;
  logits<D, T, SPLIT>(a, z, lds, m0, tn * T::TN, wave, lane);
  const int wm = wave / T::WN * 32 * T::XM, wn = wave % T::WN * 32 * T::XN;
#pragma unroll
  for (int y = 0; y < T::XN; ++y) {
    const int n = wn + 32 * y + (lane & 31), t = tn * T::TN + n;
    const bool in = t < a.rows;
    const float2 st = in ? a.stat[t] : make_float2(0.0f, INFINITY);
    const float g = in ? a.g[t] : 0.0f;
    const long target = in ? a.target[t] : -1;
    const int at = target >= 0 && target < a.vocab ? (int)target - (m0 + wm + 4 * h) : -1;
#pragma unroll
    for (int x = 0; x < T::XM; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z[x][y][i] - st.x, LOG2E, -st.y));
        // a row left out adds nothing, whatever it holds
        z[x][y][i] = g == 0.0f ? 0.0f : (at == 32 * x + (i & 3) + 8 * (i >> 2) ? p - 1.0f : p) * g;
      }
  }
  if (a.db_part) {
    float of_row[T::XN];  // 2^-k
#pragma unroll
    for (int y = 0; y < T::XN; ++y) {
      const int t = tn * T::TN + wn + 32 * y + (lane & 31);
      of_row[y] = t < a.rows ? ldexpf(1.0f, -a.shift[t]) : 0.0f;
    }
    // sums over the states: 16 registers x 32 lanes, halving the registers with four bits of the lane
    float* join = reinterpret_cast<float*>(lds);  // [WN][TM]
#pragma unroll
    for (int x = 0; x < T::XM; ++x) {
      float sums[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sums[i] = z[x][0][i] * of_row[0];
#pragma unroll
        for (int y = 1; y < T::XN; ++y) sums[i] = __builtin_fmaf(z[x][y][i], of_row[y], sums[i]);
      }
#pragma unroll
      for (int n = 8; n > 0; n >>= 1) {
        const bool up = lane & (2 * n);
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float keep = up ? sums[i + n] : sums[i], send = up ? sums[i] : sums[i + n];
          sums[i] = keep + __shfl_xor(send, 2 * n, 64);
        }
      }
      sums[0] += __shfl_xor(sums[0], 1, 64);
      const int i = (lane & 31) >> 1;
      join[wave % T::WN * T::TM + wm + 32 * x + (i & 3) + 8 * (i >> 2) + 4 * h] = sums[0];
      __builtin_amdgcn_sched_barrier(0);
    }
    lds_barrier();
    for (int m = threadIdx.x; m < T::TM && tm * T::TM + m < a.vc; m += 64 * T::WAVES) {
      float v = join[m];
#pragma unroll
      for (int w = 1; w < T::WN; ++w) v += join[w * T::TM + m];
      a.db_part[(long)tn * a.vc + tm * T::TM + m] = v;
    }
    lds_barrier();
  }
#pragma unroll 1
  for (int plane = 0; plane < (SPLIT ? 2 : 1); ++plane) {
#pragma unroll
    for (int y = 0; y < T::XN; ++y)
#pragma unroll
      for (int x = 0; x < T::XM; ++x)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          typedef typename D::type E;
          uint2 v;
          v.x = tsg_pack2<D>(z[x][y][4 * q], z[x][y][4 * q + 1]);
          v.y = tsg_pack2<D>(z[x][y][4 * q + 2], z[x][y][4 * q + 3]);
          if (SPLIT) {  // what is left over is the second plane
#pragma unroll
            for (int r = 0; r < 4; ++r) z[x][y][4 * q + r] -= (float)(E)z[x][y][4 * q + r];
          }
          *reinterpret_cast<uint2*>(lds + (wn + 32 * y + (lane & 31)) * ROW + (wm + 32 * x + 8 * q + 4 * h) * 2) = v;
        }
    lds_barrier();
    constexpr int CH = T::TM / 8;
#pragma unroll
    for (int k = 0; k < T::TN * CH / (64 * T::WAVES); ++k) {
      const int id = k * 64 * T::WAVES + threadIdx.x, n = id / CH, c = id % CH, t = tn * T::TN + n;
      if (t < a.rows && tm * T::TM + c * 8 < a.ldz)
        *reinterpret_cast<tsg_u4*>(a.dz + plane * a.dz_plane + ((long)t * a.ldz + tm * T::TM + c * 8) * 2) = *reinterpret_cast<const tsg_u4*>(lds + n * ROW + c * 16);
    }
    lds_barrier();
  }
}

// dW of the piece: rows v, columns k', summed over the states
template <typename D, typename T, typename OUT>
__global__ __launch_bounds__(64 * T::WAVES, 2) void xent_dw_kernel(XentArgs a, int tiles_m, int tiles_n) {
  constexpr bool SPLIT = __is_same(OUT, float);
  __shared__ __attribute__((aligned(1024))) char lds[2 * T::STAGE];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
  int tm, tn;
  tile_of(blockIdx.x % (tiles_m * tiles_n), tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
  const int split_id = blockIdx.x / (tiles_m * tiles_n), t0 = split_id * a.dw_len, len = min(a.dw_len, a.rows - t0);
  Acc<T> acc;
  zero_acc<T>(acc);
  const Operand A = {a.dz + (t0 * a.ldz + tm * T::TM) * 2, a.ldz * 2, a.dz_plane, len, (int)a.ldz - tm * T::TM, nullptr};
  const Operand B = {a.hd + t0 * a.hd_row + (long)tn * T::TN * 2, a.hd_row, a.hd_plane, len, a.hidden - tn * T::TN, a.used + t0 / 64};
  if (len > 0) product<D, T, true, true, true>(acc, lds, A, B, len, SPLIT ? 3 : 1, wave, lane);
  const DzUnit unit = dz_unit(*a.gmax, a.hd_by);
  const int wm = wave / T::WN * 32 * T::XM, wn = wave % T::WN * 32 * T::XN;
#pragma unroll
  for (int x = 0; x < T::XM; ++x)
#pragma unroll
    for (int y = 0; y < T::XN; ++y)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int m = tm * T::TM + wm + 32 * x + (i & 3) + 8 * (i >> 2) + 4 * h, k = tn * T::TN + wn + 32 * y + (lane & 31);
        if (m < a.vc && k < a.hidden) {
          if (a.dw_part) a.dw_part[((long)split_id * a.vc + m) * a.hidden + k] = acc[x][y][i];
          else reinterpret_cast<OUT*>(a.dw + (long)(a.v0 + m) * a.dw_row)[k] = (OUT)unit.of(acc[x][y][i]);
        }
      }
}

// dh: rows t, columns k', summed over a stretch of the piece; the stretches' sums are added up over the pieces
template <typename D, typename T, bool SPLIT>
__global__ __launch_bounds__(64 * T::WAVES, 2) void xent_dh_kernel(XentArgs a, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[2 * T::STAGE];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5;
  const int split_id = blockIdx.x / (tiles_m * tiles_n);
  int tm, tn;
  tile_of(blockIdx.x % (tiles_m * tiles_n), tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
  const int c0 = split_id * a.split_len, len = min(a.split_len, a.vc - c0);
  Acc<T> acc;
  zero_acc<T>(acc);
  if (len > 0) {
    // dz is zero behind the vocabulary up to a multiple of 64, W ends at its last row
    const Operand A = {a.dz + ((long)tm * T::TM * a.ldz + c0) * 2, a.ldz * 2, a.dz_plane, a.rows - tm * T::TM, (len + 7) / 8 * 8, nullptr};
    const Operand B = {a.w + (long)(a.v0 + c0) * a.w_row + (long)tn * T::TN * 2, a.w_row, a.w_plane, len, a.hidden - tn * T::TN, nullptr};
    product<D, T, false, true>(acc, lds, A, B, len, SPLIT ? 3 : 1, wave, lane);
  }
  const int wm = wave / T::WN * 32 * T::XM, wn = wave % T::WN * 32 * T::XN;
  float* out = a.dh_part + (long)split_id * a.rows * a.hidden;
#pragma unroll
  for (int x = 0; x < T::XM; ++x)
#pragma unroll
    for (int y = 0; y < T::XN; ++y)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = tm * T::TM + wm + 32 * x + (i & 3) + 8 * (i >> 2) + 4 * h, k = tn * T::TN + wn + 32 * y + (lane & 31);
        if (t < a.rows && k < a.hidden) {
          float* p = out + (long)t * a.hidden + k;
          *p = a.first ? acc[x][y][i] : *p + acc[x][y][i];
        }
      }
}

// A gradient from its stretches' sums: [splits][n / hidden][hidden] f32 -> rows of OUT, in units of dz and, per row, of 2^-shift.
// Four elements per thread; PARTS of the workgroup's waves share the stretches (1 or 4).
template <typename OUT, int PARTS>
__global__ __launch_bounds__(256) void xent_join_grad_kernel(const float* from, int splits, long n, int hidden, OUT* out, long out_row, const unsigned* gmax,
                                                             const float* other, const int* shift) {
  constexpr int WIDE = 256 / PARTS;
  __shared__ float4 join[PARTS][WIDE];
  const int part = threadIdx.x / WIDE, lane = threadIdx.x % WIDE;
  const long i = ((long)blockIdx.x * WIDE + lane) * 4;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (i < n)
#pragma unroll 4
    for (int p = part; p < splits; p += PARTS) {
      const float4 v = *reinterpret_cast<const float4*>(from + p * n + i);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  if (PARTS > 1) {
    join[part][lane] = s;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int p = 1; p < PARTS; ++p) {
      const float4 v = join[p][lane];
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  if (i >= n) return;
  const DzUnit unit = dz_unit(*gmax, other);
  const int k = shift ? shift[i / hidden] : 0;
  OUT* to = out + (i / hidden) * out_row + i % hidden;
  OUT v[4] = {(OUT)unit.of(s.x, k), (OUT)unit.of(s.y, k), (OUT)unit.of(s.z, k), (OUT)unit.of(s.w, k)};
  if (sizeof(OUT) == 4) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(v);
  else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(v);
}

template <typename OUT> __global__ __launch_bounds__(256) void xent_db_out_kernel(XentArgs a, OUT* db, int tiles_n) {
  __shared__ float join[4][64];
  const int part = threadIdx.x >> 6, lane = threadIdx.x & 63, v = blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (v < a.vc)
#pragma unroll 4
    for (int t = part; t < tiles_n; t += 4) s += a.db_part[(long)t * a.vc + v];
  join[part][lane] = s;
  __syncthreads();
  if (part || v >= a.vc) return;
  s = (join[0][lane] + join[1][lane]) + (join[2][lane] + join[3][lane]);
  db[a.v0 + v] = (OUT)dz_unit(*a.gmax).of(s);
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
    m = fmaxf(m, fmaxf(fmaxf(weight_of(v.x), weight_of(v.y)), fmaxf(weight_of(v.z), weight_of(v.w))));
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

// ---- the states times 2^-k of their rows, for dW where upstream gradients differ: a power of two and exact, until it reaches the type's
// smallest numbers.  f16 and f32's planes begin at 2^15 for the largest state, so an element 2^-29 of the largest in state and gradient
// together still has 11 bits; bf16 reaches further by itself.
struct Fold {
  const char* h;
  long row;             // bytes
  int rows, chunks;     // of 8 elements
  const float* g;       // rows that are left out (0) may hold anything: they have no say
  const int* shift;
  float* amax;          // [blocks], f16 only
  const float* scale;   // f32 only: what the forward multiplied its planes by
  float* by;            // f16 only, out: what the states were multiplied by
  char* out;
  long plane;           // f32 only
};
template <typename D> __device__ __forceinline__ void fold_load(const Fold& a, long i, float (&v)[8]) {
  typedef typename D::type T;
  const T* x = reinterpret_cast<const T*>(a.h + (i / a.chunks) * a.row) + (i % a.chunks) * 8;
  T e[8];
#pragma unroll
  for (int b = 0; b < (int)sizeof(T) * 8; b += 16) *reinterpret_cast<uint4*>(reinterpret_cast<char*>(e) + b) = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(x) + b);
#pragma unroll
  for (int n = 0; n < 8; ++n) v[n] = (float)e[n];
}
__global__ __launch_bounds__(256) void xent_fold_max_kernel(Fold a) {
  __shared__ float join[4];
  float m = 0.0f;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < (long)a.rows * a.chunks; i += (long)gridDim.x * 256) {
    if (a.g[i / a.chunks] == 0.0f) continue;
    float v[8];
    fold_load<TsgF16>(a, i, v);
#pragma unroll
    for (int n = 0; n < 8; ++n) m = fmaxf(m, weight_of(v[n]));
  }
  m = tsg_wave_max(m);
  if ((threadIdx.x & 63) == 0) join[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) a.amax[blockIdx.x] = fmaxf(fmaxf(join[0], join[1]), fmaxf(join[2], join[3]));
}
template <typename D> __global__ __launch_bounds__(256) void xent_fold_kernel(Fold a) {
  constexpr bool SPLIT = __is_same(D, TsgF32);
  typedef typename D::type T;
  float by = SPLIT ? *a.scale : 1.0f;
  if constexpr (__is_same(D, TsgF16)) {
    __shared__ float join[4];
    float m = 0.0f;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += 256) m = fmaxf(m, a.amax[i]);
    m = tsg_wave_max(m);
    if ((threadIdx.x & 63) == 0) join[threadIdx.x >> 6] = m;
    __syncthreads();
    by = scale_of(__float_as_uint(fmaxf(fmaxf(join[0], join[1]), fmaxf(join[2], join[3]))));
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.by = by;
  }
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < (long)a.rows * a.chunks; i += (long)gridDim.x * 256) {
    float v[8];
    fold_load<D>(a, i, v);
    const int k = a.shift[i / a.chunks];
    tsg_u4 hi, lo;
#pragma unroll
    for (int n = 0; n < 8; ++n) v[n] = ldexpf(v[n] * by, -k);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if constexpr (SPLIT) {
        hi[n] = tsg_pack2<TsgF16>(v[2 * n], v[2 * n + 1]);
        lo[n] = tsg_pack2<TsgF16>(v[2 * n] - (float)(_Float16)v[2 * n], v[2 * n + 1] - (float)(_Float16)v[2 * n + 1]);
      } else {
        hi[n] = tsg_pack2<D>(v[2 * n], v[2 * n + 1]);
      }
    }
    *reinterpret_cast<tsg_u4*>(a.out + i * 16) = hi;
    if constexpr (SPLIT) *reinterpret_cast<tsg_u4*>(a.out + a.plane + i * 16) = lo;
  }
}

// ------------------------------------------------------------------------------------------------------ host side
struct Layout {
  size_t gmax, amax, planes, h_plane, w_plane, part, zt, g, shift, used, fold, fold_amax, fold_by, dz, dz_plane, db, dh, dw, total;
  int vc, splits, split_len, dh_shape, dw_shape, dw_splits, dw_len;
};
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// The largest tile that still gives every CU a workgroup (256 x 256 fill one, of 128 x 128 two fit), else the next
enum Shape { FEW, MID, BIG };
Shape shape_of(int64_t m, int64_t n, int64_t times = 1) {
  if ((int64_t)tsg_cdiv(m, Big::TM) * tsg_cdiv(n, Big::TN) * times >= 256) return BIG;
  if ((int64_t)tsg_cdiv(m, Mid::TM) * tsg_cdiv(n, Mid::TN) * times >= 256) return MID;
  return FEW;
}
constexpr int PLANE_BLOCKS = 512;
// dz of a piece takes at most a quarter of the logits, within these bounds (but 256 vocabulary rows at least): large pieces fill the chip, small
// ones keep the memory of a call far below the logits'.  Forward and backward, and the peak with the gradients, by the bound:
//                               128 MiB          256              384              768              2 GiB
//   8192 x 40307 x 256, f32     5.56 ms 0.30 GB  2.93 0.50        2.83 0.57        2.75 0.90        2.70 1.63 (all in one piece; logits 1.32 GB)
//   16384 x 50021 x 1024, bf16  7.48    0.41     6.99 0.50        6.99 0.67        7.19 1.24        6.95 1.84 (likewise; 1.64 GB)
//   67062 x 11096 x 256, f32                     9.58 0.51        8.43 0.65        7.30 1.06        6.94 1.83 (2.98 GB)
//   30000 x 500000 x 128, f32                    130  0.88        115  1.03        107  1.43        101  2.74 (60 GB)
constexpr size_t DZ_LEAST = (size_t)384 << 20, DZ_MOST = (size_t)2 << 30;

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
    l.part = take((size_t)tsg_cdiv(V, shape_of(V, T) == FEW ? Few::TM : shape_of(V, T) == MID ? Mid::TM : Big::TM) * T * 8);
    l.zt = take(T * 4);
  } else {
    const size_t each = f32 ? 4 : 2;
    size_t budget = T * V * each / 4;
    budget = budget < DZ_LEAST ? DZ_LEAST : budget > DZ_MOST ? DZ_MOST : budget;
    size_t vc = budget / (T * each) / 256 * 256;
    if (vc < 256) vc = 256;
    const size_t all = (V + 63) / 64 * 64;
    if (vc > all) vc = all;
    if (vc > ((size_t)1 << 21)) vc = (size_t)1 << 21;  // 256 rows of dz stay below 2^31 bytes
    const size_t pieces = (all + vc - 1) / vc;  // even pieces
    if (pieces > 1) vc = ((all + pieces - 1) / pieces + 255) / 256 * 256;
    l.vc = (int)vc;
    l.dz_plane = f32 ? up256(T * vc * 2) : 0;
    l.dz = take(f32 ? 2 * l.dz_plane : T * vc * 2);
    l.g = take(T * 4);
    l.shift = take(T * 4);
    l.used = take((T + 63) / 64 * 8);
    if (d->reduction == 0) {
      l.fold = take(f32 ? 2 * l.h_plane : T * K * 2);
      l.fold_amax = take(PLANE_BLOCKS * 4);
      l.fold_by = take(4);
    }
    l.db = d->bias ? take((size_t)tsg_cdiv(T, 64) * vc * 4) : 0;
    // dh has few tiles and a long sum: cut it until the chip is full, in stretches of 128 entries at least
    l.dh_shape = T >= 2048 ? BIG : T > 64 ? MID : FEW;
    const int tm = l.dh_shape == BIG ? Big::TM : l.dh_shape == MID ? Mid::TM : Few::TM;
    const size_t tiles = (size_t)tsg_cdiv(T, tm) * tsg_cdiv(K, tm);
    size_t s = ((l.dh_shape == BIG ? 256 : 512) + tiles - 1) / tiles;
    if (s > vc / 128) s = vc / 128;
    if (s < 1) s = 1;
    l.split_len = (int)(((vc + s - 1) / s + TK - 1) / TK * TK);
    l.splits = (int)((vc + l.split_len - 1) / l.split_len);
    l.dh = take((size_t)l.splits * T * K * 4);
    // dW of a narrow state has few tiles too (40307 x 256: 158 of 256 x 256): cut the rows where that leaves the CUs less idle, each
    // cut priced at 2 % for the sums it writes and reads again.  A narrow piece has a handful (1280 x 256: 5): cut until they fill the chip
    // once, in stretches of 512 rows at least; the small tiles it would take else are slow over a long sum
    // (67062 rows, f32: 1280 x 256 in 64 x 64 tiles 3115 us; 2304 x 256, twice the products, cut: 274).
    l.dw_shape = shape_of((int64_t)vc, (int64_t)K);
    l.dw_splits = 1;
    const int64_t big = (int64_t)tsg_cdiv(vc, Big::TM) * tsg_cdiv(K, Big::TN);
    if (big < 768 && T >= 2048) {
      if (big >= 32) {
        double best = 1e9;
        for (int c = 1; c <= 8 && T / c >= 1024; ++c) {
          const double cost = (double)((big * c + 255) / 256) / c + 0.02 * c;
          if (cost < best) best = cost, l.dw_splits = c;
        }
      } else {
        l.dw_splits = (int)(T / 512 < (size_t)(256 / big) ? T / 512 : 256 / big);
      }
      l.dw_shape = BIG;
    }
    l.dw_len = (int)(((T + l.dw_splits - 1) / l.dw_splits + 63) / 64 * 64);
    l.dw = l.dw_splits > 1 ? take((size_t)l.dw_splits * vc * K * 4) : 0;
  }
  l.total = at;
  return l;
}

int check_xent(const tsg_xent_desc* d, bool backward) {
  if (!d) return TSG_E_INVALID;
  if (d->dtype != TSG_F32 && d->dtype != TSG_BF16 && d->dtype != TSG_F16) return TSG_E_INVALID;
  if (d->n_rows < 0 || d->n_vocab <= 0 || d->hidden <= 0 || d->reduction < 0 || d->reduction > 2) return TSG_E_INVALID;
  if (d->n_rows > 0x7fffff00L || d->n_vocab > 0x7fffff00L) return TSG_E_LIMIT;
  if ((int64_t)tsg_cdiv(d->n_rows, 64) * tsg_cdiv(d->n_vocab, 64) > 0x7fffffffL) return TSG_E_LIMIT;
  if (d->n_rows * (int64_t)d->hidden > ((int64_t)1 << 36)) return TSG_E_LIMIT;
  if (d->hidden % 8) return TSG_E_INVALID;
  const int epc = d->dtype == TSG_F32 ? 4 : 8;
  if (!d->h || !d->w || !d->target || !d->stats || (uintptr_t)d->h % 16 || (uintptr_t)d->w % 16 || (uintptr_t)d->stats % 8) return TSG_E_INVALID;
  if (d->h_row < d->hidden || d->w_row < d->hidden || d->h_row % epc || d->w_row % epc) return TSG_E_INVALID;
  if (d->h_row * 4 >= (1 << 23) || d->w_row * 4 >= (1 << 23)) return TSG_E_LIMIT;  // offsets inside a tile are 32-bit
  if (!backward && !d->row_loss) return TSG_E_INVALID;
  if (!backward && d->reduction && !d->loss) return TSG_E_INVALID;
  if (d->dtype == TSG_F32 && !d->scales) return TSG_E_INVALID;
  if (backward && (!d->d_loss || !d->dh || !d->dw || (d->bias && !d->dbias))) return TSG_E_INVALID;
  if (backward && (d->dh_row < d->hidden || d->dw_row < d->hidden || d->dh_row % 4 || d->dw_row % 4 || (uintptr_t)d->dh % 16 || (uintptr_t)d->dw % 16)) return TSG_E_INVALID;
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
  a.bias = (const char*)d->bias;
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

// upstream gradients per row differ: dW's states carry 2^-k
void make_fold(const tsg_xent_desc* d, XentArgs& a, const Layout& l, hipStream_t s) {
  char* ws = (char*)d->workspace;
  Fold f = {};
  f.h = (const char*)d->h, f.row = d->h_row * (d->dtype == TSG_F32 ? 4 : 2), f.rows = a.rows, f.chunks = d->hidden / 8;
  f.g = a.g, f.shift = a.shift, f.amax = (float*)(ws + l.fold_amax), f.scale = d->scales, f.by = (float*)(ws + l.fold_by);
  f.out = ws + l.fold, f.plane = (long)l.h_plane;
  const int64_t want = ((int64_t)f.rows * f.chunks + 255) / 256;
  const dim3 grid((unsigned)(want > PLANE_BLOCKS ? PLANE_BLOCKS : want)), block(256);
  a.hd = f.out, a.hd_row = d->hidden * 2L, a.hd_plane = d->dtype == TSG_F32 ? f.plane : 0;
  if (d->dtype == TSG_F32) {
    hipLaunchKernelGGL(xent_fold_kernel<TsgF32>, grid, block, 0, s, f);
  } else if (d->dtype == TSG_BF16) {
    hipLaunchKernelGGL(xent_fold_kernel<TsgBf16>, grid, block, 0, s, f);
  } else {
    hipLaunchKernelGGL(xent_fold_max_kernel, grid, block, 0, s, f);
    hipLaunchKernelGGL(xent_fold_kernel<TsgF16>, grid, block, 0, s, f);
    a.hd_by = f.by;
  }
}

// f(Tile<...>) for the shape
template <typename F> void with_tile(int shape, F f) {
  if (shape == BIG) f(Big());
  else if (shape == MID) f(Mid());
  else f(Few());
}

template <typename D, bool SPLIT> int launch_stat(const XentArgs& a, hipStream_t s) {
  int tm = 0;
  with_tile(shape_of(a.vocab, a.rows), [&](auto t) {
    typedef decltype(t) T;
    tm = tsg_cdiv(a.vocab, T::TM);
    const int tn = tsg_cdiv(a.rows, T::TN);
    hipLaunchKernelGGL((xent_stat_kernel<D, T, SPLIT>), dim3((unsigned)(tm * tn)), dim3(64 * T::WAVES), 0, s, a, tm, tn);
  });
  return tm;
}

template <typename D, typename OUT> void backward_piece(XentArgs a, const tsg_xent_desc* d, const Layout& l, hipStream_t s) {
  constexpr bool SPLIT = __is_same(OUT, float);
  int tt = 0;
  with_tile(shape_of(a.vc, a.rows), [&](auto t) {
    typedef decltype(t) T;
    tt = tsg_cdiv(a.rows, T::TN);
    const int tv = tsg_cdiv(a.vc, T::TM);
    hipLaunchKernelGGL((xent_dz_kernel<D, T, SPLIT>), dim3((unsigned)(tv * tt)), dim3(64 * T::WAVES), 0, s, a, tv, tt);
  });
  with_tile(l.dw_shape, [&](auto t) {
    typedef decltype(t) T;
    const int tv = tsg_cdiv(a.vc, T::TM), tk = tsg_cdiv(a.hidden, T::TN);
    hipLaunchKernelGGL((xent_dw_kernel<D, T, OUT>), dim3((unsigned)(tv * tk * l.dw_splits)), dim3(64 * T::WAVES), 0, s, a, tv, tk);
  });
  with_tile(l.dh_shape, [&](auto t) {
    typedef decltype(t) T;
    const int tr = tsg_cdiv(a.rows, T::TM), tk = tsg_cdiv(a.hidden, T::TN);
    hipLaunchKernelGGL((xent_dh_kernel<D, T, SPLIT>), dim3((unsigned)(tr * tk * l.splits)), dim3(64 * T::WAVES), 0, s, a, tr, tk);
  });
  if (d->bias) hipLaunchKernelGGL(xent_db_out_kernel<OUT>, dim3(tsg_cdiv(a.vc, 64)), dim3(256), 0, s, a, (OUT*)d->dbias, tt);
  auto join = [&](const float* from, int splits, long n, OUT* out, long out_row, const float* other, const int* shift) {
    if (splits >= 16)
      hipLaunchKernelGGL((xent_join_grad_kernel<OUT, 4>), dim3((unsigned)((n / 4 + 63) / 64)), dim3(256), 0, s, from, splits, n, a.hidden, out, out_row, a.gmax, other, shift);
    else
      hipLaunchKernelGGL((xent_join_grad_kernel<OUT, 1>), dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, s, from, splits, n, a.hidden, out, out_row, a.gmax, other, shift);
  };
  if (a.dw_part) join(a.dw_part, l.dw_splits, (long)a.vc * a.hidden, (OUT*)d->dw + (long)a.v0 * d->dw_row, d->dw_row, a.hd_by, nullptr);
  if (a.v0 + a.vc >= a.vocab) join(a.dh_part, l.splits, (long)a.rows * a.hidden, (OUT*)d->dh, d->dh_row, SPLIT ? a.scales + 1 : nullptr, a.shift);
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
  const int tm = d->dtype == TSG_BF16  ? launch_stat<TsgBf16, false>(a, s)
                 : d->dtype == TSG_F16 ? launch_stat<TsgF16, false>(a, s)
                                       : launch_stat<TsgF16, true>(a, s);
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
  a.shift = (int*)(ws + l.shift);
  a.used = (unsigned long long*)(ws + l.used);
  a.hd = a.h, a.hd_row = a.h_row, a.hd_plane = a.h_plane, a.hd_by = d->dtype == TSG_F32 ? d->scales : nullptr;
  a.dz = ws + l.dz, a.dz_plane = (long)l.dz_plane;
  a.db_part = d->bias ? (float*)(ws + l.db) : nullptr;
  a.dh_part = (float*)(ws + l.dh);
  a.splits = l.splits, a.split_len = l.split_len;
  a.dw_part = l.dw_splits > 1 ? (float*)(ws + l.dw) : nullptr;
  a.dw_len = l.dw_len;
  a.dw = (char*)d->dw, a.dw_row = d->dw_row * (d->dtype == TSG_F32 ? 4 : 2);
  a.ldz = l.vc;
  if (d->dtype == TSG_F32) make_planes(d, a, l, true, s);
  hipLaunchKernelGGL(xent_grad_kernel, dim3(1), dim3(1024), 0, s, a, d->d_loss, d->reduction);
  if (d->reduction == 0) make_fold(d, a, l, s);
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
