// Causal attention over packed sequences with grouped heads: forward, backward, and the form for few query rows.
//
//   p_ij = exp(scale (q_i . k_j - m_i)) / l_i,  o_i = sum_j p_ij v_j          over the keys j that row i sees
//   delta_i = do_i . o_i,  dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i                       sums over the heads of a group too
//
// Sequences lie one behind the other (q_ptr / k_ptr).  Row t of sequence s sees keys [k0, k0 + (t - q0) + (lk - lq) + 1):
// a contiguous interval of the packed keys, and both ends grow with t.  So a tile of query rows is simply a stretch of
// the packed rows, whatever sequences it crosses: it walks the union of its rows' intervals and masks by the row's own.
// Trajectories of a few dozen positions fill a tile that way.  The same holds for a tile of keys and the query
// rows that see them.  No lengths are needed on the host.  Rows of no sequence give zeros.
//
// Tile kernels (16-bit types, dim <= 256): a workgroup of four waves owns 128 rows, 32 per wave; the wave computes the TRANSPOSED
// score tile (A = keys, B = its rows), so that a lane holds one row: the softmax statistics are one register per
// lane, and the probabilities feed the next product as they stand (tsg_mma.h).  Scores, statistics and outputs are held
// in f32; p and ds are rounded to the operand type for the matrix cores (nearest even, 2^-9 relative for bf16, which is
// what the output's own rounding costs too); for f32 operands nothing is rounded.
// The backward is two kernels, one per output side (dq; dk and dv), each recomputing the scores: seven products instead
// of five, no atomics, and results that do not depend on the order of workgroups.
// 4 sequences of 2.5-4 k positions, 16 heads over 4, 128 wide, bf16: forward 236 us (775 TFLOP/s), dq 301 us (910, three products), dk and dv
// 458 us (800, four products) and 29 us for joining the stretches; a large bf16 matrix product of the library: 1129.  Matrix cores busy 37, 46 and
// 38 % of the time, vector units (exponentials, packing, masks) 39, 36 and 29 %, both at once 10-14 %, LDS 20-31 %, 1.5-1.7 waves a SIMD at work.
#include "tsg_mma.h"

namespace {

struct AttnArgs {
  int n_seq, heads, kv_heads, group, dim, chunks;
  int n_q, n_k;
  const int* q_ptr;
  const int* k_ptr;
  const char *q, *k, *v, *o, *d_o;
  char* rest;    // [n_q][heads][dim] 16-bit, or null: what the rounding of out left over (o + rest is out to 2^-16)
  char *out, *dq, *dk, *dv;
  long q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, do_row, do_head, dq_row, dq_head, dk_row, dk_head, dv_row,
      dv_head;   // bytes
  float2* stat;  // [heads][n_q]: largest product q.k of the row, log2 of the sum over it; (0, +inf) where a row sees nothing
  float* delta;  // [heads][n_q]
  float scale, scale2;
  int n_split;
  float* part;   // rows kernel: [n_q][heads][n_split][dim + 2]; dk and dv: [2][n_split][n_k][kv_heads][dim]
};

// The sequence that position t belongs to, -1 for none (empty sequences share their start with the next one).  One position,
// alike in all lanes of a wave: every lane probes, so 4096 sequences take two loads one behind the other.
__device__ __forceinline__ int starts_until(const int* ptr, int n_seq, int t) {  // how many starts are <= t
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n_seq;
  while (lo < hi) {
    const int w = (hi - lo + 64) / 65, at = lo + (lane + 1) * w - 1;
    const int n = __popcll(__ballot(at < hi && ptr[at < hi ? at : lo] <= t));
    lo += n * w;
    hi = min(hi, lo + w - 1);
  }
  return lo;
}
__device__ __forceinline__ int seq_from(const int* ptr, int n_seq, int s, int t) {  // s: starts_until of a position before t
  for (int n = 0; n < 8 && s < n_seq && ptr[s] <= t; ++n) ++s;
  int hi = s < n_seq && ptr[s] <= t ? n_seq : s;  // not among the next few: bisect
  while (s < hi) {
    const int mid = (s + hi) >> 1;
    if (ptr[mid] <= t) s = mid + 1;
    else hi = mid;
  }
  return (s > 0 && t < ptr[s]) ? s - 1 : -1;
}
__device__ __forceinline__ int clamp_to(long v, int n) { return v < 0 ? 0 : (v > n ? n : (int)v); }

// keys [lo, hi) that query row t sees; always inside [0, n_k], whatever the pointers hold.  t0 <= t: alike in the wave
__device__ __forceinline__ void keys_of_row(const AttnArgs& a, int t0, int t, int& lo, int& hi) {
  lo = hi = 0;
  const int from = starts_until(a.q_ptr, a.n_seq, t0);
  if (t >= a.n_q) return;
  const int s = seq_from(a.q_ptr, a.n_seq, from, t);
  if (s < 0) return;
  const long q1 = a.q_ptr[s + 1], k0 = a.k_ptr[s], k1 = a.k_ptr[s + 1];
  const long end = k1 - (q1 - 1 - t);  // the last row sees the last key
  lo = clamp_to(k0, a.n_k);
  hi = clamp_to(end < k1 ? end : k1, a.n_k);
  if (hi <= lo) lo = hi = 0;
}
// query rows [lo, hi) that see key j
__device__ __forceinline__ void rows_of_key(const AttnArgs& a, int j0, int j, int& lo, int& hi) {
  lo = hi = 0;
  const int from = starts_until(a.k_ptr, a.n_seq, j0);
  if (j >= a.n_k) return;
  const int s = seq_from(a.k_ptr, a.n_seq, from, j);
  if (s < 0) return;
  const long q0 = a.q_ptr[s], q1 = a.q_ptr[s + 1], k1 = a.k_ptr[s + 1];
  const long first = q1 - (k1 - j);
  lo = clamp_to(first > q0 ? first : q0, a.n_q);
  hi = clamp_to(q1, a.n_q);
  if (hi <= lo) lo = hi = 0;
}

// Interval bounds over a wave (lanes W apart hold the same row) and over the workgroup
struct Bounds {
  int wave_lo, wave_hi;  // union of the wave's intervals; empty: wave_lo >= wave_hi
  int in_lo, in_hi;      // intersection; empty when a row of the wave is empty
  int lo, hi;            // union over the workgroup
};
template <int W> __device__ __forceinline__ Bounds wave_bounds(int lo, int hi) {
  Bounds b;
  const bool none = hi <= lo;
  int ulo = none ? 0x7fffffff : lo, uhi = none ? 0 : hi, ilo = none ? 0x7fffffff : lo, ihi = none ? 0 : hi;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    ulo = min(ulo, __shfl_xor(ulo, o, 64));
    uhi = max(uhi, __shfl_xor(uhi, o, 64));
    ilo = max(ilo, __shfl_xor(ilo, o, 64));
    ihi = min(ihi, __shfl_xor(ihi, o, 64));
  }
  b.wave_lo = __builtin_amdgcn_readfirstlane(ulo);
  b.wave_hi = __builtin_amdgcn_readfirstlane(uhi);
  b.in_lo = __builtin_amdgcn_readfirstlane(ilo);
  b.in_hi = __builtin_amdgcn_readfirstlane(ihi);
  return b;
}
template <int W> __device__ __forceinline__ Bounds bounds_of(int lo, int hi, int wave, int* shared /* [8] */) {
  Bounds b = wave_bounds<W>(lo, hi);
  if ((threadIdx.x & 63) == 0) shared[wave] = b.wave_lo, shared[4 + wave] = b.wave_hi;
  __syncthreads();
  b.lo = __builtin_amdgcn_readfirstlane(min(min(shared[0], shared[1]), min(shared[2], shared[3])));
  b.hi = __builtin_amdgcn_readfirstlane(max(max(shared[4], shared[5]), max(shared[6], shared[7])));
  return b;
}

__device__ __forceinline__ tsg_u4 chunk_of(const char* row, int c, bool ok) {
  tsg_u4 v = {0u, 0u, 0u, 0u};
  if (ok) v = *reinterpret_cast<const tsg_u4*>(row + c * 16);
  return v;
}
// operand fragments of one row per lane, straight from memory; zeros outside
template <int PARTS, int NF> __device__ __forceinline__ void load_frags(tsg_u4 (&f)[NF], const char* row, bool ok, int chunks, int h) {
#pragma unroll
  for (int s = 0; s < NF; ++s) {
    const int c = PARTS * s + h;
    f[s] = chunk_of(row, c, ok && c < chunks);
  }
}

template <typename D> __device__ __forceinline__ float frag_dot(tsg_u4 a, tsg_u4 b) {
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (TsgElem<D>::BYTES == 4) {
      s += __uint_as_float(a[w]) * __uint_as_float(b[w]);
    } else {
      typedef typename D::type T;
      typedef T T2 __attribute__((ext_vector_type(2)));
      const unsigned aw = a[w], bw = b[w];
      const T2 x = __builtin_bit_cast(T2, TsgElem<D>::BYTES == 4 ? 0u : aw), y = __builtin_bit_cast(T2, TsgElem<D>::BYTES == 4 ? 0u : bw);
      s += (float)x.x * (float)y.x + (float)x.y * (float)y.y;
    }
  }
  return s;
}
template <> __device__ __forceinline__ float frag_dot<TsgF32>(tsg_u4 a, tsg_u4 b) {
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) s += __uint_as_float(a[w]) * __uint_as_float(b[w]);
  return s;
}

// four neighbouring elements of a row, f32 -> element type
template <typename D> __device__ __forceinline__ void store4(char* at, float x, float y, float z, float w) {
  uint2 v;
  v.x = tsg_pack2<D>(x, y);
  v.y = tsg_pack2<D>(z, w);
  *reinterpret_cast<uint2*>(at) = v;
}
template <> __device__ __forceinline__ void store4<TsgF32>(char* at, float x, float y, float z, float w) {
  *reinterpret_cast<float4*>(at) = make_float4(x, y, z, w);
}
// transposed accumulators [dim][row] -> one row per lane; REST: what the rounding left over instead
template <typename D, int ND, bool REST = false>
__device__ __forceinline__ void store_rows(const typename TsgElem<D>::Acc (&acc)[ND], char* row, float by, int dim, int h) {
  typedef TsgElem<D> E;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int g = 0; g < E::REGS / 4; ++g) {
      const int d = E::W * dt + 8 * g + 4 * h;
      float x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = acc[dt][4 * g + r] * by;
        if (REST) x[r] -= (float)(typename E::T)x[r];
      }
      if (d < dim) store4<D>(row + d * E::BYTES, x[0], x[1], x[2], x[3]);
    }
}

template <typename D, int ND> __device__ __forceinline__ void store_sums(const typename TsgElem<D>::Acc (&acc)[ND], float* row, float by, int dim, int h) {
  typedef TsgElem<D> E;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int g = 0; g < E::REGS / 4; ++g) {
      const int d = E::W * dt + 8 * g + 4 * h;
      if (d < dim) *reinterpret_cast<float4*>(row + d) = make_float4(acc[dt][4 * g] * by, acc[dt][4 * g + 1] * by, acc[dt][4 * g + 2] * by, acc[dt][4 * g + 3] * by);
    }
}

template <int W> __device__ __forceinline__ float parts_max(float v) {
#pragma unroll
  for (int o = W; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
template <int W> __device__ __forceinline__ float parts_sum(float v) {
#pragma unroll
  for (int o = W; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// The second product of a tile multiplies p = 0 (ds = 0) with the operand rows that a row must not see, and 0 times an infinity or NaN
// is NaN: one broken trajectory would spoil its neighbours in the tile.  Only tiles that mask have such pairs.  So a kernel
// whose sums are not all finite walks its tiles once more (SEEN): in tiles that mask, elements that are not finite then
// reach exactly the rows that see them (a count of them per sum, a third product), and all other sums are formed with zeros in
// their place.  Finite operands pay one look at the sums; rows that see such an element hold NaN or infinities as they should.
// The second walk starts from the arguments and an index that the compiler cannot connect with the first one's: nothing is held for it.
__device__ __forceinline__ void tsg_again(int& tid) { asm volatile("" : "+v"(tid)); }
template <int NW> __device__ __forceinline__ bool any_wave(float zero, int wave, int* slot /* [NW], used once */) {
  const bool bad = __any(!(zero == 0.0f));
  if (NW == 1) return bad;
  if ((threadIdx.x & 63) == 0) slot[wave] = bad;
  __syncthreads();  // and all waves are done with the tiles
  int n = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) n |= slot[w];
  return __builtin_amdgcn_readfirstlane(n) != 0;
}
template <typename A, int N> __device__ __forceinline__ float zero_of(const A (&acc)[N], float z = 0.0f) {  // NaN if any is not finite
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < (int)(sizeof(A) / 4); ++i) z = __builtin_fmaf(acc[n][i], 0.0f, z);
  return z;
}
// the word's elements that are not finite: ones; the others: as they are
template <typename D> __device__ __forceinline__ void split_bad(unsigned w, unsigned& good, unsigned& bad) {
  constexpr bool BF = __is_same(D, TsgBf16);
  constexpr unsigned E = BF ? 0x7f80u : 0x7c00u, ONE = BF ? 0x3f80u : 0x3c00u;
  const bool lo = (w & E) == E, hi = (w & (E << 16)) == E << 16;
  good = (lo ? 0u : w & 0xffffu) | (hi ? 0u : w & 0xffff0000u);
  bad = (lo ? ONE : 0u) | (hi ? ONE << 16 : 0u);
}
template <typename D, int CH>
__device__ __forceinline__ void mma_seen(const TsgAccB<D>& p, const TsgAccB<D>& sees, unsigned col, int block, int offset, tsg_f32x16& acc) {
  const unsigned at = col ^ (block * 64);
  __builtin_amdgcn_sched_barrier(0);  // one block at a time: this walk must not cost the other one registers
  tsg_f32x16 extra, count;
#pragma unroll
  for (int i = 0; i < 16; ++i) extra[i] = count[i] = 0.0f;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const tsg_u4 x = TsgAccB<D>::template frag<CH>(at, offset, t);
    tsg_u4 good, lost, ones;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      unsigned g, b;
      split_bad<D>(x[w], g, b);
      good[w] = g, lost[w] = x[w] & ~g, ones[w] = b;
    }
    tsg_mma<D>(good, p.v[t], acc);
    tsg_mma<D>(lost, p.v[t], extra);
    tsg_mma<D>(ones, sees.v[t], count);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] += count[i] > 0.0f ? extra[i] : 0.0f;
  __builtin_amdgcn_sched_barrier(0);
}
// which of the accumulator's rows, 8 (i / 4) + 4 h + i % 4 from a tile's start, lie in [first, last); first and last: less 4 h
template <typename D> __device__ __forceinline__ TsgAccB<D> sees_of(int first, int last) {
  tsg_f32x16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int at = (i & 3) + 8 * (i >> 2);
    s[i] = at >= first && at < last ? 1.0f : 0.0f;
  }
  TsgAccB<D> b;
  b.set(s);
  return b;
}
// in a branch that is seldom taken: keeps the compiler from running both sides and selecting
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// f16 holds 2^-14 to 2^16 with all its bits, and ds = p (dp - delta) is as small or large as the upstream gradients are: those of a mean over
// thousands of positions, or of a scaled loss, leave it.  So a lane's ds (dq: a row's, dk: a key's) carry a power of two 2^up, which starts
// above anything and comes down, the sums so far with it, when one of them passes 2^15; the gradient is freed of it when it is written.
// p of the backward, at most 1 and as small as a sequence is long, is carried 2^P_UP for dv.  bf16 has f32's exponents.
// 4 sequences of 2.5-4 k positions, 16 heads over 4, 128 wide, f16: 841 us for the backward, 785 without (bf16: 740).
constexpr float P_UP = 14.0f, DS_UP = 60.0f;  // |d_out| <= 2^16, |v| <= 2^16, 256 wide: |ds| <= 2^41, and 2^101 is a number
template <typename D> constexpr bool lifted() { return __is_same(D, TsgF16); }
// by what the lane's ds have to come down, as a power of two: 0 for most.  Lanes 32 apart hold the same row or key.
__device__ __forceinline__ int ds_down(const tsg_f32x16& ds) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(ds[i]));
  if (!__any(top > 0x1p15f)) return 0;
  keep_branch();
  top = parts_max<32>(top);
  int e = 0;
  if (top > 0x1p15f && top < INFINITY) frexpf(top, &e), e -= 13;  // to [2^12, 2^13)
  return e;
}
template <typename D> constexpr int rows_per_wg() { return TsgElem<D>::BYTES == 4 ? 16 : 128; }

// ------------------------------------------------------------------------------------------------- forward, tiles
template <typename D, int DP, int BK, bool SEEN>
__device__ __forceinline__ float attn_fwd_tiles(const AttnArgs& a, int tid, char* lds, int* edge) {
  typedef TsgElem<D> E;
  typedef typename E::Acc Acc;
  constexpr int W = E::W, PARTS = 64 / W, CH = DP / E::EPC, NF = CH / PARTS, ND = DP / W, NB = BK / W, TILE = BK * CH * 16;
  const int wave = tid >> 6, lane = tid & 63, h = lane / W;
  const unsigned row0 = tsg_lds_addr(lds) + TsgLane<D, CH>::row(lane), col0 = tsg_lds_addr(lds) + TsgLane<D, CH>::col(lane);
  const int tiles = gridDim.x / a.heads;
  const int tile = tiles - 1 - (int)(blockIdx.x / a.heads), head = blockIdx.x % a.heads;  // late rows see most keys: first
  const int kvh = head / a.group;
  const int w0 = __builtin_amdgcn_readfirstlane(tile * (4 * W) + wave * W), t = w0 + lane % W;
  // the row's own operands first: their way here covers the search for its sequence
  tsg_u4 qf[NF];
  load_frags<PARTS>(qf, a.q + (long)t * a.q_row + head * a.q_head, t < a.n_q, a.chunks, h);
  int lo, hi;
  keys_of_row(a, w0, t, lo, hi);
  const Bounds b = bounds_of<W>(lo, hi, wave, edge);
  Acc acc[ND];
  float m, l;
  const char* kbase = a.k + kvh * a.k_head;
  const char* vbase = a.v + kvh * a.v_head;
  TsgLoader<BK, CH, 4> kl, vl;
  kl.init(a.k_row, a.chunks, tsg_lds_addr(lds), wave, lane);
  vl.init(a.v_row, a.chunks, tsg_lds_addr(lds) + TILE, wave, lane);
  auto fetch = [&](int k0, int buf) {
    kl.load(kbase + (long)k0 * a.k_row, b.hi - k0, a.chunks * 16, buf * 2 * TILE);
    vl.load(vbase + (long)k0 * a.v_row, b.hi - k0, a.chunks * 16, buf * 2 * TILE);
  };
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < E::REGS; ++i) acc[dt][i] = 0.0f;
  m = -INFINITY, l = 0.0f;
  if (b.lo < b.hi) fetch(b.lo, 0);
  tsg_settle(qf);
  for (int k0 = b.lo, buf = 0; k0 < b.hi; k0 += BK, buf ^= 1) {
    tsg_dma_wait();
    __syncthreads();
    if (k0 + BK < b.hi) fetch(k0 + BK, buf ^ 1);
    if (k0 >= b.wave_hi || k0 + BK <= b.wave_lo) continue;  // nothing for this wave: uniform, the barriers are above
    const unsigned row = tsg_opaque(row0) + buf * 2 * TILE, col = tsg_opaque(col0) + buf * 2 * TILE;
    __builtin_amdgcn_s_setprio(1);  // matrix phases ahead of the other wave's softmax: 2 % of the forward
    Acc z[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < E::REGS; ++i) z[n][i] = 0.0f;
#pragma unroll
      for (int s = 0; s < NF; ++s) tsg_mma<D>(tsg_row_frag<D>(row, s, W * n * CH * 16), qf[s], z[n]);
    }
    tsg_interleave<NB * NF, NB * NF, 6, 1>();
    __builtin_amdgcn_s_setprio(0);
    if (k0 < b.in_lo || k0 + BK > b.in_hi) {
      keep_branch();
      const int first = lo - k0 - 4 * h, last = hi - k0 - 4 * h;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < E::REGS; ++i) {
          const int key = W * n + (i & 3) + 8 * (i >> 2);
          if (key < first || key >= last) z[n][i] = -INFINITY;
        }
    }
    float top = m;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < E::REGS; ++i) top = fmaxf(top, z[n][i]);
    top = parts_max<W>(top);
    // A row's reference m follows its maximum only when that has run 2^8 ahead: the sums and products of p <= 2^8 are as
    // exact as those of p <= 1, and most tiles then leave the 32 x dim accumulators alone.
    if (__any((top - m) * a.scale2 > 8.0f)) {
      keep_branch();
      const float fade = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - top) * a.scale2);
      l *= fade;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int i = 0; i < E::REGS; ++i) acc[dt][i] *= fade;
      m = top;
    }
    const float off = m == -INFINITY ? 0.0f : m;  // nothing seen yet: exp2(-inf) = 0, not NaN
    // One fused operation takes the reference off, where the scaling cannot overflow, and what rounding m scale2 leaves over goes
    // into the row's logarithm at the end; else it comes off before the scaling (products of the type's lowest value stay finite).
    if (a.scale2 <= 1.0f) {
      const float off2 = off * a.scale2;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < E::REGS; ++i) z[n][i] = __builtin_fmaf(z[n][i], a.scale2, -off2);
    } else {
      keep_branch();
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < E::REGS; ++i) z[n][i] = (z[n][i] - off) * a.scale2;
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < E::REGS; ++i) {
        z[n][i] = __builtin_amdgcn_exp2f(z[n][i]);
        l += z[n][i];
      }
      __builtin_amdgcn_s_setprio(1);
      TsgAccB<D> p;
      p.set(z[n]);
      if constexpr (SEEN) {
        const TsgAccB<D> sees = sees_of<D>(lo - k0 - W * n - 4 * h, hi - k0 - W * n - 4 * h);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) mma_seen<D, CH>(p, sees, col, dt, TILE + W * n * CH * 16, acc[dt]);
      } else {
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) p.template mma<CH>(col, dt, TILE + W * n * CH * 16, acc[dt]);
      }
    }
    if constexpr (!SEEN) tsg_interleave<NB * ND * 4, NB * ND * 2, 8, 2>();
    __builtin_amdgcn_s_setprio(0);
  }
  const float zero = zero_of(acc);
  l = parts_sum<W>(l);
  if (t < a.n_q) {
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    store_rows<D, ND>(acc, a.out + (long)t * a.o_row + head * a.o_head, by, a.dim, h);
    if (a.rest) store_rows<D, ND, true>(acc, a.rest + ((long)t * a.heads + head) * a.dim * E::BYTES, by, a.dim, h);
    const float left = a.scale2 <= 1.0f ? __builtin_fmaf(m, a.scale2, -(m * a.scale2)) : 0.0f;
    if (h == 0) a.stat[(long)head * a.n_q + t] = l == 0.0f ? make_float2(0.0f, INFINITY) : make_float2(m, __builtin_amdgcn_logf(l) - left);
  }
  return zero;
}
template <typename D, int DP, int BK>
__global__ __launch_bounds__(256, DP > 128 ? 1 : DP > 64 ? 2 : 3) void attn_fwd_kernel(AttnArgs a) {
  constexpr int CH = DP / TsgElem<D>::EPC, TILE = BK * CH * 16;
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];
  __shared__ int edge[8], redo[4];
  int tid = threadIdx.x;
  if (any_wave<4>(attn_fwd_tiles<D, DP, BK, false>(a, tid, lds, edge), tid >> 6, redo)) {
    tsg_again(tid);
    attn_fwd_tiles<D, DP, BK, true>(a, tid, lds, edge);
  }
}

// ------------------------------------------------------------------------------------------------ backward, tiles: dq
template <typename D, int DP, int BK, bool REST, bool SEEN>
__device__ __forceinline__ float attn_dq_tiles(const AttnArgs& a, int tid, char* lds, int* edge) {
  typedef TsgElem<D> E;
  typedef typename E::Acc Acc;
  constexpr int W = E::W, PARTS = 64 / W, CH = DP / E::EPC, NF = CH / PARTS, ND = DP / W, NB = BK / W, TILE = BK * CH * 16;
  const int wave = tid >> 6, lane = tid & 63, h = lane / W;
  const unsigned row0 = tsg_lds_addr(lds) + TsgLane<D, CH>::row(lane), col0 = tsg_lds_addr(lds) + TsgLane<D, CH>::col(lane);
  const int tiles = gridDim.x / a.heads;
  const int tile = tiles - 1 - (int)(blockIdx.x / a.heads), head = blockIdx.x % a.heads;
  const int kvh = head / a.group;
  const int w0 = __builtin_amdgcn_readfirstlane(tile * (4 * W) + wave * W), t = w0 + lane % W;
  tsg_u4 qf[NF], gf[NF];
  load_frags<PARTS>(qf, a.q + (long)t * a.q_row + head * a.q_head, t < a.n_q, a.chunks, h);
  load_frags<PARTS>(gf, a.d_o + (long)t * a.do_row + head * a.do_head, t < a.n_q, a.chunks, h);
  float delta = 0.0f;
  float2 st = make_float2(0.0f, INFINITY);
  {
    const char* orow = a.o + (long)t * a.o_row + head * a.o_head;
#pragma unroll
    for (int s = 0; s < NF; ++s) {
      const int c = PARTS * s + h;
      const bool ok = t < a.n_q && c < a.chunks;
      delta += frag_dot<D>(chunk_of(orow, c, ok), gf[s]);
      if (a.rest) delta += frag_dot<D>(chunk_of(a.rest + ((long)t * a.heads + head) * a.dim * E::BYTES, c, ok), gf[s]);
    }
    delta = parts_sum<W>(delta);
    if (t < a.n_q) {
      st = a.stat[(long)head * a.n_q + t];
      if (h == 0) a.delta[(long)head * a.n_q + t] = delta;  // the dk / dv kernel, next on the stream, reads it
    }
  }
  int lo, hi;
  keys_of_row(a, w0, t, lo, hi);
  const Bounds b = bounds_of<W>(lo, hi, wave, edge);
  Acc acc[ND];
  const char* kbase = a.k + kvh * a.k_head;
  const char* vbase = a.v + kvh * a.v_head;
  TsgLoader<BK, CH, 4> kl, vl;
  kl.init(a.k_row, a.chunks, tsg_lds_addr(lds), wave, lane);
  vl.init(a.v_row, a.chunks, tsg_lds_addr(lds) + TILE, wave, lane);
  auto fetch = [&](int k0, int buf) {
    kl.load(kbase + (long)k0 * a.k_row, b.hi - k0, a.chunks * 16, buf * 2 * TILE);
    vl.load(vbase + (long)k0 * a.v_row, b.hi - k0, a.chunks * 16, buf * 2 * TILE);
  };
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < E::REGS; ++i) acc[dt][i] = 0.0f;
  if (b.lo < b.hi) fetch(b.lo, 0);
  tsg_settle(qf);
  tsg_settle(gf);
  float up = DS_UP;
  if constexpr (lifted<D>()) st.y -= up;  // exp2 then gives p 2^up
  asm volatile("" : "+v"(st.x), "+v"(st.y), "+v"(delta));
  for (int k0 = b.lo, buf = 0; k0 < b.hi; k0 += BK, buf ^= 1) {
    tsg_dma_wait();
    __syncthreads();
    if (k0 + BK < b.hi) fetch(k0 + BK, buf ^ 1);
    if (k0 >= b.wave_hi || k0 + BK <= b.wave_lo) continue;
    const unsigned row = tsg_opaque(row0) + buf * 2 * TILE, col = tsg_opaque(col0) + buf * 2 * TILE;
    constexpr int UNROLL = SEEN ? 1 : NB;
    const bool edge_tile = k0 < b.in_lo || k0 + BK > b.in_hi;
#pragma unroll UNROLL
    for (int n = 0; n < NB; ++n) {
      Acc z, dp;
#pragma unroll
      for (int i = 0; i < E::REGS; ++i) z[i] = 0.0f, dp[i] = -delta;  // dp - delta comes out of the product
#pragma unroll
      for (int s = 0; s < NF; ++s) {
        tsg_mma<D>(tsg_row_frag<D>(row, s, W * n * CH * 16), qf[s], z);
        tsg_mma<D>(tsg_row_frag<D>(row, s, TILE + W * n * CH * 16), gf[s], dp);
      }
      tsg_interleave<2 * NF, 2 * NF, 6, 1>();
#pragma unroll
      for (int i = 0; i < E::REGS; ++i) z[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i] - st.x, a.scale2, -st.y)) * dp[i];
      if (edge_tile) {
        keep_branch();
        const int first = lo - k0 - W * n - 4 * h, last = hi - k0 - W * n - 4 * h;
#pragma unroll
        for (int i = 0; i < E::REGS; ++i) {
          const int key = (i & 3) + 8 * (i >> 2);
          if (key < first || key >= last) z[i] = 0.0f;
        }
      }
      if constexpr (lifted<D>()) {
        const int down = ds_down(z);
        if (__any(down)) {
          keep_branch();
          const float by = ldexpf(1.0f, -down);
          up -= down, st.y += down;
#pragma unroll
          for (int i = 0; i < E::REGS; ++i) z[i] *= by;
#pragma unroll
          for (int dt = 0; dt < ND; ++dt)
#pragma unroll
            for (int i = 0; i < E::REGS; ++i) acc[dt][i] *= by;
        }
      }
      TsgAccB<D> ds;
      ds.set(z);
      if constexpr (SEEN) {
        const TsgAccB<D> sees = sees_of<D>(lo - k0 - W * n - 4 * h, hi - k0 - W * n - 4 * h);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) mma_seen<D, CH>(ds, sees, col, dt, W * n * CH * 16, acc[dt]);
      } else {
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) ds.template mma<CH>(col, dt, W * n * CH * 16, acc[dt]);
        tsg_interleave<ND * 4, ND * 2, 8, 2>();
        if (REST && edge_tile) {
          keep_branch();
          ds.set_rest(z);
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) ds.template mma<CH>(col, dt, W * n * CH * 16, acc[dt]);
        }
      }
    }
  }
  const float zero = zero_of(acc);
  if (t < a.n_q)
    store_rows<D, ND>(acc, a.dq + (long)t * a.dq_row + head * a.dq_head, lifted<D>() ? a.scale * __builtin_amdgcn_exp2f(-up) : a.scale, a.dim, h);
  return zero;
}
// REST: a gradient of a short sequence is the sum of few products, and the rounding of ds costs as much there as the output's own (error 1.48
// to 1.52 times that of sums in 32 bits, rounded once).  In tiles that mask, where short sequences lie, the rest of ds is multiplied as well: 1.05
// to 1.26 times.  Sequences of 1024 positions and more in the mean do without: 1.44 to 1.46 there, for 16 and 30 us of 303 and 465 (dq, dk and dv
// of 4 sequences of 2.5-4 k positions, 16 heads over 4, 128 wide), which the branch costs every tile.
template <typename D, int DP, int BK, bool REST>
__global__ __launch_bounds__(256, DP > 128 ? 1 : DP > 64 ? 2 : 3) void attn_dq_kernel(AttnArgs a) {
  constexpr int CH = DP / TsgElem<D>::EPC, TILE = BK * CH * 16;
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];
  __shared__ int edge[8], redo[4];
  int tid = threadIdx.x;
  if (any_wave<4>(attn_dq_tiles<D, DP, BK, REST, false>(a, tid, lds, edge), tid >> 6, redo)) {
    tsg_again(tid);
    attn_dq_tiles<D, DP, BK, REST, true>(a, tid, lds, edge);
  }
}

// ------------------------------------------------------------------------------------------ backward, tiles: dk and dv
// PART 0: both; 1: dv only; 2: dk only (256 wide: keys, values and both sums do not fit the registers at once)
// VL: the values' fragments are read from LDS in every step instead of held in registers, which then suffice without spills
// (128 wide at two waves a SIMD, 256 wide at one).
template <typename D, int DP, int BQ, int PART, bool VL, bool REST, bool SEEN>
__device__ __forceinline__ float attn_dkv_tiles(const AttnArgs& a, int tid, char* lds, int* edge, float (*stat)[3][BQ]) {
  typedef TsgElem<D> E;
  typedef typename E::Acc Acc;
  constexpr int W = E::W, PARTS = 64 / W, CH = DP / E::EPC, NF = CH / PARTS, ND = DP / W, NB = BQ / W, TILE = BQ * CH * 16;
  const int wave = tid >> 6, lane = tid & 63, h = lane / W;
  const unsigned row0 = tsg_lds_addr(lds) + TsgLane<D, CH>::row(lane), col0 = tsg_lds_addr(lds) + TsgLane<D, CH>::col(lane);
  // early keys are seen by most rows: first.  With n_split > 1 the walk over the rows is cut into that many stretches.
  const int split = blockIdx.x / a.kv_heads % a.n_split, tile = blockIdx.x / a.kv_heads / a.n_split, kvh = blockIdx.x % a.kv_heads;
  const int w0 = __builtin_amdgcn_readfirstlane(tile * (4 * W) + wave * W), j = w0 + lane % W;
  tsg_u4 kf[NF], vf[PART == 1 || VL ? 1 : NF];
  load_frags<PARTS>(kf, a.k + (long)j * a.k_row + kvh * a.k_head, j < a.n_k, a.chunks, h);
  if constexpr (PART != 1 && VL) {
    // the wave's own rows: no other wave reads them, and the first step waits for them
    TsgLoader<W, CH, 1> vl;
    vl.init(a.v_row, a.chunks, tsg_lds_addr(lds) + 4 * TILE + wave * W * CH * 16, 0, lane);
    const int j0 = tile * (4 * W) + wave * W;
    vl.load(a.v + (long)j0 * a.v_row + kvh * a.v_head, a.n_k - j0, a.chunks * 16, 0);
  } else if constexpr (PART != 1) load_frags<PARTS>(vf, a.v + (long)j * a.v_row + kvh * a.v_head, j < a.n_k, a.chunks, h);
  int lo, hi;
  rows_of_key(a, w0, j, lo, hi);
  const Bounds b = bounds_of<W>(lo, hi, wave, edge);
  Acc dk[PART == 1 ? 1 : ND], dv[PART == 2 ? 1 : ND];
  // the walk: for every head of the group the row tiles [b.lo, b.hi), as one sequence of steps
  const int per = b.lo < b.hi ? (b.hi - b.lo + BQ - 1) / BQ : 0, all = per * a.group;
  const int first = (int)((long)all * split / a.n_split), steps = (int)((long)all * (split + 1) / a.n_split) - first;
  struct Step {
    int head, t0;
  };
  auto after = [&](Step p) {
    p.t0 += BQ;
    if (p.t0 >= b.hi) p.t0 = b.lo, ++p.head;
    return p;
  };
  TsgLoader<BQ, CH, 4> ql, gl;
  ql.init(a.q_row, a.chunks, tsg_lds_addr(lds), wave, lane);
  gl.init(a.do_row, a.chunks, tsg_lds_addr(lds) + TILE, wave, lane);
  auto fetch = [&](Step p, int buf) {
    ql.load(a.q + p.head * a.q_head + (long)p.t0 * a.q_row, b.hi - p.t0, a.chunks * 16, buf * 2 * TILE);
    gl.load(a.d_o + p.head * a.do_head + (long)p.t0 * a.do_row, b.hi - p.t0, a.chunks * 16, buf * 2 * TILE);
  };
  auto stat_of = [&](Step p, float2& st, float& delta) {
    const int t = p.t0 + tid;
    st = make_float2(0.0f, INFINITY), delta = 0.0f;
    if (tid < BQ && t < b.hi) st = a.stat[(long)p.head * a.n_q + t], delta = a.delta[(long)p.head * a.n_q + t];
  };
  auto stat_to = [&](int buf, float2 st, float delta) {
    if (tid < BQ) stat[buf][0][tid] = st.x, stat[buf][1][tid] = lifted<D>() ? st.y - P_UP : st.y, stat[buf][2][tid] = delta;
  };
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < E::REGS; ++i) {
      if constexpr (PART != 1) dk[dt][i] = 0.0f;
      if constexpr (PART != 2) dv[dt][i] = 0.0f;
    }
  float2 st = make_float2(0.0f, INFINITY);
  float delta = 0.0f;
  float up = __builtin_amdgcn_exp2f(DS_UP - P_UP);  // ds carry this and p's 2^P_UP
  Step now = {kvh * a.group + (steps ? first / per : 0), b.lo + (steps ? first % per : 0) * BQ};
  if (steps) {
    fetch(now, 0);
    stat_of(now, st, delta);
    stat_to(0, st, delta);
    if (steps > 1) stat_of(after(now), st, delta);  // held until the next step's buffer is free
  }
  tsg_settle(kf);
  if constexpr (PART != 1 && !VL) tsg_settle(vf);
  for (int step = 0, buf = 0; step < steps; ++step, buf ^= 1) {
    tsg_dma_wait();
    __syncthreads();
    const int t0 = now.t0;
    now = after(now);
    if (step + 1 < steps) {
      stat_to(buf ^ 1, st, delta);
      if (step + 2 < steps) stat_of(after(now), st, delta);  // before the tile's loads: a wait for these does not drain those
      fetch(now, buf ^ 1);
    }
    if (t0 >= b.wave_hi || t0 + BQ <= b.wave_lo) continue;
    const unsigned row = tsg_opaque(row0) + buf * 2 * TILE, col = tsg_opaque(col0) + buf * 2 * TILE;
    const unsigned vrow = tsg_opaque(row0) + 4 * TILE + wave * W * CH * 16;
    constexpr int UNROLL = SEEN ? 1 : NB;
    const bool edge_tile = t0 < b.in_lo || t0 + BQ > b.in_hi;
#pragma unroll UNROLL
    for (int n = 0; n < NB; ++n) {
      Acc z, dp;
#pragma unroll
      for (int g = 0; g < E::REGS / 4; ++g) {
        z[4 * g] = z[4 * g + 1] = z[4 * g + 2] = z[4 * g + 3] = 0.0f;
        if constexpr (PART != 1) {
          const float4 dl = *reinterpret_cast<const float4*>(&stat[buf][2][W * n + 8 * g + 4 * h]);
          dp[4 * g] = -dl.x, dp[4 * g + 1] = -dl.y, dp[4 * g + 2] = -dl.z, dp[4 * g + 3] = -dl.w;  // dp - delta comes out of the product
        }
      }
#pragma unroll
      for (int s = 0; s < NF; ++s) {
        tsg_mma<D>(tsg_row_frag<D>(row, s, W * n * CH * 16), kf[s], z);
        if constexpr (PART != 1)
          tsg_mma<D>(tsg_row_frag<D>(row, s, TILE + W * n * CH * 16),
                     VL ? tsg_row_frag<D>(vrow, s, 0) : vf[VL ? 0 : s], dp);
      }
      tsg_interleave<(PART == 1 ? 1 : VL ? 3 : 2) * NF, (PART == 1 ? 1 : 2) * NF, 6, PART != 1 && VL ? 2 : 1>();
#pragma unroll
      for (int g = 0; g < E::REGS / 4; ++g) {
        const float4 ms = *reinterpret_cast<const float4*>(&stat[buf][0][W * n + 8 * g + 4 * h]);
        const float4 ls = *reinterpret_cast<const float4*>(&stat[buf][1][W * n + 8 * g + 4 * h]);
        const float mv[4] = {ms.x, ms.y, ms.z, ms.w}, lv[4] = {ls.x, ls.y, ls.z, ls.w};
#pragma unroll
        for (int r = 0; r < 4; ++r) z[4 * g + r] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[4 * g + r] - mv[r], a.scale2, -lv[r]));
      }
      if (edge_tile) {
        keep_branch();
        const int first = lo - t0 - W * n - 4 * h, last = hi - t0 - W * n - 4 * h;
#pragma unroll
        for (int i = 0; i < E::REGS; ++i) {
          const int t = (i & 3) + 8 * (i >> 2);
          if (t < first || t >= last) {
            z[i] = 0.0f;
            if constexpr (PART != 1) dp[i] = 0.0f;
          }
        }
      }
      // dp becomes ds
      auto to_ds = [&]() {
#pragma unroll
        for (int i = 0; i < E::REGS; ++i) dp[i] *= lifted<D>() ? z[i] * up : z[i];
        if constexpr (lifted<D>()) {
          const int down = ds_down(dp);
          if (__any(down)) {
            keep_branch();
            const float by = ldexpf(1.0f, -down);
            up *= by;
#pragma unroll
            for (int i = 0; i < E::REGS; ++i) dp[i] *= by;
#pragma unroll
            for (int dt = 0; dt < (PART == 1 ? 1 : ND); ++dt)
#pragma unroll
              for (int i = 0; i < E::REGS; ++i) dk[dt][i] *= by;
          }
        }
      };
      if constexpr (SEEN) {
        TsgAccB<D> pb, sb;
        pb.set(z);
        if constexpr (PART != 1) {
          to_ds();
          sb.set(dp);
        }
        const TsgAccB<D> sees = sees_of<D>(lo - t0 - W * n - 4 * h, hi - t0 - W * n - 4 * h);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          if constexpr (PART != 2) mma_seen<D, CH>(pb, sees, col, dt, TILE + W * n * CH * 16, dv[dt]);
          if constexpr (PART != 1) mma_seen<D, CH>(sb, sees, col, dt, W * n * CH * 16, dk[dt]);
        }
        continue;
      }
      if constexpr (PART != 2) {
        TsgAccB<D> pb;
        pb.set(z);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) pb.template mma<CH>(col, dt, TILE + W * n * CH * 16, dv[dt]);
      }
      if constexpr (PART != 1) {
        to_ds();
        TsgAccB<D> sb;
        sb.set(dp);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) sb.template mma<CH>(col, dt, W * n * CH * 16, dk[dt]);
        if (REST && edge_tile) {
          keep_branch();
          sb.set_rest(dp);
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) sb.template mma<CH>(col, dt, W * n * CH * 16, dk[dt]);
        }
      }
    }
  }
  float zero = 0.0f;
  if constexpr (PART != 1) zero = zero_of(dk, zero);
  if constexpr (PART != 2) zero = zero_of(dv, zero);
  const float k_by = lifted<D>() ? __builtin_amdgcn_exp2f(-P_UP) / up : 1.0f, v_by = lifted<D>() ? __builtin_amdgcn_exp2f(-P_UP) : 1.0f;
  if (j < a.n_k && a.n_split > 1) {
    float* p = a.part + (((long)split * a.n_k + j) * a.kv_heads + kvh) * a.dim;
    if constexpr (PART != 1) store_sums<D, ND>(dk, p, k_by, a.dim, h);
    if constexpr (PART != 2) store_sums<D, ND>(dv, p + (long)a.n_split * a.n_k * a.kv_heads * a.dim, v_by, a.dim, h);
  } else if (j < a.n_k) {
    if constexpr (PART != 1) store_rows<D, ND>(dk, a.dk + (long)j * a.dk_row + kvh * a.dk_head, a.scale * k_by, a.dim, h);
    if constexpr (PART != 2) store_rows<D, ND>(dv, a.dv + (long)j * a.dv_row + kvh * a.dv_head, v_by, a.dim, h);
  }
  return zero;
}
template <typename D, int DP, int BQ, int PART, bool VL, bool REST>
__global__ __launch_bounds__(256, DP > 128 ? 1 : DP > 64 ? 2 : 3) void attn_dkv_kernel(AttnArgs a) {
  constexpr int W = TsgElem<D>::W, CH = DP / TsgElem<D>::EPC, TILE = BQ * CH * 16;
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE + (VL ? 4 * W * CH * 16 : 0)];
  __shared__ __attribute__((aligned(16))) float stat[2][3][BQ];  // maximum, log2 of the sum, delta
  __shared__ int edge[8], redo[4];
  int tid = threadIdx.x;
  if (any_wave<4>(attn_dkv_tiles<D, DP, BQ, PART, VL, REST, false>(a, tid, lds, edge, stat), tid >> 6, redo)) {
    // one after the other: with both it would need more registers than the first walk
    if constexpr (PART != 2) {
      tsg_again(tid);
      attn_dkv_tiles<D, DP, BQ, 1, false, false, true>(a, tid, lds, edge, stat);
    }
    if constexpr (PART == 0) __syncthreads();
    if constexpr (PART != 1) {
      tsg_again(tid);
      attn_dkv_tiles<D, DP, BQ, 2, VL, false, true>(a, tid, lds, edge, stat);
    }
  }
}

// ------------------------------------------------------------------------------------------ f32: 16 rows, 64 wide a wave
// The f32 matrix cores are a sixteenth as fast as the 16-bit ones: operands straight from the caches keep them fed (32 bytes a
// clock per CU), and what costs is idle waves.  So a workgroup owns only 16 rows, which see little more than they need
// (trajectories of a few dozen positions: three blocks of 16 keys), and its waves share the work of every block evenly: each has
// 64 of the width, forms its part of the 16 x 16 products q.k, and, once the parts have met in LDS, its 64 columns of the
// sums.  A wave then holds 16 registers of each operand, so five to eight workgroups a CU cover the loads.
// Row fragments as in tsg_mma.h.  Column fragments are read 16 bytes a lane: row m of product e of four stands for column
// 4 m + e, so that one load serves four products and a lane's results are 16 bytes side by side.
// Buffers bound the operands: rows behind the interval and chunks behind the width read as zeros.
// 2048 sequences of 2-64 positions, 256 wide: forward 80 us, dq 113 us, dk and dv 138 us; the operands and results alone are 110 us of a large
// copy, but each kernel reads all operands again.  Bound by the loads: the matrix cores work 24-29 % of the time, vector units 16-20 %.
struct Rows16 {  // one block of 16 rows, 64 columns
  __amdgpu_buffer_rsrc_t d;
  unsigned row, col, stride;  // the lane's byte offsets: its row fragment, its column fragment
  int chunks, left;           // chunks of the width; row fragments of this lane
  __device__ __forceinline__ Rows16(long row_bytes, int n_chunks, int wave, int lane) {
    stride = (unsigned)row_bytes, chunks = n_chunks, left = n_chunks - 16 * wave - (lane >> 4);
    row = (lane & 15) * stride + wave * 256 + (lane >> 4) * 16;
    col = (lane >> 4) * 4 * stride + wave * 256 + (lane & 15) * 16;
  }
  __device__ __forceinline__ void at(const char* base, int rows) {
    const int n = rows < 16 ? rows : 16;
    d = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, n > 0 ? (n - 1) * (int)stride + chunks * 16 : 0, 0x00020000);
  }
  __device__ __forceinline__ void rows(tsg_u4 (&f)[4]) const {
#pragma unroll
    for (int s = 0; s < 4; ++s)
      f[s] = __builtin_bit_cast(tsg_u4, __builtin_amdgcn_raw_buffer_load_b128(d, 4 * s < left ? (int)(row + s * 64) : (int)0x80000000, 0, 0));
  }
  // f[i]: row 4 h + i; columns behind the width only reach sums that are not stored
  __device__ __forceinline__ void cols(tsg_f4 (&f)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __builtin_bit_cast(tsg_f4, __builtin_amdgcn_raw_buffer_load_b128(d, (int)(col + i * stride), 0, 0));
  }
};
typedef tsg_f4 Sum16[4];
__device__ __forceinline__ tsg_f4 dot16(const tsg_u4 (&a)[4], const tsg_u4 (&b)[4], tsg_f4 z) {
#pragma unroll
  for (int s = 0; s < 4; ++s) tsg_mma<TsgF32>(a[s], b[s], z);
  return z;
}
__device__ __forceinline__ void add16(Sum16& acc, const tsg_f4 (&v)[4], const tsg_f4& p) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][e], p[i], acc[e], 0, 0, 0);
}
// the same, and elements that are not finite reach only the sums of rows that see them (mma_seen)
__device__ __forceinline__ void add16_seen(Sum16& acc, const tsg_f4 (&v)[4], const tsg_f4& p, int first, int last) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    tsg_f4 extra = {0.0f, 0.0f, 0.0f, 0.0f}, count = extra;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = v[i][e];
      asm volatile("" : "+v"(x));  // here and not earlier: registers
      const bool bad = (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
      acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(bad ? 0.0f : x, p[i], acc[e], 0, 0, 0);
      extra = __builtin_amdgcn_mfma_f32_16x16x4f32(bad ? x : 0.0f, p[i], extra, 0, 0, 0);
      count = __builtin_amdgcn_mfma_f32_16x16x4f32(bad ? 1.0f : 0.0f, i >= first && i < last ? 1.0f : 0.0f, count, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[e][i] += count[i] > 0.0f ? extra[i] : 0.0f;
    __builtin_amdgcn_sched_barrier(0);
  }
}
__device__ __forceinline__ void zero16(Sum16& acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = tsg_f4{0.0f, 0.0f, 0.0f, 0.0f};
}
__device__ __forceinline__ void store16(const Sum16& acc, char* row, float by, int dim, int wave, int h) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = 64 * wave + 16 * h + 4 * i;
    if (c < dim) *reinterpret_cast<float4*>(row + c * 4) = make_float4(acc[0][i] * by, acc[1][i] * by, acc[2][i] * by, acc[3][i] * by);
  }
}
// the waves' parts of a value, summed in the same order by all of them; slot: another one than the last call's
template <int NW, typename V> __device__ __forceinline__ V over_waves(V (*slot)[64], V part, int wave, int lane) {
  if (NW == 1) return part;
  slot[wave][lane] = part;
  __syncthreads();
  V sum = slot[0][lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) sum += slot[w][lane];
  return sum;
}

template <int NW, bool SEEN> __device__ __forceinline__ float attn_f32_fwd_tiles(const AttnArgs& a, int tid, tsg_f4 (*meet)[NW][64]) {
  const int wave = tid >> 6, lane = tid & 63, h = lane >> 4;
  const int tiles = gridDim.x / a.heads;
  const int t0 = (tiles - 1 - (int)(blockIdx.x / a.heads)) * 16, head = blockIdx.x % a.heads, kvh = head / a.group;
  const int t = t0 + (lane & 15);
  tsg_u4 qf[4];
  Rows16 q(a.q_row, a.chunks, wave, lane), k(a.k_row, a.chunks, wave, lane), v(a.v_row, a.chunks, wave, lane);
  q.at(a.q + (long)t0 * a.q_row + head * a.q_head, a.n_q - t0);
  q.rows(qf);
  int lo, hi;
  keys_of_row(a, t0, t, lo, hi);
  const Bounds b = wave_bounds<16>(lo, hi);
  Sum16 acc;
  float m, l;
  zero16(acc);
  m = -INFINITY, l = 0.0f;
  for (int k0 = b.wave_lo, buf = 0; k0 < b.wave_hi; k0 += 16, buf ^= 1) {
    tsg_u4 kf[4];
    tsg_f4 vf[4];
    k.at(a.k + kvh * a.k_head + (long)k0 * a.k_row, b.wave_hi - k0);
    v.at(a.v + kvh * a.v_head + (long)k0 * a.v_row, b.wave_hi - k0);
    k.rows(kf);
    v.cols(vf);
    tsg_f4 z = over_waves<NW>(meet[buf], dot16(kf, qf, tsg_f4{0.0f, 0.0f, 0.0f, 0.0f}), wave, lane);
    if (k0 < b.in_lo || k0 + 16 > b.in_hi) {
      keep_branch();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k0 + 4 * h + i < lo || k0 + 4 * h + i >= hi) z[i] = -INFINITY;
    }
    const float top = parts_max<16>(fmaxf(fmaxf(m, fmaxf(z[0], z[1])), fmaxf(z[2], z[3])));
    if (__any((top - m) * a.scale2 > 8.0f)) {  // as in attn_fwd_kernel
      keep_branch();
      const float fade = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - top) * a.scale2);
      l *= fade;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= fade;
      m = top;
    }
    const float off = m == -INFINITY ? 0.0f : m;
    // the reference comes off before the scaling: all of z - m's bits, and products of the type's lowest value stay finite
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      z[i] = __builtin_amdgcn_exp2f((z[i] - off) * a.scale2);
      l += z[i];
    }
    if constexpr (SEEN) add16_seen(acc, vf, z, lo - k0 - 4 * h, hi - k0 - 4 * h);
    else add16(acc, vf, z);
  }
  const float zero = zero_of(acc);
  l = parts_sum<16>(l);
  if (t < a.n_q) {
    store16(acc, a.out + (long)t * a.o_row + head * a.o_head, l == 0.0f ? 0.0f : 1.0f / l, a.dim, wave, h);
    if (tid < 16) a.stat[(long)head * a.n_q + t] = l == 0.0f ? make_float2(0.0f, INFINITY) : make_float2(m, __builtin_amdgcn_logf(l));
  }
  return zero;
}
template <int NW> __global__ __launch_bounds__(64 * NW, 4) void attn_f32_fwd_kernel(AttnArgs a) {
  __shared__ tsg_f4 meet[2][NW][64];
  __shared__ int redo[NW];
  int tid = threadIdx.x;
  if (any_wave<NW>(attn_f32_fwd_tiles<NW, false>(a, tid, meet), tid >> 6, redo)) {
    tsg_again(tid);
    attn_f32_fwd_tiles<NW, true>(a, tid, meet);
  }
}

template <int NW, bool SEEN> __device__ __forceinline__ float attn_f32_dq_tiles(const AttnArgs& a, int tid, tsg_f4 (*meet)[NW][64], float (*meet_delta)[64]) {
  const int wave = tid >> 6, lane = tid & 63, h = lane >> 4;
  const int tiles = gridDim.x / a.heads;
  const int t0 = (tiles - 1 - (int)(blockIdx.x / a.heads)) * 16, head = blockIdx.x % a.heads, kvh = head / a.group;
  const int t = t0 + (lane & 15);
  tsg_u4 qf[4], gf[4];
  float delta = 0.0f;
  {
    Rows16 q(a.q_row, a.chunks, wave, lane), g(a.do_row, a.chunks, wave, lane), o(a.o_row, a.chunks, wave, lane);
    q.at(a.q + (long)t0 * a.q_row + head * a.q_head, a.n_q - t0);
    g.at(a.d_o + (long)t0 * a.do_row + head * a.do_head, a.n_q - t0);
    o.at(a.o + (long)t0 * a.o_row + head * a.o_head, a.n_q - t0);
    tsg_u4 of[4];
    q.rows(qf);
    g.rows(gf);
    o.rows(of);
#pragma unroll
    for (int s = 0; s < 4; ++s) delta += frag_dot<TsgF32>(of[s], gf[s]);
  }
  int lo, hi;
  keys_of_row(a, t0, t, lo, hi);
  const Bounds b = wave_bounds<16>(lo, hi);
  delta = over_waves<NW>(meet_delta, parts_sum<16>(delta), wave, lane);
  float2 st = make_float2(0.0f, INFINITY);
  if (t < a.n_q) {
    st = a.stat[(long)head * a.n_q + t];
    if (tid < 16) a.delta[(long)head * a.n_q + t] = delta;  // the dk / dv kernel, next on the stream, reads it
  }
  Sum16 acc;
  Rows16 k(a.k_row, a.chunks, wave, lane), v(a.v_row, a.chunks, wave, lane);
  zero16(acc);
  for (int k0 = b.wave_lo, buf = 0; k0 < b.wave_hi; k0 += 16, buf ^= 2) {
    tsg_u4 kf[4], vf[4];
    tsg_f4 kc[4];
    k.at(a.k + kvh * a.k_head + (long)k0 * a.k_row, b.wave_hi - k0);
    v.at(a.v + kvh * a.v_head + (long)k0 * a.v_row, b.wave_hi - k0);
    k.rows(kf);
    v.rows(vf);
    if constexpr (!SEEN) k.cols(kc);
    tsg_f4 z = dot16(kf, qf, tsg_f4{0.0f, 0.0f, 0.0f, 0.0f}), dp = dot16(vf, gf, tsg_f4{0.0f, 0.0f, 0.0f, 0.0f});
    if (NW > 1) meet[buf][wave][lane] = z;
    dp = over_waves<NW>(meet[buf + 1], dp, wave, lane);
    if (NW > 1) {
      z = meet[buf][0][lane];
#pragma unroll
      for (int w = 1; w < NW; ++w) z += meet[buf][w][lane];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i] - st.x, a.scale2, -st.y)) * (dp[i] - delta);
    if (k0 < b.in_lo || k0 + 16 > b.in_hi) {
      keep_branch();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k0 + 4 * h + i < lo || k0 + 4 * h + i >= hi) z[i] = 0.0f;
    }
    if constexpr (SEEN) {
      __builtin_amdgcn_sched_barrier(0);
      k.cols(kc);
      add16_seen(acc, kc, z, lo - k0 - 4 * h, hi - k0 - 4 * h);
    } else {
      add16(acc, kc, z);
    }
  }
  const float zero = zero_of(acc);
  if (t < a.n_q) store16(acc, a.dq + (long)t * a.dq_row + head * a.dq_head, a.scale, a.dim, wave, h);
  return zero;
}
template <int NW> __global__ __launch_bounds__(64 * NW, 4) void attn_f32_dq_kernel(AttnArgs a) {
  __shared__ tsg_f4 meet[4][NW][64];
  __shared__ int redo[NW];
  __shared__ float meet_delta[NW][64];
  int tid = threadIdx.x;
  if (any_wave<NW>(attn_f32_dq_tiles<NW, false>(a, tid, meet, meet_delta), tid >> 6, redo)) {
    tsg_again(tid);
    attn_f32_dq_tiles<NW, true>(a, tid, meet, meet_delta);
  }
}

template <int NW, bool SEEN> __device__ __forceinline__ float attn_f32_dkv_tiles(const AttnArgs& a, int tid, tsg_f4 (*meet)[NW][64]) {
  const int wave = tid >> 6, lane = tid & 63, h = lane >> 4;
  const int split = blockIdx.x / a.kv_heads % a.n_split, j0 = blockIdx.x / a.kv_heads / a.n_split * 16, kvh = blockIdx.x % a.kv_heads;
  const int j = j0 + (lane & 15);
  tsg_u4 kf[4], vf[4];
  {
    Rows16 k(a.k_row, a.chunks, wave, lane), v(a.v_row, a.chunks, wave, lane);
    k.at(a.k + (long)j0 * a.k_row + kvh * a.k_head, a.n_k - j0);
    v.at(a.v + (long)j0 * a.v_row + kvh * a.v_head, a.n_k - j0);
    k.rows(kf);
    v.rows(vf);
  }
  int lo, hi;
  rows_of_key(a, j0, j, lo, hi);
  const Bounds b = wave_bounds<16>(lo, hi);
  Sum16 dk, dv;
  const int per = b.wave_lo < b.wave_hi ? (b.wave_hi - b.wave_lo + 15) / 16 : 0, all = per * a.group;
  const int first = (int)((long)all * split / a.n_split), last = (int)((long)all * (split + 1) / a.n_split);
  Rows16 q(a.q_row, a.chunks, wave, lane), g(a.do_row, a.chunks, wave, lane);
  zero16(dk);
  zero16(dv);
  int head = kvh * a.group + (all ? first / per : 0), t0 = b.wave_lo + (all ? first % per : 0) * 16;
  for (int step = first, buf = 0; step < last; ++step, buf ^= 2) {
    tsg_u4 qf[4], gf[4];
    tsg_f4 qc[4], gc[4];
    q.at(a.q + head * a.q_head + (long)t0 * a.q_row, b.wave_hi - t0);
    g.at(a.d_o + head * a.do_head + (long)t0 * a.do_row, b.wave_hi - t0);
    q.rows(qf);
    g.rows(gf);
    if constexpr (!SEEN) g.cols(gc), q.cols(qc);
    float2 st[4];
    float delta[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long at = (long)head * a.n_q + min(t0 + 4 * h + i, b.wave_hi - 1);  // rows behind the interval are masked below
      st[i] = a.stat[at];
      delta[i] = a.delta[at];
    }
    tsg_f4 z = dot16(qf, kf, tsg_f4{0.0f, 0.0f, 0.0f, 0.0f}), dp = dot16(gf, vf, tsg_f4{0.0f, 0.0f, 0.0f, 0.0f});
    if (NW > 1) meet[buf][wave][lane] = z;
    dp = over_waves<NW>(meet[buf + 1], dp, wave, lane);
    if (NW > 1) {
      z = meet[buf][0][lane];
#pragma unroll
      for (int w = 1; w < NW; ++w) z += meet[buf][w][lane];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      z[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i] - st[i].x, a.scale2, -st[i].y));
      dp[i] = z[i] * (dp[i] - delta[i]);
    }
    if (t0 < b.in_lo || t0 + 16 > b.in_hi) {
      keep_branch();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t0 + 4 * h + i < lo || t0 + 4 * h + i >= hi) z[i] = dp[i] = 0.0f;
    }
    if constexpr (SEEN) {
      __builtin_amdgcn_sched_barrier(0);
      g.cols(gc);
      add16_seen(dv, gc, z, lo - t0 - 4 * h, hi - t0 - 4 * h);
      q.cols(qc);
      add16_seen(dk, qc, dp, lo - t0 - 4 * h, hi - t0 - 4 * h);
    } else {
      add16(dv, gc, z);
      add16(dk, qc, dp);
    }
    t0 += 16;
    if (t0 >= b.wave_hi) t0 = b.wave_lo, ++head;
  }
  const float zero = zero_of(dk, zero_of(dv));
  if (j >= a.n_k) return zero;
  if (a.n_split > 1) {
    char* p = reinterpret_cast<char*>(a.part + (((long)split * a.n_k + j) * a.kv_heads + kvh) * a.dim);
    store16(dk, p, 1.0f, a.dim, wave, h);
    store16(dv, p + (long)a.n_split * a.n_k * a.kv_heads * a.dim * 4, 1.0f, a.dim, wave, h);
  } else {
    store16(dk, a.dk + (long)j * a.dk_row + kvh * a.dk_head, a.scale, a.dim, wave, h);
    store16(dv, a.dv + (long)j * a.dv_row + kvh * a.dv_head, 1.0f, a.dim, wave, h);
  }
  return zero;
}
template <int NW> __global__ __launch_bounds__(64 * NW, 3) void attn_f32_dkv_kernel(AttnArgs a) {
  __shared__ tsg_f4 meet[4][NW][64];
  __shared__ int redo[NW];
  int tid = threadIdx.x;
  if (any_wave<NW>(attn_f32_dkv_tiles<NW, false>(a, tid, meet), tid >> 6, redo)) {
    tsg_again(tid);
    attn_f32_dkv_tiles<NW, true>(a, tid, meet);
  }
}

// dk and dv from the stretches' sums: four elements per thread, blockIdx.y 0: dk, 1: dv
template <typename D> __global__ __launch_bounds__(256) void attn_dkv_join_kernel(AttnArgs a) {
  const long all = (long)a.n_k * a.kv_heads * a.dim, i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= all) return;
  const float* p = a.part + (long)blockIdx.y * a.n_split * all + i;
  float4 s = *reinterpret_cast<const float4*>(p);
  for (int n = 1; n < a.n_split; ++n) {
    const float4 v = *reinterpret_cast<const float4*>(p + n * all);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  const int d = (int)(i % a.dim), kvh = (int)(i / a.dim % a.kv_heads);
  const long j = i / a.dim / a.kv_heads;
  const float by = blockIdx.y ? 1.0f : a.scale;
  char* to = blockIdx.y ? a.dv + j * a.dv_row + kvh * a.dv_head : a.dk + j * a.dk_row + kvh * a.dk_head;
  store4<D>(to + d * TsgElem<D>::BYTES, s.x * by, s.y * by, s.z * by, s.w * by);
}

// --------------------------------------------------------------------------------- few rows: one row, keys split
// One workgroup per (query row, key-value head, stretch of its heads, split of its keys).  LPR lanes hold a key (16 bytes
// each, NC of them), so a wave reads 64 / LPR keys at once; every such lane group keeps its own running maximum, sum and
// weighted values for the G heads that share the key, joined at the end through LDS, and over the splits by
// attn_join_kernel.  Bound by reading the keys and values once: 48 sequences of 700-9001 keys, 32 heads over 8, 128 wide, bf16: 195 us and 8 us for
// the join, 4.7 TB/s in all.
template <typename D> __device__ __forceinline__ float chunk_dot(tsg_u4 a, tsg_u4 b, float s) {  // two products an instruction
  typedef typename D::type T;
  typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const unsigned x = a[w], y = b[w];
    if constexpr (__is_same(D, TsgBf16)) s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(T2, x), __builtin_bit_cast(T2, y), s, false);
    else s = __builtin_amdgcn_fdot2(__builtin_bit_cast(T2, x), __builtin_bit_cast(T2, y), s, false);
  }
  return s;
}
template <> __device__ __forceinline__ float chunk_dot<TsgF32>(tsg_u4 a, tsg_u4 b, float s) {
#pragma unroll
  for (int w = 0; w < 4; ++w) s = __builtin_fmaf(__uint_as_float(a[w]), __uint_as_float(b[w]), s);
  return s;
}
template <typename D> __device__ __forceinline__ void chunk_to_f32(tsg_u4 u, float (&v)[TsgElem<D>::EPC]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const unsigned x = u[w];
    if constexpr (TsgElem<D>::BYTES == 4) {
      v[w] = __uint_as_float(x);
    } else {
      typedef typename D::type T;
      typedef T T2 __attribute__((ext_vector_type(2)));
      const T2 p = __builtin_bit_cast(T2, x);
      v[2 * w] = (float)p.x;
      v[2 * w + 1] = (float)p.y;
    }
  }
}
// sum over the LPR lanes of a key: inside a row of 16 lanes by DPP (no trip through LDS), beyond it by shuffles
template <int LPR> __device__ __forceinline__ float over_lanes(float v) {
  v += tsg_dpp<0xB1>(v);
  v += tsg_dpp<0x4E>(v);
  v += tsg_dpp<0x141>(v);
  if (LPR > 8) v += tsg_dpp<0x140>(v);
#pragma unroll
  for (int w = 16; w < LPR; w <<= 1) v += __shfl_xor(v, w, 64);
  return v;
}

template <typename D, int LPR, int NC, int G>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnArgs a) {
  constexpr int EPC = TsgElem<D>::EPC, NE = EPC * NC, PER = 64 / LPR, GROUPS = 4 * PER, U = G * NE > 32 ? 2 : 4;
  __shared__ float st_m[GROUPS][G], st_l[GROUPS][G];
  __shared__ float st_o[4][G][LPR * NE];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, part = lane % LPR, grp = wave * PER + lane / LPR;
  const int stretches = (a.group + G - 1) / G;
  int bid = blockIdx.x;
  const int split = bid % a.n_split;
  bid /= a.n_split;
  const int st = bid % stretches;
  bid /= stretches;
  const int kvh = bid % a.kv_heads, t = bid / a.kv_heads;
  const int head0 = kvh * a.group + st * G, n_heads = min(G, a.group - st * G);
  int lo, hi;
  keys_of_row(a, t, t, lo, hi);
  const long span = hi - lo;
  const int j0 = lo + (int)(span * split / a.n_split), j1 = lo + (int)(span * (split + 1) / a.n_split);
  tsg_u4 qv[G][NC];
  float o[G][NE], m[G], l[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -INFINITY, l[g] = 0.0f;
    const char* row = a.q + (long)t * a.q_row + (head0 + g) * a.q_head;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int ch = part + c * LPR;
      tsg_u4 u = {0u, 0u, 0u, 0u};
      if (g < n_heads && ch < a.chunks) u = *reinterpret_cast<const tsg_u4*>(row + ch * 16);
      qv[g][c] = u;
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) o[g][e] = 0.0f;
  }
  const char* kb = a.k + kvh * a.k_head;
  const char* vb = a.v + kvh * a.v_head;
  for (int j = j0 + grp; j < j1; j += GROUPS * U) {
    tsg_u4 kr[U][NC], vr[U][NC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int jj = min(j + u * GROUPS, j1 - 1);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int ch = min(part + c * LPR, a.chunks - 1);  // lanes behind the width read its last chunk, and drop it below
        kr[u][c] = *reinterpret_cast<const tsg_u4*>(kb + (long)jj * a.k_row + ch * 16);
        vr[u][c] = *reinterpret_cast<const tsg_u4*>(vb + (long)jj * a.v_row + ch * 16);
      }
    }
    if (a.chunks < LPR * NC) {
      keep_branch();
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (part + c * LPR >= a.chunks) {
#pragma unroll
          for (int u = 0; u < U; ++u) kr[u][c] = vr[u][c] = tsg_u4{0u, 0u, 0u, 0u};
        }
    }
    if (j + (U - 1) * GROUPS >= j1) {  // a key behind the end was read again: its value must not enter, not even times 0
      keep_branch();
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j + u * GROUPS >= j1) {
#pragma unroll
          for (int c = 0; c < NC; ++c) vr[u][c] = tsg_u4{0u, 0u, 0u, 0u};
        }
    }
    float z[G][U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) s = chunk_dot<D>(kr[u][c], qv[g][c], s);
        s = over_lanes<LPR>(s);
        z[g][u] = j + u * GROUPS >= j1 ? -INFINITY : s;
      }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float top = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) top = fmaxf(top, z[g][u]);
      const float off = top == -INFINITY ? 0.0f : top;
      const float fade = __builtin_amdgcn_exp2f((m[g] - off) * a.scale2);
      m[g] = top;
      l[g] *= fade;
#pragma unroll
      for (int e = 0; e < NE; ++e) o[g][e] *= fade;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        z[g][u] = __builtin_amdgcn_exp2f((z[g][u] - off) * a.scale2);
        l[g] += z[g][u];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float v[EPC];
        chunk_to_f32<D>(vr[u][c], v);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < EPC; ++e) o[g][c * EPC + e] = __builtin_fmaf(z[g][u], v[e], o[g][c * EPC + e]);
      }
  }
  // join the lane groups: common maximum, then sums over the groups of a wave (shuffles) and over the waves (LDS)
  if (part == 0)
#pragma unroll
    for (int g = 0; g < G; ++g) st_m[grp][g] = m[g], st_l[grp][g] = l[g];
  __syncthreads();
  float top[G], sum[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float v = -INFINITY;
#pragma unroll 4
    for (int x = 0; x < GROUPS; ++x) v = fmaxf(v, st_m[x][g]);
    top[g] = v;
    const float off = v == -INFINITY ? 0.0f : v;
    float s = 0.0f;
#pragma unroll 4
    for (int x = 0; x < GROUPS; ++x) s += st_l[x][g] * __builtin_amdgcn_exp2f((st_m[x][g] - off) * a.scale2);
    sum[g] = s;
    const float by = __builtin_amdgcn_exp2f((m[g] - off) * a.scale2);
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      float v2 = o[g][e] * by;
#pragma unroll
      for (int w = LPR; w < 64; w <<= 1) v2 += __shfl_xor(v2, w, 64);
      if (lane < LPR) st_o[wave][g][(part + (e / EPC) * LPR) * EPC + e % EPC] = v2;
    }
  }
  __syncthreads();
  for (int x = tid; x < G * a.dim; x += 256) {
    const int g = x / a.dim, d = x % a.dim;
    if (g >= n_heads) break;
    const float v = (st_o[0][g][d] + st_o[1][g][d]) + (st_o[2][g][d] + st_o[3][g][d]);
    float sg = 0.0f, tg = 0.0f;
#pragma unroll
    for (int y = 0; y < G; ++y)
      if (y == g) sg = sum[y], tg = top[y];
    if (a.n_split == 1) {
      typedef typename D::type T;
      const float x = v * (sg == 0.0f ? 0.0f : 1.0f / sg);
      reinterpret_cast<T*>(a.out + (long)t * a.o_row + (head0 + g) * a.o_head)[d] = (T)x;
      if (a.rest) reinterpret_cast<T*>(a.rest)[((long)t * a.heads + head0 + g) * a.dim + d] = (T)(x - (float)(T)x);
      if (d == 0) a.stat[(long)(head0 + g) * a.n_q + t] = sg == 0.0f ? make_float2(0.0f, INFINITY) : make_float2(tg, __builtin_amdgcn_logf(sg));
    } else {
      float* p = a.part + (((long)t * a.heads + head0 + g) * a.n_split + split) * (a.dim + 2);
      p[d] = v;
      if (d == 0) p[a.dim] = tg, p[a.dim + 1] = sg;
    }
  }
}

// one wave per (row, head): the splits' maxima, sums and weighted values
template <typename D> __global__ __launch_bounds__(64) void attn_join_kernel(AttnArgs a) {
  const int t = blockIdx.x / a.heads, head = blockIdx.x % a.heads, lane = threadIdx.x;
  const float* p = a.part + ((long)t * a.heads + head) * a.n_split * (a.dim + 2);
  float top = -INFINITY;
  for (int s = lane; s < a.n_split; s += 64) top = fmaxf(top, p[(long)s * (a.dim + 2) + a.dim]);
  top = tsg_wave_max(top);
  const float off = top == -INFINITY ? 0.0f : top;
  float l = 0.0f;
  for (int s = lane; s < a.n_split; s += 64)
    l += p[(long)s * (a.dim + 2) + a.dim + 1] * __builtin_amdgcn_exp2f((p[(long)s * (a.dim + 2) + a.dim] - off) * a.scale2);
  l = tsg_wave_sum(l);
  const float by = l == 0.0f ? 0.0f : 1.0f / l;
  typedef typename D::type T;
  for (int d = lane; d < a.dim; d += 64) {
    float v = 0.0f;
    for (int s = 0; s < a.n_split; ++s)
      v += p[(long)s * (a.dim + 2) + d] * __builtin_amdgcn_exp2f((p[(long)s * (a.dim + 2) + a.dim] - off) * a.scale2);
    v *= by;
    reinterpret_cast<T*>(a.out + (long)t * a.o_row + head * a.o_head)[d] = (T)v;
    if (a.rest) reinterpret_cast<T*>(a.rest)[((long)t * a.heads + head) * a.dim + d] = (T)(v - (float)(T)v);
  }
  if (lane == 0) a.stat[(long)head * a.n_q + t] = l == 0.0f ? make_float2(0.0f, INFINITY) : make_float2(top, __builtin_amdgcn_logf(l));
}

// -------------------------------------------------------------------------------- backward for heads wider than 256
// One wave per row (dq) or key (dk, dv), lanes over the width.  Heads this wide are the largest recurrent states only.
constexpr int WIDE = 8;  // elements per lane: dim <= 512
template <typename T> __device__ __forceinline__ void load_wide(float (&x)[WIDE], const char* row, int dim, int lane) {
#pragma unroll
  for (int e = 0; e < WIDE; ++e) x[e] = lane + 64 * e < dim ? (float)reinterpret_cast<const T*>(row)[lane + 64 * e] : 0.0f;
}
template <typename T> __device__ __forceinline__ void store_wide(const float (&x)[WIDE], char* row, float by, int dim, int lane) {
#pragma unroll
  for (int e = 0; e < WIDE; ++e)
    if (lane + 64 * e < dim) reinterpret_cast<T*>(row)[lane + 64 * e] = (T)(x[e] * by);
}
__device__ __forceinline__ float dot_wide(const float (&x)[WIDE], const float (&y)[WIDE]) {
  float s = 0.0f;
#pragma unroll
  for (int e = 0; e < WIDE; ++e) s += x[e] * y[e];
  return tsg_wave_sum_u(s);
}
template <typename D> __global__ __launch_bounds__(64) void attn_wide_dq_kernel(AttnArgs a) {
  typedef typename D::type T;
  const int t = blockIdx.x / a.heads, head = blockIdx.x % a.heads, kvh = head / a.group, lane = threadIdx.x;
  int lo, hi;
  keys_of_row(a, t, t, lo, hi);
  float q[WIDE], g[WIDE], x[WIDE], acc[WIDE];
  load_wide<T>(q, a.q + (long)t * a.q_row + head * a.q_head, a.dim, lane);
  load_wide<T>(g, a.d_o + (long)t * a.do_row + head * a.do_head, a.dim, lane);
  load_wide<T>(x, a.o + (long)t * a.o_row + head * a.o_head, a.dim, lane);
  float delta = dot_wide(g, x);
  if (a.rest) {
    load_wide<T>(x, a.rest + ((long)t * a.heads + head) * a.dim * sizeof(T), a.dim, lane);
    delta += dot_wide(g, x);
  }
  const float2 st = a.stat[(long)head * a.n_q + t];
  if (lane == 0) a.delta[(long)head * a.n_q + t] = delta;
#pragma unroll
  for (int e = 0; e < WIDE; ++e) acc[e] = 0.0f;
  for (int j = lo; j < hi; ++j) {
    load_wide<T>(x, a.v + (long)j * a.v_row + kvh * a.v_head, a.dim, lane);
    const float dp = dot_wide(g, x);
    load_wide<T>(x, a.k + (long)j * a.k_row + kvh * a.k_head, a.dim, lane);
    const float ds = __builtin_amdgcn_exp2f(__builtin_fmaf(dot_wide(q, x) - st.x, a.scale2, -st.y)) * (dp - delta);
#pragma unroll
    for (int e = 0; e < WIDE; ++e) acc[e] += ds * x[e];
  }
  store_wide<T>(acc, a.dq + (long)t * a.dq_row + head * a.dq_head, a.scale, a.dim, lane);
}
template <typename D> __global__ __launch_bounds__(64) void attn_wide_dkv_kernel(AttnArgs a) {
  typedef typename D::type T;
  const int j = blockIdx.x / a.kv_heads, kvh = blockIdx.x % a.kv_heads, lane = threadIdx.x;
  int lo, hi;
  rows_of_key(a, j, j, lo, hi);
  float k[WIDE], v[WIDE], x[WIDE], dk[WIDE], dv[WIDE];
  load_wide<T>(k, a.k + (long)j * a.k_row + kvh * a.k_head, a.dim, lane);
  load_wide<T>(v, a.v + (long)j * a.v_row + kvh * a.v_head, a.dim, lane);
#pragma unroll
  for (int e = 0; e < WIDE; ++e) dk[e] = dv[e] = 0.0f;
  for (int head = kvh * a.group; head < (kvh + 1) * a.group; ++head)
    for (int t = lo; t < hi; ++t) {
      load_wide<T>(x, a.d_o + (long)t * a.do_row + head * a.do_head, a.dim, lane);
      const float dp = dot_wide(v, x) - a.delta[(long)head * a.n_q + t];
      float q[WIDE];
      load_wide<T>(q, a.q + (long)t * a.q_row + head * a.q_head, a.dim, lane);
      const float2 st = a.stat[(long)head * a.n_q + t];
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(dot_wide(q, k) - st.x, a.scale2, -st.y));
#pragma unroll
      for (int e = 0; e < WIDE; ++e) {
        dv[e] += p * x[e];
        dk[e] += p * dp * q[e];
      }
    }
  store_wide<T>(dk, a.dk + (long)j * a.dk_row + kvh * a.dk_head, a.scale, a.dim, lane);
  store_wide<T>(dv, a.dv + (long)j * a.dv_row + kvh * a.dv_head, 1.0f, a.dim, lane);
}

// ------------------------------------------------------------------------------------------------------ host side
int rows_g(int group) { return group >= 8 ? 8 : (group >= 4 ? 4 : (group >= 2 ? 2 : 1)); }

// The rows kernel reads a row's keys once per row; a tile kernel once per 128 rows, but spends 128 rows' worth of matrix
// work on them.  Rows of one sequence share their keys, so the tile form wins as soon as a sequence has a few dozen rows,
// and also where there are no more keys than rows around (short sequences lie side by side in a tile).
bool use_rows(const tsg_attn_desc* d) {
  if (d->dim > 256) return true;
  return d->n_k >= 8 * d->n_q && d->n_q < 16 * (int64_t)d->n_seq;
}
int splits_of(const tsg_attn_desc* d) {
  const int64_t wgs = d->n_q * (int64_t)d->kv_heads * tsg_cdiv(d->heads / d->kv_heads, rows_g(d->heads / d->kv_heads));
  int64_t n = (2048 + wgs - 1) / wgs;
  const int64_t mean = d->n_k / (d->n_seq > 0 ? d->n_seq : 1);
  if (n > mean / 128) n = mean / 128;
  return (int)(n < 1 ? 1 : (n > 1024 ? 1024 : n));
}
size_t workspace_of(const tsg_attn_desc* d) {
  if (!use_rows(d)) return 0;
  const int n = splits_of(d);
  return n == 1 ? 0 : (size_t)d->n_q * d->heads * n * (d->dim + 2) * 4;
}

// A tile of keys walks every row that sees it, for all heads of its group: the first keys of a long sequence walk twice the mean,
// and a workgroup's walk is one chain.  Cut until there are three rounds of workgroups, but no shorter than eight steps of
// 64 rows in the mean; the sums then meet in f32 (4 sequences of 2.5-4 k positions, 16 heads over 4, 128 wide).
int dkv_splits_of(const tsg_attn_desc* d) {
  if (d->dim > 256 || d->n_seq <= 0) return 1;
  const int64_t wgs = (int64_t)tsg_cdiv(d->n_k, d->dtype == TSG_F32 ? 16 : 128) * d->kv_heads;
  const int64_t steps = d->n_q / d->n_seq * (d->heads / d->kv_heads) / 64 / 2;
  int64_t n = wgs ? 1536 / wgs : 1;
  if (n > steps / 8) n = steps / 8;
  return (int)(n < 1 ? 1 : (n > 16 ? 16 : n));
}
size_t backward_workspace_of(const tsg_attn_desc* d) {
  const int n = dkv_splits_of(d);
  return n == 1 ? 0 : (size_t)2 * n * d->n_k * d->kv_heads * d->dim * 4;
}

int check_attn(const tsg_attn_desc* d, bool backward) {
  if (!d) return TSG_E_INVALID;
  if (d->dtype != TSG_F32 && d->dtype != TSG_BF16 && d->dtype != TSG_F16) return TSG_E_INVALID;
  if (d->n_seq < 0 || d->n_q < 0 || d->n_k < 0 || d->heads <= 0 || d->kv_heads <= 0 || d->dim <= 0) return TSG_E_INVALID;
  if (d->heads % d->kv_heads) return TSG_E_INVALID;
  if (!(d->scale > 0.0f) || !(d->scale < INFINITY)) return TSG_E_INVALID;
  const int bytes = d->dtype == TSG_F32 ? 4 : 2, epc = 16 / bytes;
  if (d->dim > 512 || d->n_q > 0x7ffffff0L || d->n_k > 0x7ffffff0L) return TSG_E_LIMIT;
  if (d->n_q * (int64_t)d->heads > 0x7fffffffL || d->n_k * (int64_t)d->kv_heads > 0x7fffffffL) return TSG_E_LIMIT;
  if (d->dim % epc) return TSG_E_INVALID;
  if (!d->q_ptr || !d->k_ptr || !d->stats || (uintptr_t)d->stats % 8) return TSG_E_INVALID;
  const void* p[9] = {d->q, d->k, d->v, d->out, backward ? d->d_out : nullptr, backward ? d->dq : nullptr,
                      backward ? d->dk : nullptr, backward ? d->dv : nullptr, nullptr};
  const int64_t s[16] = {d->q_row, d->q_head, d->k_row, d->k_head, d->v_row, d->v_head, d->out_row, d->out_head,
                         backward ? d->d_out_row : 0, backward ? d->d_out_head : 0, backward ? d->dq_row : 0, backward ? d->dq_head : 0,
                         backward ? d->dk_row : 0, backward ? d->dk_head : 0, backward ? d->dv_row : 0, backward ? d->dv_head : 0};
  for (int i = 0; i < (backward ? 8 : 4); ++i)
    if (!p[i] || (uintptr_t)p[i] % 16) return TSG_E_INVALID;
  for (int i = 0; i < 16; ++i)
    if (s[i] % epc || s[i] < 0) return TSG_E_INVALID;
  if (backward && !d->delta) return TSG_E_INVALID;
  for (int i = 0; i < 16; i += 2)
    if (s[i] * bytes >= (1 << 24)) return TSG_E_LIMIT;  // offsets inside a tile of 64 rows are 32-bit
  if ((uintptr_t)d->out_rest % 16) return TSG_E_INVALID;
  return 0;
}

AttnArgs args_of(const tsg_attn_desc* d) {
  AttnArgs a;
  const long b = d->dtype == TSG_F32 ? 4 : 2;
  a.n_seq = d->n_seq, a.heads = d->heads, a.kv_heads = d->kv_heads, a.group = d->heads / d->kv_heads;
  a.dim = d->dim, a.chunks = (int)(d->dim * b / 16);
  a.n_q = (int)d->n_q, a.n_k = (int)d->n_k;
  a.q_ptr = d->q_ptr, a.k_ptr = d->k_ptr;
  a.q = (const char*)d->q, a.k = (const char*)d->k, a.v = (const char*)d->v, a.o = (const char*)d->out, a.d_o = (const char*)d->d_out;
  a.out = (char*)d->out, a.dq = (char*)d->dq, a.dk = (char*)d->dk, a.dv = (char*)d->dv;
  a.q_row = d->q_row * b, a.q_head = d->q_head * b, a.k_row = d->k_row * b, a.k_head = d->k_head * b;
  a.v_row = d->v_row * b, a.v_head = d->v_head * b, a.o_row = d->out_row * b, a.o_head = d->out_head * b;
  a.do_row = d->d_out_row * b, a.do_head = d->d_out_head * b, a.dq_row = d->dq_row * b, a.dq_head = d->dq_head * b;
  a.dk_row = d->dk_row * b, a.dk_head = d->dk_head * b, a.dv_row = d->dv_row * b, a.dv_head = d->dv_head * b;
  a.stat = (float2*)d->stats, a.delta = d->delta;
  a.scale = d->scale, a.scale2 = d->scale * 1.44269504088896340736f;
  a.rest = d->dtype == TSG_F32 ? nullptr : (char*)d->out_rest;
  a.n_split = 1;
  a.part = (float*)d->workspace;
  return a;
}

template <typename D, int LPR, int NC> void launch_rows(const AttnArgs& a, hipStream_t s) {
  const int g = rows_g(a.group);
  const dim3 grid((unsigned)((long)a.n_q * a.kv_heads * tsg_cdiv(a.group, g) * a.n_split)), block(256);
  if (g == 8) {
    if constexpr (NC == 1) hipLaunchKernelGGL((attn_rows_kernel<D, LPR, NC, 8>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attn_rows_kernel<D, LPR, NC, 4>), dim3(grid.x / tsg_cdiv(a.group, 8) * tsg_cdiv(a.group, 4)), block, 0, s, a);
  } else if (g == 4) hipLaunchKernelGGL((attn_rows_kernel<D, LPR, NC, 4>), grid, block, 0, s, a);
  else if (g == 2) hipLaunchKernelGGL((attn_rows_kernel<D, LPR, NC, 2>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((attn_rows_kernel<D, LPR, NC, 1>), grid, block, 0, s, a);
}

template <typename D> int forward_of(const tsg_attn_desc* d, hipStream_t s) {
  AttnArgs a = args_of(d);
  if (use_rows(d)) {
    a.n_split = splits_of(d);
    if ((long)a.n_q * a.kv_heads * tsg_cdiv(a.group, rows_g(a.group)) * 2 * a.n_split > 0x7fffffffL) return TSG_E_LIMIT;
    constexpr int F = TsgElem<D>::BYTES / 2;  // 1: 16-bit types, 2: f32
    if (a.dim <= 64) launch_rows<D, 8 * F, 1>(a, s);
    else if (a.dim <= 128) launch_rows<D, 16 * F, 1>(a, s);
    else if (a.dim <= 256) launch_rows<D, 32 * F, 1>(a, s);
    else launch_rows<D, 64, F>(a, s);
    if (a.n_split > 1) hipLaunchKernelGGL(attn_join_kernel<D>, dim3((unsigned)((long)a.n_q * a.heads)), dim3(64), 0, s, a);
  } else {
    const dim3 grid((unsigned)(tsg_cdiv(a.n_q, rows_per_wg<D>()) * a.heads)), block(256);
    if constexpr (__is_same(D, TsgF32)) {
      if (a.dim <= 64) hipLaunchKernelGGL(attn_f32_fwd_kernel<1>, grid, dim3(64), 0, s, a);
      else if (a.dim <= 128) hipLaunchKernelGGL(attn_f32_fwd_kernel<2>, grid, dim3(128), 0, s, a);
      else hipLaunchKernelGGL(attn_f32_fwd_kernel<4>, grid, block, 0, s, a);
    } else {
      if (a.dim <= 64) hipLaunchKernelGGL((attn_fwd_kernel<D, 64, 64>), grid, block, 0, s, a);
      else if (a.dim <= 128) hipLaunchKernelGGL((attn_fwd_kernel<D, 128, 64>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((attn_fwd_kernel<D, 256, 32>), grid, block, 0, s, a);
    }
  }
  TSG_LAUNCH_CHECK();
  return 0;
}

template <typename D, bool REST> void launch_backward(const AttnArgs& a, dim3 gq, dim3 gk, hipStream_t s) {
  const dim3 block(256);
  if (a.n_q) {
    if (a.dim <= 64) hipLaunchKernelGGL((attn_dq_kernel<D, 64, 64, REST>), gq, block, 0, s, a);
    else if (a.dim <= 128) hipLaunchKernelGGL((attn_dq_kernel<D, 128, 64, REST>), gq, block, 0, s, a);
    else hipLaunchKernelGGL((attn_dq_kernel<D, 256, 32, REST>), gq, block, 0, s, a);
  }
  if (a.n_k) {
    if (a.dim <= 64) hipLaunchKernelGGL((attn_dkv_kernel<D, 64, 32, 0, REST || lifted<D>(), REST>), gk, block, 0, s, a);  // the rest, and the powers of two, take the values' registers
    else if (a.dim <= 128) hipLaunchKernelGGL((attn_dkv_kernel<D, 128, 32, 0, true, REST>), gk, block, 0, s, a);
    else {
      hipLaunchKernelGGL((attn_dkv_kernel<D, 256, 32, 1, false, false>), gk, block, 0, s, a);
      hipLaunchKernelGGL((attn_dkv_kernel<D, 256, 32, 2, true, REST>), gk, block, 0, s, a);
    }
  }
}

template <typename D> int backward_of(const tsg_attn_desc* d, hipStream_t s) {
  AttnArgs a = args_of(d);
  a.n_split = dkv_splits_of(d);
  const dim3 block(256);
  if (a.dim > 256) {
    if (a.n_q) hipLaunchKernelGGL(attn_wide_dq_kernel<D>, dim3((unsigned)((long)a.n_q * a.heads)), dim3(64), 0, s, a);
    if (a.n_k) hipLaunchKernelGGL(attn_wide_dkv_kernel<D>, dim3((unsigned)((long)a.n_k * a.kv_heads)), dim3(64), 0, s, a);
    TSG_LAUNCH_CHECK();
    return 0;
  }
  constexpr int R = rows_per_wg<D>();
  const dim3 gq((unsigned)(tsg_cdiv(a.n_q, R) * a.heads)), gk((unsigned)(tsg_cdiv(a.n_k, R) * a.kv_heads * a.n_split));
  if constexpr (__is_same(D, TsgF32)) {
    if (a.n_q) {
      if (a.dim <= 64) hipLaunchKernelGGL(attn_f32_dq_kernel<1>, gq, dim3(64), 0, s, a);
      else if (a.dim <= 128) hipLaunchKernelGGL(attn_f32_dq_kernel<2>, gq, dim3(128), 0, s, a);
      else hipLaunchKernelGGL(attn_f32_dq_kernel<4>, gq, block, 0, s, a);
    }
    if (a.n_k) {
      if (a.dim <= 64) hipLaunchKernelGGL(attn_f32_dkv_kernel<1>, gk, dim3(64), 0, s, a);
      else if (a.dim <= 128) hipLaunchKernelGGL(attn_f32_dkv_kernel<2>, gk, dim3(128), 0, s, a);
      else hipLaunchKernelGGL(attn_f32_dkv_kernel<4>, gk, block, 0, s, a);
    }
  } else {
    if (d->n_q < 1024 * (int64_t)d->n_seq) launch_backward<D, true>(a, gq, gk, s);
    else launch_backward<D, false>(a, gq, gk, s);
  }
  if (a.n_k && a.n_split > 1)
    hipLaunchKernelGGL(attn_dkv_join_kernel<D>, dim3((unsigned)(((long)a.n_k * a.kv_heads * a.dim / 4 + 255) / 256), 2), block, 0, s, a);
  TSG_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" int tsg_attn_workspace(const tsg_attn_desc* d, size_t* forward_bytes_host, size_t* backward_bytes_host) {
  if (!d || !forward_bytes_host || !backward_bytes_host) return TSG_E_INVALID;
  if (d->n_q < 0 || d->n_k < 0 || d->dim <= 0 || d->heads <= 0 || d->kv_heads <= 0 || d->heads % d->kv_heads) return TSG_E_INVALID;
  *forward_bytes_host = d->n_q ? workspace_of(d) : 0;
  *backward_bytes_host = d->n_k ? backward_workspace_of(d) : 0;
  return 0;
}

extern "C" int tsg_attn_forward(const tsg_attn_desc* d, void* stream) {
  if (d && d->n_q == 0 && d->heads > 0) return 0;
  const int rc = check_attn(d, false);
  if (rc) return rc;
  const size_t need = workspace_of(d);
  if (need && (!d->workspace || d->workspace_bytes < need)) return TSG_E_TOO_SMALL;
  hipStream_t s = (hipStream_t)stream;
  return d->dtype == TSG_F32 ? forward_of<TsgF32>(d, s) : (d->dtype == TSG_BF16 ? forward_of<TsgBf16>(d, s) : forward_of<TsgF16>(d, s));
}

extern "C" int tsg_attn_backward(const tsg_attn_desc* d, void* stream) {
  if (d && d->n_q == 0 && d->n_k == 0) return 0;
  const int rc = check_attn(d, true);
  if (rc) return rc;
  const size_t need = backward_workspace_of(d);
  if (need && (!d->workspace || (uintptr_t)d->workspace % 16 || d->workspace_bytes < need)) return TSG_E_TOO_SMALL;
  hipStream_t s = (hipStream_t)stream;
  return d->dtype == TSG_F32 ? backward_of<TsgF32>(d, s) : (d->dtype == TSG_BF16 ? backward_of<TsgBf16>(d, s) : backward_of<TsgF16>(d, s));
}
