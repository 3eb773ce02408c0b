// Attention over packed sequences (gfx950): out = softmax(scale q k^T) v for sequences of different lengths that lie one
// behind the other in [tokens, heads, dim] tensors, with grouped heads, causal or not, in fp16, bf16 and fp32.
//
// One pass over the keys with a running maximum and sum (softmax in the log2 domain, fp32).  Orientation: S^T = K Q^T puts
// the keys on the accumulator registers and the query on the lane, so maximum and sum are taken in registers plus one
// exchange of the lane halves, and the exponentiated tile is already the B operand of O^T += V^T P^T: accumulator element i
// of lane half h is key 8 (i / 4) + 4 h + i % 4, and the V^T fragments are read in that order of keys.
//
// A row is one query of one head; the rows of a key head's group are taken together (row r = query r / group, head
// r % group), so K and V are read once for the group and a single query still fills `group` rows.
//
// Bounds, and what was reached (16-bit heads unless said otherwise; a large matrix product reaches 1390 TFLOP/s here):
//   many rows: the products and the exponentials, which share a wave's issue.  A 32x32x16 product takes 32 clocks of the matrix
//     unit; four vector instructions beside it add 5 in one wave and 2 with two waves on the SIMD, eight add 19 and 13 (a score
//     block needs 5.5 to a product with heads of 128, 12 with heads of 64).  Heads of 128 (64 rows a wave, one wave a SIMD,
//     its loop pipelined): 1020 TFLOP/s on a causal prompt of 16384 (16 / 4 heads), 920 on 8 causal prompts of 4096 (32 / 8); heads
//     of 64 (two waves a SIMD), where a score has half the products to its exponential: 960 on 8 x 4096 tokens (12 heads); images
//     of 1 .. 2305 tokens 640, of which a fifth is rows that do not fill a tile.  64 rows a wave, because K and V come from LDS:
//     with 32 the reads alone would take as long as the products.  Heads of 80: 660 on 3 x 4097, 2305, 3137 tokens (16 heads; 96
//     output columns, bank conflicts in half of the LDS cycles).
//   few rows on keys that are there already (up to 512 queries on 900 .. 8077 keys): 250, the grid's bounds leave blocks empty.
//   single queries: the bytes of K and V.  64 on 4096 keys each 5.7 TB/s, 16 on 1 .. 16000 keys 4.7 (a copy: 5.0); fp32 3.0.
//   fp32: six bf16 products for one (below), 178 on 32 x 785 tokens, 213 on 8 x 4096 (12 heads of 64), where the fp32 instruction
//     reached 105 .. 140.
#include "common.h"

namespace {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct AttArgs {
  const void *q, *k, *v; void* out; float* sums;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;
  const int32_t *starts_q, *starts_k;
  int tokens_q, tokens_k, sequences, heads, kv_heads, group, dim, causal;
  float c_log2;                      // |scale| log2(e), positive: masked scores are -inf before it is applied
  uint32_t q_keep, q_flip;           // bits of q that stay, and that turn: a negative scale negates q, a zero one clears it
  int clear;                         // rows before the first and behind the last sequence: 1 zero in out, 2 -inf in sums
  int pairs, replicas, together, tiles, splits, chunk;    // the grid (launch())
  float* part_o; float* part_ml;     // a split key axis: each part's weighted mean, and its maximum and sum
};

// ---- the three types: a 16-byte fragment, its products, and P
template <class T> struct Num;
template <> struct Num<_Float16> {
  typedef half8 frag;
  static constexpr bool wide = false;              // (odd(): does a word hold an infinity or NaN?)
  __device__ static f32x16 mfma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  __device__ static uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, half2v{(_Float16)a, (_Float16)b}); }
  __device__ static bool odd(uint32_t w) { return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u; }
};
template <> struct Num<__bf16> {
  typedef bf8 frag;
  static constexpr bool wide = false;
  __device__ static f32x16 mfma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  __device__ static uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf2)); }
  __device__ static bool odd(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
};
template <> struct Num<float> {
  typedef f32x4 frag;
  static constexpr bool wide = true;
  __device__ static bool odd(uint32_t w) { return (w & 0x7f800000u) == 0x7f800000u; }
  // four products of two: lane half h holds four neighbouring entries of the contraction
  __device__ static f32x16 mfma(frag a, frag b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// fp32 on the bf16 products: x = h + m + l, three bf16 values of 8 bits each, exactly where l is not under the smallest normal
// number (h and m cut off, no rounding, so that no finite x overflows), and x y = h h + (h m + m h) + (m m + h l + l h), smallest
// first; what is left out, m l + l m + l l, has the product's sign and is under 2^-21 of it (m < 2^-7 x, l < 2^-15 x): eight half-steps
// of fp32, where a chain of D fp32 products may lose D.  Calls of at most 32 rows take the fp32 instruction, so the last digits of a
// row are other ones there.
// Six products of 2.5 PFLOP/s peak against the 157 TFLOP/s of the fp32 instruction.  An infinity or NaN makes NaN, which the
// end of the kernel looks for.
struct Thirds { bf8 h, m, l; };
__device__ inline Thirds thirds(const float (&x)[8]) {
  u32x4 h, m, l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t a[2][3];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      a[i][0] = __builtin_bit_cast(uint32_t, x[2 * j + i]);
      const float r = x[2 * j + i] - __builtin_bit_cast(float, a[i][0] & 0xffff0000u);
      a[i][1] = __builtin_bit_cast(uint32_t, r);
      const float q = r - __builtin_bit_cast(float, a[i][1] & 0xffff0000u);
      a[i][2] = __builtin_bit_cast(uint32_t, q);
    }
    h[j] = __builtin_amdgcn_perm(a[1][0], a[0][0], 0x07060302u);       // the upper halves of two words
    m[j] = __builtin_amdgcn_perm(a[1][1], a[0][1], 0x07060302u);
    l[j] = __builtin_amdgcn_perm(a[1][2], a[0][2], 0x07060302u);
  }
  return {__builtin_bit_cast(bf8, h), __builtin_bit_cast(bf8, m), __builtin_bit_cast(bf8, l)};
}
__device__ inline f32x16 product(const Thirds& a, const Thirds& b, f32x16 c) {
  c = Num<__bf16>::mfma(a.l, b.h, c);
  c = Num<__bf16>::mfma(a.h, b.l, c);
  c = Num<__bf16>::mfma(a.m, b.m, c);
  c = Num<__bf16>::mfma(a.m, b.h, c);
  c = Num<__bf16>::mfma(a.h, b.m, c);
  return Num<__bf16>::mfma(a.h, b.h, c);
}

// ---- a tile of keys in LDS: rows of NS steps of 32 bytes (S = 2 NS slots of 16), slots moved by the row so that the reads
// of neighbouring rows meet different banks: XOR where S is a power of two, rotation otherwise.
template <int NS> struct Slots {
  static constexpr int S = 2 * NS, P = 32 * NS;
  static constexpr bool pow2 = (S & (S - 1)) == 0;
  static constexpr int gcd16(int x) { return x % 16 == 0 ? 16 : x % 8 == 0 ? 8 : x % 4 == 0 ? 4 : x % 2 == 0 ? 2 : 1; }
  static constexpr int period = 16 / gcd16(S);
  // K: 16 rows of one slot column
  __device__ static int k_turn(int row) { return ((row & 31) / period) % S; }
  // V, 16-bit transposed reads: four rows of 64 bytes; fp32: two rows, four apart, of 128 bytes
  template <bool WIDE> __device__ static int v_turn(int row) {
    if (WIDE) return (S % 4 == 0 && S >= 16) ? 8 * ((row >> 2) & 1) : 0;
    return S % 16 == 0 ? 4 * (row & 3) : S % 8 == 0 ? 4 * ((row & 3) >> 1) : 0;
  }
  __device__ static int place(int slot, int turn) {
    if (pow2) return slot ^ turn;
    const int p = slot + turn;
    return p >= S ? p - S : p;
  }
  __device__ static int slot_at(int place_, int turn) {      // the inverse
    if (pow2) return place_ ^ turn;
    const int p = place_ - turn;
    return p < 0 ? p + S : p;
  }
};

__device__ inline uint32_t first_lane(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// 16 bytes per lane from a buffer into LDS at `at` (uniform) + 16 * lane; an offset behind the descriptor's end writes zeros.  As
// assembly because the compiler, which cannot tell the tiles apart, waits for every transfer in flight before it reads any of
// them; the kernel's own waits order both.  It writes no register but M0 (one wait state between that and its use).
__device__ inline void to_lds(u32x4 rsrc, uint32_t offset, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(first_lane(at)), "v"(offset), "s"(rsrc) : "memory", "m0");
}
template <int N> __device__ inline void wait_transfers() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ inline void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// the larger of the two lane halves' values, in both
__device__ inline float halves_max(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t lower = p[0], upper = p[1];       // (a bit cast of p[1] itself reads p[0])
  return fmaxf(__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper));
}

constexpr float NO_MAX = -3.0e38f;     // of a row that has seen no key: finite, so that no difference of infinities arises

// NS: steps of 32 bytes of a row (dim rounded up); NQ: blocks of 32 rows per wave; WQ x WK waves: over rows x over keys;
// KB: blocks of 32 keys per wave and tile
template <class T, int NS, int NQ, int WQ, int WK, int KB>
struct Shape {
  static constexpr int W = WQ * WK, THREADS = 64 * W, ROWS = 32 * NQ * WQ, KEYS = 32 * KB * WK;
  static constexpr int P = 32 * NS, S = 2 * NS, TILE = KEYS * P;           // bytes of K (or V) of a tile
  static constexpr int E = 16 / (int)sizeof(T);                            // entries of a slot
  static constexpr int DB = (NS * 2 * E + 31) / 32;                        // blocks of 32 entries of the output
  static constexpr int BUF = 2 * TILE;
  static constexpr bool SPLIT = sizeof(T) == 4 && WQ > 1;                  // fp32 in thirds; few rows: the fp32 instruction
  static constexpr bool RING = sizeof(T) == 2 && WQ > 1 && 4 * BUF + 256 <= 160 * 1024;  // the pipelined loop: four tiles; else two
  static constexpr int BUFS = RING ? 4 : 2;
  static constexpr int JOIN = WK > 1 ? (WK - 1) * WQ * NQ * 64 * (DB * 16 + 2) * 4 : 0;
  // SPLIT: V's three planes, K's, then the fp32 tile that they are made of
  static constexpr int PLANE = TILE / 2, STAGE = 6 * PLANE;
  static constexpr int LDS = SPLIT ? STAGE + BUF : BUFS * BUF + 256 > JOIN ? BUFS * BUF + 256 : JOIN;
  // registers: queries, output, two blocks of scores, weights, K and V fragments, the rest
  static constexpr int REGS = SPLIT ? NQ * (NS * 6 + DB * 16 + 40) + 56 : NQ * (NS * 4 + DB * 16 + (RING ? 32 : 16) + (sizeof(T) == 2 ? 8 : 0)) + (RING ? 2 * NS * 4 : 16) + 40;
  static constexpr int WAVES = REGS <= 128 && LDS <= 40960 ? 4 : REGS <= 168 && LDS <= 54000 ? 3 : REGS <= 256 && LDS <= 81920 ? 2 : 1;
  static constexpr int NI = TILE / 1024;                                   // transfers of 64 x 16 bytes per tile of K (or V)
  static constexpr int NJ = (NI + W - 1) / W;
};

// Rows [first, last) of a wave once more, key by key, over the keys that each sees alone: where values that some row does not see
// are infinite or NaN, and where a sum of finite scores and weights came out infinite or NaN.  That happens to finite values too:
// the sums below weigh them up to 2^8 (rescale()), n keys add up, and from FLT_MAX / (2^8 n) on they leave the range though their
// weighted mean does not; and to an infinite value whose weight is 0 in the tensor's type (fp16: under 2^-25) and not in fp32.
// Here weights are at most 2^-K with 2^K > n, exactly scaled, and stay fp32, so that no finite value overflows.  Lane -> key for
// the scores, -> entries of the head for the sum.  Not made to be fast: 4096 causal tokens, 16 / 4 heads of 128 bf16, every row done
// again 68 ms (0.12 without).
template <class T, int DMAX>
__device__ inline void again(const AttArgs& a, int split, int begin, int end, int q0, int nq, int k0, int nk, int kvh, int first, int last, int lane) {
  constexpr int ND = (DMAX + 63) / 64;
  for (int row = first; row < last; ++row) {
    const int i = row / a.group, hh = kvh * a.group + row - i * a.group;
    const int seen = min(end, a.causal ? min(max(i + nk - nq + 1, 0), nk) : nk);
    const T* q = static_cast<const T*>(a.q) + (int64_t)(q0 + i) * a.q_tok + (int64_t)hh * a.q_head;
    float m = NO_MAX, l = 0.f, o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = 0.f;
    const float c = a.q_keep ? (a.q_flip ? -a.c_log2 : a.c_log2) : 0.f;
    const int bits = 32 - __builtin_clz(max(seen - begin, 1));               // K
    const float down = __builtin_bit_cast(float, (uint32_t)(127 - bits) << 23), up = __builtin_bit_cast(float, (uint32_t)(127 + bits) << 23);
    for (int key = begin; key < seen; key += 64) {
      const int n = min(64, seen - key);
      float s = -__builtin_inff();
      if (lane < n) {
        const T* k = static_cast<const T*>(a.k) + (int64_t)(k0 + key + lane) * a.k_tok + (int64_t)kvh * a.k_head;
        float dot = 0.f;
        for (int d = 0; d < a.dim; ++d) dot = __builtin_fmaf((float)q[d], (float)k[d], dot);
        s = dot * c;
      }
      const float m_new = fmaxf(m, wave_max(s)), corr = __builtin_amdgcn_exp2f(m - m_new), p = __builtin_amdgcn_exp2f(s - m_new);
      l = l * corr + wave_sum(p);
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= corr;
      for (int j = 0; j < n; ++j) {
        const float w = __shfl(p, j, 64) * down;
        const T* v = static_cast<const T*>(a.v) + (int64_t)(k0 + key + j) * a.v_tok + (int64_t)kvh * a.v_head;
#pragma unroll
        for (int d = 0; d < ND; ++d)
          if (lane + 64 * d < a.dim) o[d] = __builtin_fmaf(w, (float)v[lane + 64 * d], o[d]);
      }
      m = m_new;
    }
    const size_t at = (size_t)(q0 + i) * a.heads + hh;
    const float inv = l == 0.f ? 0.f : 1.0f / l * up;
    if (a.splits > 1) {
      const size_t part = (size_t)split * a.tokens_q * a.heads + at;
      if (lane == 0) { a.part_ml[2 * part] = m; a.part_ml[2 * part + 1] = l; }
#pragma unroll
      for (int d = 0; d < ND; ++d)
        if (lane + 64 * d < a.dim) a.part_o[part * a.dim + lane + 64 * d] = o[d] * inv;
    } else {
      T* out = static_cast<T*>(a.out) + (int64_t)(q0 + i) * a.o_tok + (int64_t)hh * a.o_head;
#pragma unroll
      for (int d = 0; d < ND; ++d)
        if (lane + 64 * d < a.dim) out[lane + 64 * d] = (T)(o[d] * inv);
      if (a.sums && lane == 0) a.sums[at] = l == 0.f ? -__builtin_inff() : 0.69314718055994530942f * (m + __builtin_amdgcn_logf(l));
    }
  }
}

// Infinite or NaN outputs of rows whose sums are numbers: do the rows have to be done again?  Not where the values that they see hold
// a NaN, or an infinity that passes as it is: the outputs then are what they should be (and repeating them would take a hundred
// times as long as the rest of the call).  Lane -> column.
template <class T, bool THIRDS>
__device__ inline bool unexplained(const AttArgs& a, int begin, int end, int nq, int k0, int nk, int kvh, int last, int lane) {
  bool nan = false, inf = false;
  const int seen = min(end, a.causal ? min(max((last - 1) / a.group + nk - nq + 1, 0), nk) : nk);
  for (int d = lane; d < a.dim; d += 64) {
    const T* v = static_cast<const T*>(a.v) + (int64_t)(k0 + begin) * a.v_tok + (int64_t)kvh * a.v_head + d;
#pragma unroll 4
    for (int key = begin; key < seen; ++key, v += a.v_tok) {
      const float x = (float)*v;
      nan |= x != x;
      inf |= __builtin_fabsf(x) == __builtin_inff();
    }
  }
  // an infinity has no thirds, and fp16 may have rounded its weight to 0
  if (__builtin_amdgcn_ballot_w64(inf)) return THIRDS || __is_same(T, _Float16);
  return __builtin_amdgcn_ballot_w64(nan) == 0;
}

template <class T, int NS, int NQ, int WQ, int WK, int KB>
__global__ __launch_bounds__(64 * WQ * WK, (Shape<T, NS, NQ, WQ, WK, KB>::WAVES)) void packed_attention_kernel(const AttArgs a) {
  typedef Shape<T, NS, NQ, WQ, WK, KB> G;
  typedef Slots<NS> L;
  typedef Num<T> N;
  typedef typename N::frag frag;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  constexpr int S = G::S, P = G::P, DB = G::DB, E = G::E;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wq = wave % WQ, wk = wave / WQ;

  // block -> (pair of sequence and key head, tile of rows, part of the keys).  Blocks go to the 8 XCDs in turn; every eighth
  // pair belongs to an XCD (pairs are taken `replicas` times to make their number divisible by 8), so that the blocks which share
  // K and V share an L2 and each XCD has its share of every sequence; `together` pairs take turns, tile by tile.  Their order
  // turns by one from tile to tile: an XCD deals its blocks to four shader engines in turn, and a fixed order of pairs of
  // different lengths would give the long ones to the same engine every time.
  const unsigned per_xcd = (unsigned)(a.pairs * a.replicas) / 8, units = (unsigned)(a.tiles * a.splits);
  const unsigned id = blockIdx.x / 8, first = id / (a.together * units) * a.together;
  const unsigned width = min((unsigned)a.together, per_xcd - first), in_group = id - first * units;
  const int unit = (int)(in_group / width);
  const unsigned vp = (first + (in_group + unit) % width) * 8 + blockIdx.x % 8;
  const int split = unit % a.splits;
  const int pair = (int)(vp / (unsigned)a.replicas), replica = (int)(vp % (unsigned)a.replicas);
  const int kvh = pair % a.kv_heads;
  int seq = pair / a.kv_heads, q0, q1, k0, k1;
  if (a.sequences > 1 && a.sequences <= 64) {
    // the sequence with the seq-th most keys: long ones first, so that the last blocks to run are the short ones
    const int s = min(lane, a.sequences - 1);
    const int qf = a.starts_q[s], qt = a.starts_q[s + 1], kf = a.starts_k[s], kt = a.starts_k[s + 1];
    const int vq0 = min(max(qf, 0), a.tokens_q), vq1 = min(max(qt, vq0), a.tokens_q);
    const int vk0 = min(max(kf, 0), a.tokens_k), vk1 = min(max(kt, vk0), a.tokens_k);
    const int keys = vk1 - vk0, all = __builtin_amdgcn_readfirstlane(keys);
    if (__builtin_amdgcn_ballot_w64(keys != all)) {
      int place = 0;
      for (int i = 0; i < a.sequences; ++i) {
        const int other = __builtin_amdgcn_readlane(keys, i);
        place += other > keys || (other == keys && i < lane);
      }
      seq = __builtin_ctzll(__builtin_amdgcn_ballot_w64(place == seq && lane < a.sequences));
    }
    q0 = __builtin_amdgcn_readlane(vq0, seq);
    q1 = __builtin_amdgcn_readlane(vq1, seq);
    k0 = __builtin_amdgcn_readlane(vk0, seq);
    k1 = __builtin_amdgcn_readlane(vk1, seq);
  } else {
    q0 = min(max(a.starts_q[seq], 0), a.tokens_q);
    q1 = min(max(a.starts_q[seq + 1], q0), a.tokens_q);
    k0 = min(max(a.starts_k[seq], 0), a.tokens_k);
    k1 = min(max(a.starts_k[seq + 1], k0), a.tokens_k);
  }
  const int nq = q1 - q0, nk = k1 - k0, rows = nq * a.group;
  if (a.clear && unit == 0 && replica == 0) {                              // what lies before the first and behind the last sequence
    const int width = a.group * a.dim;
    auto wipe = [&](int first, int last) {
      for (int64_t i = tid; i < (int64_t)(last - first) * width; i += G::THREADS) {
        const int64_t t = first + i / width;
        const int e = (int)(i % width), hh = kvh * a.group + e / a.dim;
        if (a.clear & 1) static_cast<T*>(a.out)[t * a.o_tok + hh * a.o_head + e % a.dim] = (T)0.f;
        if ((a.clear & 2) && a.sums && e % a.dim == 0) a.sums[t * a.heads + hh] = -__builtin_inff();
      }
    };
    if (seq == 0) wipe(0, q0);
    if (seq == a.sequences - 1) wipe(q1, a.tokens_q);
  }
  const int split_begin = split * a.chunk;
  if (split > 0 && split_begin >= nk) return;                              // nothing reads this part (join_kernel)
  const int split_end = split == a.splits - 1 ? nk : min(nk, split_begin + a.chunk);

  // transfers: lane -> (row, slot) of the tile, the address of the slot's entries behind the tile's first row
  const uint32_t ks_bytes = (uint32_t)(a.k_tok * sizeof(T)), vs_bytes = (uint32_t)(a.v_tok * sizeof(T));
  uint32_t koff[G::NJ], voff[G::NJ];
#pragma unroll
  for (int j = 0; j < G::NJ; ++j) {
    const int chunk = (wave + G::W * j) * 64 + lane, row = chunk / S, place = chunk - row * S;
    const int ks = G::SPLIT ? place : L::slot_at(place, L::k_turn(row)), vs = G::SPLIT ? place : L::slot_at(place, L::template v_turn<N::wide>(row));
    koff[j] = ks * E < a.dim ? (uint32_t)row * ks_bytes + ks * 16 : 0x80000000u;      // behind the head: reads as zero
    voff[j] = vs * E < a.dim ? (uint32_t)row * vs_bytes + vs * 16 : 0x80000000u;
  }
  const uint8_t* const kbase = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.k) + (int64_t)k0 * a.k_tok + kvh * a.k_head);
  const uint8_t* const vbase = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.v) + (int64_t)k0 * a.v_tok + kvh * a.v_head);
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  // tile of keys `key` .. : rows behind the sequence read as zero (the descriptor ends with its last entry)
  auto fetch = [&](int key, int buffer) {
    const int left = min(nk - key, G::KEYS);
    const uint64_t kb = (uint64_t)kbase + (uint64_t)key * ks_bytes, vb = (uint64_t)vbase + (uint64_t)key * vs_bytes;
    const uint32_t kn = (uint32_t)(left - 1) * ks_bytes + a.dim * sizeof(T), vn = (uint32_t)(left - 1) * vs_bytes + a.dim * sizeof(T);
    const u32x4 kr = {first_lane((uint32_t)kb), first_lane((uint32_t)(kb >> 32)), first_lane(kn), 0x00020000u};
    const u32x4 vr = {first_lane((uint32_t)vb), first_lane((uint32_t)(vb >> 32)), first_lane(vn), 0x00020000u};
    const uint32_t dst = lds_base + (G::SPLIT ? G::STAGE : 0) + buffer * G::BUF;
#pragma unroll
    for (int j = 0; j < G::NJ; ++j) {
      const int n = wave + G::W * j;
      if (G::NI % G::W == 0 || n < G::NI) {
        to_lds(kr, koff[j], dst + n * 1024);
        to_lds(vr, voff[j], dst + G::TILE + n * 1024);
      }
    }
  };

  // causal: the tiles with the most keys first, so that the last blocks to run are the short ones
  const int place = (unit / a.splits) * a.replicas + replica;
  for (int tile = a.causal ? a.tiles * a.replicas - 1 - place : place; (int64_t)tile * G::ROWS < rows; tile += a.tiles * a.replicas) {
    const int tile_row = tile * G::ROWS, wave_row = tile_row + wq * 32 * NQ;
    // keys that a row sees: the first `lim` of its sequence
    auto limit = [&](int row) {
      const int i = row / a.group;
      return a.causal ? min(max(i + nk - nq + 1, 0), nk) : nk;
    };
    const int block_last = min(tile_row + G::ROWS, rows) - 1;
    const int key_end = min(split_end, limit(block_last));
    const bool active = wave_row < rows;
    bool odd_values = false;                       // an infinity or NaN among values that not every row of the wave sees
    const int lim_least = active ? limit(wave_row) : 0, lim_most = active ? min(key_end, limit(min(wave_row + 32 * NQ, rows) - 1)) : 0;
    int lim[NQ];
    frag qf[G::SPLIT ? 1 : NQ][G::SPLIT ? 1 : NS];
    Thirds qt[G::SPLIT ? NQ : 1][G::SPLIT ? NS / 2 : 1];
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      const int row = wave_row + 32 * b + r, i = row / a.group, hh = kvh * a.group + row - i * a.group;
      lim[b] = row < rows ? limit(row) : 0;
      const T* src = static_cast<const T*>(a.q) + (int64_t)(q0 + i) * a.q_tok + (int64_t)hh * a.q_head;
      auto words = [&](int d) {                    // 16 bytes of the row from entry d on
        frag z = {};
        u32x4 w = __builtin_bit_cast(u32x4, row < rows && d < a.dim ? *reinterpret_cast<const frag*>(src + d) : z);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = (w[j] & a.q_keep) ^ a.q_flip;
        return w;
      };
      if constexpr (G::SPLIT) {
#pragma unroll
        for (int s = 0; s < NS / 2; ++s) {
          const f32x4 lo = __builtin_bit_cast(f32x4, words(16 * s + 8 * h)), hi = __builtin_bit_cast(f32x4, words(16 * s + 8 * h + 4));
          const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          qt[b][s] = thirds(x);
        }
      } else {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          u32x4 w = words((2 * s + h) * E);
          if constexpr (G::WAVES == 1 && !N::wide) asm volatile("" : "+a"(w));       // in the accumulation registers, which the products read in place
          qf[b][s] = __builtin_bit_cast(frag, w);
        }
      }
    }
    f32x16 o[NQ][DB];
    float m_run[NQ], l_run[NQ];
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      m_run[b] = NO_MAX;
      l_run[b] = 0.f;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][d][i] = 0.f;
    }

    const int kturn = L::k_turn(r);
    const int vq = (lane & 15) >> 2, vp = lane & 3, vg = (lane >> 4) & 1;
    // S^T of 32 keys, from LDS row `krow` of a tile on
    auto scores = [&](const uint8_t* Kt, int krow, f32x16 (&sc)[NQ]) {
      const uint8_t* krp = Kt + (krow + r) * P;
#pragma unroll
      for (int b = 0; b < NQ; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[b][i] = 0.f;
      if constexpr (G::SPLIT) {                    // Kt: K's planes
        typedef Slots<NS / 2> H;
        const int turn = H::k_turn(r);
#pragma unroll
        for (int s = 0; s < NS / 2; ++s) {
          const uint8_t* at = Kt + r * (P / 2) + H::place(2 * s + h, turn) * 16;
          const Thirds k = {*reinterpret_cast<const bf8*>(at), *reinterpret_cast<const bf8*>(at + G::PLANE), *reinterpret_cast<const bf8*>(at + 2 * G::PLANE)};
#pragma unroll
          for (int b = 0; b < NQ; ++b) sc[b] = product(k, qt[b][s], sc[b]);
        }
      } else {
        frag kf[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) kf[s] = *reinterpret_cast<const frag*>(krp + L::place(2 * s + h, kturn) * 16);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int b = 0; b < NQ; ++b) sc[b] = N::mfma(kf[s], qf[b][s], sc[b]);
      }
    };
    // key: the block's first; some row of the wave does not see all of its keys
    auto mask = [&](const uint8_t* Vt, int krow, int key, f32x16 (&sc)[NQ]) {
#pragma unroll
      for (int b = 0; b < NQ; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[b][i] = key + 8 * (i >> 2) + 4 * h + (i & 3) < lim[b] ? sc[b][i] : -__builtin_inff();
      // A masked score has p = 0, but 0 times an infinity or NaN is NaN: rows of a wave that meets one here are done again
      bool odd = false;
      if constexpr (G::SPLIT) {                    // Vt: V's planes; the first shows them
#pragma unroll
        for (int j = 0; j < NS / 2; ++j) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(Vt + j * 1024 + lane * 16);
          odd |= Num<__bf16>::odd(w[0]) | Num<__bf16>::odd(w[1]) | Num<__bf16>::odd(w[2]) | Num<__bf16>::odd(w[3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(Vt + krow * P + j * 1024 + lane * 16);
          odd |= N::odd(w[0]) | N::odd(w[1]) | N::odd(w[2]) | N::odd(w[3]);
        }
      }
      if (__builtin_amdgcn_ballot_w64(odd)) odd_values = true;
      asm volatile("" ::: "memory");                   // (keeps this a branch: as selects it would cost every block)
    };
    auto maxima = [&](const f32x16 (&sc)[NQ], float (&top)[NQ]) {
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        top[b] = sc[b][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top[b] = fmaxf(top[b], sc[b][i]);
        top[b] = halves_max(top[b]) * a.c_log2;
      }
    };
    // The sums keep an older maximum until one is 2^8 ahead of it: weights up to 256 cost no digits (they are rounded relative
    // to themselves) and o is rescaled a few times per row instead of in most blocks
    auto rescale = [&](const float (&top)[NQ]) {
#pragma unroll
      for (int b = 0; b < NQ; ++b)
        if (__builtin_amdgcn_ballot_w64(top[b] > m_run[b] + 8.0f)) {
          const float m_new = fmaxf(m_run[b], top[b]), corr = __builtin_amdgcn_exp2f(m_run[b] - m_new);
          l_run[b] *= corr;
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][d][i] *= corr;
          m_run[b] = m_new;
        }
    };
    // Weights: fp32 in the sum; rounded to the tensor's type (16-bit) for the product with the values, as the matrix instructions
    // take them: half a step, 2^-8 or 2^-11 relative, of each weight, next to the same of the result
    auto weights = [&](f32x16 (&sc)[NQ], frag (&pf)[NQ][2]) {
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][i], a.c_log2, -m_run[b]));
        float part[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) part[i] = (sc[b][i] + sc[b][4 + i]) + (sc[b][8 + i] + sc[b][12 + i]);
        l_run[b] += (part[0] + part[1]) + (part[2] + part[3]);
        if constexpr (!N::wide) {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = N::pack(sc[b][8 * ks + 2 * j], sc[b][8 * ks + 2 * j + 1]);
            asm volatile("" : "+v"(w));                // here, beside the products of the next scores, and not where it is used
            pf[b][ks] = __builtin_bit_cast(frag, w);
          }
        }
      }
    };
    // V^T fragments of 32 keys.  Transposed reads: lane 4 q + p of a 16-lane group addresses key row q, entries 4 p .. of the
    // group's 16, and gets column (lane & 15) of the 4 x 16 block; the groups take (entries 0 .. 15, 16 .. 31) x (lane halves)
    auto value_at = [&](const uint8_t* Vt, int krow, int d, int ks) {
      typedef Slots<G::SPLIT ? NS / 2 : NS> H;
      u32x4 w;
#pragma unroll
      for (int j2 = 0; j2 < 2; ++j2) {
        const int row = krow + 16 * ks + 8 * j2 + 4 * h + vq;
        const uint8_t* at = Vt + row * H::P + H::place(4 * d + 2 * vg + (vp >> 1), H::template v_turn<false>(4 * h + vq)) * 16 + 8 * (vp & 1);
        const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at)));
        w[2 * j2] = x[0];
        w[2 * j2 + 1] = x[1];
      }
      return w;
    };
    // O^T += V^T P^T
    auto values = [&](const uint8_t* Vt, int krow, const f32x16 (&sc)[NQ], const frag (&pf)[NQ][2]) {
      if constexpr (G::SPLIT) {
        Thirds pt[NQ][2];
#pragma unroll
        for (int b = 0; b < NQ; ++b)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = sc[b][8 * ks + i];
            pt[b][ks] = thirds(x);
          }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const Thirds v = {__builtin_bit_cast(bf8, value_at(Vt, 0, d, ks)), __builtin_bit_cast(bf8, value_at(Vt + G::PLANE, 0, d, ks)),
                              __builtin_bit_cast(bf8, value_at(Vt + 2 * G::PLANE, 0, d, ks))};
#pragma unroll
            for (int b = 0; b < NQ; ++b) o[b][d] = product(v, pt[b][ks], o[b][d]);
          }
        return;
      }
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        if constexpr (N::wide) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int row = krow + 8 * (i >> 2) + 4 * h + (i & 3);
            const float vf = *reinterpret_cast<const float*>(Vt + row * P + L::place(8 * d + (r >> 2), L::template v_turn<true>(4 * h)) * 16 + (r & 3) * 4);
#pragma unroll
            for (int b = 0; b < NQ; ++b) o[b][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, sc[b][i], o[b][d], 0, 0, 0);
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const frag vf = __builtin_bit_cast(frag, value_at(Vt, krow, d, ks));
#pragma unroll
            for (int b = 0; b < NQ; ++b) o[b][d] = N::mfma(vf, pf[b][ks], o[b][d]);
          }
        }
      }
    };

    const int tiles = key_end > split_begin ? (key_end - split_begin + G::KEYS - 1) / G::KEYS : 0;
    if constexpr (G::RING) {
      // Pipelined: block j's exponentials run beside the products of block j + 1's scores, its values beside their maxima.
      // Tiles t + 1 and t + 2 are in flight while t is read; the buffer of t + 3 is the one of t - 1, which every wave has
      // left when it passes the barrier in front of the last block of t.
      constexpr int COUNT = 2 * (G::NI / G::W);        // transfers of a tile per wave (some waves issue two more: they wait longer)
      const int blocks = (key_end - split_begin + 31) / 32, mine = (lim_most - split_begin + 31) / 32;
#pragma unroll
      for (int t = 0; t < 3; ++t)
        if (t < tiles) fetch(split_begin + t * G::KEYS, t);
      wait_transfers<0>();
      barrier();
      f32x16 sa[NQ], sb[NQ];
      if (mine > 0) {
        float top[NQ];
        scores(lds, 0, sa);
        if (split_begin + 32 > lim_least) mask(lds + G::TILE, 0, split_begin, sa);
        maxima(sa, top);
        rescale(top);
      }
      auto step = [&](int j, f32x16 (&now)[NQ], f32x16 (&next)[NQ]) {
        const int t = j / KB;
        if (j % KB == KB - 1 && t + 1 < tiles) {       // the next block lies in the next tile
          if (t + 2 < tiles) wait_transfers<COUNT>();
          else wait_transfers<0>();
          barrier();
          if (t + 3 < tiles) fetch(split_begin + (t + 3) * G::KEYS, (t + 3) & 3);
        }
        if (j >= mine) return;
        const uint8_t* Vt = lds + (t & 3) * G::BUF + G::TILE;
        const int tn = (j + 1) / KB, krow = (j % KB) * 32, krow_n = ((j + 1) % KB) * 32, key_n = split_begin + (j + 1) * 32;
        const uint8_t* Kn = lds + (tn & 3) * G::BUF;   // behind the last block: what is there, for nothing
        frag pf[NQ][2];
        float top[NQ];
        u32x4 vf[DB][2];
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) vf[d][ks] = value_at(Vt, krow, d, ks);
        scores(Kn, krow_n, next);
        weights(now, pf);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {              // read beside the scores' products, not after them
            if constexpr (G::WAVES == 1) asm volatile("" : "+a"(vf[d][ks]));
            else asm volatile("" : "+v"(vf[d][ks]));
          }
        const bool more = j + 1 < mine;
        if (more && key_n + 32 > lim_least) mask(Kn + G::TILE, krow_n, key_n, next);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int b = 0; b < NQ; ++b) o[b][d] = N::mfma(__builtin_bit_cast(frag, vf[d][ks]), pf[b][ks], o[b][d]);
        maxima(next, top);
        if (more) rescale(top);
      };
      for (int j = 0; j < blocks; j += 2) {
        step(j, sa, sb);
        if (j + 1 < blocks) step(j + 1, sb, sa);
      }
    } else if constexpr (G::SPLIT) {
      // A tile of 32 keys arrives in fp32; each thread cuts its share of it into thirds once for the whole block, and the next tile
      // is on its way while this one's planes are multiplied (each wave cutting every tile for itself: 402 us instead of 344
      // for 32 images of 785 tokens).
      static_assert(KB == 1 && WK == 1, "");
      typedef Slots<NS / 2> H;
      if (tiles) fetch(split_begin, 0);
      for (int t = 0; t < tiles; ++t) {
        wait_transfers<0>();
        barrier();                                 // the tile is there; the planes of the last one are read
#pragma unroll
        for (int c = tid; c < 64 * NS; c += G::THREADS) {
          const bool value = c < 32 * NS;
          const int at = value ? c : c - 32 * NS, row = at / NS, slot = at - row * NS;
          const uint8_t* from = lds + G::STAGE + (value ? G::TILE : 0) + row * P + slot * 32;
          const f32x4 lo = *reinterpret_cast<const f32x4*>(from), hi = *reinterpret_cast<const f32x4*>(from + 16);
          const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          const Thirds y = thirds(x);
          uint8_t* to = lds + (value ? 0 : 3 * G::PLANE) + row * (P / 2) + H::place(slot, value ? H::template v_turn<false>(row) : H::k_turn(row)) * 16;
          *reinterpret_cast<bf8*>(to) = y.h;
          *reinterpret_cast<bf8*>(to + G::PLANE) = y.m;
          *reinterpret_cast<bf8*>(to + 2 * G::PLANE) = y.l;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier();
        if (t + 1 < tiles) fetch(split_begin + (t + 1) * G::KEYS, 0);
        const int key = split_begin + t * G::KEYS;
        if (key >= lim_most) continue;
        f32x16 sc[NQ];
        frag pf[NQ][2];
        float top[NQ];
        scores(lds + 3 * G::PLANE, 0, sc);
        if (key + 32 > lim_least) mask(lds, 0, key, sc);
        maxima(sc, top);
        rescale(top);
        weights(sc, pf);
        values(lds, 0, sc, pf);
      }
    } else {
      if (tiles) fetch(split_begin, 0);
      for (int t = 0; t < tiles; ++t) {
        wait_transfers<0>();
        barrier();
        if (t + 1 < tiles) fetch(split_begin + (t + 1) * G::KEYS, (t + 1) & 1);
        const uint8_t* Kt = lds + (t & 1) * G::BUF;
#pragma unroll 1
        for (int kb = 0; kb < KB; ++kb) {
          const int krow = (wk * KB + kb) * 32, key = split_begin + t * G::KEYS + krow;
          if (key >= lim_most) continue;
          f32x16 sc[NQ];
          frag pf[NQ][2];
          float top[NQ];
          scores(Kt, krow, sc);
          if (key + 32 > lim_least) mask(Kt + G::TILE, krow, key, sc);
          maxima(sc, top);
          rescale(top);
          weights(sc, pf);
          values(Kt + G::TILE, krow, sc, pf);
        }
      }
    }

    // ---- the lane halves' sums, then the waves that took other keys
#pragma unroll
    for (int b = 0; b < NQ; ++b) l_run[b] += __shfl_xor(l_run[b], 32, 64);
    if constexpr (WK > 1) {
      __syncthreads();
      float* const mine = reinterpret_cast<float*>(lds) + (size_t)((wk - 1) * WQ + wq) * NQ * 64 * (DB * 16 + 2);
      if (wk > 0) {
#pragma unroll
        for (int b = 0; b < NQ; ++b) {
          float* p = mine + b * 64 * (DB * 16 + 2) + lane;
          p[0] = m_run[b];
          p[64] = l_run[b];
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) p[64 * (2 + d * 16 + i)] = o[b][d][i];
        }
      }
      __syncthreads();
      if (wk == 0) {
#pragma unroll
        for (int w = 1; w < WK; ++w)
#pragma unroll
          for (int b = 0; b < NQ; ++b) {
            const float* p = reinterpret_cast<const float*>(lds) + ((size_t)((w - 1) * WQ + wq) * NQ + b) * 64 * (DB * 16 + 2) + lane;
            const float m_new = fmaxf(m_run[b], p[0]);
            const float ca = __builtin_amdgcn_exp2f(m_run[b] - m_new), cb = __builtin_amdgcn_exp2f(p[0] - m_new);
            l_run[b] = l_run[b] * ca + p[64] * cb;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
              for (int i = 0; i < 16; ++i) o[b][d][i] = o[b][d][i] * ca + p[64 * (2 + d * 16 + i)] * cb;
            m_run[b] = m_new;
          }
      }
    }
    // Outputs that are not finite: again(), unless the values explain them.  A sum that is NaN says that a score was; thirds make one of
    // an infinite score, the others are right
    bool not_finite = false;
    if (wk == 0) {
      bool odd = false, sum_odd = false;
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        const bool there = wave_row + 32 * b + r < rows, number = l_run[b] == l_run[b];
        float part[4] = {0.f, 0.f, 0.f, 0.f};      // NaN if an entry is not finite
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) part[i & 3] = __builtin_fmaf(o[b][d][i], 0.f, part[i & 3]);
        const float zero = (part[0] + part[1]) + (part[2] + part[3]);
        odd |= there && number && zero != zero;
        sum_odd |= there && !number;
      }
      not_finite = __builtin_amdgcn_ballot_w64(odd) != 0;
      if (G::SPLIT && __builtin_amdgcn_ballot_w64(sum_odd)) odd_values = true;
    }
    if constexpr (WK > 1) {
      __syncthreads();
      int* const flag = reinterpret_cast<int*>(lds);
      if (tid == 0) *flag = 0;
      __syncthreads();
      if (odd_values && lane == 0) *flag = 1;      // WQ is 1 here: the block's waves share the rows
      __syncthreads();
      odd_values = *flag != 0;
    }
    if (wk == 0) {
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        const int row = wave_row + 32 * b + r;
        if (row >= rows) continue;
        const int i = row / a.group, hh = kvh * a.group + row - i * a.group;
        const float inv = l_run[b] == 0.f ? 0.f : 1.0f / l_run[b];
        if (a.splits > 1) {
          const size_t at = (size_t)split * a.tokens_q * a.heads + (size_t)(q0 + i) * a.heads + hh;
          float* dst = a.part_o + at * a.dim;
          if (h == 0) {
            a.part_ml[2 * at] = m_run[b];
            a.part_ml[2 * at + 1] = l_run[b];
          }
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int e = 32 * d + 8 * j + 4 * h;
              if (e < a.dim) *reinterpret_cast<f32x4*>(dst + e) = f32x4{o[b][d][4 * j] * inv, o[b][d][4 * j + 1] * inv, o[b][d][4 * j + 2] * inv, o[b][d][4 * j + 3] * inv};
            }
        } else {
          T* dst = static_cast<T*>(a.out) + (int64_t)(q0 + i) * a.o_tok + (int64_t)hh * a.o_head;
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int e = 32 * d + 8 * j + 4 * h;
              const float x[4] = {o[b][d][4 * j] * inv, o[b][d][4 * j + 1] * inv, o[b][d][4 * j + 2] * inv, o[b][d][4 * j + 3] * inv};
              if (e < a.dim) {
                if constexpr (N::wide) *reinterpret_cast<f32x4*>(dst + e) = f32x4{x[0], x[1], x[2], x[3]};
                else *reinterpret_cast<u32x2*>(dst + e) = u32x2{N::pack(x[0], x[1]), N::pack(x[2], x[3])};
              }
            }
          if (a.sums && h == 0)
            a.sums[(size_t)(q0 + i) * a.heads + hh] = l_run[b] == 0.f ? -__builtin_inff() : 0.69314718055994530942f * (m_run[b] + __builtin_amdgcn_logf(l_run[b]));
        }
      }
    }
    // (behind the normal output, which again() overwrites: in front of it the scan's scalar registers cost 2 % of the whole)
    if (wk == 0 && (odd_values || not_finite)) {
      const int last = min(wave_row + 32 * NQ, rows);
      wait_transfers<0>();
      if (odd_values || unexplained<T, G::SPLIT>(a, split_begin, split_end, nq, k0, nk, kvh, last, lane))
        again<T, DB * 32>(a, split, split_begin, split_end, q0, nq, k0, nk, kvh, wave_row, last, lane);
    }
    __syncthreads();                 // the next tile's transfers overwrite what these waves may still read
  }
}

// Joins the parts of a split key axis: a block per row; eight groups of 32 lanes take every eighth part, lane -> four entries (and four
// more, up to 256).  The parts' maxima and sums: lane -> part.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(const AttArgs a) {
  __shared__ float weight[64];
  __shared__ __attribute__((aligned(16))) float all[8][260];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const int token = (int)(row / a.heads), hh = (int)(row - (int64_t)token * a.heads);
  // the sequence that holds the token: the first whose (clamped, as above) range does
  int seq = -1;
  for (int s0 = 0; s0 < a.sequences && seq < 0; s0 += 64) {
    const int s = s0 + lane;
    bool here = false;
    if (s < a.sequences) {
      const int q0 = min(max(a.starts_q[s], 0), a.tokens_q), q1 = min(max(a.starts_q[s + 1], q0), a.tokens_q);
      here = token >= q0 && token < q1;
    }
    const unsigned long long m = __builtin_amdgcn_ballot_w64(here);
    if (m) seq = s0 + __builtin_ctzll(m);
  }
  if (seq < 0) return;                                           // outside every sequence: left as it is (the whole block)
  const int k0 = min(max(a.starts_k[seq], 0), a.tokens_k), nk = min(max(a.starts_k[seq + 1], k0), a.tokens_k) - k0;
  const int parts = max(1, min(a.splits, (nk + a.chunk - 1) / a.chunk));            // at most 64
  const size_t step = (size_t)a.tokens_q * a.heads;
  float m = NO_MAX, l = 0.f;
  if (lane < parts) {
    const float* ml = a.part_ml + 2 * (lane * step + row);
    m = ml[0];
    l = ml[1];
  }
  // the parts hold means: their weights add up to 1, so what is finite stays so
  const float top = wave_max(m), w = lane < parts ? l * __builtin_amdgcn_exp2f(m - top) : 0.f;
  l = wave_sum(w);
  if (tid < 64) weight[tid] = l == 0.f ? 0.f : w / l;
  __syncthreads();
  const int grp = tid >> 5, e = (tid & 31) * 4;
  f32x4 x0 = {0.f, 0.f, 0.f, 0.f}, x1 = x0;
  for (int s = grp; s < parts; s += 8) {
    const float* p = a.part_o + (s * step + row) * a.dim;
    const float ws = weight[s];
    f32x4 y0 = x0, y1 = x0;
    if (e < a.dim) y0 = *reinterpret_cast<const f32x4*>(p + e);
    if (e + 128 < a.dim) y1 = *reinterpret_cast<const f32x4*>(p + e + 128);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (e < a.dim) x0[j] += y0[j] * ws;
      if (e + 128 < a.dim) x1[j] += y1[j] * ws;
    }
  }
  *reinterpret_cast<f32x4*>(&all[grp][e]) = x0;
  *reinterpret_cast<f32x4*>(&all[grp][e + 128]) = x1;
  __syncthreads();
  if (tid < a.dim) {
    float x = 0.f;
#pragma unroll
    for (int g = 0; g < 8; ++g) x += all[g][tid];
    static_cast<T*>(a.out)[(int64_t)token * a.o_tok + (int64_t)hh * a.o_head + tid] = (T)x;
  }
  if (a.sums && tid == 0) a.sums[row] = l == 0.f ? -__builtin_inff() : 0.69314718055994530942f * (top + __builtin_amdgcn_logf(l));
}

// ---- the launch plan: what ac_attention_packed and its workspace size agree on
struct Plan { int kind, rows, tiles, splits, chunk, keys; };   // kind 0: 256 rows, 1: 128 rows, 2: 32 rows and split keys, 3: 128 rows on two waves

template <class T> int plan_steps(int dim) {                    // NS of the instance that holds `dim`
  const int per = 32 / (int)sizeof(T), need = (dim + per - 1) / per;
  const int have16[] = {2, 3, 4, 5, 6, 8, 10, 12, 16}, have32[] = {4, 6, 8, 10, 12, 16, 24, 32};
  if (sizeof(T) == 4) { for (int n : have32) if (n >= need) return n; }
  else { for (int n : have16) if (n >= need) return n; }
  return 0;
}

Plan make_plan(const ac_attention_args* p) {
  const int group = p->heads / p->kv_heads;
  // the caller's bounds, at least the averages (a bound that is too small must not make the parts of a split axis many)
  auto bound = [&](int hint, int64_t tokens) {
    const int64_t mean = (tokens + p->sequences - 1) / p->sequences;
    return max((int64_t)1, min(max((int64_t)hint, mean), tokens));
  };
  const int64_t max_q = bound(p->max_q, p->tokens_q), max_k = bound(p->max_k, p->tokens_k);
  const int64_t rows = max_q * group, pairs = (int64_t)p->sequences * p->kv_heads;
  const bool wide = p->type == AC_F32;
  const int bytes = p->dim * (wide ? 4 : 2);
  Plan r;
  r.kind = rows <= 32 ? 2 : (wide || bytes > 256 || pairs * ((rows + 255) / 256) < 2 * ac_device_cus()) ? 1 : 0;
  // Heads of more than 128 bytes have one wave on a SIMD: blocks of two waves halve what is left over at the end of sequences and
  // of the launch, for twice the transfers.  8 prompts of 1 .. 4096, 32 / 8 heads of 128 (1700 blocks of 256 rows): 457 -> 431 us;
  // 8 prompts of 4096 (4096 blocks): 1196 -> 1222 us.
  if (r.kind == 0 && bytes > 128 && p->tokens_q * (int64_t)p->heads / 256 < 8 * ac_device_cus()) r.kind = 3;
  r.rows = r.kind == 2 ? 32 : r.kind != 0 ? 128 : 256;
  r.keys = r.kind == 2 && wide && bytes <= 256 ? 128 : 64;
  // (a launch may not have 2^32 threads: many sequences under a loose bound get fewer blocks, which walk over the tiles)
  r.tiles = (int)max((int64_t)1, min((rows + r.rows - 1) / r.rows, (1LL << 22) / pairs));
  // The key axis is split where the rows alone would leave CUs idle, into parts of 256 keys or more: so many that a CU gets about
  // four (16-bit; fp32 six) blocks.  Two waves on tiles of 64 keys, 64 KB of LDS: two blocks of a CU cover each other's start and
  // end.  16 queries on 64 .. 16000 keys, 32 / 8 heads of 128: 90 us, against 106 with four waves on 128 keys; 64 queries on 4096
  // keys each: 183 us (5.9 TB/s) against 196.
  const int64_t blocks = pairs * r.tiles, want = (wide ? 6LL : 4LL) * ac_device_cus();
  int64_t splits = blocks >= want / 2 ? 1 : min((want + blocks - 1) / blocks, (max_k + 255) / 256);
  splits = max((int64_t)1, min((int64_t)64, splits));
  r.chunk = (int)(((max_k + splits - 1) / splits + r.keys - 1) / r.keys * r.keys);
  r.splits = (int)((max_k + r.chunk - 1) / r.chunk);
  return r;
}

template <class T, int NS, int NQ, int WQ, int WK, int KB>
int launch(const AttArgs& a, hipStream_t stream) {
  typedef Shape<T, NS, NQ, WQ, WK, KB> G;
  static unsigned long long done = 0;
  if (int rc = ac_set_max_lds(reinterpret_cast<const void*>(&packed_attention_kernel<T, NS, NQ, WQ, WK, KB>), G::LDS, &done)) return rc;
  const int64_t blocks = (int64_t)a.pairs * a.replicas * a.tiles * a.splits;       // under 2^24 (make_plan, check)
  hipLaunchKernelGGL((packed_attention_kernel<T, NS, NQ, WQ, WK, KB>), dim3((unsigned)blocks), dim3(G::THREADS), G::LDS, stream, a);
  return AC_OK;
}

template <class T, int NS>
int launch_kind(const AttArgs& a, int kind, hipStream_t stream) {
  constexpr bool big = NS * 32 > 256;                            // rows of more than 256 bytes: smaller tiles
  if constexpr (!Num<T>::wide && !big) {
    if (kind == 0) return launch<T, NS, 2, 4, 1, 2>(a, stream);
    if (kind == 3) return launch<T, NS, 2, 2, 1, 1>(a, stream);
  }
  if (kind == 2) {
    if constexpr (NS * 32 > 512) return launch<T, NS, 1, 1, 1, 1>(a, stream);
    else if constexpr (big) return launch<T, NS, 1, 1, 2, 1>(a, stream);
    else return launch<T, NS, 1, 1, Num<T>::wide ? 4 : 2, 1>(a, stream);
  }
  if constexpr (NS * 32 > 512) return launch<T, NS, 1, 4, 1, 1>(a, stream);
  else return launch<T, NS, 1, 4, 1, big || Num<T>::wide ? 1 : 2>(a, stream);
}

template <class T>
int launch_type(const AttArgs& a, int kind, hipStream_t stream) {
  int rc = AC_EINVAL;
  if constexpr (sizeof(T) == 4) {
    switch (plan_steps<T>(a.dim)) {
      case 4: rc = launch_kind<T, 4>(a, kind, stream); break;
      case 6: rc = launch_kind<T, 6>(a, kind, stream); break;
      case 8: rc = launch_kind<T, 8>(a, kind, stream); break;
      case 10: rc = launch_kind<T, 10>(a, kind, stream); break;
      case 12: rc = launch_kind<T, 12>(a, kind, stream); break;
      case 16: rc = launch_kind<T, 16>(a, kind, stream); break;
      case 24: rc = launch_kind<T, 24>(a, kind, stream); break;
      case 32: rc = launch_kind<T, 32>(a, kind, stream); break;
    }
  } else {
    switch (plan_steps<T>(a.dim)) {
      case 2: rc = launch_kind<T, 2>(a, kind, stream); break;
      case 3: rc = launch_kind<T, 3>(a, kind, stream); break;
      case 4: rc = launch_kind<T, 4>(a, kind, stream); break;
      case 5: rc = launch_kind<T, 5>(a, kind, stream); break;
      case 6: rc = launch_kind<T, 6>(a, kind, stream); break;
      case 8: rc = launch_kind<T, 8>(a, kind, stream); break;
      case 10: rc = launch_kind<T, 10>(a, kind, stream); break;
      case 12: rc = launch_kind<T, 12>(a, kind, stream); break;
      case 16: rc = launch_kind<T, 16>(a, kind, stream); break;
    }
  }
  if (rc != AC_OK) return rc;
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.tokens_q * a.heads;
    hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)rows), dim3(256), 0, stream, a);
  }
  return AC_OK;
}

int check(const ac_attention_args* p) {
  AC_REQUIRE(p, "ac_attention_packed: null arguments");
  AC_REQUIRE(p->type == AC_F32 || p->type == AC_F16 || p->type == AC_BF16, "ac_attention_packed: unknown type %d", p->type);
  AC_REQUIRE(p->heads >= 1 && p->kv_heads >= 1 && p->heads % p->kv_heads == 0, "ac_attention_packed: %d heads cannot share %d key heads", p->heads, p->kv_heads);
  AC_REQUIRE(p->dim >= 8 && p->dim <= 256 && p->dim % 8 == 0, "ac_attention_packed: head dim %d must be a multiple of 8, 8 .. 256", p->dim);
  AC_REQUIRE(p->sequences >= 0 && p->tokens_q >= 0 && p->tokens_k >= 0, "ac_attention_packed: negative count");
  const int64_t most = (1LL << 31) - 256;                        // (each count first: their products then fit 64 bits)
  AC_REQUIRE(p->tokens_q < most && p->tokens_k < most && p->tokens_q * (p->heads / p->kv_heads) < most && p->tokens_q * p->heads < (1LL << 32),
             "ac_attention_packed: too many tokens");
  AC_REQUIRE(p->scale - p->scale == 0.f, "ac_attention_packed: the scale is not finite");
  AC_REQUIRE((int64_t)p->sequences * p->kv_heads < (1LL << 21), "ac_attention_packed: too many sequences (2^21 with one key head)");
  return AC_OK;
}

}  // namespace

extern "C" size_t ac_attention_packed_workspace_bytes(const ac_attention_args* p) {
  if (check(p) != AC_OK || p->sequences == 0 || p->tokens_q == 0) return 0;
  const Plan r = make_plan(p);
  if (r.splits <= 1) return 0;
  const size_t rows = (size_t)r.splits * p->tokens_q * p->heads;
  return align_up(rows * p->dim * 4, 256) + align_up(rows * 8, 256);
}

extern "C" int ac_attention_packed(const ac_attention_args* p, void* ws, size_t ws_bytes, void* stream_) {
  if (int rc = check(p)) return rc;
  if (p->sequences == 0 || p->tokens_q == 0) return AC_OK;
  AC_REQUIRE(p->q && p->out && p->starts_q && p->starts_k && (p->tokens_k == 0 || (p->k && p->v)), "ac_attention_packed: null pointer");
  AC_REQUIRE((((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->out) & 15) == 0 && (((uintptr_t)p->starts_q | (uintptr_t)p->starts_k | (uintptr_t)p->sums) & 3) == 0,
             "ac_attention_packed: q, k, v and out must be 16-byte aligned");
  const int64_t strides[] = {p->q_token, p->q_head, p->k_token, p->k_head, p->v_token, p->v_head, p->out_token, p->out_head};
  const int entries = p->type == AC_F32 ? 4 : 8;
  for (int64_t s : strides) AC_REQUIRE(s >= 0 && s % entries == 0, "ac_attention_packed: strides must be non-negative multiples of 16 bytes");
  AC_REQUIRE(p->k_token < (1 << 20) && p->v_token < (1 << 20), "ac_attention_packed: a key's stride must stay under 2^20 entries");
  const Plan r = make_plan(p);
  const size_t need = ac_attention_packed_workspace_bytes(p);
  if (need && (!ws || ws_bytes < need)) return ac_fail(AC_EWORKSPACE, "ac_attention_packed: workspace %zu < %zu", ws ? ws_bytes : (size_t)0, need);
  AC_REQUIRE(!need || ((uintptr_t)ws & 15) == 0, "ac_attention_packed: the workspace must be 16-byte aligned");
  AttArgs a;
  a.q = p->q; a.k = p->k; a.v = p->v; a.out = p->out; a.sums = p->sums;
  a.q_tok = p->q_token; a.q_head = p->q_head; a.k_tok = p->k_token; a.k_head = p->k_head;
  a.v_tok = p->v_token; a.v_head = p->v_head; a.o_tok = p->out_token; a.o_head = p->out_head;
  a.starts_q = p->starts_q; a.starts_k = p->starts_k;
  a.tokens_q = (int)p->tokens_q; a.tokens_k = (int)p->tokens_k; a.sequences = p->sequences; a.heads = p->heads; a.kv_heads = p->kv_heads;
  a.group = p->heads / p->kv_heads; a.dim = p->dim; a.causal = p->causal; a.clear = p->clear;
  a.c_log2 = p->scale == 0.f ? 1.f : fabsf(p->scale) * 1.44269504088896340736f;
  a.q_keep = p->scale == 0.f ? 0u : ~0u;
  a.q_flip = p->scale < 0.f ? (p->type == AC_F32 ? 0x80000000u : 0x80008000u) : 0u;
  a.pairs = p->sequences * p->kv_heads;
  a.replicas = a.pairs % 8 == 0 ? 1 : a.pairs % 4 == 0 ? 2 : a.pairs % 2 == 0 ? 4 : 8;
  // Causal: tiles differ by up to their number in work, and eight pairs in turn, longest tiles first, end within a tile of
  // each other (16 heads of 128, 4 x 4096: 394 -> 326 us).  Otherwise one pair after the other: the fewest streams of keys through an L2.
  a.together = a.causal ? 8 : 1;
  a.tiles = (r.tiles + a.replicas - 1) / a.replicas; a.splits = r.splits; a.chunk = r.chunk;
  a.part_o = static_cast<float*>(ws);
  a.part_ml = need ? reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + align_up((size_t)r.splits * p->tokens_q * p->heads * p->dim * 4, 256)) : nullptr;
  int rc = p->type == AC_F32 ? launch_type<float>(a, r.kind, as_stream(stream_))
         : p->type == AC_F16 ? launch_type<_Float16>(a, r.kind, as_stream(stream_)) : launch_type<__bf16>(a, r.kind, as_stream(stream_));
  if (rc != AC_OK) return rc;
  return ac_check_launch("ac_attention_packed");
}
