// Rotary positions of packed queries and keys (gfx950).
//
// Pair i of a head turns by theta = position * frequency[i]: (a, b) -> m (a cos - b sin, b cos + a sin).  In the half layout
// the pair is (i, i + part/2), in the interleaved one (2i, 2i + 1), counted from `offset`; the rest of the head passes.
// Cosines and sines: theta and its remainder by pi/2 in fp64 (a position of 4e6 leaves an fp32 angle no digit behind the
// point), then Taylor polynomials on [-pi/4, pi/4] in fp32 (first dropped terms 7e-12 and 1.2e-10, below half an fp32 step),
// so the factors are right to fp32 rounding up to angles of 2^28, where the fp64 product's own rounding (2^-53 of the angle) comes to
// half an fp32 step.  They are computed once per token and pair into LDS and used by every head; products and sums are fp32, the
// result is rounded to the tensor's type once.
//
// Bound: memory; each element is read once and written once, nothing else is of size.  131072 tokens x 40 heads of 128 in bf16 (2.7
// GB) 486 us, 5.5 TB/s; 24571 x 40 in fp16, half of each interleaved, 93 us, 5.4; a copy of 1 GB reaches 5.0.  Narrower accesses cost
// more: 24 of 128 entries in halves (12 pairs: two entries at a time) 244 us for 24571 x 40.
#include "common.h"

namespace {

struct RotaryArgs {
  const void* src[2]; void* dst[2];              // q, k
  int64_t s_tok[2], s_head[2], d_tok[2], d_head[2];
  int heads[2];
  const void* positions; int64_t pos_axis; int pos64;
  const double* freq;
  int64_t tokens;
  int dim, part, offset, axes, group;            // group: tokens per block
  float amplitude; int inverse;
};

// cos and sin of a fp64 angle, to fp32
__device__ inline void cos_sin(double x, float& c, float& s) {
  const double n = __builtin_rint(x * 0.63661977236758134308);               // 2 / pi
  double r = __builtin_fma(-n, 1.5707963267948965580, x);                     // pi/2, its head and its rest
  r = __builtin_fma(-n, 6.1232339957367660e-17, r);
  const float t = (float)r, u = t * t;
  float ps = __builtin_fmaf(u, -2.50521083854417187751e-8f, 2.75573192239858906526e-6f);      // 1/11!, 1/9!, ...
  ps = __builtin_fmaf(u, ps, -1.98412698412698412698e-4f);
  ps = __builtin_fmaf(u, ps, 8.33333333333333333333e-3f);
  ps = __builtin_fmaf(u, ps, -1.66666666666666666667e-1f);
  const float sn = __builtin_fmaf(u * t, ps, t);
  float pc = __builtin_fmaf(u, -2.75573192239858906526e-7f, 2.48015873015873015873e-5f);      // 1/10!, 1/8!, ...
  pc = __builtin_fmaf(u, pc, -1.38888888888888888889e-3f);
  pc = __builtin_fmaf(u, pc, 4.16666666666666666667e-2f);
  pc = __builtin_fmaf(u, pc, -0.5f);
  const float cs = __builtin_fmaf(u, pc, 1.0f);
  const int quarter = (int)((long long)n & 3);
  const float a = (quarter & 1) ? sn : cs, b = (quarter & 1) ? cs : sn;
  c = (quarter == 1 || quarter == 2) ? -a : a;
  s = (quarter >= 2) ? -b : b;
}

template <class T, int VEC> struct Pack { typedef T type __attribute__((ext_vector_type(VEC))); };
template <class T> struct Pack<T, 1> { typedef T type; };
// One block: `group` tokens, all heads of q and k.  A unit is VEC elements of a head that pass, VEC neighbours that turn
// (interleaved) or VEC pairs (half); thread -> (row, unit), a row being one head of one token.  With VEC = 1 an interleaved pair
// is a unit of two accesses too (one thread has to own both entries: q may turn in place).
template <class T, int VEC, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  extern __shared__ float table[];               // [group][pairs] cosines, then as many sines
  const int pairs = a.part / 2, per_axis = pairs / a.axes;
  const int64_t t0 = (int64_t)blockIdx.x * a.group;
  const int n = (int)min((int64_t)a.group, a.tokens - t0);
  float* const cosines = table;
  float* const sines = table + a.group * pairs;
  constexpr bool TWO = HALF || VEC == 1;         // a unit that turns has its second entries elsewhere
  const int apart = HALF ? pairs : 1;
  const int turning = TWO ? pairs / VEC : a.part / VEC, units = turning + (a.dim - a.part) / VEC;
  const int wide = min(units, 256), rows_at_once = 256 / wide;
  const int r0 = threadIdx.x / wide, u0 = threadIdx.x - r0 * wide;
  typedef typename Pack<T, VEC>::type raw;
  const int heads = a.heads[0] + a.heads[1], rows = n * heads;
  const int before = a.offset / VEC;
  // units in the order of their places (neighbouring lanes, neighbouring addresses); where a unit is two accesses, the second's place is skipped
  auto turns = [&](int u) { return u >= before && u - before < turning; };
  raw x, y;
  T* dst;
  int tok;
  auto fetch = [&](int u, int row) {
    int at = TWO && u - before >= turning ? u * VEC + pairs : u * VEC;
    if (TWO && !HALF && turns(u)) at += u - before;
    tok = row / heads;
    const int hh = row - tok * heads, which = hh >= a.heads[0], h = which ? hh - a.heads[0] : hh;
    const T* src = static_cast<const T*>(a.src[which]) + (t0 + tok) * a.s_tok[which] + h * a.s_head[which] + at;
    dst = static_cast<T*>(a.dst[which]) + (t0 + tok) * a.d_tok[which] + h * a.d_head[which] + at;
    x = *reinterpret_cast<const raw*>(src);
    if (TWO && turns(u)) y = *reinterpret_cast<const raw*>(src + apart);
  };
  // The first entries are on their way while the table is made: 65536 tokens x 40 heads of 128 bf16, half of each interleaved, 285 ->
  // 238 us; 25120 x 24 heads of 64 fp32 55 -> 49; all of each, half layout, 236 (two rows at a time, behind the table) -> 242.
  const bool mine = r0 < rows_at_once && u0 < units && r0 < rows;
  if (mine) fetch(u0, r0);
  for (int i = threadIdx.x; i < n * pairs; i += 256) {
    const int t = i / pairs, p = i - t * pairs;
    const int64_t at = (int64_t)(p / per_axis) * a.pos_axis + t0 + t;
    const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[at] : (double)static_cast<const int32_t*>(a.positions)[at];
    float c, s;
    cos_sin(pos * a.freq[p], c, s);
    cosines[i] = c * a.amplitude;
    sines[i] = (a.inverse ? -s : s) * a.amplitude;
  }
  __syncthreads();
  if (!mine) return;
  for (int u = u0; u < units; u += wide) {
    for (int row = r0; row < rows; row += rows_at_once) {
      if (u != u0 || row != r0) fetch(u, row);
      raw* const out = reinterpret_cast<raw*>(dst);
      if (!turns(u)) { *out = x; continue; }
      constexpr int P = TWO ? VEC : VEC / 2;       // pairs of a unit
      const float* c = cosines + tok * pairs + (u - before) * P;
      const float* s = sines + tok * pairs + (u - before) * P;
      if constexpr (TWO) {
        raw ox, oy;
        if constexpr (VEC == 1) {
          ox = (T)((float)x * c[0] - (float)y * s[0]);
          oy = (T)((float)y * c[0] + (float)x * s[0]);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            ox[i] = (T)((float)x[i] * c[i] - (float)y[i] * s[i]);
            oy[i] = (T)((float)y[i] * c[i] + (float)x[i] * s[i]);
          }
        }
        *out = ox;
        *reinterpret_cast<raw*>(dst + apart) = oy;
      } else {
        raw o;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          o[2 * i] = (T)((float)x[2 * i] * c[i] - (float)x[2 * i + 1] * s[i]);
          o[2 * i + 1] = (T)((float)x[2 * i + 1] * c[i] + (float)x[2 * i] * s[i]);
        }
        *out = o;
      }
    }
  }
}

template <class T, int VEC>
void launch(const RotaryArgs& a, bool half, unsigned blocks, size_t lds, hipStream_t stream) {
  if (half) hipLaunchKernelGGL((rotary_kernel<T, VEC, true>), dim3(blocks), dim3(256), lds, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, VEC, false>), dim3(blocks), dim3(256), lds, stream, a);
}

template <class T>
void launch_vec(const RotaryArgs& a, int vec, bool half, unsigned blocks, size_t lds, hipStream_t stream) {
  constexpr int WIDE = 16 / sizeof(T);
  if (vec == WIDE) launch<T, WIDE>(a, half, blocks, lds, stream);
  else if (vec >= 2) launch<T, 2>(a, half, blocks, lds, stream);
  else launch<T, 1>(a, half, blocks, lds, stream);
}

}  // namespace

extern "C" int ac_rotary(const ac_rotary_args* r, void* stream) {
  AC_REQUIRE(r, "ac_rotary: null arguments");
  AC_REQUIRE(r->type == AC_F32 || r->type == AC_F16 || r->type == AC_BF16, "ac_rotary: unknown type %d", r->type);
  AC_REQUIRE(r->layout == AC_ROTARY_HALF || r->layout == AC_ROTARY_INTERLEAVED, "ac_rotary: unknown layout %d", r->layout);
  AC_REQUIRE(r->tokens >= 0 && r->heads[0] >= 1 && r->heads[1] >= 0, "ac_rotary: bad counts");
  AC_REQUIRE(r->dim >= 1 && r->dim <= 1024, "ac_rotary: head dim %d must be in 1 .. 1024", r->dim);
  AC_REQUIRE(r->axes >= 1 && r->part >= 2 && r->axes <= r->part / 2 && r->part % (2 * r->axes) == 0,
             "ac_rotary: part=%d must be a positive multiple of 2 * axes (2 * %d)", r->part, r->axes);
  AC_REQUIRE(r->offset >= 0 && r->part <= r->dim && r->offset <= r->dim - r->part, "ac_rotary: entries %d .. %lld lie outside a head of %d", r->offset,
             (long long)r->offset + r->part, r->dim);
  AC_REQUIRE((int64_t)r->heads[0] + r->heads[1] <= 1 << 20, "ac_rotary: too many heads");
  if (r->tokens == 0) return AC_OK;
  AC_REQUIRE(r->positions && r->frequencies, "ac_rotary: null pointer");
  AC_REQUIRE(((uintptr_t)r->frequencies & 7) == 0 && ((uintptr_t)r->positions & (r->positions64 ? 7 : 3)) == 0, "ac_rotary: misaligned positions or frequencies");
  const int size = r->type == AC_F32 ? 4 : 2;
  const bool half = r->layout == AC_ROTARY_HALF;
  AC_REQUIRE(half || r->offset % 2 == 0, "ac_rotary: interleaved pairs need an even offset");
  RotaryArgs a;
  // the widest access that every address allows: 16 bytes, two elements or one (the stride of an axis of one addresses nothing)
  int64_t all = half ? (int64_t)r->part / 2 : r->part;
  all |= r->offset | r->dim;
  for (int i = 0; i < 2; ++i) {
    a.src[i] = r->src[i]; a.dst[i] = r->dst[i]; a.heads[i] = r->heads[i];
    a.s_tok[i] = r->src_token[i]; a.s_head[i] = r->src_head[i]; a.d_tok[i] = r->dst_token[i]; a.d_head[i] = r->dst_head[i];
    if (!r->heads[i]) continue;
    AC_REQUIRE(r->src[i] && r->dst[i], "ac_rotary: null pointer");
    AC_REQUIRE(((uintptr_t)r->src[i] | (uintptr_t)r->dst[i]) % size == 0, "ac_rotary: misaligned tensor");
    all |= (int64_t)((uintptr_t)r->src[i] / size) | (int64_t)((uintptr_t)r->dst[i] / size);
    if (r->tokens > 1) all |= r->src_token[i] | r->dst_token[i];
    if (r->heads[i] > 1) all |= r->src_head[i] | r->dst_head[i];
  }
  const int wide = 16 / size;
  const int vec = all % wide == 0 ? wide : all % 2 == 0 ? 2 : 1;
  a.positions = r->positions; a.pos_axis = r->position_axis; a.pos64 = r->positions64; a.freq = r->frequencies;
  a.tokens = r->tokens; a.dim = r->dim; a.part = r->part; a.offset = r->offset; a.axes = r->axes;
  a.amplitude = r->amplitude; a.inverse = r->inverse;
  // tokens per block: about 1024 accesses for its 256 threads (65536 tokens x 40 heads of 128 bf16: 239 us with 512 or 1024, 254 with
  // 2048; 25120 x 24 heads of 64 fp32: 52, 49, 50), fewer where that would leave CUs idle
  const int64_t per_token = (int64_t)(r->heads[0] + r->heads[1]) * (r->dim / vec);
  int64_t group = max((int64_t)1, min((int64_t)16, 1024 / per_token));
  while (group > 1 && (r->tokens + group - 1) / group < 4 * ac_device_cus()) group /= 2;
  a.group = (int)group;
  const size_t lds = (size_t)group * r->part * sizeof(float);                 // 16 x 1024 x 4 = 64 KB at most
  // (a launch may not have 2^32 threads: 2^20 blocks of 256 each, one after the other)
  const int64_t most = group << 20;
  for (int64_t t = 0; t < r->tokens; t += most) {
    a.tokens = min(r->tokens - t, most);
    a.positions = static_cast<const uint8_t*>(r->positions) + t * (r->positions64 ? 8 : 4);
    for (int i = 0; i < 2; ++i) if (a.heads[i]) {
      a.src[i] = static_cast<const uint8_t*>(r->src[i]) + t * a.s_tok[i] * size;
      a.dst[i] = static_cast<uint8_t*>(r->dst[i]) + t * a.d_tok[i] * size;
    }
    const unsigned blocks = (unsigned)((a.tokens + group - 1) / group);
    if (r->type == AC_F32) launch_vec<float>(a, vec, half, blocks, lds, as_stream(stream));
    else if (r->type == AC_F16) launch_vec<_Float16>(a, vec, half, blocks, lds, as_stream(stream));
    else launch_vec<__bf16>(a, vec, half, blocks, lds, as_stream(stream));
  }
  return ac_check_launch("ac_rotary");
}
