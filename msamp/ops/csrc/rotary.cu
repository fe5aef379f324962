// Rotary positions: each pair (x1, x2) of the first `part` elements of a head is turned by the angle position * freq[pair],
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin     (the gradient: by the negative angle),
// pairs (i, i + part / 2) of a head, or (2 i, 2 i + 1) when interleaved; the other elements are copied.
//
// The angle is taken in 64 bits, in turns, and reduced to (-1/2, 1/2] before it is rounded to 32 bits: at position 10^6 a 32-bit
// angle is off by 0.06.  Sine and cosine belong to a token, not to a head, so a CTA computes those of its tokens once
// (in shared memory) and takes all heads of both tensors through them.  Bound by memory: one read and one write of every head.
#include <initializer_list>

#include "common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPart = 1024;
constexpr int kMaxTokens = 4;

struct RotTensor {
  const void* x;
  void* y;
  int64_t x_sb, x_ss, x_sh, y_sb, y_ss, y_sh;    // element strides: batch, sequence, head; the elements of a head are adjacent
  int heads;
};
struct RotParams {
  RotTensor t[2];
  const double* freqs;       // [part / 2], radians per position
  const void* positions;     // int32 or int64, or null: the index in the sequence
  int64_t p_sb, p_ss;
  int pos64, batch, seq, dim, part, per_cta, inplace;
  float sign;
};

// What a thread takes of a head at once: VEC, a 16-byte vector of pairs (interleaved), or one of first and one of second elements; else a pair.
// In the last slots of a head, elements that are only copied.
template <typename T, bool INTER, bool VEC>
struct Slot {
  static constexpr int V = VEC ? 16 / sizeof(T) : 1;
  Bytes16 a, b;
  T sa, sb;
  __device__ __forceinline__ void load(const T* x, int slot, int turn, int half, int part) {
    const bool copy = slot >= turn;
    const int at = copy ? part + (slot - turn) * V : (INTER && !VEC ? 2 * slot : slot * V);
    const int second = INTER ? at + 1 : at + half;    // of a pair in two places
    if constexpr (VEC) {
      a = *reinterpret_cast<const Bytes16*>(x + at);
      if (!INTER && !copy) b = *reinterpret_cast<const Bytes16*>(x + second);
    } else {
      sa = x[at];
      if (!copy) sb = x[second];
    }
  }
  __device__ __forceinline__ void store(T* y, const float2* cs, int slot, int turn, int half, int part) {
    const bool copy = slot >= turn;
    const int at = copy ? part + (slot - turn) * V : (INTER && !VEC ? 2 * slot : slot * V);
    const int second = INTER ? at + 1 : at + half;
    if constexpr (VEC) {
      if (!copy) {
        T* ea = reinterpret_cast<T*>(&a);
        T* eb = reinterpret_cast<T*>(&b);
        if constexpr (INTER) {
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            const float2 w = cs[(slot * V + j) / 2];
            const float x1 = to_f32<T>(ea[j]), x2 = to_f32<T>(ea[j + 1]);
            ea[j] = from_f32<T>(x1 * w.x - x2 * w.y);
            ea[j + 1] = from_f32<T>(x2 * w.x + x1 * w.y);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float2 w = cs[slot * V + j];
            const float x1 = to_f32<T>(ea[j]), x2 = to_f32<T>(eb[j]);
            ea[j] = from_f32<T>(x1 * w.x - x2 * w.y);
            eb[j] = from_f32<T>(x2 * w.x + x1 * w.y);
          }
          *reinterpret_cast<Bytes16*>(y + second) = b;
        }
      }
      *reinterpret_cast<Bytes16*>(y + at) = a;
    } else {
      if (copy) {
        y[at] = sa;
      } else {
        const float2 w = cs[slot];
        const float x1 = to_f32<T>(sa), x2 = to_f32<T>(sb);
        y[at] = from_f32<T>(x1 * w.x - x2 * w.y);
        y[second] = from_f32<T>(x2 * w.x + x1 * w.y);
      }
    }
  }
};

// The CTA's work is a list of (token, head, slot); a thread takes every 256th and counts up in mixed radix instead of dividing.  Its first
// loads are under way while the angles are worked out.  Six CTAs an SM (40 registers; the interleaved vector forms spill one of them, 4 bytes
// in and out) and two loads in flight a thread measure the same (L2 flushed before each call): 8192 tokens x 40 heads of 128, bf16, 39 us,
// interleaved 43, half of each head 41; a copy of the same bytes takes 33 us.  With divisions for every item it took 37, 53 and 51 us.
// Far from memory's time: narrow parts.  Where half of the part is no whole number of vectors, everything goes one element at a time, what
// is only copied as well (6000 tokens x 32 heads of 80, part 20, bf16: 62 us, a copy 16); with vectors but few of them a CTA is mostly its
// chain of offsets, barrier, angles, barrier, store (3069 tokens x 24 heads of 64, part 16, fp16: 10 us for the 3 of its bytes).
template <typename T, bool INTER, bool VEC>
__global__ void __launch_bounds__(kThreads, 6) rotary_kernel(const RotParams p) {
  extern __shared__ float2 s_cs[];    // [per_cta][half] cosine, signed sine
  __shared__ int64_t s_at[2][2][kMaxTokens];    // offsets of the tokens: tensor, x or y
  constexpr int V = VEC ? 16 / sizeof(T) : 1;
  const int half = p.part / 2;
  const int64_t tokens = (int64_t)p.batch * p.seq, t0 = (int64_t)blockIdx.x * p.per_cta;
  const int n_tok = (int)min((int64_t)p.per_cta, tokens - t0);
  if (threadIdx.x < 4 * n_tok) {
    const int j = threadIdx.x >> 2, tensor = (threadIdx.x >> 1) & 1;
    const int64_t b = (t0 + j) / p.seq, s = (t0 + j) - b * p.seq;
    const RotTensor& t = p.t[tensor];
    s_at[tensor][threadIdx.x & 1][j] = threadIdx.x & 1 ? b * t.y_sb + s * t.y_ss : b * t.x_sb + s * t.x_ss;
  }
  __syncthreads();
  // slots of a head: vectors (or elements) of its pairs, then of what is only copied
  const int turn = VEC && INTER ? p.part / V : half / V;
  const int slots = turn + (p.inplace ? 0 : (p.dim - p.part) / V);
  const int heads0 = p.t[0].heads, heads = heads0 + p.t[1].heads;
  int slot = threadIdx.x % slots, h = threadIdx.x / slots, tok = h / heads;
  h -= tok * heads;
  const int d_slot = kThreads % slots, d_rest = kThreads / slots, d_h = d_rest % heads, d_tok = d_rest / heads;
  auto advance = [&]() {
    slot += d_slot;
    h += d_h;
    tok += d_tok;
    if (slot >= slots) {
      slot -= slots;
      ++h;
    }
    if (h >= heads) {
      h -= heads;
      ++tok;
    }
  };
  Slot<T, INTER, VEC> x;
  T* y;
  int at_slot, at_tok;
  auto load = [&]() {
    y = nullptr;
    if (tok >= n_tok) return;
    const int second = h >= heads0;
    const RotTensor& t = p.t[second];
    const int64_t k = h - (second ? heads0 : 0);
    x.load(reinterpret_cast<const T*>(t.x) + s_at[second][0][tok] + k * t.x_sh, slot, turn, half, p.part);
    y = reinterpret_cast<T*>(t.y) + s_at[second][1][tok] + k * t.y_sh;
    at_slot = slot;
    at_tok = tok;
    advance();
  };
  load();
  for (int i = threadIdx.x; i < n_tok * half; i += kThreads) {
    const int j = i / half;
    const int64_t b = (t0 + j) / p.seq, s = (t0 + j) - b * p.seq;
    double pos = (double)s;
    if (p.positions) {
      const int64_t at = b * p.p_sb + s * p.p_ss;
      pos = p.pos64 ? (double)reinterpret_cast<const int64_t*>(p.positions)[at] : (double)reinterpret_cast<const int*>(p.positions)[at];
    }
    double turns = pos * p.freqs[i - j * half] * 0.15915494309189533577;    // 1 / (2 pi)
    turns -= rint(turns);
    float sn, cs;
    sincospif((float)(2.0 * turns), &sn, &cs);
    s_cs[i] = make_float2(cs, sn * p.sign);
  }
  __syncthreads();
  while (y) {
    x.store(y, s_cs + at_tok * half, at_slot, turn, half, p.part);
    load();
  }
}

}    // namespace

// x0 [batch, seq, heads0, dim] -> y0 and x1 [batch, seq, heads1, dim] -> y1 (heads1 may be 0).  y may be x itself with the same strides;
// otherwise the two must not overlap.  The arguments come as one block of 64-bit fields, which a caller in Python packs several times faster
// than it passes thirty arguments.
struct RotaryArgs {
  const void* x0;
  void* y0;
  const void* x1;
  void* y1;
  int64_t strides[12];    // (batch, seq, head) element strides of x0, y0, x1, y1
  const double* freqs;
  const void* positions;
  int64_t pos64, p_sb, p_ss;    // positions are int64 (else int32); their strides
  int64_t batch, seq, heads0, heads1, dim, part, interleaved, inverse, dtype;
};
MSAMP_API int msamp_rotary(const RotaryArgs* a, void* stream_) {
  MSAMP_REQUIRE(a, "rotary: no arguments");
  const void *x0 = a->x0, *x1 = a->x1;
  void *y0 = a->y0, *y1 = a->y1;
  const int64_t* strides = a->strides;
  const double* freqs = a->freqs;
  for (int64_t v : {a->batch, a->seq, a->heads0, a->heads1, a->dim, a->part}) MSAMP_REQUIRE(v >= 0 && v <= 0x7fffffff, "rotary: size %lld", (long long)v);
  const int batch = (int)a->batch, seq = (int)a->seq, heads0 = (int)a->heads0, heads1 = (int)a->heads1, dim = (int)a->dim, part = (int)a->part;
  const int dtype = (int)a->dtype;
  const bool interleaved = a->interleaved != 0, inverse = a->inverse != 0;
  MSAMP_REQUIRE(part >= 2 && part % 2 == 0 && part <= dim && part <= kMaxPart, "rotary: part %d of a head of %d (even, at most %d)", part, dim, kMaxPart);
  MSAMP_REQUIRE(freqs, "rotary: no frequencies");
  if (batch == 0 || seq == 0 || heads0 + heads1 == 0) return MSAMP_OK;
  RotParams p = {};
  const bool in0 = heads0 == 0 || x0 == y0, in1 = heads1 == 0 || x1 == y1;
  p.inplace = in0 && in1;
  const void *px[2] = {x0, x1};
  void* py[2] = {y0, y1};
  const int heads[2] = {heads0, heads1};
  int64_t each = 0;    // every stride and address, OR-ed: vectors need all of them to be multiples of 16 bytes
  const int size = dtype == DT_F32 ? 4 : 2;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = strides + 6 * i;
    if (heads[i] > 0) {
      MSAMP_REQUIRE(px[i] && py[i], "rotary: null pointer");
      if (px[i] == py[i]) MSAMP_REQUIRE(s[0] == s[3] && s[1] == s[4] && s[2] == s[5], "rotary: in place with other strides");
      for (int k = 0; k < 6; ++k) each |= s[k] * size;
      each |= (int64_t)(uintptr_t)px[i] | (int64_t)(uintptr_t)py[i];
    }
    p.t[i] = RotTensor{px[i], py[i], s[0], s[1], s[2], s[3], s[4], s[5], heads[i]};
  }
  p.freqs = freqs; p.positions = a->positions; p.pos64 = a->pos64 != 0; p.p_sb = a->p_sb; p.p_ss = a->p_ss;
  p.batch = batch; p.seq = seq; p.dim = dim; p.part = part; p.sign = inverse ? -1.0f : 1.0f;
  const int half = part / 2;
  // tokens of a CTA: an angle for every thread, but one token each while that leaves SMs without work
  p.per_cta = half >= kThreads ? 1 : kThreads / half < kMaxTokens ? kThreads / half : kMaxTokens;
  while (p.per_cta > 1 && (int64_t)batch * seq < (int64_t)p.per_cta * 2 * msamp_sm_count()) p.per_cta /= 2;
  const int64_t tokens = (int64_t)batch * seq, grid = (tokens + p.per_cta - 1) / p.per_cta;
  MSAMP_REQUIRE(grid <= 0x7fffffff, "rotary: too many tokens");
  const int v = 16 / size;
  const bool vec = each % 16 == 0 && dim % v == 0 && (interleaved ? part % v == 0 : half % v == 0);
  const int smem = p.per_cta * half * (int)sizeof(float2);
  cudaStream_t stream = (cudaStream_t)stream_;
  MSAMP_DISPATCH_HP(dtype, T, {
    if (vec && interleaved)  rotary_kernel<T, true, true><<<(unsigned)grid, kThreads, smem, stream>>>(p);
    else if (vec)            rotary_kernel<T, false, true><<<(unsigned)grid, kThreads, smem, stream>>>(p);
    else if (interleaved)    rotary_kernel<T, true, false><<<(unsigned)grid, kThreads, smem, stream>>>(p);
    else                     rotary_kernel<T, false, false><<<(unsigned)grid, kThreads, smem, stream>>>(p);
  });
  return msamp_check_launch("msamp_rotary");
}
