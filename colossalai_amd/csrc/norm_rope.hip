// A packed projection [q | k | v], split, its query and key heads normed, weighted and rotated, in one pass; and its backward pass.
//
//   u = x / sqrt(mean(x^2) + eps),  y = R_p (w * u)         (a head x of D channels at position p; values are copied)
//   g = w * R_p^T dy,  dx = (g - u mean(g u)) / sqrt(..),  dw = sum over tokens and heads of (R_p^T dy) * u
//
// R_p turns the pairs (i, i + D/2) by the angles of p, from a float32 table of cosines and sines. All arithmetic is float32; a
// result is rounded to its type once.
//
// Bound by memory: forward and backward read and write every value once. A wave takes a token: the lanes of a head (D / 16 of
// them, 8 channels of each half a lane, 16-byte loads) form its sums by exchanges among themselves, 64 / lanes heads at a time,
// and the token's angles and the weights stay in registers over all its heads. The weights' gradients are summed in registers over a
// block's tokens, then in LDS, and the blocks' sums meet in a second launch, always in the same order. In the backward, blocks take queries
// or keys, so that one weight and its gradient are in registers.
// 4 x 8192 tokens, 32/8 heads of 128 in bfloat16: forward 178 us (4.5 TB/s), backward 237 (4.8; with both kinds in a block 343, without the next
// head's values on their way 275). As elementary operations both take 7400 us.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.h"

namespace cai {
namespace {

constexpr int NR_BLOCK = 256, NR_WAVES = NR_BLOCK / WAVE;

struct half16 { unsigned short bits; };   // float16 as it is stored
struct brain16 { unsigned short bits; };

DEV_INLINE float to_f32(unsigned short bits, brain16*) { return bf2f(bits); }
DEV_INLINE float to_f32(unsigned short bits, half16*) { return (float)__builtin_bit_cast(_Float16, bits); }
DEV_INLINE unsigned short from_f32(float v, brain16*) { return f2bf(v); }
DEV_INLINE unsigned short from_f32(float v, half16*) { return __builtin_bit_cast(unsigned short, (_Float16)v); }

template <typename T>
struct Eight {   // 8 neighbouring values as they are stored
  short8 raw;
  DEV_INLINE void load(const T* p) { raw = *reinterpret_cast<const short8*>(p); }
  DEV_INLINE void store(T* p) const { *reinterpret_cast<short8*>(p) = raw; }
  DEV_INLINE float get(int i) const { return to_f32((unsigned short)raw[i], (T*)nullptr); }
  DEV_INLINE void set(int i, float v) { raw[i] = (short)from_f32(v, (T*)nullptr); }
};
template <>
struct Eight<float> {
  float4v raw[2];
  DEV_INLINE void load(const float* p) { raw[0] = *reinterpret_cast<const float4v*>(p); raw[1] = *reinterpret_cast<const float4v*>(p + 4); }
  DEV_INLINE void store(float* p) const { *reinterpret_cast<float4v*>(p) = raw[0]; *reinterpret_cast<float4v*>(p + 4) = raw[1]; }
  DEV_INLINE float get(int i) const { return raw[i >> 2][i & 3]; }
  DEV_INLINE void set(int i, float v) { raw[i >> 2][i & 3] = v; }
};

DEV_INLINE float scalar(const float* p) { return *p; }
template <typename T> DEV_INLINE float scalar(const T* p) { return to_f32(p->bits, (T*)nullptr); }

template <int L>
DEV_INLINE float lanes_sum(float v) {
#pragma unroll
  for (int off = L / 2; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// What both passes are told.
struct Heads {
  long tokens;
  int seq, Hq, Hkv, D, rows;           // rows of the table
  long x_batch, x_token;               // strides of the packed projection
  const float* table;
  const int* positions;                // or null: a token's place in its sequence
  const void *wq, *wk;
  bool narrow_weights;                 // of the activations' type, else float32
  float eps;
};

// The channels of a lane: 8 from `at` on in each half, if it has any.
template <typename T>
DEV_INLINE void load_weight(float (&w)[16], const void* from, bool narrow, int at, int half, bool on) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = at + (i & 7) + (i < 8 ? 0 : half);
    w[i] = !on ? 0.0f : narrow ? scalar((const T*)from + c) : ((const float*)from)[c];
  }
}

// Cosines and sines of a token's angles; a position that the table does not have gives NaN.
DEV_INLINE void load_angles(float (&c)[8], float (&s)[8], const Heads& h, long token, int ss, int at, int half, bool on) {
  const int p = h.positions ? h.positions[token] : ss;
  if (!on) return;
  if (p < 0 || p >= h.rows) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = s[i] = __builtin_nanf("");
    return;
  }
  Eight<float> cv, sv;
  cv.load(h.table + (long)p * h.D + at);
  sv.load(h.table + (long)p * h.D + half + at);
#pragma unroll
  for (int i = 0; i < 8; ++i) { c[i] = cv.get(i); s[i] = sv.get(i); }
}

template <typename T, int L>
__global__ __launch_bounds__(NR_BLOCK) void norm_rope_fwd_kernel(T* __restrict__ q, T* __restrict__ k, T* __restrict__ v,
                                                                 const T* __restrict__ x, Heads h) {
  constexpr int SIDE = WAVE / L;   // heads at a time
  const int lane = threadIdx.x & 63, l = lane & (L - 1), side = lane / L, half = h.D / 2, at = l * 8;
  const bool on = at < half;
  const int all = h.Hq + 2 * h.Hkv;
  float wq[16], wk[16];
  load_weight<T>(wq, h.wq, h.narrow_weights, at, half, on);
  load_weight<T>(wk, h.wk, h.narrow_weights, at, half, on);
  const float inv_d = 1.0f / (float)h.D;
  for (long token = (long)blockIdx.x * NR_WAVES + (threadIdx.x >> 6); token < h.tokens; token += (long)gridDim.x * NR_WAVES) {
    const long bb = token / h.seq;
    const int ss = (int)(token % h.seq);
    const T* row = x + bb * h.x_batch + ss * h.x_token;
    float c[8], s[8];
    load_angles(c, s, h, token, ss, at, half, on);
#pragma unroll 2
    for (int head = side; head < all; head += SIDE) {
      Eight<T> lo, hi;
      if (on) {
        lo.load(row + (long)head * h.D + at);
        hi.load(row + (long)head * h.D + half + at);
      }
      const bool is_q = head < h.Hq;
      T* to = is_q ? q + (token * h.Hq + head) * h.D
              : head < h.Hq + h.Hkv ? k + (token * h.Hkv + head - h.Hq) * h.D : v + (token * h.Hkv + head - h.Hq - h.Hkv) * h.D;
      float sum = 0.0f;
      if (on) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += lo.get(i) * lo.get(i) + hi.get(i) * hi.get(i);
      }
      sum = lanes_sum<L>(sum);
      if (!on) continue;
      if (head < h.Hq + h.Hkv) {
        const float r = 1.0f / sqrtf(sum * inv_d + h.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = lo.get(i) * r * (is_q ? wq[i] : wk[i]), b = hi.get(i) * r * (is_q ? wq[8 + i] : wk[8 + i]);
          lo.set(i, a * c[i] - b * s[i]);
          hi.set(i, b * c[i] + a * s[i]);
        }
      }
      lo.store(to + at);
      hi.store(to + half + at);
    }
  }
}

// dw [blocks, 2, D]: sums of the blocks of queries (blockIdx.y == 0) and of those of keys, which copy the values' gradients too.
template <typename T, int L>
__global__ __launch_bounds__(NR_BLOCK) void norm_rope_bwd_kernel(T* __restrict__ dx, float* __restrict__ dw, const T* __restrict__ dq,
                                                                 const T* __restrict__ dk, const T* __restrict__ dv,
                                                                 const T* __restrict__ x, Heads h) {
  constexpr int SIDE = WAVE / L;
  __shared__ float lds[NR_WAVES][L * 16];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, l = lane & (L - 1), side = lane / L, half = h.D / 2, at = l * 8;
  const bool on = at < half, keys = blockIdx.y != 0;
  const int all = h.Hq + 2 * h.Hkv, first = keys ? h.Hq : 0, heads = keys ? h.Hkv : h.Hq;
  float w[16], g[16];
  load_weight<T>(w, keys ? h.wk : h.wq, h.narrow_weights, at, half, on);
#pragma unroll
  for (int i = 0; i < 16; ++i) g[i] = 0.0f;
  const float inv_d = 1.0f / (float)h.D;
  for (long token = (long)blockIdx.x * NR_WAVES + wid; token < h.tokens; token += (long)gridDim.x * NR_WAVES) {
    const long bb = token / h.seq;
    const int ss = (int)(token % h.seq);
    const T* row = x + bb * h.x_batch + ss * h.x_token + (long)first * h.D + at;
    const T* grad = (keys ? dk : dq) + token * heads * h.D + at;
    T* out = dx + (token * all + first) * h.D + at;
    float c[8], s[8];
    load_angles(c, s, h, token, ss, at, half, on);
    // the next head's values are on their way while a head is worked on, where they are two bytes (else they take a wave's room)
    constexpr bool AHEAD = sizeof(T) == 2;
    Eight<T> lo, hi, glo, ghi, lo2, hi2, glo2, ghi2;
    auto load = [&](int head, Eight<T>& a, Eight<T>& b, Eight<T>& c, Eight<T>& d) {
      if (!on || head >= heads) return;
      a.load(row + (long)head * h.D);
      b.load(row + (long)head * h.D + half);
      c.load(grad + (long)head * h.D);
      d.load(grad + (long)head * h.D + half);
    };
    if (AHEAD) load(side, lo2, hi2, glo2, ghi2);
#pragma unroll 1
    for (int head = side; head < heads; head += SIDE) {
      if (AHEAD) {
        lo = lo2, hi = hi2, glo = glo2, ghi = ghi2;
        load(head + SIDE, lo2, hi2, glo2, ghi2);
      } else {
        load(head, lo, hi, glo, ghi);
      }
      float sum = 0.0f, dot = 0.0f, a[16];
      if (on) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = glo.get(i), r = ghi.get(i), u = lo.get(i), v = hi.get(i);
          a[i] = p * c[i] + r * s[i];
          a[8 + i] = r * c[i] - p * s[i];
          sum += u * u + v * v;
          dot += a[i] * w[i] * u + a[8 + i] * w[8 + i] * v;
        }
      }
      sum = lanes_sum<L>(sum);
      dot = lanes_sum<L>(dot);
      if (!on) continue;
      const float r = 1.0f / sqrtf(sum * inv_d + h.eps), m = dot * inv_d * r * r;
      Eight<T> olo, ohi;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = lo.get(i), v = hi.get(i);
        olo.set(i, r * (a[i] * w[i] - u * m));
        ohi.set(i, r * (a[8 + i] * w[8 + i] - v * m));
        g[i] += a[i] * (u * r);
        g[8 + i] += a[8 + i] * (v * r);
      }
      olo.store(out + (long)head * h.D);
      ohi.store(out + (long)head * h.D + half);
    }
    if (!keys || !on) continue;
    for (int head = side; head < heads; head += SIDE) {
      Eight<T> lo, hi;
      const T* from = dv + (token * heads + head) * h.D + at;
      lo.load(from);
      hi.load(from + half);
      T* to = out + (long)(heads + head) * h.D;
      lo.store(to);
      hi.store(to + half);
    }
  }
  // the heads beside each other, then the waves
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int off = L; off < WAVE; off <<= 1) g[i] += __shfl_xor(g[i], off);
    if (side == 0 && on) lds[wid][at + (i & 7) + (i < 8 ? 0 : half)] = g[i];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < h.D; j += NR_BLOCK) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NR_WAVES; ++i) sum += lds[i][j];
    dw[((long)blockIdx.x * 2 + keys) * h.D + j] = sum;
  }
}

// The blocks' sums, 32 columns x 32 groups of blocks a block; columns [0, D) are the query weight's.
template <typename T>
__global__ __launch_bounds__(1024) void norm_rope_dw_kernel(void* __restrict__ dwq, void* __restrict__ dwk, const float* __restrict__ part,
                                                            int parts, int D, bool narrow) {
  __shared__ float lds[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
  float sum = 0.0f;
  if (col < 2 * D) {
#pragma unroll 8
    for (int p = g; p < parts; p += 32) sum += part[(long)p * 2 * D + col];
  }
  lds[g][c] = sum;
  __syncthreads();
  if (g == 0 && col < 2 * D) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) total += lds[i][c];
    void* to = col < D ? dwq : dwk;
    const int at = col < D ? col : col - D;
    if constexpr (!std::is_same<T, float>::value) {
      if (narrow) {
        ((T*)to)[at].bits = from_f32(total, (T*)nullptr);
        return;
      }
    }
    ((float*)to)[at] = total;
  }
}

// =============================================================== host side

bool known(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

Heads heads_of(const at::Tensor& x, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& table,
               const c10::optional<at::Tensor>& positions, int64_t Hq, int64_t Hkv, double eps) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 3 && known(x.scalar_type()), "qkv_norm_rope: qkv must be bfloat16, float16 or float32 [B, S, (Hq + 2 Hkv) D]");
  TORCH_CHECK(wq.dim() == 1 && wk.dim() == 1 && wq.numel() == wk.numel() && wq.scalar_type() == wk.scalar_type() &&
              (wq.scalar_type() == x.scalar_type() || wq.scalar_type() == at::kFloat) && wq.is_contiguous() && wk.is_contiguous(),
              "qkv_norm_rope: both weights must be [D], of qkv's type or float32");
  const int64_t D = wq.numel();
  TORCH_CHECK(D % 16 == 0 && D >= 16 && D <= 512, "qkv_norm_rope: head sizes are multiples of 16 up to 512, got ", D);
  TORCH_CHECK(Hq > 0 && Hkv > 0 && x.size(2) == (Hq + 2 * Hkv) * D, "qkv_norm_rope: qkv has ", x.size(2), " channels, ", Hq, " + 2 * ", Hkv,
              " heads of ", D, " have ", (Hq + 2 * Hkv) * D);
  TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kFloat && table.is_contiguous() && table.size(1) == D,
              "qkv_norm_rope: table must be contiguous float32 [positions, D]");
  const int64_t tokens = x.size(0) * x.size(1);
  TORCH_CHECK(tokens < (1L << 31), "qkv_norm_rope: too many tokens");
  if (positions.has_value()) {
    TORCH_CHECK(positions->scalar_type() == at::kInt && positions->is_contiguous() && positions->numel() == tokens,
                "qkv_norm_rope: positions must be int32, one a token");
  } else {
    TORCH_CHECK(x.size(1) <= table.size(0), "qkv_norm_rope: ", x.size(1), " positions, the table has ", table.size(0));
  }
  for (const at::Tensor& t : {wq, wk, table, positions.value_or(table)})
    TORCH_CHECK(t.device() == x.device(), "qkv_norm_rope: tensors on ", x.device(), " and ", t.device());
  Heads h;
  h.tokens = tokens;
  h.seq = (int)std::max<int64_t>(x.size(1), 1);
  h.Hq = (int)Hq;
  h.Hkv = (int)Hkv;
  h.D = (int)D;
  h.rows = (int)std::min<int64_t>(table.size(0), INT_MAX);
  h.x_batch = x.stride(0);
  h.x_token = x.stride(1);
  h.table = table.data_ptr<float>();
  h.positions = positions.has_value() ? positions->data_ptr<int>() : nullptr;
  h.wq = wq.data_ptr();
  h.wk = wk.data_ptr();
  h.narrow_weights = wq.scalar_type() != at::kFloat;
  h.eps = (float)eps;
  return h;
}

bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// rows that 16-byte loads fit
at::Tensor dense_rows(const at::Tensor& x) {
  const int64_t per = 16 / x.element_size();
  if (x.stride(2) == 1 && x.stride(0) % per == 0 && x.stride(1) % per == 0 && aligned(x)) return x;
  return x.clone(at::MemoryFormat::Contiguous);
}
at::Tensor dense(const at::Tensor& x) { return x.is_contiguous() && aligned(x) ? x : x.clone(at::MemoryFormat::Contiguous); }

#define NR_LANES(T, D, ...)                                                             \
  do {                                                                                  \
    if ((D) <= 32) { using S = T; constexpr int L = 2; __VA_ARGS__; }                    \
    else if ((D) <= 64) { using S = T; constexpr int L = 4; __VA_ARGS__; }               \
    else if ((D) <= 128) { using S = T; constexpr int L = 8; __VA_ARGS__; }              \
    else if ((D) <= 256) { using S = T; constexpr int L = 16; __VA_ARGS__; }             \
    else { using S = T; constexpr int L = 32; __VA_ARGS__; }                             \
  } while (0)
#define NR_DISPATCH(type, D, ...)                                \
  do {                                                           \
    if ((type) == at::kFloat) NR_LANES(float, D, __VA_ARGS__);    \
    else if ((type) == at::kHalf) NR_LANES(half16, D, __VA_ARGS__); \
    else NR_LANES(brain16, D, __VA_ARGS__);                       \
  } while (0)

}  // namespace

std::vector<at::Tensor> norm_rope_fwd(at::Tensor qkv, at::Tensor wq, at::Tensor wk, at::Tensor table,
                                      c10::optional<at::Tensor> positions, int64_t Hq, int64_t Hkv, double eps) {
  TORCH_CHECK(qkv.is_cuda() && qkv.dim() == 3, "qkv_norm_rope: qkv must be [B, S, (Hq + 2 Hkv) D]");
  const c10::DeviceGuard guard(qkv.device());
  const at::Tensor x = dense_rows(qkv);
  for (at::Tensor* t : {&wq, &wk, &table}) *t = dense(*t);
  const Heads h = heads_of(x, wq, wk, table, positions, Hq, Hkv, eps);
  const auto q = at::empty({x.size(0), x.size(1), Hq, h.D}, x.options()), k = at::empty({x.size(0), x.size(1), Hkv, h.D}, x.options());
  const auto v = at::empty_like(k);
  if (h.tokens == 0) return {q, k, v};
  auto stream = at::hip::getCurrentHIPStream();
  NR_DISPATCH(x.scalar_type(), h.D, {
    hipLaunchKernelGGL((norm_rope_fwd_kernel<S, L>), dim3(capped_grid((h.tokens + NR_WAVES - 1) / NR_WAVES, 4096)), dim3(NR_BLOCK), 0,
                       stream.stream(), (S*)q.data_ptr(), (S*)k.data_ptr(), (S*)v.data_ptr(), (const S*)x.data_ptr(), h);
  });
  HIP_CHECK_LAST();
  return {q, k, v};
}

std::vector<at::Tensor> norm_rope_bwd(at::Tensor dq_in, at::Tensor dk_in, at::Tensor dv_in, at::Tensor qkv, at::Tensor wq, at::Tensor wk,
                                      at::Tensor table, c10::optional<at::Tensor> positions, int64_t Hq, int64_t Hkv, double eps) {
  TORCH_CHECK(qkv.is_cuda() && qkv.dim() == 3, "qkv_norm_rope: qkv must be [B, S, (Hq + 2 Hkv) D]");
  const c10::DeviceGuard guard(qkv.device());
  const at::Tensor x = dense_rows(qkv), dq = dense(dq_in), dk = dense(dk_in), dv = dense(dv_in);
  for (at::Tensor* t : {&wq, &wk, &table}) *t = dense(*t);
  const Heads h = heads_of(x, wq, wk, table, positions, Hq, Hkv, eps);
  for (const at::Tensor& t : {dq, dk, dv})
    TORCH_CHECK(t.device() == x.device() && t.scalar_type() == x.scalar_type() && t.numel() == h.tokens * h.D * (t.is_same(dq) ? Hq : Hkv),
                "qkv_norm_rope: gradients have the outputs' shapes and type");
  const auto dx = at::empty({x.size(0), x.size(1), x.size(2)}, x.options()), dwq = at::empty_like(wq), dwk = at::empty_like(wk);
  // Three tokens a wave make up for a block's weights and sums, while there are blocks for every CU. Three waves a SIMD, which every type and
  // head size has the registers for (150 to 168), are 768 blocks, 384 of each kind, at once: a few more would wait for all of them. With 384, and with
  // the 391, 475 and 571 of 4700, 5700 and 6850 tokens: 16/4 heads of 64 in bfloat16 20 to 24 us and 27 to 29, 8/8 of 128 23 to 29 and 28 to 32, 32/8
  // of 128 38 to 49 and 38 to 51, 16/4 of 256 39 to 51 and 40 to 53, 4/2 of 512 in float16 29 to 37 and 36 to 43, in float32 12/4 of 96 27 to 36 and
  // 33 to 39, 16/4 of 32 20 to 24 and 27 to 29, 32/8 of 128 the same. Many even the kinds' shares out (4 x 8192 tokens, 32/8 heads of 128: 1024 236
  // us, 384 of each 325)
  const long one = (h.tokens + NR_WAVES - 1) / NR_WAVES, some = std::min<long>({one, 1024, std::max<long>(256, one / 3)});
  const int grid = (int)(some > 384 && some < 576 ? 384 : some);
  const auto part = at::empty({(long)grid * 2 * h.D}, x.options().dtype(at::kFloat));
  auto stream = at::hip::getCurrentHIPStream();
  NR_DISPATCH(x.scalar_type(), h.D, {
    if (grid > 0)
      hipLaunchKernelGGL((norm_rope_bwd_kernel<S, L>), dim3(grid, 2), dim3(NR_BLOCK), 0, stream.stream(), (S*)dx.data_ptr(), part.data_ptr<float>(),
                         (const S*)dq.data_ptr(), (const S*)dk.data_ptr(), (const S*)dv.data_ptr(), (const S*)x.data_ptr(), h);
    HIP_CHECK_LAST();
    hipLaunchKernelGGL((norm_rope_dw_kernel<S>), dim3((2 * h.D + 31) / 32), dim3(1024), 0, stream.stream(), dwq.data_ptr(), dwk.data_ptr(),
                       part.data_ptr<float>(), grid, h.D, h.narrow_weights);
  });
  HIP_CHECK_LAST();
  return {dx, dwq, dwk};
}

}  // namespace cai
