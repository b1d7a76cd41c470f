// The chosen experts of few tokens, their matrices in microscaled 4-bit numbers (`mx4.h`): a whole layer in two kernels, for steps of at most
// 16 tokens and 128 (token, choice) pairs.
//
//   up:    y[pair][f] = act(gate_e x', up_e x') in bfloat16: a workgroup owns 16 gate rows and the 16 up rows beside them of one chosen expert.
//   down:  out[t][n] (+)= sum over t's choices of w down_e y': a workgroup owns 16 output rows of every chosen expert, one after the other, so
//          nothing is left to add up behind it.
//
// x' and y' are the rows in E2M3, made in registers on the way (`mx6_block`).  In both kernels the 16 columns of the 16x16x128 instruction are the
// step's tokens, whoever's turn it is: a token that has not chosen the expert is a column of zeros and asks for nothing.  So every chosen
// expert's matrices are read once, whatever the number of its tokens, and the down kernel weighs what an instruction gives by the token's weight and
// adds it up in registers.  Sums are in 32 bits in an order that the sizes and the choices fix.
// What bounds both is the stream of the chosen matrices, 17/32 of a byte a value.
#include <algorithm>
#include <type_traits>

#include "mx4.h"

#define MF_MOE_ACT_CLAMPED 0        // as in moe.hip; 1: silu

__device__ __forceinline__ float expert_gate(float g, float u, float limit, int act) {
  return act == MF_MOE_ACT_CLAMPED ? clamped_gate(g, u, limit) : g / (1.0f + expf(-g)) * u;
}

// The pairs of a step, two to a lane, and which of them are of one expert.
struct Pairs {
  int c0, c1;
  __device__ __forceinline__ void load(const int* __restrict__ chosen, int n_pairs, int lane) {
    c0 = lane < n_pairs ? chosen[lane] : -1;
    c1 = lane + 64 < n_pairs ? chosen[lane + 64] : -1;
  }
};
// Token t's choices among the pairs of the masks: bit k is its choice k.
__device__ __forceinline__ unsigned long long choices_of(unsigned long long m0, unsigned long long m1, int t, int top) {
  const int lo = t * top;
  const unsigned long long all = lo < 64 ? (m0 >> lo) | (lo ? m1 << (64 - lo) : 0ull) : lo < 128 ? m1 >> (lo - 64) : 0ull;
  return all & (top == 64 ? ~0ull : (1ull << top) - 1);
}

// grid (tiles of 16 f, experts or pairs): by_pair: the workgroup's expert is that of pair blockIdx.y, if no earlier pair has it
template <typename XT, bool VEC, int NW>
__global__ __launch_bounds__(NW * 64) void experts_up_kernel(const XT* __restrict__ x, const uint4* __restrict__ codes,
                                                             const unsigned* __restrict__ powers, const int* __restrict__ chosen,
                                                             bf16* __restrict__ y, int T, int top, int E, int by_pair, int K, int tiles,
                                                             int steps, int groups, float limit, int act) {
  constexpr int D = sizeof(XT) == 2 ? 3 : 2, W = sizeof(XT) * 8;
  __shared__ __attribute__((aligned(16))) float red[NW][16][36];
  __shared__ int first_of[16];
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Pairs p;
  p.load(chosen, T * top, lane);
  int e = blockIdx.y;
  if (by_pair) e = blockIdx.y < 64 ? __builtin_amdgcn_readlane(p.c0, blockIdx.y) : __builtin_amdgcn_readlane(p.c1, blockIdx.y - 64);
  if (e < 0 || e >= E) return;
  const unsigned long long m0 = __ballot(p.c0 == e), m1 = __ballot(p.c1 == e);
  if (!(m0 | m1)) return;
  if (by_pair && (m0 ? __builtin_ctzll(m0) : 64 + __builtin_ctzll(m1)) != (int)blockIdx.y) return;
  const unsigned long long mine = r16 < T ? choices_of(m0, m1, r16, top) : 0ull;
  if (wid == 0 && g == 0) first_of[r16] = mine ? r16 * top + __builtin_ctzll(mine) : -1;
  const XT* row = x + (size_t)(mine ? r16 : 0) * K;
  const int k_end = mine ? K : 0;
  const size_t tile0 = ((size_t)e * tiles + blockIdx.x) * 2;
  const uint4* wt = codes + tile0 * steps * 64 + lane;
  const unsigned* wp = powers + tile0 * groups * 64 + lane;
  floatx4 acc[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
  uint4 w[D][2];
  unsigned pw[D][2], words[D][W];
  auto load = [&](int s, int t) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      w[s][j] = wt[((size_t)j * steps + t) * 64];
      pw[s][j] = wp[((size_t)j * groups + (t >> 2)) * 64];
    }
    mx_load_block<VEC>(row, t * 128 + g * 32, k_end, words[s]);
  };
  auto multiply = [&](int s, int t) {
    unsigned power;
    const intx8 b = mx6_operand(mx6_block(words[s], power));
#pragma unroll
    for (int j = 0; j < 2; ++j)
      acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_operand(w[s][j]), b, acc[j], MX_FP4, MX_FP6, 0,
                                                                (int)(pw[s][j] >> (8 * (t & 3))), 0, (int)power);
  };
  const int n = (steps - wid + NW - 1) / NW;
#pragma unroll
  for (int s = 0; s < D; ++s)
    if (s < n) load(s, wid + s * NW);
  for (int base = 0; base < n; base += D) {
#pragma unroll
    for (int s = 0; s < D; ++s)
      if (base + s < n) {
        multiply(s, wid + (base + s) * NW);
        if (base + s + D < n) load(s, wid + (base + s + D) * NW);
      }
  }
  // D[f][t]: t = lane % 16, f = 4 (lane / 16) + r
  *reinterpret_cast<floatx4*>(&red[wid][r16][4 * g]) = acc[0];
  *reinterpret_cast<floatx4*>(&red[wid][r16][16 + 4 * g]) = acc[1];
  __syncthreads();
  if (threadIdx.x < 256) {
    const int t = threadIdx.x >> 4, f = threadIdx.x & 15, pair = first_of[t];
    if (pair >= 0) {
      float gate = 0.f, up = 0.f;
#pragma unroll
      for (int q = 0; q < NW; ++q) {
        gate += red[q][t][f];
        up += red[q][t][16 + f];
      }
      y[(size_t)pair * tiles * 16 + blockIdx.x * 16 + f] = (bf16)expert_gate(gate, up, limit, act);      // (past F: zeros)
    }
  }
}

// grid (tiles of 16 n).  y: rows of F16 values, a multiple of 16, zeros past F
template <typename XT, typename OT, int NW>
__global__ __launch_bounds__(NW * 64) void experts_down_kernel(const bf16* __restrict__ y, const uint4* __restrict__ codes,
                                                               const unsigned* __restrict__ powers, const int* __restrict__ chosen,
                                                               const float* __restrict__ weights, const XT* __restrict__ x,
                                                               OT* __restrict__ out, int T, int top, int E, int F16, int N, int tiles, int steps,
                                                               int groups, int add, int hands_on) {
  constexpr int D = 3;
  __shared__ __attribute__((aligned(16))) float red[NW][16][20];
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Pairs p;
  p.load(chosen, T * top, lane);
  const int n = (steps - wid + NW - 1) / NW;                       // steps of this wave in every expert: wid, wid + NW, ...
  // the pairs of experts that are still to come
  unsigned long long left0 = __ballot(p.c0 >= 0 && p.c0 < E), left1 = __ballot(p.c1 >= 0 && p.c1 < E);
  // the loads' place: an expert, this lane's row and weight there, a step
  const uint4* wt = nullptr;
  const unsigned* wp = nullptr;
  const bf16* row = y;
  float weight = 0.f;
  int k_end = 0, i = n;                                            // (i == n: the next expert's turn)
  bool more = n > 0;
  auto next = [&]() {                                              // false: nothing is left
    if (i == n) {
      if (!(left0 | left1)) return false;
      const int e = left0 ? __builtin_amdgcn_readlane(p.c0, __builtin_ctzll(left0)) : __builtin_amdgcn_readlane(p.c1, __builtin_ctzll(left1));
      const unsigned long long m0 = __ballot(p.c0 == e), m1 = __ballot(p.c1 == e);
      left0 &= ~m0;
      left1 &= ~m1;
      unsigned long long mine = r16 < T ? choices_of(m0, m1, r16, top) : 0ull;
      row = y + (size_t)(mine ? r16 * top + __builtin_ctzll(mine) : 0) * F16;
      k_end = mine ? F16 : 0;
      weight = 0.f;
      for (; mine; mine &= mine - 1) weight += weights[r16 * top + __builtin_ctzll(mine)];     // (an expert chosen twice: both weights)
      const size_t tile = (size_t)e * tiles + blockIdx.x;
      wt = codes + tile * steps * 64 + lane;
      wp = powers + tile * groups * 64 + lane;
      i = 0;
    }
    return true;
  };
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
  uint4 w[D];
  unsigned pw[D], words[D][16];
  float share[D];
  bool have[D];
  auto load = [&](int s) {
    have[s] = more = more && next();
    if (have[s]) {
      const int t = wid + i * NW;
      w[s] = wt[(size_t)t * 64];
      pw[s] = wp[(size_t)(t >> 2) * 64] >> (8 * (t & 3));
      mx_load_block<true>(row, t * 128 + g * 32, k_end, words[s]);
      share[s] = weight;
      ++i;
    }
  };
  auto multiply = [&](int s) {
    unsigned power;
    const intx8 b = mx6_operand(mx6_block(words[s], power));
    const floatx4 z = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_operand(w[s]), b, floatx4{0.f, 0.f, 0.f, 0.f}, MX_FP4, MX_FP6, 0,
                                                                       (int)pw[s], 0, (int)power);
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[r] = fmaf(share[s], z[r], sum[r]);
  };
#pragma unroll
  for (int s = 0; s < D; ++s) load(s);
  bool any = true;
  while (any) {
    any = false;
#pragma unroll
    for (int s = 0; s < D; ++s)
      if (have[s]) {
        multiply(s);
        load(s);
        any = true;
      }
  }
  // D[n][t]: t = lane % 16, n = 4 (lane / 16) + r
  *reinterpret_cast<floatx4*>(&red[wid][r16][4 * g]) = sum;
  __syncthreads();
  if (threadIdx.x < 256) {
    const int t = threadIdx.x >> 4, c = threadIdx.x & 15, col = blockIdx.x * 16 + c;
    if (t < T && col < N) {
      const size_t at = (size_t)t * N + col;
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < NW; ++q) v += red[q][t][c];
      if (hands_on)
        for (int k = 0; k < top; ++k)
          if (chosen[t * top + k] >= E) v = fmaf(weights[t * top + k], to_f32(x[at]), v);
      out[at] = from_f32<OT>(add ? to_f32(out[at]) + v : v);
    }
  }
}

// x [T][K] (bfloat16 or float32); gate_up: the stored [E][2 tiles of 16][K], gate and up tiles in turn; down: the stored [E][N][F]; chosen, weights
// [T][top]; y: scratch of T top ceil16(F) bfloat16; out [T][N] float32 (added to with `add`) or bfloat16.  Choices outside 0 .. E - 1 add nothing, or
// with hands_on (from E on, N == K) their token's x.
MF_API int mf_mx4_moe(const void* x, int is_bf16, const void* gate_up, const void* gate_up_powers, const void* down, const void* down_powers,
                      const int* chosen, const float* weights, void* y, void* out, int out_bf16, int T, int top, int E, int F, int K, int N,
                      float limit, int act, int add, int hands_on, hipStream_t stream) {
  if (T < 1 || T > 16 || top < 1 || top > 64 || T * top > 128 || E < 1 || F < 1 || K < 1 || N < 1 || (hands_on && N != K) || (add && out_bf16))
    return (int)hipErrorInvalidValue;
  const int up_tiles = (F + 15) / 16, up_steps = (K + 127) / 128, up_groups = (K + 511) / 512;
  const int tiles = (N + 15) / 16, steps = (F + 127) / 128, groups = (F + 511) / 512;
  const bool vec = (uintptr_t)x % 16 == 0 && K % (is_bf16 ? 8 : 4) == 0;
  const int by_pair = T * top < E;
  auto up = [&](auto T0, auto VEC) {
    using XT = decltype(T0);
    experts_up_kernel<XT, decltype(VEC)::value, 8><<<dim3(up_tiles, by_pair ? T * top : E), 512, 0, stream>>>(
        (const XT*)x, (const uint4*)gate_up, (const unsigned*)gate_up_powers, chosen, (bf16*)y, T, top, E, by_pair, K, up_tiles, up_steps, up_groups,
        limit, act);
  };
  if (is_bf16) vec ? up(bf16{}, std::true_type{}) : up(bf16{}, std::false_type{});
  else vec ? up(float{}, std::true_type{}) : up(float{}, std::false_type{});
  const int rc = mf_launch_status();
  if (rc) return rc;
  auto behind = [&](auto T0, auto O0) {
    using XT = decltype(T0);
    using OT = decltype(O0);
    experts_down_kernel<XT, OT, 16><<<tiles, 1024, 0, stream>>>((const bf16*)y, (const uint4*)down, (const unsigned*)down_powers, chosen, weights,
                                                              (const XT*)x, (OT*)out, T, top, E, up_tiles * 16, N, tiles, steps, groups, add, hands_on);
  };
  if (is_bf16) out_bf16 ? behind(bf16{}, bf16{}) : behind(bf16{}, float{});
  else out_bf16 ? behind(float{}, bf16{}) : behind(float{}, float{});
  return mf_launch_status();
}
