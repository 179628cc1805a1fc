// Dropout's random bits: Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", SC 2011), a bijection of a 128-bit counter under a 64-bit key. Each round multiplies two
// words of the counter by constants and mixes the halves of the products with the other two words and the
// key, which advances by a Weyl step. A mask needs no storage: whoever knows (key, counter) forms it again.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace b2c {
namespace dev {

struct Philox4 {
  uint32_t w[4];
};

__host__ __device__ __forceinline__ Philox4 philox(uint64_t lo, uint64_t hi, uint64_t key) {
  uint32_t c0 = (uint32_t)lo, c1 = (uint32_t)(lo >> 32), c2 = (uint32_t)hi, c3 = (uint32_t)(hi >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// Dropout's parameters as the kernels take them: keep iff bits >= threshold (0: everything is kept).
struct Drop {
  uint64_t seed, stream;
  uint32_t threshold;
  float scale;
};

// The eight 16-bit fields of one counter are elements 8 i .. 8 i + 7.
__device__ __forceinline__ bool kept(const Philox4& w, int j, uint32_t threshold) {
  return ((w.w[j >> 1] >> ((j & 1) * 16)) & 0xffffu) >= threshold;
}

// Which of elements e .. e + N - 1 are kept (N at most 8), as bits: they lie in one counter's fields or in two neighbouring
// counters'. One copy of the rounds, run once or twice.
template <int N>
__device__ __forceinline__ uint32_t kept_bits(const Drop& d, uint64_t e) {
  const int o = (int)(e & 7);
  uint32_t m = 0;
#pragma unroll 1
  for (int i = 0; i <= (o + N > 8); i++) {
    const Philox4 w = philox((e >> 3) + i, d.stream, d.seed);
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) b |= (uint32_t)kept(w, j, d.threshold) << j;
    m |= b << (8 * i);
  }
  return m >> o;
}

}  // namespace dev
}  // namespace b2c
