// The 4-bit key/value cache: where its bytes are, and device functions shared by the kernels that write and read it.
//
// A slab is 16 tokens of one head, 18 D bytes: codes of the keys (8 D), codes of the values (8 D), scales and zero points of
// the keys (D), of the values (D).  The order inside is that of the registers of mma.m16n8k16 with the cache as the 16-row
// operand: a lane (g = lane / 4, t = lane % 4) finds its codes in one contiguous piece, and masking a word with 0x000f000f
// gives two neighbours along the contraction as the two halves of a register (channels for q.k, tokens for p.v).
//   keys    [plane][token 16][t 4][j][b 2][a 4]        channel 128 plane + 32 j + 8 t + 2 a + b, a and b within a word
//   values  [plane][half 2][g 8][t 4][j][odd 2][p 4]   token 8 half + 2 t + odd, channel 128 plane + 32 j + 4 g + p
//   keys    [token 16][group] {fp16 scale, fp16 1024 + zero point}
//   values  [pair 8][group] {scale, scale, 1024 + zero point, 1024 + zero point} (even token, odd token)
// (codes are nibbles, a plane is 128 channels or all 64 of a head of 64, a group 64 channels).  A group's value is
// s (c - z) with c, z in 0..15 and s of 7 significant bits, at least 2^-18 and at most 4352: exact in fp16.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace atlas {

constexpr int KV_SLAB = 16;                  // tokens
constexpr float KV_MIN_SCALE = 0x1p-18f;     // s (c - z) is a multiple of 2^-24, the spacing of the smallest fp16 numbers
constexpr float KV_MAX_SCALE = 4352.0f;      // 15 s stays below the largest fp16 number (groups that span more than 15 s lose their upper end)
constexpr float KV_MAX_VALUE = 15.0f * KV_MAX_SCALE;

__host__ __device__ constexpr int kv_slab_bytes(int d) { return 18 * d; }
// Offsets within a slab.
__host__ __device__ constexpr int kv_value_codes(int d) { return 8 * d; }
__host__ __device__ constexpr int kv_key_params(int d) { return 16 * d; }
__host__ __device__ constexpr int kv_value_params(int d) { return 17 * d; }
// Byte of the word that holds channels 8 w .. 8 w + 7 of a token's key.
__host__ __device__ constexpr int kv_key_word(int d, int token, int w) {
    return d == 64 ? token * 32 + (w & 3) * 8 + (w >> 2) * 4 : (w >> 4) * 1024 + token * 64 + (w & 3) * 16 + ((w >> 2) & 3) * 4;
}
// Byte of the unit of two that holds channels 4 u .. 4 u + 3 of a token's value (from the start of the values' codes).
__host__ __device__ constexpr int kv_value_unit(int d, int token, int u) {
    const int lane = (u & 7) * 4 + (token & 7) / 2;
    return d == 64 ? (token >> 3) * 256 + lane * 8 + (u >> 3) * 4 + (token & 1) * 2
                   : (u >> 5) * 1024 + (token >> 3) * 512 + lane * 16 + ((u >> 3) & 3) * 4 + (token & 1) * 2;
}

int check_kv_shape(int64_t num_pages, int64_t kv_heads, int64_t head_dim, int64_t page_size, const char *what);

// Launches a kernel that waits for the one in front itself (griddepcontrol.wait), so that its start overlaps with that one's end.
template <typename... Parameters, typename... Arguments>
int launch_early(void (*kernel)(Parameters...), dim3 grid, int threads, int smem, cudaStream_t stream, const char *what, Arguments... arguments) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    return check_cuda(cudaLaunchKernelEx(&config, kernel, Parameters(arguments)...), what);
}
// Nothing is read before the kernels in front have ended; what follows may start then, and wait in turn.
inline __device__ void wait_for_front() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace atlas
