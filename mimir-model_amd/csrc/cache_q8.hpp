// The 8-bit key-value cache: int8 values with one float32 scale for each
// block of 32 entries and kv head, for keys and for values.
//
// A block of a kv head is one record of 64 * DP bytes (DP: d padded to a
// multiple of 64): 32 keys, then 32 values, a byte each holding value + 128.
// Inside, the bytes lie in the order in which the lanes of a wave read them
// as operands of v_mfma_f32_16x16x32_f16, 16 bytes a lane, so that a load of
// 64 lanes is 1 KiB without a gap and no lane moves bytes to another:
//   keys    [2 key tiles][DP/64][lane][16]: lane 16 g + r holds the dims
//           64 c + 16 g .. +15 of key r of the tile;
//   values  [DP/32][lane][2 dim tiles][8]: lane 16 g + m holds dim 32 c +
//           16 dt + m of keys 4 g .. 4 g + 3 of both key tiles, the keys whose
//           weights the same lane holds after the score product.
// Byte + 128 costs the attention one byte permute and one packed add for two
// values: 0x6400 | byte is the f16 number 1024 + byte.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mimg {

constexpr int Q8C_BLOCK = 32;
constexpr int Q8C_MAX_D = 256;
// The smallest scale of a block that is not all zeros: its reciprocal and
// weights of 2^15 times it stay in float32's range.
#define Q8C_FLOOR 0x1p-96f

// A block's scales; bit e of kbad (vbad): entry e has a key (value) that is not
// finite (stored as zero; what sees it gets NaN).
struct __align__(16) Q8Meta {
    float ks, vs;
    uint32_t kbad, vbad;
};

__host__ __device__ __forceinline__ int q8c_dp(int d) { return (d + 63) & ~63; }
__host__ __device__ __forceinline__ int64_t q8c_blocks(int64_t context) { return (context + Q8C_BLOCK - 1) / Q8C_BLOCK; }
// Byte offset of block b of kv head hk, and of its scales.
__host__ __device__ __forceinline__ int64_t q8c_record(int64_t nb, int hk, int64_t b, int dp) {
    return ((int64_t)hk * nb + b) * (2 * Q8C_BLOCK) * dp;
}
__host__ __device__ __forceinline__ int64_t q8c_meta(int64_t nb, int Hkv, int hk, int64_t b, int dp) {
    return (int64_t)Hkv * nb * (2 * Q8C_BLOCK) * dp + ((int64_t)hk * nb + b) * (int64_t)sizeof(Q8Meta);
}
__host__ __device__ __forceinline__ int64_t q8c_bytes(int Hkv, int64_t context, int dp) {
    return (int64_t)Hkv * q8c_blocks(context) * (2 * Q8C_BLOCK * dp + (int64_t)sizeof(Q8Meta));
}
// Byte of dim d of entry e (0..31) inside a record's keys, and its values.
__host__ __device__ __forceinline__ int q8c_kbyte(int e, int d, int dp) {
    return ((((e >> 4) * (dp >> 6) + (d >> 6)) << 6) + (((d >> 4) & 3) << 4) + (e & 15)) * 16 + (d & 15);
}
__host__ __device__ __forceinline__ int q8c_vbyte(int e, int d) {
    return (((d >> 5) << 6) + (((e >> 2) & 3) << 4) + (d & 15)) * 16 + ((d >> 4) & 1) * 8 + ((e >> 4) << 2) + (e & 3);
}

}  // namespace mimg
