// Writing and reading the 8-bit key/value cache (layout: kv8.h).
//
// Each 64-token block of a head is held as 8-bit codes times one power of two: scale = 2^k with the smallest k for
// which the block's largest magnitude fits the code's range (448 for e4m3, 127 for int8), code = round to nearest
// even of x * 2^-k.  Power-of-two scales make x * 2^-k exact (the only rounding is the one to the code), make every
// stored value exact in bf16, and let the attention kernel fold a scale into an exponent.  They cost e4m3 nothing
// (its steps are relative) and int8 at most one of its eight bits.
//
// Masked tokens are stored as zeros and do not enter the scale, so padding cannot coarsen its block; infinities
// saturate and do not enter the scale either; a NaN stays a NaN in e4m3 and becomes 0 in int8, which has none.  In a block of
// nearly the largest bf16 values the largest codes would stand for 2^128: they become the next lower ones, so that every held
// value of a finite or infinite input is finite.
#include "kv8.h"

namespace {

constexpr int THREADS = 256;

// exponent k of a block's scale
template <int TYPE>
__device__ __forceinline__ int scale_exponent(float amax) {
    if (amax == 0.f) return 0;
    const unsigned u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127;
    const unsigned frac = u & 0x7FFFFFu;
    // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
    const int k = TYPE == LLADA_KV_E4M3 ? e - 8 + (frac > 0x600000u) : e - 6 + (frac > 0x7E0000u);
    return k < -126 ? -126 : k;          // keeps the scale and its inverse normal numbers
}

// the largest exponent whose every code stands for a finite bf16 value (448 * 2^119, 127 * 2^121); at the one above it, codes
// end at 240 and 63
template <int TYPE>
constexpr int TOP_EXPONENT = TYPE == LLADA_KV_E4M3 ? 119 : 121;
template <int TYPE>
__device__ __forceinline__ float code_limit(int k) {
    return TYPE == LLADA_KV_E4M3 ? (k > TOP_EXPONENT<TYPE> ? 240.f : 448.f) : (k > TOP_EXPONENT<TYPE> ? 63.f : 127.f);
}

__device__ __forceinline__ float power_of_two(int k) { return __uint_as_float((unsigned)(k + 127) << 23); }

// Four values -> four codes of magnitude up to `limit`.  RAW: the block holds finite values alone and its scale is not the
// topmost (then |x inv| is within the code's range by the choice of the scale).
template <int TYPE, bool RAW>
__device__ __forceinline__ unsigned encode4(float a, float b, float c, float d, float inv, float limit) {
    float x[4] = {a, b, c, d};
    if constexpr (TYPE == LLADA_KV_E4M3) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] *= inv;
            if (!RAW) x[i] = x[i] != x[i] ? x[i] : __builtin_amdgcn_fmed3f(x[i], -limit, limit);
        }
        int r = 0;
        r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], r, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], r, true);
        return (unsigned)r;
    } else {
        // 1.5 * 2^23 + y: the sum's last bit stands for 1, so the addition rounds y to the nearest integer, ties to even,
        // and leaves it in two's complement in the low byte (x inv is exact: one rounding)
        unsigned u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!RAW) x[i] = x[i] != x[i] ? 0.f : __builtin_amdgcn_fmed3f(x[i] * inv, -limit, limit);
            u[i] = __float_as_uint(RAW ? __builtin_fmaf(x[i], inv, 12582912.f) : x[i] + 12582912.f);
        }
        const unsigned lo = __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x0C0C0400u);
        return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
}

template <int TYPE>
__device__ __forceinline__ float decode(unsigned word, int byte) {
    if constexpr (TYPE == LLADA_KV_E4M3) {
        switch (byte) {
            case 0: return __builtin_amdgcn_cvt_f32_fp8((int)word, 0);
            case 1: return __builtin_amdgcn_cvt_f32_fp8((int)word, 1);
            case 2: return __builtin_amdgcn_cvt_f32_fp8((int)word, 2);
            default: return __builtin_amdgcn_cvt_f32_fp8((int)word, 3);
        }
    } else {
        return (float)(signed char)(word >> (8 * byte));
    }
}

// entry e (0 .. 7) of four words of bf16 pairs
__device__ __forceinline__ float entry(u32x4 w, int e) { return __uint_as_float((e & 1) ? (w[e >> 1] & 0xFFFF0000u) : (w[e >> 1] << 16)); }

typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
__device__ __forceinline__ u16x2 halves(unsigned w) { return __builtin_bit_cast(u16x2, w); }

// x: four keys x 8 dims of the keys and of the values; their codes into the tile's LDS image.
template <int TYPE, bool RAW>
__device__ __forceinline__ void encode_tile(const u32x4 (&x)[2][4], const int (&k)[2], unsigned char* codes, int kg, int dg) {
    const float ik = power_of_two(-k[0]), iv = power_of_two(-k[1]), lk = code_limit<TYPE>(k[0]), lv = code_limit<TYPE>(k[1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u32x2 w;
        w[0] = encode4<TYPE, RAW>(entry(x[0][i], 0), entry(x[0][i], 1), entry(x[0][i], 2), entry(x[0][i], 3), ik, lk);
        w[1] = encode4<TYPE, RAW>(entry(x[0][i], 4), entry(x[0][i], 5), entry(x[0][i], 6), entry(x[0][i], 7), ik, lk);
        *(u32x2*)(codes + kv8_key_offset(kg * 4 + i, dg * 8)) = w;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        *(unsigned*)(codes + KV8_CODES + kv8_value_offset(kg * 4, dg * 8 + e)) =
            encode4<TYPE, RAW>(entry(x[1][0], e), entry(x[1][1], e), entry(x[1][2], e), entry(x[1][3], e), iv, lv);
}

// One workgroup = one (sequence, head, block): thread (kg, dg) holds keys 4 kg .. + 3 and dims 8 dg .. + 7 of the keys
// and of the values, as bf16 pairs (what a cache holds is exact in bf16).  Bound by memory, 4 bytes in and 2 out per
// channel, once the arithmetic is out of its way: the largest magnitude is taken on packed 16-bit patterns (2
// instructions for two elements), and a block without infinities, NaNs and values at the top of bf16, known from that
// maximum, needs no clamp: under three instructions an element.  The codes cross the LDS once to leave as whole 1-KiB runs.
// Measured, 32 heads: 16 x 4096 tokens 253 us e4m3 (1.61 GB: 6.4 TB/s; a copy on this card moves 4.9, which reads as much
// as it writes), 8 x 1150 int8 45 us (0.23 GB; 54 with the clamp and float maxima), 1 x 384 5 us (launch and one round trip).
template <int TYPE>
__global__ void __launch_bounds__(THREADS) kv8_write_kernel(const bf16_t* __restrict__ rows, int64_t row_stride,
                                                            const uint8_t* __restrict__ key_mask, float* __restrict__ scales,
                                                            unsigned char* __restrict__ tiles, int seq_len, int n_heads,
                                                            int n_blocks, int start, int len, int first_block,
                                                            int touched) {
    __shared__ __attribute__((aligned(16))) unsigned char codes[KV8_TILE];
    __shared__ unsigned red[2][THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int kg = tid >> 4, dg = tid & 15;
    unsigned item = blockIdx.x;
    const int h = (int)(item % (unsigned)n_heads);
    item /= (unsigned)n_heads;
    const int t = first_block + (int)(item % (unsigned)touched);
    const int b = (int)(item / (unsigned)touched);
    const int64_t tile = ((int64_t)b * n_heads + h) * n_blocks + t;
    unsigned char* const dst = tiles + (size_t)tile * KV8_TILE;
    float* const sc = scales + tile * 2;
    const int d = n_heads * KV8_HD;
    const int key0 = t * KV8_TOKENS + kg * 4;
    const int t_end = min(seq_len, (t + 1) * KV8_TOKENS);
    const bool partial = start > t * KV8_TOKENS || start + len < t_end;      // (uniform)

    // every load first: rows clamped into the range, what does not count is replaced below
    u32x4 x[2][4];
    uint8_t m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = min(max(key0 + i - start, 0), len - 1);
        const bf16_t* p = rows + ((size_t)b * len + row) * row_stride + d + h * KV8_HD + dg * 8;
        x[0][i] = __builtin_nontemporal_load((const u32x4*)p);
        x[1][i] = __builtin_nontemporal_load((const u32x4*)(p + d));
        m[i] = key_mask ? key_mask[(size_t)b * seq_len + min(key0 + i, seq_len - 1)] : (uint8_t)1;
    }
    if (partial) {       // the block's other tokens as the cache holds them
        const float sk = sc[0], sv = sc[1];
        u32x2 kw[4];
        unsigned vw[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) kw[i] = *(const u32x2*)(dst + kv8_key_offset(kg * 4 + i, dg * 8));
#pragma unroll
        for (int e = 0; e < 8; ++e) vw[e] = *(const unsigned*)(dst + KV8_CODES + kv8_value_offset(kg * 4, dg * 8 + e));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = key0 + i;
            if (key >= start && key < start + len) continue;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                x[0][i][w] = pack_bf16x2(decode<TYPE>(kw[i][w >> 1], (2 * w) & 3) * sk, decode<TYPE>(kw[i][w >> 1], (2 * w + 1) & 3) * sk);
                x[1][i][w] = pack_bf16x2(decode<TYPE>(vw[2 * w], i) * sv, decode<TYPE>(vw[2 * w + 1], i) * sv);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (key0 + i >= seq_len || m[i] == 0) x[0][i] = x[1][i] = (u32x4){0u, 0u, 0u, 0u};

    // largest magnitude of the block: of all patterns first, of the finite ones where that is not finite
    auto largest = [&](bool finite_only, int o) {
        u16x2 most = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                u16x2 a = halves(x[o][i][w] & 0x7FFF7FFFu);
                if (finite_only) a = (u16x2){a[0] < 0x7F80 ? a[0] : (unsigned short)0, a[1] < 0x7F80 ? a[1] : (unsigned short)0};
                most = __builtin_elementwise_max(most, a);
            }
        unsigned v = most[0] > most[1] ? most[0] : most[1];
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) {
            const unsigned u = (unsigned)__shfl_xor((int)v, s);
            v = v > u ? v : u;
        }
        return v;
    };
    auto block_largest = [&](bool finite_only, unsigned (&out)[2]) {
        const unsigned a = largest(finite_only, 0), c = largest(finite_only, 1);
        if (lane == 0) {
            red[0][wave] = a;
            red[1][wave] = c;
        }
        __syncthreads();                 // also: every old code of this tile has been read
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            out[o] = red[o][0];
#pragma unroll
            for (int w = 1; w < THREADS / 64; ++w) out[o] = out[o] > red[o][w] ? out[o] : red[o][w];
        }
    };
    unsigned most[2];
    block_largest(false, most);
    const bool raw = most[0] < 0x7F80u && most[1] < 0x7F80u;      // (uniform)
    if (!raw) {
        __syncthreads();
        block_largest(true, most);
    }
    const int k[2] = {scale_exponent<TYPE>(__uint_as_float(most[0] << 16)), scale_exponent<TYPE>(__uint_as_float(most[1] << 16))};
    if (raw && k[0] <= TOP_EXPONENT<TYPE> && k[1] <= TOP_EXPONENT<TYPE>)
        encode_tile<TYPE, true>(x, k, codes, kg, dg);
    else
        encode_tile<TYPE, false>(x, k, codes, kg, dg);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KV8_TILE / (16 * THREADS); ++i) {
        const int at = (i * THREADS + tid) * 16;
        *(u32x4*)(dst + at) = *(const u32x4*)(codes + at);
    }
    if (tid < 2) sc[tid] = power_of_two(k[tid]);
}

// The values a layer of the cache stands for, as bf16 rows (exact: at most seven significant bits times a power of two).
// Bound by the rows it writes, 16 bytes a lane: 16 x 4096 tokens of 32 heads 350 us (1.61 GB: 4.6 TB/s), 8 x 1150 int8 32.5 us.
template <int TYPE>
__global__ void __launch_bounds__(THREADS) kv8_read_kernel(const float* __restrict__ scales,
                                                           const unsigned char* __restrict__ tiles, bf16_t* __restrict__ k_out,
                                                           bf16_t* __restrict__ v_out, int seq_len, int n_heads, int n_blocks) {
    __shared__ __attribute__((aligned(16))) unsigned char codes[KV8_TILE];
    const int tid = threadIdx.x, kg = tid >> 4, dg = tid & 15;
    unsigned item = blockIdx.x;
    const int h = (int)(item % (unsigned)n_heads);
    item /= (unsigned)n_heads;
    const int t = (int)(item % (unsigned)n_blocks);
    const int b = (int)(item / (unsigned)n_blocks);
    const int64_t tile = ((int64_t)b * n_heads + h) * n_blocks + t;
    const unsigned char* const src = tiles + (size_t)tile * KV8_TILE;
    const float sk = scales[tile * 2], sv = scales[tile * 2 + 1];
#pragma unroll
    for (int i = 0; i < KV8_TILE / (16 * THREADS); ++i) {
        const int at = (i * THREADS + tid) * 16;
        *(u32x4*)(codes + at) = *(const u32x4*)(src + at);
    }
    __syncthreads();
    unsigned vw[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) vw[e] = *(const unsigned*)(codes + KV8_CODES + kv8_value_offset(kg * 4, dg * 8 + e));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int key = t * KV8_TOKENS + kg * 4 + i;
        if (key >= seq_len) continue;
        const u32x2 kw = *(const u32x2*)(codes + kv8_key_offset(kg * 4 + i, dg * 8));
        u32x4 a, c;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            a[w] = pack_bf16x2(decode<TYPE>(kw[w >> 1], (2 * w) & 3) * sk, decode<TYPE>(kw[w >> 1], (2 * w + 1) & 3) * sk);
            c[w] = pack_bf16x2(decode<TYPE>(vw[2 * w], i) * sv, decode<TYPE>(vw[2 * w + 1], i) * sv);
        }
        const size_t at = ((size_t)b * seq_len + key) * ((size_t)n_heads * KV8_HD) + (size_t)h * KV8_HD + dg * 8;
        __builtin_nontemporal_store(a, (u32x4*)(k_out + at));
        __builtin_nontemporal_store(c, (u32x4*)(v_out + at));
    }
}

}  // namespace

extern "C" size_t llada_kv8_layer_bytes(int32_t n_seq, int32_t seq_len, int32_t n_heads) {
    if (n_seq <= 0 || seq_len <= 0 || n_heads <= 0) return 0;
    const int64_t n_tiles = (int64_t)n_seq * n_heads * kv8_blocks(seq_len);
    return kv8_scale_bytes(n_tiles) + (size_t)n_tiles * KV8_TILE;
}

extern "C" int llada_kv8_write(const void* qkv, int64_t row_stride, const uint8_t* key_mask, void* cache, int32_t kv_type,
                               int32_t n_seq, int32_t seq_len, int32_t n_heads, int32_t start, int32_t len, void* stream) {
    LLADA_CHECK_ARG(qkv && cache, "kv8_write: null argument");
    LLADA_CHECK_ARG(n_seq > 0 && seq_len > 0 && n_heads > 0, "kv8_write: bad shape");
    LLADA_CHECK_ARG(start >= 0 && len > 0 && (int64_t)start + len <= seq_len, "kv8_write: rows %d .. %lld of %d", start,
                    (long long)start + len, seq_len);
    LLADA_CHECK_ARG(row_stride >= (int64_t)3 * n_heads * KV8_HD && row_stride % 8 == 0 && ((uintptr_t)qkv & 15) == 0,
                    "kv8_write: rows hold [Q | K | V] and start at 16-byte boundaries");
    LLADA_CHECK_ARG(((uintptr_t)cache & 255) == 0, "kv8_write: cache must be 256-byte aligned");
    LLADA_CHECK_SUPPORTED(kv_type == LLADA_KV_E4M3 || kv_type == LLADA_KV_INT8, "kv8_write: unknown cache type %d", kv_type);
    const int64_t n_blocks = kv8_blocks(seq_len);
    const int64_t n_tiles = (int64_t)n_seq * n_heads * n_blocks;
    const int first = start / KV8_TOKENS, touched = (start + len - 1) / KV8_TOKENS - first + 1;
    const int64_t grid = (int64_t)n_seq * n_heads * touched;
    LLADA_CHECK_SUPPORTED(grid * THREADS < (1LL << 32), "kv8_write: grid too large (a launch ends at 2^32 threads)");
    float* scales = (float*)cache;
    unsigned char* tiles = (unsigned char*)cache + kv8_scale_bytes(n_tiles);
    auto kernel = kv_type == LLADA_KV_E4M3 ? kv8_write_kernel<LLADA_KV_E4M3> : kv8_write_kernel<LLADA_KV_INT8>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(THREADS), 0, (hipStream_t)stream, (const bf16_t*)qkv, row_stride,
                       key_mask, scales, tiles, seq_len, n_heads, (int)n_blocks, start, len, first, touched);
    LLADA_CHECK_LAUNCH("kv8_write_kernel");
    return LLADA_OK;
}

extern "C" int llada_kv8_read(const void* cache, int32_t kv_type, void* k_out, void* v_out, int32_t n_seq, int32_t seq_len,
                              int32_t n_heads, void* stream) {
    LLADA_CHECK_ARG(cache && k_out && v_out, "kv8_read: null argument");
    LLADA_CHECK_ARG(n_seq > 0 && seq_len > 0 && n_heads > 0, "kv8_read: bad shape");
    LLADA_CHECK_ARG(((uintptr_t)cache & 255) == 0 && (((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0,
                    "kv8_read: cache must be 256-byte, outputs 16-byte aligned");
    LLADA_CHECK_SUPPORTED(kv_type == LLADA_KV_E4M3 || kv_type == LLADA_KV_INT8, "kv8_read: unknown cache type %d", kv_type);
    const int64_t n_blocks = kv8_blocks(seq_len);
    const int64_t n_tiles = (int64_t)n_seq * n_heads * n_blocks;
    LLADA_CHECK_SUPPORTED(n_tiles * THREADS < (1LL << 32), "kv8_read: grid too large (a launch ends at 2^32 threads)");
    const float* scales = (const float*)cache;
    const unsigned char* tiles = (const unsigned char*)cache + kv8_scale_bytes(n_tiles);
    auto kernel = kv_type == LLADA_KV_E4M3 ? kv8_read_kernel<LLADA_KV_E4M3> : kv8_read_kernel<LLADA_KV_INT8>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_tiles), dim3(THREADS), 0, (hipStream_t)stream, scales, tiles, (bf16_t*)k_out,
                       (bf16_t*)v_out, seq_len, n_heads, (int)n_blocks);
    LLADA_CHECK_LAUNCH("kv8_read_kernel");
    return LLADA_OK;
}
