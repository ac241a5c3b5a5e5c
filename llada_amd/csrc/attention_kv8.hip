// Bidirectional attention over the 8-bit key/value cache (layout: kv8.h), head_dim 128, bf16 queries and output.
//
//   out[q] = sum_k p_qk v_k / sum_k p_qk,   p_qk = exp(q . k / sqrt(128) - m_q)
//
// over the sequence's unmasked tokens; the tokens of [blk_start, blk_start + blk_len) come from fresh bf16 rows instead
// of the cache (a block-cached denoise step recomputes them).  A query whose sequence has no unmasked token gets zeros.
//
// A wave holds 32 queries and sweeps 64-key tiles: S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16_bf16, a query's
// scores in one lane pair.  Few queries meet each key here, so the sweep is bound by memory and then by the vector pipe,
// not by the matrix pipe, and the cache's tile order is chosen for that: a wave loads the codes of a tile with sixteen
// contiguous 1-KiB loads straight into operand registers, the next tile's keys while this tile's softmax and values are
// worked on and the next tile's values during the next scores; there is no LDS staging and no barrier in the loop.
// Codes become bf16 exactly (e4m3: one conversion for two codes; int8: three instructions for two); a tile's
// key scale goes into the multiplier of the scores, its value scale, a power of two 2^e, into the exponent of the
// probabilities (p 2^e = 2^(s - m + e)), so neither costs an instruction per element.  Their sum is taken back by 2^-e: it would
// lose the keys whose p 2^e the exponential flushes (below 2^-126), so no more than 2^-64 or 2^64 goes in before the sum: the
// outputs have a unit, a power of two, and e counts from there.  Larger scales raise the unit (outputs stay finite up to the
// largest bf16 values), smaller ones go into the probabilities in bf16, after the sum (what flushes there is below 2^-117 of a
// unit); a wave that has summed nothing takes a tiny tile's scale for its unit.
// (Fresh rows carry no scale; like the bf16 attention's, sums over them are finite for values up to 2^96.)
//
// Measured, 32 heads, us a call among others (the kernel traced alone, with the profiler's gaps, takes 1 to 8 % more): 32
// queries on 32 x 4096 tokens 186 (1.08 GB: 5.8 TB/s, the memory's rate), on 8 x 384 9.3 and on 1 x 384 9.2 (kernels 9.7
// and 8.0, latency: a few tiles a wave), 64 on 8 x 1150 int8 24 (one workgroup a CU: the wave's own chain of load, convert,
// scores, exponentials, values), 1 on 5 x 2049 int8 19.7 (likewise), 321 on 8 x 769 55 (0.59 PFLOP/s: the chain again, two
// waves a SIMD, each loading and converting every tile for itself, 1.5 rounds of workgroups), 256 on 16 x 2176 181 in a
// graph (0.81 PFLOP/s).  Keeping extreme value scales and scores right costs all others up to 2 % (8 x 512, 128 queries: 4 %).
// Tried and dropped: workgroups of 8 waves (level or slower, but for 64 queries on 8 x 1150: 25.0 us against
// the 27.5 of that time), a fresh tile in halves of 32 keys with one half's exponentials under the other's products
// (level; on cached tiles its registers spill), raised wave priority around the products (level), fresh tiles last (a
// seventh slower), the next values fetched before the next keys are waited for (256 queries on 16 x 2176 166 / 161 us,
// but 32 on 8 x 384 7.8 / 8.3 and 32 on 1 x 4096 21.8 / 23.4).
//
// Scores, running maximum, sums and outputs are float32; P is rounded to bf16 once for the matrix unit, like the keys' and
// values' bf16 forms it multiplies (at most 2^-8 of a term, averaged over the terms).
#include "kv8.h"

namespace {

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;
typedef __attribute__((address_space(3))) void* lds_void_ptr;
typedef const __attribute__((address_space(1))) void* gbl_void_ptr;

constexpr int QW = 32;                       // queries of a wave
constexpr int NW = 4;                        // waves of a workgroup
constexpr int OROW = KV8_HD * 4 + 16;        // bytes of a float32 output row in LDS (16 bytes of padding)
constexpr int SLICE = QW * OROW;             // one wave's result in LDS

template <int TYPE>
__device__ __forceinline__ bf16x8 codes_to_bf16(unsigned a, unsigned b) {
    bf16x8 r;
    if constexpr (TYPE == LLADA_KV_E4M3) {
        const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
        const bf16x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
        const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
        const bf16x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
        r = (bf16x8){x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
    } else {
        // (opaque to the optimiser, which would otherwise carry a prefetched tile around the loop as 256 converted
        // floats instead of 32 words of codes, in scratch memory)
        asm("" : "+v"(a), "+v"(b));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            r[i] = (__bf16)(float)(signed char)(a >> (8 * i));
            r[4 + i] = (__bf16)(float)(signed char)(b >> (8 * i));
        }
    }
    return r;
}

struct Kv8Attn {
    const bf16_t* q;
    int64_t q_stride;
    const float* scales;
    const unsigned char* tiles;
    const uint8_t* key_mask;
    bf16_t* out;
    const bf16_t* blk;        // fresh [Q | K | V] rows, or null
    int64_t blk_stride;
    float* part_o;            // key splits: [split][row][d] float32, unnormalised
    float* part_ml;           // [split][row][head][2]: running maximum (log2 domain), sum
    int64_t n_rows;
    int n_q, seq_len, n_heads, n_blocks, n_qblocks;
    int blk_start, blk_len;
    int skip_from, skipped;   // cached tiles [skip_from, skip_from + skipped) lie inside the fresh block
    int n_cached, n_units;    // tiles to sweep: cached ones, then fresh ones
    int splits, per_split;
    float scale_log2e;
};

// A wave's state over the tiles it has swept.
struct Softmax {
    f32x16 o[4];              // in units of 2^unit
    float m, l;
    int unit;
    bool far;                 // some query's maximum is past FAR
};

// A fused s sc - m leaves up to half a step of m in the exponent, the same for all keys: harmless until that nears the
// exponent's range, for maxima of 2^30.  Past FAR the product is rounded before the difference, as it was for m: nothing is left.
constexpr float FAR = 16777216.f;

// The most of a tile's value scale that goes into the exponent of its probabilities: these then stay normal numbers
// down to 2^-62 of the largest, and finite.
constexpr int FOLD = 64;

// One tile's scores -> probabilities, the running maximum and sum brought up to date.  s: raw scores (lane: query
// lane & 31; register 4 c + e of s[kb]: key 32 kb + 8 c + 4 (lane >> 5) + e); valid: bit per key; sc: multiplier into the
// log2 domain; ve: exponent put into the probabilities (at most FOLD either way, so that the sum misses no key that counts),
// inv_vs: 2^-ve; over: the outputs' unit has risen by 2^over; under: what the probabilities take besides ve, after their sum.
__device__ __forceinline__ void softmax_tile(f32x16 (&s)[2], uint64_t valid, float sc, float ve, float inv_vs, int over, int under, Softmax& w,
                                             bf16x8 (&pb)[2][2], int hg) {
    if (valid != ~0ull) {
        const uint64_t mine = valid >> (4 * hg);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!((mine >> (kb * 32 + 8 * (i >> 2) + (i & 3))) & 1)) s[kb][i] = -INFINITY;   // selected, not added: a masked NaN is gone
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32)) * sc;
    // the reference maximum moves only when it has risen by more than 2^8: the 64 multiplies of the
    // accumulators are then rare, and probabilities up to 2^8 are as exact as those below 1
    const float m_cand = fmaxf(w.m, mx);
    if ((__builtin_amdgcn_ballot_w64(m_cand > w.m + 8.0f) | (unsigned)over) != 0) {
        float alpha = __builtin_amdgcn_exp2f(w.m - (m_cand == -INFINITY ? 0.f : m_cand));
        w.m = m_cand;
        w.far = __builtin_amdgcn_ballot_w64(fabsf(m_cand) > FAR && m_cand != -INFINITY) != 0;
        w.l *= alpha;
        alpha = __builtin_ldexpf(alpha, -over);
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) w.o[db][e] *= alpha;
    }
    if (__builtin_expect(w.far, 0)) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kb][e] *= sc;
        sc = 1.f;
    }
    const float off = ve - (w.m == -INFINITY ? 0.f : w.m);
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e], sc, off));
            sum += p;
            pb[kb][e >> 3][e & 7] = (__bf16)p;
        }
    w.l = __builtin_fmaf(sum, inv_vs, w.l);
    if (under != 0) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) pb[kb][e >> 3][e & 7] = (__bf16)__builtin_ldexpf((float)pb[kb][e >> 3][e & 7], under);
    }
}

// NQ query groups of 32 and 4 / NQ key groups per workgroup: few queries -> the waves share the queries and deal the
// tiles among themselves, their results merged once at the end; many -> each wave has queries of its own and the waves
// meet a tile's codes in the CU's cache.
template <int TYPE, int NQ>
__global__ void __launch_bounds__(NW * 64, 2) attn_kv8_kernel(const Kv8Attn a) {
    constexpr int NK = NW / NQ;
    __shared__ __attribute__((aligned(16))) unsigned char lds[NW * SLICE + NW * QW * 8];
    float* const ml = (float*)(lds + NW * SLICE);           // [wave][query][2]

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, hg = lane >> 5;
    const int qg = wave % NQ, kg = wave / NQ;
    // consecutive workgroups go to the 8 XCDs in turn: the query blocks of one head, which read the same
    // tiles, are made consecutive items of one XCD and meet in its L2
    int qb, h, b, ks;
    {
        const int nt = gridDim.x, bid = blockIdx.x;
        const int xcd = bid & 7, per = nt >> 3, rem = nt & 7;
        int item = (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + (bid >> 3);
        qb = ks = 0;
        if (a.n_qblocks > 1) {
            qb = item % a.n_qblocks;
            item /= a.n_qblocks;
        }
        if (a.splits > 1) {
            ks = item % a.splits;
            item /= a.splits;
        }
        h = item % a.n_heads;
        b = item / a.n_heads;
    }
    const int d = a.n_heads * KV8_HD;
    const int q0 = (qb * NQ + qg) * QW;
    const int64_t tile0 = ((int64_t)b * a.n_heads + h) * a.n_blocks;
    const unsigned char* const tiles = a.tiles + (size_t)tile0 * KV8_TILE + lane * 16;
    const float* const scales = a.scales + tile0 * 2;
    const uint8_t* const mask = a.key_mask ? a.key_mask + (size_t)b * a.seq_len : nullptr;
    const int blk_end = a.blk_start + a.blk_len;

    // lane holds Q[q0 + r][64 hg + 8 i .. + 7]: the contraction runs over the dims in the order of the key codes
    bf16x8 qf[8];
    {
        const int q = min(q0 + r, a.n_q - 1);
        const bf16_t* qp = a.q + ((size_t)b * a.n_q + q) * (size_t)a.q_stride + h * KV8_HD + hg * 64;
#pragma unroll
        for (int i = 0; i < 8; ++i) qf[i] = *(const bf16x8*)(qp + i * 8);
    }
    Softmax w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) w.o[i][e] = 0.f;
    w.m = -INFINITY;
    w.l = 0.f;
    w.unit = 0;
    w.far = false;

    // units of this workgroup: [u_begin, u_end) of the fresh tiles, then the cached ones; unit u_begin + i is key group i % NK's
    const int n_fresh = a.n_units - a.n_cached;
    const int u_begin = ks * a.per_split, u_end = min(a.n_units, u_begin + a.per_split);
    const int c_begin = max(u_begin, n_fresh);
    const bool idle = q0 >= a.n_q;                                      // (a wave behind the last query only helps to fetch)
    int u = idle ? u_end : c_begin + ((kg - (c_begin - u_begin)) & (NK - 1));           // this wave's first cached one

    // The first cached tile's keys are fetched ahead of everything else.
    auto tile_of = [&](int i) { i -= n_fresh; return i < a.skip_from ? i : i + a.skipped; };
    u32x4 kc[8], vc[8];
    auto load_keys = [&](int t) {
#pragma unroll
        for (int i = 0; i < 8; ++i) kc[i] = *(const u32x4*)(tiles + (size_t)t * KV8_TILE + i * 1024);
    };
    auto load_values = [&](int t) {
#pragma unroll
        for (int i = 0; i < 8; ++i) vc[i] = *(const u32x4*)(tiles + (size_t)t * KV8_TILE + KV8_CODES + i * 1024);
    };
    // which keys of tile t this kernel takes from the cache
    auto live_keys = [&](int t, uint8_t m) {
        const int key = t * KV8_TOKENS + lane;
        return __builtin_amdgcn_ballot_w64(key < a.seq_len && m != 0 && !(key >= a.blk_start && key < blk_end));
    };
    auto mask_byte = [&](int t) -> uint8_t { return mask ? mask[min(t * KV8_TOKENS + lane, a.seq_len - 1)] : (uint8_t)1; };

    int t = 0;
    uint8_t mb = 0;
    float ks_next = 1.f, vs_next = 1.f;
    if (u < u_end) {
        t = tile_of(u);
        if constexpr (NK > 1) load_keys(t);
        mb = mask_byte(t);
        ks_next = scales[2 * t];
        vs_next = scales[2 * t + 1];
    }

    // Fresh tiles are bf16 rows, and rows of values have to be read transposed: they cross the LDS, which the cached tiles leave
    // idle.  They come first, while the first cached tile is on its way.  All waves bring them in by LDS-DMA, keys and values
    // of two tiles at a time (one key group: the next tile under the work on this one; several: a round of two, a tile for
    // each of two groups).
    // 16-byte chunk c of key row k stands at c ^ (k & 15), 64-byte slot s of value row k at s ^ (k & 3): applied to the
    // source address, so that no read meets a bank twice.
    constexpr int FRESH = 2 * KV8_TOKENS * 256;                         // bytes of a tile
    constexpr int AHEAD = NK == 1 ? 1 : 2;                              // tiles of a round
    static_assert(2 * FRESH <= NW * SLICE, "two tiles fit the slices");
    auto fetch_fresh = [&](int f, int buf) {
        const bf16_t* const rows = a.blk + (size_t)b * a.blk_len * (size_t)a.blk_stride + h * KV8_HD + d;
        const int f0 = f * KV8_TOKENS, row0 = lane >> 4, at = lane & 15;
#pragma unroll
        for (int i = 0; i < 32 / NW; ++i) {
            const int piece = wave + i * NW, is_v = piece >> 4;         // 0 .. 15: four key rows each, 16 .. 31: value rows
            const int row = (piece & 15) * 4 + row0;
            const int chunk = is_v ? ((((at >> 2) ^ (row & 3)) << 2) | (at & 3)) : (at ^ (row & 15));
            const bf16_t* src = rows + (is_v ? d : 0) + (size_t)min(f0 + row, a.blk_len - 1) * (size_t)a.blk_stride + chunk * 8;
            __builtin_amdgcn_global_load_lds((gbl_void_ptr)src, (lds_void_ptr)(lds + buf * FRESH + piece * 1024), 16, 0, 0);
        }
    };
    const int f_end = min(u_end, n_fresh);
    int f_next = u_begin;                                               // first fresh tile of the next round
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (f_next + i < f_end) fetch_fresh(f_next + i, i);
    for (int buf = 0; f_next < f_end; f_next += AHEAD) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                // this wave's pieces have landed
        __syncthreads();                                                // everyone's
        const int f = NK == 1 ? f_next : f_next + ((kg + u_begin - f_next) & (NK - 1));     // this wave's tile of the two
        const int f0 = f * KV8_TOKENS;
        if (NK == 1 && f + 1 < f_end) fetch_fresh(f + 1, buf ^ 1);      // (the buffer of the last round is no longer read)
        if (!idle && f < min(f_next + AHEAD, f_end)) {
            unsigned char* const k_lds = lds + (NK == 1 ? buf : f - f_next) * FRESH;
            unsigned char* const v_lds = k_lds + KV8_TOKENS * 256;
            const int fk = f0 + lane;
            const uint64_t there = a.blk_len - f0 >= 64 ? ~0ull : (1ull << (a.blk_len - f0)) - 1;
            const uint64_t unmasked = __builtin_amdgcn_ballot_w64(mask == nullptr || fk >= a.blk_len || mask[min(a.blk_start + fk, a.seq_len - 1)] != 0);
            if ((unmasked & there) != there) {                          // what stands under a masked token, and the copies of
                                                                        // the last row behind the block: zeros
                // (waves of several query groups write the same zeros to a tile of theirs, each before its own reads)
#pragma unroll
                for (int i = 0; i < KV8_TOKENS / 4; ++i)
                    if (!(((unmasked & there) >> (i * 4 + (lane >> 4))) & 1)) *(u32x4*)(v_lds + i * 1024 + lane * 16) = (u32x4){0u, 0u, 0u, 0u};
            }
            // One key group: reads go out four products ahead (left to itself, the compiler saves registers and waits out each
            // read alone); several: their registers hold the first cached tile's keys.
            auto hold = [] { if constexpr (NK == 1) __builtin_amdgcn_sched_barrier(0); };
            f32x16 s[2];
            bf16x8 kf[2][4];
            auto read_keys = [&](int g) {                               // of products 4 g .. + 3: keys 32 (g >> 1) .., dims 32 (g & 1) .. of each half
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    kf[g & 1][i] = *(const bf16x8*)(k_lds + ((g >> 1) * 32 + r) * 256 + (((8 * hg + 4 * (g & 1) + i) ^ (r & 15)) * 16));
            };
            read_keys(0);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (g < 3) read_keys(g + 1);
                hold();
                if ((g & 1) == 0) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[g >> 1][e] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[g >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[g & 1][i], qf[4 * (g & 1) + i], s[g >> 1], 0, 0, 0);
                hold();
            }
            bf16x8 pb[2][2];
            softmax_tile(s, unmasked & there, a.scale_log2e, 0.f, 1.f, 0, 0, w, pb, hg);
            const int q4 = (lane & 15) >> 2, p4 = lane & 3, g1 = (lane >> 4) & 1;
            const unsigned char* const vrow = v_lds + (4 * hg + q4) * 256 + 32 * g1 + 8 * p4;
            s16x4 vf[2][4][2];
            auto read_values = [&](int g) {                             // of keys 16 g .. + 15
#pragma unroll
                for (int db = 0; db < 4; ++db) {
                    const unsigned char* p = vrow + g * 16 * 256 + ((db * 64) ^ (q4 * 64));
                    vf[g & 1][db][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p);
                    vf[g & 1][db][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p + 8 * 256));
                }
            };
            read_values(0);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (g < 3) read_values(g + 1);
                hold();
#pragma unroll
                for (int db = 0; db < 4; ++db) {
                    const s16x8 v = __builtin_shufflevector(vf[g & 1][db][0], vf[g & 1][db][1], 0, 1, 2, 3, 4, 5, 6, 7);
                    w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), pb[g >> 1][g & 1], w.o[db], 0, 0, 0);
                }
                hold();
            }
        }
        if constexpr (NK == 1) {
            buf ^= 1;
        } else if (f_next + AHEAD < f_end) {
            __syncthreads();                                            // both tiles have been read
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (f_next + AHEAD + i < f_end) fetch_fresh(f_next + AHEAD + i, i);
        }
    }
    // ---- cached tiles ----
    if (u < u_end) {
        if constexpr (NK == 1) load_keys(t);
        load_values(t);
    }
    for (; u < u_end; u += NK) {
        const uint64_t valid = live_keys(t, mb);
        const float kscale = ks_next, vscale = vs_next;
        const int tn = u + NK < u_end ? tile_of(u + NK) : t;      // (the last tile is fetched once more and dropped)
        f32x16 s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        codes_to_bf16<TYPE>(kc[kb * 4 + j][2 * half], kc[kb * 4 + j][2 * half + 1]), qf[2 * j + half], s[kb], 0, 0, 0);
        load_keys(tn);
        mb = mask_byte(tn);
        ks_next = scales[2 * tn];
        vs_next = scales[2 * tn + 1];
        bf16x8 pb[2][2];
        // value scale 2^(e + unit), e uniform and, values of ordinary sizes all over, never past FOLD
        int e = __builtin_amdgcn_readfirstlane((int)(__float_as_uint(vscale) >> 23)) - 127 - w.unit, over = 0, under = 0;
        if (__builtin_expect((unsigned)(e + FOLD) > 2u * FOLD, 0)) {
            if (__builtin_amdgcn_ballot_w64(w.m != -INFINITY) == 0) {               // nothing has been summed: any unit will do
                w.unit += e;
                e = 0;
            } else if (e > 0) {
                over = e - FOLD;
                w.unit += over;
                e = FOLD;
            } else {
                under = e + FOLD;
                e = -FOLD;
            }
        }
        softmax_tile(s, valid, a.scale_log2e * kscale, (float)e, __uint_as_float((unsigned)(127 - e) << 23), over, under, w, pb, hg);
        if (valid != ~0ull) {          // zero codes under masked keys: 0 * NaN would reach the sums
            const uint64_t mine = valid >> (4 * hg);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned nib = (unsigned)(mine >> (kb * 32 + 8 * i)) & 15u;
                    const unsigned keep = ((nib * 0x00204081u) & 0x01010101u) * 255u;
#pragma unroll
                    for (int db = 0; db < 4; ++db) vc[db * 2 + kb][i] &= keep;
                }
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int ss = 0; ss < 2; ++ss)
#pragma unroll
                for (int db = 0; db < 4; ++db)
                    w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        codes_to_bf16<TYPE>(vc[db * 2 + kb][2 * ss], vc[db * 2 + kb][2 * ss + 1]), pb[kb][ss], w.o[db], 0, 0, 0);
        load_values(tn);
        t = tn;
    }

    unsigned char* const slice = lds + wave * SLICE;

    // ---- the key groups' results meet in LDS and are summed at their common maximum ----
    float l_tot = w.l + __shfl_xor(w.l, 32);
    if (w.unit != 0) {
        // The unit is taken back, and what keeps the outputs and their sum over all groups finite goes into the reference
        // maximum: |o| 2^unit <= l 2^128, so with l brought to 2^-8 at most, 64 groups' outputs add up below 2^126.
        const int g = l_tot > 0.f ? __builtin_amdgcn_frexp_expf(l_tot) + 8 : 0;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) w.o[db][i] = __builtin_ldexpf(w.o[db][i], w.unit - g);
        l_tot = __builtin_ldexpf(l_tot, -g);
        w.m += (float)g;
    }
    if (f_end > u_begin) __syncthreads();                               // the fresh tiles have been read
    if (hg == 0) {
        ml[(wave * QW + r) * 2] = w.m;
        ml[(wave * QW + r) * 2 + 1] = l_tot;
    }
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *(f32x4*)(slice + r * OROW + (db * 32 + 8 * c + 4 * hg) * 4) =
                (f32x4){w.o[db][4 * c], w.o[db][4 * c + 1], w.o[db][4 * c + 2], w.o[db][4 * c + 3]};
    __syncthreads();
    // wave kg of a query group writes 32 / NK of its queries: 16 lanes a row, 8 dims a lane
#pragma unroll
    for (int i = 0; i < QW / NK / 4; ++i) {
        const int row = kg * (QW / NK) + i * 4 + (lane >> 4), c = lane & 15;
        float m[NK], l[NK], mr = -INFINITY;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            m[k] = ml[((k * NQ + qg) * QW + row) * 2];
            l[k] = ml[((k * NQ + qg) * QW + row) * 2 + 1];
            mr = fmaxf(mr, m[k]);
        }
        const float mu = mr == -INFINITY ? 0.f : mr;
        float lr = 0.f;
        f32x4 x0 = {0.f, 0.f, 0.f, 0.f}, x1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const float f = __builtin_amdgcn_exp2f(m[k] - mu);
            const unsigned char* p = lds + (k * NQ + qg) * SLICE + row * OROW + c * 32;
            lr += l[k] * f;
            x0 += *(const f32x4*)p * f;
            x1 += *(const f32x4*)(p + 16) * f;
        }
        const int q = q0 + row;
        if (q >= a.n_q) continue;
        const int64_t orow = (int64_t)b * a.n_q + q;
        if (a.splits > 1) {
            float* po = a.part_o + ((size_t)ks * a.n_rows + orow) * d + h * KV8_HD + c * 8;
            *(f32x4*)po = x0;
            *(f32x4*)(po + 4) = x1;
            if (c == 0) {
                float* pm = a.part_ml + (((size_t)ks * a.n_rows + orow) * a.n_heads + h) * 2;
                pm[0] = mr;
                pm[1] = lr;
            }
        } else {
            const float inv = lr == 0.f ? 0.f : 1.0f / lr;              // no unmasked token: zeros
            u32x4 o;
            o[0] = pack_bf16x2(x0[0] * inv, x0[1] * inv);
            o[1] = pack_bf16x2(x0[2] * inv, x0[3] * inv);
            o[2] = pack_bf16x2(x1[0] * inv, x1[1] * inv);
            o[3] = pack_bf16x2(x1[2] * inv, x1[3] * inv);
            *(u32x4*)(a.out + (size_t)orow * d + h * KV8_HD + c * 8) = o;
        }
    }
}

// Key splits: out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s, m = max_s m_s; one thread per 4 columns.
__global__ void __launch_bounds__(256) attn_kv8_combine_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                                               bf16_t* __restrict__ out, int64_t n_rows, int n_heads, int splits) {
    const int d = n_heads * KV8_HD;
    const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (i >= n_rows * (d / 4)) return;
    const int64_t row = i / (d / 4);
    const int col = (int)(i % (d / 4)) * 4, h = col / KV8_HD;
    float m = -INFINITY;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, part_ml[((s * n_rows + row) * n_heads + h) * 2]);
    const float mu = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
        const float* pm = part_ml + ((s * n_rows + row) * n_heads + h) * 2;
        const float f = __builtin_amdgcn_exp2f(pm[0] - mu);
        const f32x4 o = *(const f32x4*)(part_o + (s * n_rows + row) * (int64_t)d + col);
        l += f * pm[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += f * o[e];
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    u32x2 w;
    w[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    w[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
    *(u32x2*)(out + row * d + col) = w;
}

constexpr int MAX_SPLITS = 16;

int g_force_nq = 0, g_force_splits = 0;     // test hook: 0 = automatic

struct Plan {
    int nq, splits;
};

// How a call's queries and tiles are dealt to waves (measured; times in us, 32 heads).
Plan pick_plan(int64_t n_seq, int n_q, int n_heads, int units, bool scratch) {
    auto workgroups = [&](int nq) { return (int64_t)((n_q + nq * QW - 1) / (nq * QW)) * n_heads * n_seq; };
    Plan p;
    // Waves that hold different queries share a tile's fetch; waves that share the queries fill more CUs.  The former while
    // every CU still has a workgroup: 64 x 640 tokens, 64 queries: 2 groups 94, 1 group 108; 4 x 2048, 128 queries: 2 groups
    // (256 workgroups) 25, 4 groups (128) 35.
    p.nq = 1;
    while (p.nq < 4 && n_q > p.nq * QW && workgroups(2 * p.nq) >= 256) p.nq *= 2;
    if (g_force_nq) p.nq = g_force_nq;
    p.splits = 1;
    if (!scratch) return p;
    // Key splits cost a second launch and a round trip of float32 partial results: up to one workgroup per CU, 16 tiles
    // each at least.  One sequence, 32 queries, unsplit / split: 1150 tokens 10.3 / 11.1, 2048: 14.5 / 14.0 (2 splits),
    // 4096: 21.6 / 15.4 (4); 4 sequences of 16384: 116 / 98 (2), 112 (4).
    const int64_t wgs = workgroups(p.nq);
    if (g_force_splits) {
        p.splits = g_force_splits < units ? g_force_splits : units;
    } else if (wgs <= 128) {
        const int64_t s = 256 / wgs;
        const int most = units / 16;
        p.splits = s < most ? (int)s : most > 1 ? most : 1;
    }
    if (p.splits > MAX_SPLITS) p.splits = MAX_SPLITS;
    return p;
}

size_t part_bytes(int64_t n_rows, int n_heads, int splits) {
    return (size_t)splits * n_rows * ((size_t)n_heads * KV8_HD * 4 + (size_t)n_heads * 8);
}

template <int TYPE>
void launch(const Kv8Attn& a, Plan p, unsigned grid, hipStream_t st) {
    if (p.nq == 1)
        hipLaunchKernelGGL((attn_kv8_kernel<TYPE, 1>), dim3(grid), dim3(NW * 64), 0, st, a);
    else if (p.nq == 2)
        hipLaunchKernelGGL((attn_kv8_kernel<TYPE, 2>), dim3(grid), dim3(NW * 64), 0, st, a);
    else
        hipLaunchKernelGGL((attn_kv8_kernel<TYPE, 4>), dim3(grid), dim3(NW * 64), 0, st, a);
}

}  // namespace

extern "C" size_t llada_attn_kv8_workspace_bytes(int32_t n_seq, int32_t n_q, int32_t seq_len, int32_t n_heads) {
    if (n_seq <= 0 || n_q <= 0 || seq_len <= 0 || n_heads <= 0) return 0;
    // + 2: a fresh block that tile borders cut at both ends sweeps up to two tiles more (start 1, 65 tokens)
    const Plan p = pick_plan(n_seq, n_q, n_heads, (int)kv8_blocks(seq_len) + 2, true);
    return p.splits > 1 ? part_bytes((int64_t)n_seq * n_q, n_heads, p.splits) : 0;
}

// tests and sweeps: query groups of a workgroup (1, 2, 4), key splits; 0 = automatic
extern "C" void llada_attn_kv8_force(int nq, int splits) {
    g_force_nq = nq;
    g_force_splits = splits;
}

extern "C" int llada_attn_kv8(const void* q, int64_t q_stride, int32_t n_q, const void* cache, int32_t kv_type,
                              const uint8_t* key_mask, void* out, int32_t n_seq, int32_t seq_len, int32_t n_heads,
                              const void* block_qkv, int64_t block_stride, int32_t block_start, int32_t block_len,
                              void* workspace, size_t workspace_bytes, void* stream) {
    LLADA_CHECK_ARG(q && cache && out, "attn_kv8: null argument");
    LLADA_CHECK_ARG(n_seq > 0 && seq_len > 0 && n_heads > 0 && n_q > 0, "attn_kv8: bad shape");
    LLADA_CHECK_ARG(q_stride >= (int64_t)n_heads * KV8_HD && q_stride % 8 == 0 && (((uintptr_t)q | (uintptr_t)out) & 15) == 0,
                    "attn_kv8: query rows cover the heads; rows start at 16-byte boundaries");
    LLADA_CHECK_ARG(((uintptr_t)cache & 255) == 0, "attn_kv8: cache must be 256-byte aligned");
    LLADA_CHECK_SUPPORTED(kv_type == LLADA_KV_E4M3 || kv_type == LLADA_KV_INT8, "attn_kv8: unknown cache type %d", kv_type);
    LLADA_CHECK_ARG(workspace == nullptr || ((uintptr_t)workspace & 15) == 0, "attn_kv8: workspace must be 16-byte aligned");
    if (block_qkv) {
        LLADA_CHECK_ARG(block_start >= 0 && block_len > 0 && (int64_t)block_start + block_len <= seq_len,
                        "attn_kv8: the block must lie inside the sequence");
        LLADA_CHECK_ARG(block_stride >= (int64_t)3 * n_heads * KV8_HD && block_stride % 8 == 0 && ((uintptr_t)block_qkv & 15) == 0,
                        "attn_kv8: block rows hold [Q | K | V] and start at 16-byte boundaries");
    }
    const int64_t n_blocks = kv8_blocks(seq_len);
    const int64_t n_tiles = (int64_t)n_seq * n_heads * n_blocks;
    Kv8Attn a;
    a.q = (const bf16_t*)q;
    a.q_stride = q_stride;
    a.scales = (const float*)cache;
    a.tiles = (const unsigned char*)cache + kv8_scale_bytes(n_tiles);
    a.key_mask = key_mask;
    a.out = (bf16_t*)out;
    a.blk = (const bf16_t*)block_qkv;
    a.blk_stride = block_stride;
    a.n_rows = (int64_t)n_seq * n_q;
    a.n_q = n_q;
    a.seq_len = seq_len;
    a.n_heads = n_heads;
    a.n_blocks = (int)n_blocks;
    a.scale_log2e = 1.4426950408889634f / sqrtf((float)KV8_HD);
    a.blk_start = block_qkv ? block_start : 0;
    a.blk_len = block_qkv ? block_len : 0;
    a.skip_from = (int)n_blocks;
    a.skipped = 0;
    int fresh = 0;
    if (block_qkv) {
        const int end = block_start + block_len;
        const int c0 = (block_start + KV8_TOKENS - 1) / KV8_TOKENS, c1 = end == seq_len ? (int)n_blocks : end / KV8_TOKENS;
        if (c1 > c0) {
            a.skip_from = c0;
            a.skipped = c1 - c0;
        }
        fresh = (block_len + KV8_TOKENS - 1) / KV8_TOKENS;
    }
    a.n_cached = (int)n_blocks - a.skipped;
    a.n_units = a.n_cached + fresh;
    const Plan plan = pick_plan(n_seq, n_q, n_heads, a.n_units, workspace != nullptr);
    a.n_qblocks = (n_q + plan.nq * QW - 1) / (plan.nq * QW);
    const int64_t wgs = (int64_t)a.n_qblocks * n_heads * n_seq;
    int splits = plan.splits;
    while (splits > 1 && part_bytes(a.n_rows, n_heads, splits) > workspace_bytes) --splits;
    a.per_split = (a.n_units + splits - 1) / splits;
    a.splits = (a.n_units + a.per_split - 1) / a.per_split;             // no empty run
    a.part_o = (float*)workspace;
    a.part_ml = a.splits > 1 ? a.part_o + (size_t)a.splits * a.n_rows * n_heads * KV8_HD : nullptr;
    LLADA_CHECK_SUPPORTED(wgs * a.splits * (NW * 64) < (1LL << 32) && (a.splits == 1 || a.n_rows * n_heads * (KV8_HD / 4) + 255 < (1LL << 32)),
                          "attn_kv8: grid too large (a launch ends at 2^32 threads)");
    hipStream_t st = (hipStream_t)stream;
    if (kv_type == LLADA_KV_E4M3)
        launch<LLADA_KV_E4M3>(a, plan, (unsigned)(wgs * a.splits), st);
    else
        launch<LLADA_KV_INT8>(a, plan, (unsigned)(wgs * a.splits), st);
    LLADA_CHECK_LAUNCH("attn_kv8_kernel");
    if (a.splits > 1) {
        const int64_t items = a.n_rows * n_heads * (KV8_HD / 4);
        hipLaunchKernelGGL(attn_kv8_combine_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st,
                           (const float*)a.part_o, (const float*)a.part_ml, a.out, a.n_rows, n_heads, a.splits);
        LLADA_CHECK_LAUNCH("attn_kv8_combine_kernel");
    }
    return LLADA_OK;
}
