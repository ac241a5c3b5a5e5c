// Sampling a token per logits row from the softmax distribution at a temperature, truncated by top-k, then top-p, then
// min-p, by inversion of one given uniform per row; alone (llada_sample_rows) and as the candidate rule of the remasking
// epilogue (llada_remask_scores_sampled).
//
// Definition, for a row's entries ordered by (logit descending, index ascending), m the largest logit:
//   w_i = exp((l_i - m) / T) in float64;  n_k = top_k (all when 0);
//   n_p = the smallest n with w_1 + .. + w_n >= top_p * (w_1 + .. + w_{n_k});  n_m = the number of w_i >= min_p (l_i - m >= T log min_p);
//   n = max(1, min(n_k, n_p, n_m));  token = the first i <= n with w_1 + .. + w_i > u * (w_1 + .. + w_n).
//
// A bf16 row has at most a few thousand DISTINCT values, and the order, the masses and every cut depend on the values
// alone (equal values are consecutive, in index order).  So nothing is sorted: a row's values are counted in LDS (one
// integer atomic per entry: exact, order-free), exponentials in float64 are taken per distinct value, 64-value chunks of
// the histogram are summed by waves in a fixed order, and the cuts and the token are found by prefix search over chunk
// totals and then inside one chunk.  The row, or half of it, stays in registers (16 x 16 bytes a lane) for the last step,
// which turns "the j-th entry of value v" into an index.
//
// The histogram has a bin for every bf16 value of magnitude in [2^-55, 2^8), or [2^-35, 2^8), of either sign and one for
// zero.  A row with another finite magnitude, an infinity of positive sign or a NaN is "irregular" (its clamped bins say
// so, at no cost to other rows) and is counted over the whole 16-bit key space in windows instead; -inf entries, NaNs
// included, have no weight and are never drawn.  A row with nothing else gives token 0 with probability 0.
//
// Bound by a CU's own work on a row, 41 to 50 thousand cycles where 1024 lanes do it: the histogram 21 to 26 (its LDS
// atomics alone 16: 64 random bins meet in the banks, 8 cycles an instruction), listing the occupied bins 4.5, their
// weights and prefixes 5, the searches 6 (one wave, a chain of scans), the place of the token 3 to 8; from a few rows a CU
// on by memory (Shape).  126464 entries: 32 rows 24 us, 256 guided 45 us (2.9 TB/s), 2048 rows 139 us (3.7 TB/s of rows).
// An irregular row is read again, entry by entry, for each window (4, or 8 by half), each cut and the token: 230 to 310 us for
// up to 256 rows, 2.6 ms for 2048.  A vocabulary masked with -1e4 or the type's lowest value makes its rows irregular, one
// masked with -inf does not.
// Tried and dropped: reading a row twice and keeping none of it (2048 rows 198 us against the 194 of rows kept whole); a
// wave-major order of the chunks (slower); four workgroups that count a quarter of a row each and a fifth that joins
// their bins and goes on (32 rows 23.4 us against 23.3 in a graph, guided 44 / 39: the second launch and the fixed
// 20 thousand cycles behind the histogram eat what the counting saves).
#include "common.h"
#include "philox.h"
#include "rowregs.h"

namespace {

constexpr int MAX_CHUNKS = 65536 / 64;
constexpr unsigned LLADA_STREAM_SAMPLE = 4u;
constexpr double MAX_TEMPERATURE = 1.0e30;

typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
typedef __attribute__((ext_vector_type(2))) short s16x2;

struct SampleArgs {
    const bf16_t* logits;
    const bf16_t* uncond;
    int64_t stride;           // elements between rows, of both
    float cfg1;
    int vocab;
    llada_sampling s;
    uint64_t seed;
    uint32_t step, row_offset;
    int64_t* tokens;          // llada_sample_rows
    float* probs;
    llada_remask_args r;      // remasking epilogue
};

// What a workgroup is made for.
//   WHOLE  1024 lanes keep the row in registers (16 x 16 bytes each), one workgroup a CU: the row is read once.
//   else   512 lanes keep the first half of the longest row, read the rest past, and read that again only when the drawn
//          entry is not in the half they hold; half the LDS, so two workgroups share a CU and one's reading goes on under
//          the other's searches.
// Both sides, us in a graph (whole / half), 126464 entries, temperature 0.8, min_p 0.02 (other parameters: within 3): 256 rows
// 30.5 / 33.1, 384 46.1 / 47.2, 512 52.1 / 50.4, 768 73.8 / 70.2, 1024 92.6 / 78.8, 2048 174.6 / 139.5; with the epilogue 256
// rows 33.8 / 37.0, 384 50.4 / 52.7, 512 56.4 / 52.6, 1024 102.3 / 88.2, 2048 193.5 / 153.3: by half from two rows a CU on.
// Guided rows of that length are always kept whole: combining is arithmetic, which a second workgroup does not hide (256
// rows 57 / 76, 2048 341 / 372 when both existed).  Rows that fit the half are held whole by it, guided ones too: 50257
// entries, 32 rows 18.2 / 15.6, 1500 rows 95 / 60; 1000 entries 16.6 / 11.7, 70 / 40.
template <bool WHOLE_>
struct Shape {
    static constexpr bool WHOLE = WHOLE_;
    static constexpr int HELD = 16;                                // chunks of 16 bytes a lane keeps
    static constexpr int THREADS = WHOLE ? 1024 : 512;
    static constexpr int NWV = THREADS / 64;
    static constexpr int SLOTS = ROW_MAX_VOCAB / 8 / THREADS;      // 16-byte chunks a lane
    // magnitudes with a bin of their own: [2^-55, 2^8), or [2^-35, 2^8)
    static constexpr unsigned MAG_HI = 0x4380, MAG_LO = WHOLE ? 0x2400 : 0x2E00;
    static constexpr int SPAN = MAG_HI - MAG_LO;                   // bin 0: below the range (zero), SPAN + 1: above
    // bin of a negative value: the sign bit stays where it is and what is between the planes holds the other shared state,
    // or the second plane follows the first
    static constexpr int NEGATIVE = WHOLE ? 0x8000 : (SPAN + 2 + 3) / 4 * 4;
    static constexpr int REGULAR_KEYS = 2 * SPAN + 1;              // descending values: SPAN positive, zero, SPAN negative
    static constexpr int RUN = WHOLE ? 16 : 24;                    // neighbouring bins a lane lists: half of the lanes a sign
    static constexpr int WINDOW = WHOLE ? 16384 : 8192;             // irregular rows: keys counted at a time
    static constexpr int REST_AT = WHOLE ? WINDOW : NEGATIVE + (SPAN + 2 + 3) / 4 * 4;   // in LDS words: the other shared state

    struct Shared {
        unsigned cnt[MAX_CHUNKS];        // entries of a chunk of 64 positions, then: entries before it
        double mass[MAX_CHUNKS];         // their weight, then: the weight before it
        double conf[NWV];                // epilogue: partial sums of the waves
        double total_mass;
        unsigned total;
        int first[NWV];
        int irregular;
        int broken;                      // epilogue: the row has a NaN or an infinity of positive sign
        int j, tied;                     // the drawn entry: the j-th of `tied` equal ones
        float value, prob;
        unsigned slot_tot[SLOTS];
        unsigned wave_tot[NWV];
        int token;
        unsigned short patterns[REGULAR_KEYS + 64];   // regular rows: the values that have entries, in order
    };
    static constexpr int LDS_WORDS = WHOLE ? NEGATIVE + (SPAN + 2 + 3) / 4 * 4 : REST_AT + (int)((sizeof(Shared) + 3) / 4);
    static_assert(RUN % 4 == 0 && SPAN % 4 == 0 && NEGATIVE % 4 == 0 && (SPAN / RUN + 1) <= THREADS / 2, "a lane's run");
    static_assert((REGULAR_KEYS + 63) / 64 <= 256 && SLOTS <= 64 && WINDOW <= REST_AT, "ranges of the scans");
    static_assert(WHOLE ? REST_AT * 4 + sizeof(Shared) <= NEGATIVE * 4 && LDS_WORDS * 4 <= 160 * 1024 : LDS_WORDS * 4 <= 80 * 1024, "LDS");
};

// irregular rows: position p of the whole key space (0 = the largest value) -> bf16 pattern
__device__ __forceinline__ unsigned full_bits(int p) {
    const unsigned k = 65535u - (unsigned)p;
    return (k & 0x8000u) ? k ^ 0x8000u : ~k & 0xFFFFu;
}

// irregular rows: key of a bf16 pattern, -1 for an entry without weight (-inf, NaN); -0 counts as +0
__device__ __forceinline__ int full_key(unsigned bits) {
    if (bits == 0x8000u) bits = 0u;
    if ((bits & 0x7FFFu) > 0x7F80u || bits == 0xFF80u) return -1;
    return 65535 - (int)((bits & 0x8000u) ? ~bits & 0xFFFFu : bits | 0x8000u);
}

// Scans and broadcasts by data-parallel moves: a few cycles a step where a shuffle through LDS takes a hundred.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned dpp(unsigned v) {      // lanes without a source get 0
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t r = (uint64_t)dpp<CTRL, ROWS>((unsigned)(b >> 32)) << 32 | dpp<CTRL, ROWS>((unsigned)b);
    return __builtin_bit_cast(double, r);
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {               // inclusive, fixed order
    v += dpp<0x111, 0xF>(v);
    v += dpp<0x112, 0xF>(v);
    v += dpp<0x114, 0xF>(v);
    v += dpp<0x118, 0xF>(v);
    v += dpp<0x142, 0xA>(v);
    v += dpp<0x143, 0xC>(v);
    return v;
}
template <class T>
__device__ __forceinline__ T lane_before(T v) { return dpp<0x138, 0xF>(v); }      // lane 0: zero
__device__ __forceinline__ unsigned from_lane(unsigned v, int at) { return (unsigned)__builtin_amdgcn_readlane((int)v, at); }
__device__ __forceinline__ double from_lane(double v, int at) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)from_lane((unsigned)(b >> 32), at) << 32 | from_lane((unsigned)b, at));
}
__device__ __forceinline__ float uniform(float v) {         // the same in every lane: into a scalar register
    return __uint_as_float((unsigned)__builtin_amdgcn_readfirstlane((int)__float_as_uint(v)));
}
__device__ __forceinline__ double wave_total(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// 2^y in float64, y <= 0: 2^rint(y) times the Taylor polynomial of 2^f = e^(f ln 2) to the 13th power, |f| <= 1/2
// (remainder below 5e-18).  The argument is formed with one rounding, so a weight is off by up to 2^-53 |y| of itself:
// what counts in a row's sums are the weights with small |y|.  Half the instructions of the library's exp, and in four
// short chains where a wave would wait out one long one.
__device__ __forceinline__ double exp2_neg(double y) {
    constexpr double L = 0.69314718055994530942;
    constexpr double C2 = L * L / 2, C3 = C2 * L / 3, C4 = C3 * L / 4, C5 = C4 * L / 5, C6 = C5 * L / 6, C7 = C6 * L / 7, C8 = C7 * L / 8,
                     C9 = C8 * L / 9, C10 = C9 * L / 10, C11 = C10 * L / 11, C12 = C11 * L / 12, C13 = C12 * L / 13;
    y = fmax(y, -1100.0);                        // (2^-1100 is 0; an infinity stays out of the polynomial)
    const double k = __builtin_rint(y), f = y - k, f2 = f * f, f4 = f2 * f2;
    const double a = __builtin_fma(__builtin_fma(C3, f, C2), f2, __builtin_fma(L, f, 1.0));
    const double b = __builtin_fma(__builtin_fma(C7, f, C6), f2, __builtin_fma(C5, f, C4));
    const double c = __builtin_fma(__builtin_fma(C11, f, C10), f2, __builtin_fma(C9, f, C8));
    const double d = __builtin_fma(C13, f, C12);
    const double p = __builtin_fma(__builtin_fma(__builtin_fma(d, f4, c), f4, b), f4, a);
    return __builtin_ldexp(p, (int)k);
}
constexpr double LOG2E = 1.44269504088896340736;

// (by value: a bit cast straight from a vector's element reads the vector's first)
__device__ __forceinline__ u16x2 halves(unsigned w) { return __builtin_bit_cast(u16x2, w); }

// generate.py:89-90 on eight entries: cfg_combine's three operations, each rounded to bf16, two entries a conversion (17
// instructions for two entries instead of 26: guided rows are bound by them)
__device__ __forceinline__ u32x4 combine(u32x4 c, u32x4 u, float cfg1) {
    typedef __attribute__((ext_vector_type(2))) float f32x2;
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    auto rounded = [](float lo, float hi) { return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){lo, hi}, bf16x2)); };
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        unsigned d = rounded(bf16lo(c[e]) - bf16lo(u[e]), bf16hi(c[e]) - bf16hi(u[e]));
        d = rounded(bf16lo(d) * cfg1, bf16hi(d) * cfg1);
        c[e] = rounded(bf16lo(u[e]) + bf16lo(d), bf16hi(u[e]) + bf16hi(d));
    }
    return c;
}

// Entries v0 .. v0 + 7 of a row as the draw sees them, one at a time: combined under guidance; -inf for what lies outside the
// row and for the entry that is taken out of everything (EOS removed before the draw).  (Indexes clamped into the row and
// no branches: the eight loads travel together.)
template <bool EPI>
__device__ __forceinline__ u32x4 row_chunk(const bf16_t* lc, const bf16_t* lu, int v0, int vocab, float cfg1, int excluded) {
    auto fetch = [&](const bf16_t* row) {
        bf16_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = row[min(max(v0 + e, 0), vocab - 1)];
        u32x4 t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = (unsigned)x[2 * e] | (unsigned)x[2 * e + 1] << 16;
        return t;
    };
    u32x4 t = fetch(lc);
    if (lu) {
        asm volatile("" : "+v"(t)::"memory");        // (one row's entries after the other's: eight registers fewer)
        t = combine(t, fetch(lu), cfg1);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int v = v0 + e;
        const bool out = v < 0 || v >= vocab || (EPI && v == excluded);
        const unsigned keep = out ? ((e & 1) ? 0x0000FFFFu : 0xFFFF0000u) : 0xFFFFFFFFu, put = out ? ((e & 1) ? 0xFF800000u : 0x0000FF80u) : 0u;
        t[e >> 1] = (t[e >> 1] & keep) | put;
    }
    return t;
}

// One more in the bins of a word's two entries.  The addresses are formed by hand where the compiler takes two instructions
// more for each word.
template <class L>
__device__ __forceinline__ void count_two(unsigned* bins, unsigned word) {
    const u16x2 idx = __builtin_elementwise_min(
        __builtin_elementwise_sub_sat(halves(word & 0x7FFF7FFFu), (u16x2)((unsigned short)(L::MAG_LO - 1))), (u16x2)((unsigned short)(L::SPAN + 1)));
    unsigned at, lo, hi;
    if constexpr (L::WHOLE)
        asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(at) : "v"(word), "s"(0x80008000u), "v"(__builtin_bit_cast(unsigned, idx)));
    else
        asm("v_pk_mad_u16 %0, %1, %2, %3" : "=v"(at) : "v"(halves(word) >> (unsigned short)15), "v"((unsigned)L::NEGATIVE * 0x00010001u), "v"(idx));
    asm("v_lshlrev_b32_sdwa %0, %2, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:WORD_0" : "=v"(lo) : "v"(at), "v"(2u));
    asm("v_lshlrev_b32_sdwa %0, %2, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:WORD_1" : "=v"(hi) : "v"(at), "v"(2u));
    atomicAdd((unsigned*)((unsigned char*)bins + lo), 1u);
    atomicAdd((unsigned*)((unsigned char*)bins + hi), 1u);
}

// 1 in each half that is zero, else 0 (by hand: the compiler turns the saturating 1 - x into compares and selects)
__device__ __forceinline__ unsigned zero_halves(unsigned x) {
    unsigned r;
    asm("v_pk_sub_u16 %0, %1, %2 clamp" : "=v"(r) : "v"(0x00010001u), "v"(x));
    return r;
}

// Draws the token of one row.  EPI: also leaves the row's confidence (rules of llada_remask_scores) in `conf`.
template <bool EPI, class L, bool GUIDED>
__device__ __forceinline__ void sample_row(const SampleArgs& a, unsigned* bins, typename L::Shared& sh, const bf16_t* lc, const bf16_t* lu, double T, int top_k,
                                           double top_p, double min_p, double u, int excl_all, const int (&excl_conf)[2], float& conf) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int THREADS = L::THREADS, NWV = L::NWV, SLOTS = L::SLOTS, HELD = L::HELD, SPAN = L::SPAN, NEGATIVE = L::NEGATIVE, WINDOW = L::WINDOW, RUN = L::RUN;
    constexpr int WINDOWS = 65536 / WINDOW;
    constexpr unsigned MAG_LO = L::MAG_LO, MAG_HI = L::MAG_HI;
    const int V = a.vocab;
    // Chunk c = lane + THREADS i (slot i) holds entries 8 c - off .. + 7, off = the row's offset from a 16-byte boundary in
    // entries, so that all but its first and last chunk are one aligned load.
    const int off = (int)(((uintptr_t)lc >> 1) & 7);
    if constexpr (!GUIDED) lu = nullptr;
    const int chunks = (V + off + 7) / 8;

    for (int i = tid; i < SPAN + 2; i += THREADS) bins[i] = bins[NEGATIVE + i] = 0u;
    if (tid < SLOTS) sh.slot_tot[tid] = 0u;
    if (tid == 0) {
        sh.irregular = 0;
        sh.broken = 0;
        sh.token = -1;
    }

    __syncthreads();

    // entries the confidence's softmax does not see although they can be drawn (generate.py:100-101)
    float lx_excl[2] = {-INFINITY, -INFINITY};
    if constexpr (EPI) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (excl_conf[i] >= 0) {
                lx_excl[i] = bf16_to_f32(lc[excl_conf[i]]);
                if (lu) lx_excl[i] = cfg_combine(lx_excl[i], bf16_to_f32(lu[excl_conf[i]]), a.cfg1);
                lx_excl[i] = uniform(lx_excl[i]);
            }
    }
    // entries of a key that this softmax sees
    auto seen = [&](unsigned n, float v) { return n - (v == lx_excl[0] ? 1u : 0u) - (v == lx_excl[1] ? 1u : 0u); };

    // Chunks that are not one load: those the row covers only in part (its first or last) and the one with the entry taken out
    // of everything.  They are fetched entry by entry, apart from the others: this code runs once a row, and what it costs
    // beside its memory time is its length.
    const int odd[3] = {off != 0 ? 0 : -1, ((V + off) & 7) != 0 ? chunks - 1 : -1, EPI && excl_all >= 0 ? (excl_all + off) >> 3 : -1};
    auto is_odd = [&](int c) { return c == odd[0] || c == odd[1] || (EPI && c == odd[2]); };
    auto each_odd = [&](auto&& f) {              // f(slot, words) in the lane that holds the chunk
        if (odd[0] < 0 && odd[1] < 0 && odd[2] < 0) return;
#pragma unroll 1
        for (int k = 0; k < 3; ++k) {
            const int c = k == 0 ? odd[0] : k == 1 ? odd[1] : odd[2];
            if (c < 0 || c % THREADS != tid || (k > 0 && c == odd[0]) || (k > 1 && c == odd[1])) continue;
            f(c / THREADS, row_chunk<EPI>(lc, lu, c * 8 - off, V, a.cfg1, excl_all));
        }
    };
    // (a uniform address and one 32-bit offset for all slots)
    auto chunk_at = [&](const bf16_t* row, int slot) { return (const u32x4*)((const char*)(row - off) + (size_t)slot * (THREADS * 16) + (unsigned)tid * 16u); };
    const u32x4 ninf = {BF16_NEG_INF2, BF16_NEG_INF2, BF16_NEG_INF2, BF16_NEG_INF2};

    // The chunks that are kept,
    u32x4 q[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int v0 = (tid + i * THREADS) * 8 - off;
        q[i] = ninf;
        if (v0 >= 0 && v0 + 8 <= V) q[i] = __builtin_nontemporal_load(chunk_at(lc, i));
    }
    each_odd([&](int slot, u32x4 t) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (i == slot) q[i] = t;
    });
    auto plain = [&](int slot) { return tid + slot * THREADS < chunks && !is_odd(tid + slot * THREADS); };
    // and the rest, read past: f(slot, words) in every lane of the workgroup (-inf where a lane has no chunk, or an odd one, which
    // comes at the end, in its lane alone), a few loads ahead
    auto rest = [&](auto&& f) {
        constexpr int AHEAD = 6;
        const int used = (chunks + THREADS - 1) / THREADS;
        if (HELD == SLOTS || used <= HELD) return;
        u32x4 next[AHEAD];
        auto fetch = [&](int slot, int i) {
            next[i] = ninf;
            if (plain(slot)) next[i] = *chunk_at(lc, slot);
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) fetch(HELD + i, i);
#pragma unroll 1
        for (int i0 = HELD; i0 < used; i0 += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const u32x4 t = next[i];
                fetch(i0 + AHEAD + i, i);
                if (i0 + i < used) f(i0 + i, t);
            }
        }
        each_odd([&](int slot, u32x4 t) {
            if (slot >= HELD) f(slot, t);
        });
    };

    // ---- the histogram, as the chunks arrive: clamped magnitudes, both signs ----
    auto count = [&](int i) {
        if (tid + i * THREADS >= chunks) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) count_two<L>(bins, q[i][e]);
    };
    if constexpr (GUIDED) {            // eight chunks of the other row are on their way while the eight before are counted
        u32x4 b[8];
        auto fetch = [&](int g) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (plain(g + i)) b[i] = __builtin_nontemporal_load(chunk_at(lu, g + i));
        };
        fetch(0);
#pragma unroll
        for (int g = 0; g < HELD; g += 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (plain(g + i)) q[g + i] = combine(q[g + i], b[i], a.cfg1);
            __builtin_amdgcn_sched_barrier(0);
            if (g + 8 < HELD) fetch(g + 8);
#pragma unroll
            for (int i = 0; i < 8; ++i) count(g + i);
            __builtin_amdgcn_sched_barrier(0);
        }
    } else {
#pragma unroll
        for (int i = 0; i < HELD; ++i) count(i);
    }
    rest([&](int i, u32x4 t) {
        if (tid + i * THREADS >= chunks) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) count_two<L>(bins, t[e]);
    });
    __syncthreads();
    if (tid == 0) bins[0] += bins[NEGATIVE];     // zero of either sign (the test below holds before and after)
    // clamped bins that hold more than what was put there for entries that do not count: zeros and -inf are as good as
    // binned, anything else makes the row irregular
    unsigned padded = (unsigned)(chunks * 8 - V) + (EPI && excl_all >= 0 ? 1u : 0u);
    if constexpr (HELD < SLOTS) {
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (odd[k] >= HELD * THREADS && (k == 0 || odd[k] != odd[0]) && (k < 2 || odd[k] != odd[1])) padded += 8u;
    }
    if (bins[0] + bins[NEGATIVE] + bins[SPAN + 1] + bins[NEGATIVE + SPAN + 1] != padded) {
        // smallest magnitude above zero, largest positive pattern, largest negative one but -inf
        const u16x2 one = {1, 1}, minus_inf = {0xFF80, 0xFF80};
        u16x2 least = {0xFFFF, 0xFFFF}, neg = {0, 0};
        s16x2 pos = {0, 0};
        auto look = [&](u32x4 t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u16x2 w = halves(t[e]);
                least = __builtin_elementwise_min(least, (w & (unsigned short)0x7FFF) - one);
                pos = __builtin_elementwise_max(pos, __builtin_bit_cast(s16x2, w));
                neg = __builtin_elementwise_max(neg, w * __builtin_elementwise_min(w ^ minus_inf, one));
            }
        };
#pragma unroll
        for (int i = 0; i < HELD; ++i) look(q[i]);
        rest([&](int, u32x4 t) { look(t); });
        const bool bad = min(least[0], least[1]) < MAG_LO - 1 || (unsigned)max(pos[0], pos[1]) >= MAG_HI ||
                         max(neg[0], neg[1]) >= 0x8000u + MAG_HI;
        if (__builtin_amdgcn_ballot_w64(bad) != 0 && lane == 0) sh.irregular = 1;
        if constexpr (EPI) {
            const bool odd_one = max(pos[0], pos[1]) >= 0x7F80 || max(neg[0], neg[1]) > 0xFF80;
            if (__builtin_amdgcn_ballot_w64(odd_one) != 0 && lane == 0) sh.broken = 1;
        }
    }
    __syncthreads();
    const bool regular = sh.irregular == 0;
    // a distance from the largest logit -> log2 of its weight (temperature 0: all but the largest weigh nothing)
    const double to_log2 = T > 0.0 ? fmin(LOG2E / T, 1.0e300) : 1.0e300;

    // An irregular row: counts one window of its keys into the bins, from memory again (such rows are rare and the
    // row's registers are better left alone).  All threads call it together.
    auto count_window = [&](int win) {
        __syncthreads();
        for (int i = tid; i < WINDOW; i += THREADS) bins[i] = 0u;
        __syncthreads();
#pragma unroll 1
        for (int c = tid; c < chunks; c += THREADS) {
            const u32x4 t = row_chunk<EPI>(lc, lu, c * 8 - off, V, a.cfg1, excl_all);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int k = full_key((e & 1) ? t[e >> 1] >> 16 : t[e >> 1] & 0xFFFFu);
                if (k >= 0 && k / WINDOW == win) atomicAdd(&bins[k & (WINDOW - 1)], 1u);
            }
        }
        __syncthreads();
    };

    // The row's values in order stand at positions 0 .. n_pos - 1: a regular row's occupied ones, gathered in a list; an
    // irregular row's whole key space.  A chunk is 64 positions.
    float m = 0.f;                   // the largest value
    int n_pos = 65536;
    struct Entries {
        unsigned n;                  // of this position
        float v;
        double dl;                   // v minus the largest (0 where there is no entry)
    };
    auto bits_at = [&](int p) { return regular ? (unsigned)sh.patterns[p] : full_bits(p); };
    auto value_at = [&](int p) { return __uint_as_float(bits_at(p) << 16); };
    auto entries_at = [&](int p) {
        const int at = min(p, n_pos - 1);
        const unsigned bits = bits_at(at), mag = bits & 0x7FFFu;
        Entries x;
        x.n = bins[regular ? (int)(mag < MAG_LO ? 0u : mag - (MAG_LO - 1u)) + (bits & 0x8000u ? NEGATIVE : 0) : (at & (WINDOW - 1))];
        if (p >= n_pos) x.n = 0u;
        x.v = __uint_as_float(bits << 16);
        const double dl = (double)x.v - (double)m;
        x.dl = x.v == m || x.n == 0u ? 0.0 : dl;
        return x;
    };
    double s_sum = 0.0;              // epilogue: sum of exp(l - m) over the row
    auto total_chunk = [&](int c) {
        const Entries x = entries_at(c * 64 + lane);
        const double ms = wave_scan(x.n * exp2_neg(x.dl * to_log2));
        const unsigned cs = wave_scan(x.n);
        if (lane == 63) {
            sh.cnt[c] = cs;
            sh.mass[c] = ms;
        }
        if (EPI && x.n) s_sum += seen(x.n, x.v) * exp2_neg(x.dl * LOG2E);
    };

    // ---- totals of the chunks: entries, weight ----
    if (regular) {
        // A lane lists the occupied ones among RUN neighbouring bins; where its part begins is a scan of the lanes' counts.  The
        // first half of the lanes take the positive plane from its top (zero the last), the others the negative one.
        const bool minus = wave >= NWV / 2;                  // (uniform)
        const int g = minus ? tid - THREADS / 2 : SPAN / RUN - tid;
        unsigned n[RUN], held = 0;
#pragma unroll
        for (int e = 0; e < RUN; e += 4) {
            const u32x4 x = *(const u32x4*)(bins + (minus ? NEGATIVE : 0) + min(max(g * RUN + e, 0), SPAN));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int bin = g * RUN + e + i;
                n[e + i] = bin <= SPAN && bin >= (minus ? 1 : 0) ? x[i] : 0u;
            }
        }
#pragma unroll
        for (int e = 0; e < RUN; ++e) held += n[e] != 0u;
        const unsigned incl = wave_scan(held);
        if (lane == 63) sh.wave_tot[wave] = incl;
        __syncthreads();
        const unsigned upto = wave_scan(lane < NWV ? sh.wave_tot[lane & (NWV - 1)] : 0u);
        n_pos = (int)from_lane(upto, NWV - 1);
        unsigned short* out = sh.patterns + (from_lane(lane_before(upto), wave) + incl - held);
        const unsigned bits0 = (minus ? 0x8000u : 0u) + MAG_LO - 1u + g * RUN;
        if (minus) {
#pragma unroll
            for (int e = 0; e < RUN; ++e)
                if (n[e]) *out++ = (unsigned short)(bits0 + e);
        } else {
#pragma unroll
            for (int e = RUN - 1; e >= 0; --e)
                if (n[e]) *out++ = (unsigned short)(e == 0 && g == 0 ? 0u : bits0 + e);
        }
        __syncthreads();
        if (n_pos > 0) m = value_at(0);
#pragma unroll 1
        for (int c = wave; c * 64 < n_pos; c += NWV) total_chunk(c);
    } else {
        bool found = false;
        for (int win = 0; win < WINDOWS; ++win) {
            count_window(win);
            const int c_lo = win * (WINDOW / 64), c_hi = c_lo + WINDOW / 64;
            if (!found) {
                int mine = 0x7fffffff;
                for (int c = c_lo + wave; c < c_hi; c += NWV) {
                    const uint64_t any = __builtin_amdgcn_ballot_w64(bins[(c * 64 + lane) & (WINDOW - 1)] != 0u);
                    if (any != 0 && mine == 0x7fffffff) mine = c * 64 + __builtin_ctzll(any);
                }
                if (lane == 0) sh.first[wave] = mine;
                __syncthreads();
                int top = 0x7fffffff;
#pragma unroll
                for (int w = 0; w < NWV; ++w) top = min(top, sh.first[w]);
                found = top != 0x7fffffff;
                if (found) m = value_at(top);
                __syncthreads();
            }
            for (int c = c_lo + wave; c < c_hi; c += NWV) total_chunk(c);
        }
    }
    const int n_chunks = (n_pos + 63) / 64;
    __syncthreads();

    // ---- exclusive prefixes over the chunks (wave 0); a regular row's stay in its registers: chunks 4 lane .. + 3 ----
    unsigned pc[4] = {0u, 0u, 0u, 0u};
    double pm[4] = {0.0, 0.0, 0.0, 0.0};
    if (wave == 0) {
        if (regular) {
            unsigned c[4];
            double w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool there = lane * 4 + i < n_chunks;
                c[i] = there ? sh.cnt[lane * 4 + i] : 0u;
                w[i] = there ? sh.mass[lane * 4 + i] : 0.0;
            }
            const unsigned ci = wave_scan(c[0] + c[1] + c[2] + c[3]);
            const double wi = wave_scan(w[0] + w[1] + w[2] + w[3]);
            pc[0] = lane_before(ci);
            pm[0] = lane_before(wi);
#pragma unroll
            for (int i = 1; i < 4; ++i) {
                pc[i] = pc[i - 1] + c[i - 1];
                pm[i] = pm[i - 1] + w[i - 1];
            }
            *(u32x4*)&sh.cnt[lane * 4] = (u32x4){pc[0], pc[1], pc[2], pc[3]};
#pragma unroll
            for (int i = 0; i < 4; ++i) sh.mass[lane * 4 + i] = pm[i];
            if (lane == 63) {
                sh.total = ci;
                sh.total_mass = wi;
            }
        } else {
            unsigned cb = 0;
            double qb = 0.0;
#pragma unroll 1
            for (int at = lane; at < MAX_CHUNKS; at += 64) {
                const unsigned c = sh.cnt[at];
                const double w = sh.mass[at];
                const unsigned ci = wave_scan(c);
                const double wi = wave_scan(w);
                sh.cnt[at] = cb + ci - c;
                sh.mass[at] = qb + lane_before(wi);
                cb += from_lane(ci, 63);
                qb += from_lane(wi, 63);
            }
            if (lane == 0) {
                sh.total = cb;
                sh.total_mass = qb;
            }
        }
    }
    __syncthreads();
    const unsigned N = sh.total;
    if (N == 0u) {                       // nothing but -inf
        if (tid == 0) {
            sh.token = 0;
            sh.prob = 0.f;
        }
        conf = __builtin_nanf("");           // (a softmax of nothing)
        __syncthreads();
        return;
    }

    // A regular row's searches run in wave 0 alone.  An irregular row's bins hold one window at a time: every wave follows
    // the search, and the window that holds a chunk is counted again when it is looked into.
    auto chunks_before = [&](auto&& test) {          // number of leading chunks whose prefixes pass the test
        int c = 0;
        if (regular) {
#pragma unroll
            for (int i = 0; i < 4; ++i) c += __popcll(__builtin_amdgcn_ballot_w64(lane * 4 + i < n_chunks && test(pc[i], pm[i])));
        } else {
#pragma unroll 1
            for (int at = lane; at < MAX_CHUNKS; at += 64) c += __popcll(__builtin_amdgcn_ballot_w64(test(sh.cnt[at], sh.mass[at])));
        }
        return c;
    };
    struct Inside {          // a chunk, entry by entry of its keys
        unsigned n, upto;    // this lane's key: entries, entries of the row up to and with it
        double w, before;    // weight of one entry, weight of the row before this key
    };
    auto look_inside = [&](int c) {
        if (!regular) count_window(c / (WINDOW / 64));
        const Entries e = entries_at(c * 64 + lane);
        Inside x;
        x.n = e.n;
        x.w = exp2_neg(e.dl * to_log2);
        x.before = sh.mass[c] + lane_before(wave_scan(x.n * x.w));
        x.upto = sh.cnt[c] + wave_scan(x.n);
        return x;
    };
    auto chunk_of_rank = [&](unsigned k) {           // chunk that holds the k-th entry (k >= 1)
        return chunks_before([&](unsigned c, double) { return c < k; }) - 1;
    };

    if (wave == 0 || !regular) {
        unsigned kept = top_k > 0 && (unsigned)top_k < N ? (unsigned)top_k : N;
        double total = sh.total_mass;                              // weight of the first `kept` entries
        if (!(T > 0.0)) kept = 1u;                                 // the largest logit, lowest index
        if (kept == 1u) {
            total = 1.0;
        } else if (kept < N) {
            const Inside x = look_inside(chunk_of_rank(kept));
            const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(x.upto >= kept && x.n != 0u));
            total = from_lane(x.before + (double)(kept - (x.upto - x.n)) * x.w, at);
        }
        if (top_p < 1.0 && kept > 1u) {
            const double x = top_p * total;
            const Inside y = look_inside(max(chunks_before([&](unsigned, double w) { return w < x; }) - 1, 0));
            // the first key of the chunk whose own entries reach x (none: x is a rounding short of the next chunk)
            const uint64_t reach = __builtin_amdgcn_ballot_w64(y.n != 0u && y.before + y.n * y.w >= x);
            if (reach != 0) {
                const int at = __builtin_ctzll(reach);
                const double w = from_lane(y.w, at), before = from_lane(y.before, at);
                const unsigned n = from_lane(y.n, at), upto = from_lane(y.upto, at);
                unsigned j = w > 0.0 ? (unsigned)fmin(fmax(ceil((x - before) / w), 1.0), (double)n) : 1u;
                while (j > 1u && before + (double)(j - 1u) * w >= x) --j;
                while (j < n && before + (double)j * w < x) ++j;
                if (upto - n + j < kept) {
                    kept = upto - n + j;
                    total = before + (double)j * w;
                }
            } else if (from_lane(y.upto, 63) < kept) {
                kept = max(from_lane(y.upto, 63), 1u);
                total = from_lane(y.before + y.n * y.w, 63);
            }
        }
        if (min_p > 0.0 && kept > 1u) {
            // the first position whose weight is below min_p: weights fall along the positions, 64 probes a round.
            // Compared before the exponential: min_p = 1 keeps exactly the entries that equal the largest, whatever T.
            const double edge = T * log(min_p);
            auto below = [&](int p) { return value_at(p) == m ? 0.0 : (double)value_at(p) - (double)m; };
            int cut = 0, hi = n_pos;
            while (cut < hi) {
                const int step = (hi - cut + 63) / 64, s = cut + (lane + 1) * step - 1;
                const uint64_t fails = __builtin_amdgcn_ballot_w64(s >= hi || below(s) < edge);
                const int f = fails ? __builtin_ctzll(fails) : 64;
                hi = min(hi, cut + (f + 1) * step - 1);
                cut = cut + f * step;
            }
            if (cut < n_pos) {
                const Inside x = look_inside(cut / 64);
                const unsigned nm = from_lane(x.upto - x.n, cut & 63);
                if (nm < kept) {
                    kept = max(nm, 1u);
                    total = nm > 0u ? from_lane(x.before, cut & 63) : 1.0;
                }
            }
        }
        const double x = u * total;
        int c = max(chunks_before([&](unsigned, double w) { return w <= x; }) - 1, 0);
        Inside y = look_inside(c);
        const uint64_t over = __builtin_amdgcn_ballot_w64(y.n != 0u && y.before + y.n * y.w > x);
        int at = 0;
        unsigned rank = from_lane(y.upto, 63) + 1u;                // 1-based; as it stands: x rounds up to the chunk's end
        if (over != 0) {
            at = __builtin_ctzll(over);
            const double w = from_lane(y.w, at), before = from_lane(y.before, at);
            const unsigned n = from_lane(y.n, at), upto = from_lane(y.upto, at);
            unsigned j = w > 0.0 ? (unsigned)fmin(fmax((x - before) / w, 0.0), (double)(n - 1u)) : 0u;
            while (j > 0u && before + (double)j * w > x) --j;
            while (j + 1u < n && before + (double)(j + 1u) * w <= x) ++j;
            rank = upto - n + j + 1u;
        }
        if (over == 0 || rank > kept) {                            // (a rounding past the last kept entry)
            rank = min(rank, kept);
            c = chunk_of_rank(rank);
            y = look_inside(c);
            at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(y.n != 0u && y.upto >= rank));
        }
        if (wave == 0 && lane == at) {
            sh.j = (int)(rank - (y.upto - y.n) - 1u);
            sh.tied = (int)y.n;
            sh.value = value_at(c * 64 + lane);
            sh.prob = (float)(y.w / total);
        }
    }
    __syncthreads();

    // ---- the j-th entry of that value, in index order ----
    const float value = sh.value;
    const unsigned bits = __float_as_uint(value) >> 16;
    const unsigned pat = bits * 0x00010001u;
    const unsigned msk = bits == 0u ? 0x7FFF7FFFu : 0xFFFFFFFFu;      // zero: either sign
    const bool single = sh.tied == 1;            // (uniform)
    auto differs = [&](unsigned w) { return (w ^ pat) & msk; };               // zero in a half: a match
    auto nearest = [&](u32x4 t) {                                             // zero in a half: a match in that half of some word
        return __builtin_elementwise_min(__builtin_elementwise_min(halves(differs(t[0])), halves(differs(t[1]))),
                                         __builtin_elementwise_min(halves(differs(t[2])), halves(differs(t[3]))));
    };
    auto any_match = [](u16x2 least) { return zero_halves(__builtin_bit_cast(unsigned, least)) != 0u; };
    auto matches = [&](u32x4 t) {                                             // sums of the packed halves: at most 4 a half
        const unsigned h = zero_halves(differs(t[0])) + zero_halves(differs(t[1])) + zero_halves(differs(t[2])) + zero_halves(differs(t[3]));
        return (h & 0xFFFFu) + (h >> 16);
    };
    // the token: the entry of chunk `slot` of this lane that matches after `skip` others
    auto take = [&](u32x4 t, int slot, unsigned skip) {
        unsigned ahead = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool match = ((e & 1) ? bf16hi(t[e >> 1]) : bf16lo(t[e >> 1])) == value;
            if (match && ahead == skip) sh.token = (tid + slot * THREADS) * 8 - off + e;
            ahead += match;
        }
    };
    const bool more = HELD < SLOTS && chunks > HELD * THREADS;                // (uniform)
    if (single) {
        int slot = -1;
#pragma unroll
        for (int g = 0; g < HELD; g += 4) {      // most waves hold no match: four chunks are ruled out at a time
            u16x2 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = nearest(q[g + i]);
            if (__builtin_amdgcn_ballot_w64(any_match(__builtin_elementwise_min(__builtin_elementwise_min(x[0], x[1]), __builtin_elementwise_min(x[2], x[3])))) == 0) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (any_match(x[i])) slot = g + i;
        }
        if (slot >= 0) {
            u32x4 t = q[0];
#pragma unroll
            for (int i = 1; i < HELD; ++i)
                if (i == slot) t = q[i];
            take(t, slot, 0u);
        }
        if (more) {
            __syncthreads();
            if (sh.token < 0)
                rest([&](int i, u32x4 t) {
                    if (any_match(nearest(t))) take(t, i, 0u);
                });
        }
    } else {
        // matches of every slot, row-wide; then of the lanes of the slot that holds the entry
#pragma unroll
        for (int i = 0; i < HELD; i += 2) {      // (two slots' totals in one scan, 16 bits each)
            const unsigned sum = wave_scan(matches(q[i]) | matches(q[i + 1]) << 16);
            if (lane == 63 && sum) {
                atomicAdd(&sh.slot_tot[i], sum & 0xFFFFu);
                atomicAdd(&sh.slot_tot[i + 1], sum >> 16);
            }
        }
        __syncthreads();
        unsigned upto = wave_scan(lane < SLOTS ? sh.slot_tot[lane & (SLOTS - 1)] : 0u);
        if (more && from_lane(upto, 63) <= (unsigned)sh.j) {      // (uniform)
            __syncthreads();
            rest([&](int i, u32x4 t) {
                const unsigned n = matches(t);
                if (n) atomicAdd(&sh.slot_tot[i], n);
            });
            __syncthreads();
            upto = wave_scan(lane < SLOTS ? sh.slot_tot[lane & (SLOTS - 1)] : 0u);
        }
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > (unsigned)sh.j));
        const unsigned left = (unsigned)sh.j - from_lane(lane_before(upto), at);
        u32x4 here = ninf;
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (i == at) here = q[i];
        if (at >= HELD && tid + at * THREADS < chunks) here = row_chunk<EPI>(lc, lu, (tid + at * THREADS) * 8 - off, V, a.cfg1, excl_all);
        const unsigned n_here = matches(here);
        const unsigned incl = wave_scan(n_here);
        if (lane == 63) sh.wave_tot[wave] = incl;
        __syncthreads();
        const unsigned waves = wave_scan(lane < NWV ? sh.wave_tot[lane & (NWV - 1)] : 0u);
        const unsigned before = from_lane(lane_before(waves), wave) + incl - n_here;
        if (left >= before && left < before + n_here) take(here, at, left - before);
    }
    __syncthreads();

    if constexpr (EPI) {
        // ---- generate.py:103-123 on the row's temperature-1 softmax, from the histogram ----
        const llada_remask_args& r = a.r;
        const int token = sh.token;
        // f(entries) for every position that has some, dealt to the threads
        auto each_position = [&](auto&& f) {
            for (int win = 0; win < (regular ? 1 : WINDOWS); ++win) {
                if (!regular) count_window(win);
                const int p_lo = regular ? 0 : win * WINDOW, p_hi = regular ? n_pos : p_lo + WINDOW;
#pragma unroll 1
                for (int p = p_lo + tid; p < p_hi; p += THREADS) {
                    const Entries x = entries_at(p);
                    if (x.n) f(x);
                }
            }
        };
        // the largest value that this softmax sees: the row's, unless that is an entry it does not see, which may stand too far
        // above the others for their exponentials to be taken from there
        float mc = m;
        if (m == lx_excl[0] || m == lx_excl[1]) {
            mc = -INFINITY;
            each_position([&](const Entries& x) {
                if (seen(x.n, x.v) != 0u) mc = fmaxf(mc, x.v);
            });
            mc = wave_reduce_max(mc);
            if (lane == 0) sh.conf[wave] = mc;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NWV; ++w) mc = fmaxf(mc, (float)sh.conf[w]);
            __syncthreads();
            s_sum = 0.0;
            each_position([&](const Entries& x) {
                if (seen(x.n, x.v) != 0u) s_sum += seen(x.n, x.v) * exp((double)x.v - (double)mc);
            });
        }
        s_sum = wave_total(s_sum);
        if (lane == 0) sh.conf[wave] = s_sum;
        __syncthreads();
        double S = 0.0;
#pragma unroll
        for (int w = 0; w < NWV; ++w) S += sh.conf[w];
        bool broken = mc == -INFINITY;               // (uniform)
        if (sh.broken != 0) {                        // does this softmax see it?
            bool any = false;
            for (int c = tid; c < chunks; c += THREADS) {
                const u32x4 t = row_chunk<EPI>(lc, lu, c * 8 - off, V, a.cfg1, excl_all);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const unsigned bits = (e & 1) ? t[e >> 1] >> 16 : t[e >> 1] & 0xFFFFu;
                    const int v = c * 8 - off + e;
                    any |= (bits == 0x7F80u || (bits & 0x7FFFu) > 0x7F80u) && v != excl_conf[0] && v != excl_conf[1];
                }
            }
            const bool in_wave = __builtin_amdgcn_ballot_w64(any) != 0;
            if (lane == 0) sh.first[wave] = in_wave;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NWV; ++w) broken |= sh.first[w] != 0;
        }
        if (broken) {
            conf = __builtin_nanf("");               // it is NaN all over
        } else if (r.remasking == LLADA_REMASK_LOW_CONFIDENCE || r.remasking == LLADA_REMASK_HIGH_CONFIDENCE) {
            const double dl = value == mc ? 0.0 : (double)value - (double)mc;
            const float pf = token == excl_conf[0] || token == excl_conf[1] ? 0.f : (float)(exp(dl) / S);
            const bool f32 = (r.flags & LLADA_FLAG_CONF_FLOAT32) != 0;
            const float p = f32 ? pf : round_bf16(pf);
            conf = r.remasking == LLADA_REMASK_LOW_CONFIDENCE ? p : (f32 ? 1.0f - p : round_bf16(1.0f - p));
        } else {
            // sum of bf16(log p) bf16(p), both rounded first, over the row: per distinct value, times its count
            const double lse = log(S);
            double es = 0.0;
            auto term = [&](double dl) {
                const float p = round_bf16((float)(exp(dl) / S)), lp = round_bf16((float)(dl - lse));
                return (double)round_bf16(lp * p);
            };
            each_position([&](const Entries& x) {
                if (seen(x.n, x.v) != 0u) es += seen(x.n, x.v) * term(m == mc ? x.dl : (double)x.v - (double)mc);
            });
            es = wave_total(es);
            __syncthreads();
            if (lane == 0) sh.conf[wave] = es;
            __syncthreads();
            double tot = 0.0;
#pragma unroll
            for (int w = 0; w < NWV; ++w) tot += sh.conf[w];
            const float t = round_bf16((float)tot);
            conf = r.remasking == LLADA_REMASK_LOW_ENTROPY ? -t : t;
        }
    }
}

// One workgroup per row.
template <bool EPI, bool WHOLE, bool GUIDED>
__global__ void __launch_bounds__(Shape<WHOLE>::THREADS, 4) sample_rows_kernel(const SampleArgs a) {
    using L = Shape<WHOLE>;
    __shared__ __attribute__((aligned(16))) unsigned lds[L::LDS_WORDS];
    typename L::Shared& sh = *(typename L::Shared*)(lds + L::REST_AT);
    const int row = blockIdx.x;
    const int tid = threadIdx.x;
    int pos = row, b = row, col = 0;
    if constexpr (EPI) {
        pos = a.r.row_pos ? a.r.row_pos[row] : row;
        b = pos / a.r.L;
        col = pos - b * a.r.L;
        if (a.r.x[pos] != a.r.mask_id || col >= a.r.block_end) return;      // the defaults stand (uniform)
    }
    double T = a.s.row_temperature ? (double)a.s.row_temperature[b] : a.s.temperature;
    if (T > MAX_TEMPERATURE) T = MAX_TEMPERATURE;
    const int top_k = a.s.row_top_k ? a.s.row_top_k[b] : a.s.top_k;
    const double top_p = a.s.row_top_p ? (double)a.s.row_top_p[b] : a.s.top_p;
    const double min_p = a.s.row_min_p ? (double)a.s.row_min_p[b] : a.s.min_p;
    double u;
    if (a.s.uniforms) {
        u = a.s.uniforms[pos];
    } else {
        uint32_t k0, k1;
        philox_key(a.seed, LLADA_STREAM_SAMPLE, k0, k1);
        const Philox4 ph = philox4x32_10(0u, (uint32_t)col, a.row_offset + (uint32_t)b, a.step, k0, k1);
        u = u53(ph.v[0], ph.v[1]);
    }
    const bf16_t* lc = a.logits + (size_t)row * (size_t)a.stride;
    const bf16_t* lu = a.uncond ? a.uncond + (size_t)row * (size_t)a.stride : nullptr;
    const int ex_all = EPI && (a.r.flags & LLADA_FLAG_LOGITS_EOS_INF) ? a.r.eos_id : -1;
    // EOT, and at temperature 0, where the noisy copy that loses EOS is the logits themselves, EOS (generate.py:100-101)
    const bool no_eot = EPI && (a.r.flags & LLADA_FLAG_CONF_EOS_EOT_INF) != 0;
    const int ex_conf[2] = {no_eot && a.r.eot_id != ex_all ? a.r.eot_id : -1,
                            no_eot && !(T > 0.0) && a.r.eos_id != ex_all && a.r.eos_id != a.r.eot_id ? a.r.eos_id : -1};
    float conf = 0.f;
    sample_row<EPI, L, GUIDED>(a, lds, sh, lc, lu, T, top_k, top_p, min_p, u, ex_all, ex_conf, conf);
    if (tid != 0) return;
    if constexpr (EPI) {
        if (a.r.remasking == LLADA_REMASK_RANDOM) {
            if (a.r.rand_scores) {
                conf = a.r.rand_scores[pos];
            } else {
                uint32_t r0, r1;
                philox_key(a.r.seed, LLADA_STREAM_REMASK, r0, r1);
                const Philox4 ph = philox4x32_10((uint32_t)col, 0u, a.row_offset + (uint32_t)b, a.step, r0, r1);
                conf = (float)(ph.v[0] >> 8) * (1.0f / 16777216.0f);
            }
        }
        a.r.x0[pos] = (int64_t)sh.token;
        a.r.confidence[pos] = conf;
    } else {
        a.tokens[row] = (int64_t)sh.token;
        if (a.probs) a.probs[row] = sh.prob;
    }
}

// x0 = x, confidence = -inf at every position; the rows' kernel overwrites the active ones
__global__ void __launch_bounds__(256) sample_defaults_kernel(const int64_t* __restrict__ x, int64_t* __restrict__ x0,
                                                              float* __restrict__ conf, int64_t n) {
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        x0[i] = x[i];
        conf[i] = -INFINITY;
    }
}

int g_force = 0;        // test hook

constexpr int32_t MAX_LAUNCH_ROWS = 1 << 21;      // of up to 1024 lanes: a launch ends at 2^32 threads

// One workgroup a row, of the kind that pays (Shape).
template <bool EPI>
void launch_rows(const SampleArgs& a, int n_rows, hipStream_t st) {
    const bool guided = a.uncond != nullptr;
    const bool fits = a.vocab <= Shape<false>::HELD * Shape<false>::THREADS * 8 - 7;      // in half a row, wherever it starts
    const bool half = fits ? g_force != 1 : !guided && (g_force ? g_force == 2 : n_rows >= 512);
    if (half && guided)
        hipLaunchKernelGGL((sample_rows_kernel<EPI, false, true>), dim3(n_rows), dim3(Shape<false>::THREADS), 0, st, a);
    else if (half)
        hipLaunchKernelGGL((sample_rows_kernel<EPI, false, false>), dim3(n_rows), dim3(Shape<false>::THREADS), 0, st, a);
    else if (guided)
        hipLaunchKernelGGL((sample_rows_kernel<EPI, true, true>), dim3(n_rows), dim3(Shape<true>::THREADS), 0, st, a);
    else
        hipLaunchKernelGGL((sample_rows_kernel<EPI, true, false>), dim3(n_rows), dim3(Shape<true>::THREADS), 0, st, a);
}

int check_sampling(const char* who, const llada_sampling* s) {
    LLADA_CHECK_ARG(s != nullptr, "%s: null sampling parameters", who);
    LLADA_CHECK_ARG(s->row_temperature || (s->temperature >= 0.0 && s->temperature <= MAX_TEMPERATURE), "%s: temperature %g", who, s->temperature);
    LLADA_CHECK_ARG(s->row_top_k || s->top_k >= 0, "%s: top_k %d", who, s->top_k);
    LLADA_CHECK_ARG(s->row_top_p || (s->top_p > 0.0 && s->top_p <= 1.0), "%s: top_p %g is outside (0, 1]", who, s->top_p);
    LLADA_CHECK_ARG(s->row_min_p || (s->min_p >= 0.0 && s->min_p <= 1.0), "%s: min_p %g is outside [0, 1]", who, s->min_p);
    return LLADA_OK;
}

}  // namespace

// tests: rows kept whole (1), kept by half where that is possible (2); 0 = automatic
extern "C" void llada_sample_rows_force(int kind) { g_force = kind; }

extern "C" int llada_sample_rows(const void* logits, const void* uncond_logits, int64_t row_stride, double cfg_scale,
                                 int32_t n_rows, int32_t vocab, const llada_sampling* sampling, uint64_t seed, uint32_t step,
                                 uint32_t row_offset, int64_t* tokens, float* probs, void* stream) {
    LLADA_CHECK_ARG(logits && tokens && n_rows > 0 && vocab > 0, "sample_rows: bad argument");
    LLADA_CHECK_ARG(row_stride >= vocab || n_rows == 1, "sample_rows: rows overlap (stride %lld, vocab %d)", (long long)row_stride, vocab);
    LLADA_CHECK_ARG((((uintptr_t)logits | (uintptr_t)uncond_logits) & 1) == 0, "sample_rows: misaligned logits");
    LLADA_CHECK_ARG(uncond_logits == nullptr || (((uintptr_t)logits ^ (uintptr_t)uncond_logits) & 15) == 0,
                    "sample_rows: uncond_logits must stand at the same offset from a 16-byte boundary as logits");
    const bool aligned = ((uintptr_t)logits & 15) == 0 && (row_stride % 8 == 0 || n_rows == 1);
    LLADA_CHECK_SUPPORTED(vocab <= ROW_MAX_VOCAB - (aligned ? 0 : 7), "sample_rows: vocab=%d: a row must fit the registers of a workgroup", vocab);
    const int rc = check_sampling("sample_rows", sampling);
    if (rc != LLADA_OK) return rc;
    SampleArgs a = {};
    a.logits = (const bf16_t*)logits;
    a.uncond = (const bf16_t*)uncond_logits;
    a.stride = row_stride;
    a.cfg1 = (float)(cfg_scale + 1.0);
    a.vocab = vocab;
    a.s = *sampling;
    a.seed = seed;
    a.step = step;
    a.row_offset = row_offset;
    a.tokens = tokens;
    a.probs = probs;
    for (int32_t done = 0;;) {
        const int32_t n = n_rows - done < MAX_LAUNCH_ROWS ? n_rows - done : MAX_LAUNCH_ROWS;
        launch_rows<false>(a, n, (hipStream_t)stream);
        LLADA_CHECK_LAUNCH("sample_rows_kernel");
        done += n;
        if (done == n_rows) return LLADA_OK;
        a.logits += (int64_t)n * row_stride;
        if (a.uncond) a.uncond += (int64_t)n * row_stride;
        if (a.s.row_temperature) a.s.row_temperature += n;
        if (a.s.row_top_k) a.s.row_top_k += n;
        if (a.s.row_top_p) a.s.row_top_p += n;
        if (a.s.row_min_p) a.s.row_min_p += n;
        if (a.s.uniforms) a.s.uniforms += n;
        a.row_offset += (uint32_t)n;
        a.tokens += n;
        if (a.probs) a.probs += n;
    }
}

extern "C" int llada_remask_scores_sampled(const llada_remask_args* args, const llada_sampling* sampling, void* stream) {
    LLADA_CHECK_ARG(args != nullptr, "remask_scores_sampled: null args");
    const llada_remask_args& r = *args;
    LLADA_CHECK_ARG(r.logits && r.x && r.x0 && r.confidence, "remask_scores_sampled: null tensor");
    LLADA_CHECK_ARG(r.n_rows > 0 && r.B > 0 && r.L > 0 && r.vocab > 0, "remask_scores_sampled: bad shape");
    LLADA_CHECK_ARG(r.row_pos != nullptr || r.n_rows == (int64_t)r.B * r.L, "remask_scores_sampled: row_pos is required unless n_rows == B*L");
    LLADA_CHECK_SUPPORTED(r.n_rows <= MAX_LAUNCH_ROWS, "remask_scores_sampled: %d rows, one launch takes %d", r.n_rows, MAX_LAUNCH_ROWS);
    LLADA_CHECK_SUPPORTED(r.vocab % 8 == 0 && r.vocab <= ROW_MAX_VOCAB, "remask_scores_sampled: vocab=%d must be a multiple of 8 up to %d", r.vocab, ROW_MAX_VOCAB);
    LLADA_CHECK_ARG((((uintptr_t)r.logits | (uintptr_t)r.uncond_logits) & 15) == 0, "remask_scores_sampled: logits must be 16-byte aligned");
    if (r.remasking < LLADA_REMASK_LOW_CONFIDENCE || r.remasking > LLADA_REMASK_RANDOM) {
        llada_set_error("remask_scores_sampled: unknown remasking rule %d", r.remasking);
        return LLADA_ERR_UNSUPPORTED;
    }
    if (r.flags & (LLADA_FLAG_LOGITS_EOS_INF | LLADA_FLAG_CONF_EOS_EOT_INF))
        LLADA_CHECK_ARG(r.eos_id >= 0 && r.eos_id < r.vocab && r.eot_id >= 0 && r.eot_id < r.vocab,
                        "remask_scores_sampled: eos/eot id outside the vocabulary");
    const int rc = check_sampling("remask_scores_sampled", sampling);
    if (rc != LLADA_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    const int64_t n = (int64_t)r.B * r.L;
    hipLaunchKernelGGL(sample_defaults_kernel, dim3((unsigned)((n + 255) / 256 < 2048 ? (n + 255) / 256 : 2048)), dim3(256), 0, st,
                       r.x, r.x0, r.confidence, n);
    LLADA_CHECK_LAUNCH("sample_defaults_kernel");
    SampleArgs a = {};
    a.logits = (const bf16_t*)r.logits;
    a.uncond = (const bf16_t*)r.uncond_logits;
    a.stride = r.vocab;
    a.cfg1 = (float)(r.cfg_scale + 1.0);
    a.vocab = r.vocab;
    a.s = *sampling;
    a.seed = r.seed;
    a.step = r.step;
    a.row_offset = r.row_offset;
    a.r = r;
    launch_rows<true>(a, r.n_rows, st);
    LLADA_CHECK_LAUNCH("sample_rows_kernel");
    return LLADA_OK;
}
