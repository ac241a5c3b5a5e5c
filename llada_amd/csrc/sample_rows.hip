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
// totals and then inside one chunk.  The row is read once and stays in registers (16 x 16 bytes a lane, 1024 lanes) for
// the last step, which turns "the j-th entry of value v" into an index.
//
// The histogram has a bin for every bf16 value of magnitude in [2^-55, 2^9) of either sign and one for zero (64 KiB).  A
// row with another finite magnitude, an infinity of positive sign or a NaN is "irregular" (its clamped bins say so, at no
// cost to other rows) and is counted over the whole 16-bit key space in four windows instead; -inf entries, NaNs
// included, have no weight and are never drawn.  A row with nothing else gives token 0 with probability 0.
#include "common.h"
#include "philox.h"
#include "rowregs.h"

namespace {

constexpr int THREADS = ROW_THREADS;                 // 1024
constexpr int SLOTS = ROW_SLOTS;                     // 16-byte chunks a lane
constexpr int NWV = THREADS / 64;
constexpr unsigned MAG_LO = 0x2400, MAG_HI = 0x4400; // magnitudes with a bin of their own: [2^-55, 2^9)
constexpr int SPAN = MAG_HI - MAG_LO;                // 8192
constexpr int PLANE = SPAN + 2;                      // bin 0: below the range (zero), SPAN + 1: above
constexpr int BINS = 2 * PLANE;                      // both signs
constexpr int REGULAR_KEYS = 2 * SPAN + 1;           // descending values: SPAN positive, zero, SPAN negative
constexpr int WINDOW = 16384;                        // irregular rows: keys counted at a time, 4 windows
constexpr int MAX_CHUNKS = 65536 / 64;
constexpr unsigned LLADA_STREAM_SAMPLE = 4u;
static_assert(WINDOW <= BINS, "a window fits the bins");

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

struct Shared {
    unsigned bins[BINS];
    unsigned cnt[MAX_CHUNKS];        // entries of a chunk of 64 keys, then: entries before it
    double mass[MAX_CHUNKS];         // their weight, then: the weight before it
    double conf[NWV];                // epilogue: partial sums of the waves
    unsigned total;
    double total_mass;
    int first[NWV];
    int irregular;
    // the drawn entry
    int key, j, tied;
    float value, prob;
    unsigned slot_tot[SLOTS];
    unsigned wave_tot[NWV];
    int token;
};

// Key s of a row's value order (0 = the largest) <-> value.  Regular rows: the histogram's own order; irregular rows: all
// bf16 patterns.
__device__ __forceinline__ float key_value(int s, bool regular) {
    if (regular) {
        if (s == SPAN) return 0.f;
        return s < SPAN ? __uint_as_float((MAG_HI - 1 - s) << 16)
                        : __uint_as_float(0x80000000u | ((MAG_LO + (s - SPAN - 1)) << 16));
    }
    const unsigned k = 65535u - (unsigned)s;
    return __uint_as_float(((k & 0x8000u) ? k ^ 0x8000u : ~k & 0xFFFFu) << 16);
}

__device__ __forceinline__ unsigned key_count(const Shared& sh, int s, bool regular) {
    if (regular) {
        if (s >= REGULAR_KEYS) return 0u;
        if (s == SPAN) return sh.bins[0] + sh.bins[PLANE];
        return s < SPAN ? sh.bins[SPAN - s] : sh.bins[PLANE + (s - SPAN)];
    }
    return sh.bins[s & (WINDOW - 1)];
}

// irregular rows: key of a bf16 pattern, -1 for an entry without weight (-inf, NaN); -0 counts as +0
__device__ __forceinline__ int full_key(unsigned bits) {
    if (bits == 0x8000u) bits = 0u;
    if ((bits & 0x7FFFu) > 0x7F80u || bits == 0xFF80u) return -1;
    return 65535 - (int)((bits & 0x8000u) ? ~bits & 0xFFFFu : bits | 0x8000u);
}

__device__ __forceinline__ double wave_scan(double v, int lane) {      // inclusive, fixed order
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double t = __shfl_up(v, o);
        if (lane >= o) v += t;
    }
    return v;
}
__device__ __forceinline__ unsigned wave_scan(unsigned v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned t = __shfl_up(v, o);
        if (lane >= o) v += t;
    }
    return v;
}
__device__ __forceinline__ double wave_total(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// (by value: a bit cast straight from a vector's element reads the vector's first)
__device__ __forceinline__ u16x2 halves(unsigned w) { return __builtin_bit_cast(u16x2, w); }

// entries v0 .. v0 + 7 of a row, -inf outside it; `vector`: v0 stands at a 16-byte boundary
__device__ __forceinline__ u32x4 load_chunk(const bf16_t* row, int v0, int vocab, bool vector) {
    if (vector && v0 >= 0 && v0 + 8 <= vocab) return __builtin_nontemporal_load((const u32x4*)(row + v0));
    u32x4 t = {BF16_NEG_INF2, BF16_NEG_INF2, BF16_NEG_INF2, BF16_NEG_INF2};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int v = v0 + e;
        if (v < 0 || v >= vocab) continue;
        const unsigned bits = row[v];
        t[e >> 1] = (e & 1) ? (t[e >> 1] & 0xFFFFu) | bits << 16 : (t[e >> 1] & 0xFFFF0000u) | bits;
    }
    return t;
}

// Draws the token of one row.  EPI: also leaves the row's confidence (rules of llada_remask_scores) in `conf`.
template <bool EPI>
__device__ __forceinline__ void sample_row(const SampleArgs& a, Shared& sh, const bf16_t* lc, const bf16_t* lu, double T, int top_k,
                                           double top_p, double min_p, double u, int excl_all, int excl_conf, float& conf) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int V = a.vocab;
    // The row in registers: chunk c = lane + 1024 i holds entries 8 c - off .. + 7, off = the row's offset from a 16-byte
    // boundary in entries, so that all but its first and last chunk are one aligned load.
    const int off = (int)(((uintptr_t)lc >> 1) & 7);
    const bool uvec = lu && (int)(((uintptr_t)lu >> 1) & 7) == off;
    const int chunks = (V + off + 7) / 8;

    for (int i = tid; i < BINS; i += THREADS) sh.bins[i] = 0u;
    if (tid < SLOTS) sh.slot_tot[tid] = 0u;
    if (tid == 0) sh.irregular = 0;

    // one chunk of the row as the draw sees it: combined under guidance; what lies outside the row, and the entry that is
    // taken out of everything (EOS removed before the draw), as -inf
    auto put = [](u32x4 t, int e, unsigned bits) {
#pragma unroll
        for (int w = 0; w < 8; ++w)
            if (w == e) t[w >> 1] = (w & 1) ? (t[w >> 1] & 0xFFFFu) | bits << 16 : (t[w >> 1] & 0xFFFF0000u) | bits;
        return t;
    };
    auto finish_chunk = [&](u32x4 t, int c) {
        const int v0 = c * 8 - off;
        if (lu) {
            const u32x4 b = load_chunk(lu, v0, V, uvec);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                t[e] = pack_bf16x2(cfg_combine(bf16lo(t[e]), bf16lo(b[e]), a.cfg1), cfg_combine(bf16hi(t[e]), bf16hi(b[e]), a.cfg1));
            if (v0 < 0 || v0 + 8 > V) {          // the combination of two -inf is a NaN
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (v0 + e < 0 || v0 + e >= V) t = put(t, e, 0xFF80u);
            }
        }
        if (EPI && excl_all >= 0 && (excl_all + off) >> 3 == c) t = put(t, (excl_all + off) & 7, 0xFF80u);
        return t;
    };
    const u32x4 ninf = {BF16_NEG_INF2, BF16_NEG_INF2, BF16_NEG_INF2, BF16_NEG_INF2};
    u32x4 q[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        const int c = tid + i * THREADS;
        q[i] = c < chunks ? load_chunk(lc, c * 8 - off, V, true) : ninf;
    }
    if (lu || (EPI && excl_all >= 0)) {
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            const int c = tid + i * THREADS;
            if (c < chunks) q[i] = finish_chunk(q[i], c);
        }
    }
    // an entry the confidence's softmax does not see although it can be drawn (generate.py:100-101)
    float lx_excl = -INFINITY;
    if (EPI && excl_conf >= 0) {
        lx_excl = bf16_to_f32(lc[excl_conf]);
        if (lu) lx_excl = cfg_combine(lx_excl, bf16_to_f32(lu[excl_conf]), a.cfg1);
    }
    // entries of a key that this softmax sees
    auto seen = [&](unsigned n, float v) { return n - (v == lx_excl ? 1u : 0u); };
    __syncthreads();

    // ---- the histogram: clamped magnitudes, both signs ----
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        if (tid + i * THREADS >= chunks) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const u16x2 w = halves(q[i][e]);
            const u16x2 mag = w & (unsigned short)0x7FFF;
            const u16x2 idx = __builtin_elementwise_min(__builtin_elementwise_sub_sat(mag, (u16x2)((unsigned short)(MAG_LO - 1))),
                                                        (u16x2)((unsigned short)(SPAN + 1)));
            const u16x2 at = (w >> (unsigned short)15) * (unsigned short)PLANE + idx;
            atomicAdd(&sh.bins[at[0]], 1u);
            atomicAdd(&sh.bins[at[1]], 1u);
        }
    }
    __syncthreads();
    // clamped bins that are not empty: zeros and -inf are as good as binned, anything else makes the row irregular
    if (sh.bins[0] + sh.bins[PLANE] + sh.bins[SPAN + 1] + sh.bins[PLANE + SPAN + 1] != 0u) {
        // smallest magnitude above zero, largest positive pattern, largest negative one but -inf
        const u16x2 one = {1, 1}, minus_inf = {0xFF80, 0xFF80};
        u16x2 least = {0xFFFF, 0xFFFF}, neg = {0, 0};
        s16x2 pos = {0, 0};
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u16x2 w = halves(q[i][e]);
                least = __builtin_elementwise_min(least, (w & (unsigned short)0x7FFF) - one);
                pos = __builtin_elementwise_max(pos, __builtin_bit_cast(s16x2, w));
                neg = __builtin_elementwise_max(neg, w * __builtin_elementwise_min(w ^ minus_inf, one));
            }
        const bool bad = min(least[0], least[1]) < MAG_LO - 1 || (unsigned)max(pos[0], pos[1]) >= MAG_HI ||
                         max(neg[0], neg[1]) >= 0x8000u + MAG_HI;
        if (__builtin_amdgcn_ballot_w64(bad) != 0 && lane == 0) sh.irregular = 1;
    }
    __syncthreads();
    const bool regular = sh.irregular == 0;
    const int n_chunks = regular ? (REGULAR_KEYS + 63) / 64 : MAX_CHUNKS;

    // An irregular row: counts one window of its keys into the bins, from memory again (such rows are rare and the
    // row's registers are better left alone).  All threads call it together.
    auto count_window = [&](int win) {
        __syncthreads();
        for (int i = tid; i < WINDOW; i += THREADS) sh.bins[i] = 0u;
        __syncthreads();
#pragma unroll 1
        for (int c = tid; c < chunks; c += THREADS) {
            const u32x4 t = finish_chunk(load_chunk(lc, c * 8 - off, V, true), c);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int k = full_key((e & 1) ? t[e >> 1] >> 16 : t[e >> 1] & 0xFFFFu);
                if (k >= 0 && k / WINDOW == win) atomicAdd(&sh.bins[k & (WINDOW - 1)], 1u);
            }
        }
        __syncthreads();
    };

    // ---- totals of the chunks: entries, weight; the largest value on the way ----
    int top_key = 0x7fffffff;
    float m = 0.f;
    double s_sum = 0.0;              // epilogue: sum of exp(l - m) over the row
    for (int win = 0; win < (regular ? 1 : 4); ++win) {
        if (!regular) count_window(win);
        const int c_lo = regular ? 0 : win * (WINDOW / 64), c_hi = regular ? n_chunks : c_lo + WINDOW / 64;
        if (top_key == 0x7fffffff) {
            int mine = 0x7fffffff;
            for (int c = c_lo + wave; c < c_hi; c += NWV) {
                const uint64_t any = __builtin_amdgcn_ballot_w64(key_count(sh, c * 64 + lane, regular) != 0u);
                if (any != 0 && mine == 0x7fffffff) mine = c * 64 + __builtin_ctzll(any);
            }
            if (lane == 0) sh.first[wave] = mine;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NWV; ++w) top_key = min(top_key, sh.first[w]);
            if (top_key != 0x7fffffff) m = key_value(top_key, regular);
            __syncthreads();
        }
        for (int c = c_lo + wave; c < c_hi; c += NWV) {
            const unsigned n = key_count(sh, c * 64 + lane, regular);
            if (__builtin_amdgcn_ballot_w64(n != 0u) == 0) {
                if (lane == 0) {
                    sh.cnt[c] = 0u;
                    sh.mass[c] = 0.0;
                }
                continue;
            }
            const float v = key_value(c * 64 + lane, regular);
            const double dl = v == m ? 0.0 : (double)v - (double)m;
            const double wgt = T > 0.0 ? exp(dl / T) : (v == m ? 1.0 : 0.0);
            const double ms = wave_scan(n ? n * wgt : 0.0, lane);
            const unsigned cs = wave_scan(n, lane);
            if (lane == 63) {
                sh.cnt[c] = cs;
                sh.mass[c] = ms;
            }
            if (EPI) s_sum += n ? seen(n, v) * exp(dl) : 0.0;
        }
    }
    __syncthreads();

    // key s: its value minus the largest, its weight
    auto distance = [&](int s) {
        const float v = key_value(s, regular);
        return v == m ? 0.0 : (double)v - (double)m;
    };
    auto weight = [&](int s) {
        const double dl = distance(s);
        return T > 0.0 ? exp(dl / T) : (dl == 0.0 ? 1.0 : 0.0);
    };

    // ---- exclusive prefixes over the chunks (one wave, 64 chunks at a time) ----
    if (wave == 0) {
        unsigned cb = 0;
        double qb = 0.0;
#pragma unroll 1
        for (int at = lane; at < (n_chunks + 63) / 64 * 64; at += 64) {
            const unsigned c = at < n_chunks ? sh.cnt[at] : 0u;
            const double w = at < n_chunks ? sh.mass[at] : 0.0;
            const unsigned ci = wave_scan(c, lane);
            const double wi = wave_scan(w, lane);
            double we = __shfl_up(wi, 1);
            if (lane == 0) we = 0.0;
            sh.cnt[at] = cb + ci - c;
            sh.mass[at] = qb + we;
            cb += __shfl(ci, 63);
            qb += __shfl(wi, 63);
        }
        if (lane == 0) {
            sh.total = cb;
            sh.total_mass = qb;
        }
    }
    __syncthreads();
    const unsigned N = sh.total;
    if (N == 0u) {                       // nothing but -inf
        if (tid == 0) {
            sh.token = 0;
            sh.prob = 0.f;
        }
        conf = 0.f;
        __syncthreads();
        return;
    }

    // An irregular row's bins hold one window: count the one that holds chunk c again (uniform over the workgroup).
    // A regular row's searches run in wave 0 alone, an irregular row's with every wave following.
    auto chunk_of_count = [&](unsigned k) {          // chunk that holds the k-th entry (k >= 1)
        int c = 0;
#pragma unroll 1
        for (int at = lane; at < (n_chunks + 63) / 64 * 64; at += 64) {
            c += __popcll(__builtin_amdgcn_ballot_w64(at < n_chunks && sh.cnt[at] < k));
        }
        return c - 1;
    };
    auto chunk_of_mass = [&](double x, bool strict) {  // last chunk whose prefix is below x (strict: at most x)
        int c = 0;
#pragma unroll 1
        for (int at = lane; at < (n_chunks + 63) / 64 * 64; at += 64) {
            const bool before = at < n_chunks && (strict ? sh.mass[at] <= x : sh.mass[at] < x);
            c += __popcll(__builtin_amdgcn_ballot_w64(before));
        }
        return c > 0 ? c - 1 : 0;
    };
    struct Inside {          // a chunk, entry by entry of its keys
        unsigned n, upto;    // this lane's key: entries, entries of the row up to and with it
        double w, before;    // weight of one entry, weight of the row before this key
    };
    auto look_inside = [&](int c) {
        if (!regular) count_window(c / (WINDOW / 64));
        Inside x;
        x.n = key_count(sh, c * 64 + lane, regular);
        x.w = x.n ? weight(c * 64 + lane) : 0.0;
        const double own = x.n ? x.n * x.w : 0.0;
        const double incl = wave_scan(own, lane);
        double ex = __shfl_up(incl, 1);
        if (lane == 0) ex = 0.0;
        x.before = sh.mass[c] + ex;
        x.upto = sh.cnt[c] + wave_scan(x.n, lane);
        return x;
    };
    // weight of the first k entries of the row (1 <= k <= N)
    auto mass_of = [&](unsigned k) {
        if (k >= N) return sh.total_mass;
        const Inside x = look_inside(chunk_of_count(k));
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(x.upto >= k && x.n != 0u));
        return __shfl(x.before + (double)(k - (x.upto - x.n)) * x.w, at);
    };

    if (wave == 0 || !regular) {
        unsigned kept = top_k > 0 && (unsigned)top_k < N ? (unsigned)top_k : N;
        if (!(T > 0.0)) kept = 1u;                                 // the largest logit, lowest index
        if (top_p < 1.0 && kept > 1u) {
            const double x = top_p * mass_of(kept);
            int c = chunk_of_mass(x, false);
            const Inside y = look_inside(c);
            // the first key of the chunk whose own entries reach x (none: x is a rounding short of the next chunk)
            const uint64_t reach = __builtin_amdgcn_ballot_w64(y.n != 0u && y.before + y.n * y.w >= x);
            if (reach != 0) {
                const int at = __builtin_ctzll(reach);
                const double w = __shfl(y.w, at), before = __shfl(y.before, at);
                const unsigned n = __shfl(y.n, at), upto = __shfl(y.upto, at);
                unsigned j = w > 0.0 ? (unsigned)fmin(fmax(ceil((x - before) / w), 1.0), (double)n) : 1u;
                while (j > 1u && before + (double)(j - 1u) * w >= x) --j;
                while (j < n && before + (double)j * w < x) ++j;
                kept = min(kept, upto - n + j);
            } else {
                kept = max(min(kept, __shfl(y.upto, 63)), 1u);
            }
        }
        if (min_p > 0.0 && kept > 1u) {
            // the first key whose weight is below min_p: weights fall with the key, 64 probes a round.  Compared before the
            // exponential: min_p = 1 keeps exactly the entries that equal the largest, whatever T.
            const double edge = T * log(min_p);
            int cut = 0, hi = regular ? REGULAR_KEYS : 65536;
            const int keys = hi;
            while (cut < hi) {
                const int step = (hi - cut + 63) / 64, s = cut + (lane + 1) * step - 1;
                const uint64_t fails = __builtin_amdgcn_ballot_w64(s >= hi || distance(s) < edge);
                const int f = fails ? __builtin_ctzll(fails) : 64;
                hi = min(hi, cut + (f + 1) * step - 1);
                cut = cut + f * step;
            }
            unsigned nm = N;
            if (cut < keys) {
                const int c = cut / 64;
                const Inside x = look_inside(c);
                nm = __shfl(x.upto - x.n, cut & 63);
            }
            kept = min(kept, nm > 0u ? nm : 1u);
        }
        const double total = mass_of(kept);
        const double x = u * total;
        const int c = chunk_of_mass(x, true);
        const Inside y = look_inside(c);
        const uint64_t over = __builtin_amdgcn_ballot_w64(y.n != 0u && y.before + y.n * y.w > x);
        unsigned rank = min(kept, __shfl(y.upto, 63) + 1u);        // 1-based; as it stands: x rounds up to the chunk's end
        if (over != 0) {
            const int at = __builtin_ctzll(over);
            const double w = __shfl(y.w, at), before = __shfl(y.before, at);
            const unsigned n = __shfl(y.n, at), upto = __shfl(y.upto, at);
            unsigned j = w > 0.0 ? (unsigned)fmin(fmax((x - before) / w, 0.0), (double)(n - 1u)) : 0u;
            while (j > 0u && before + (double)j * w > x) --j;
            while (j + 1u < n && before + (double)(j + 1u) * w <= x) ++j;
            rank = min(kept, upto - n + j + 1u);
        }
        // the key and place of that rank
        const Inside z = look_inside(chunk_of_count(rank));
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(z.n != 0u && z.upto >= rank));
        const int cz = chunk_of_count(rank);
        if (wave == 0 && lane == at) {
            sh.key = cz * 64 + lane;
            sh.j = (int)(rank - (z.upto - z.n) - 1u);
            sh.tied = (int)z.n;
            sh.value = key_value(cz * 64 + lane, regular);
            sh.prob = (float)(z.w / total);
        }
    }
    __syncthreads();

    // ---- the j-th entry of that value, in index order ----
    const float value = sh.value;
    unsigned mine[SLOTS / 4];                    // matches of each chunk, a byte each
#pragma unroll
    for (int i = 0; i < SLOTS / 4; ++i) mine[i] = 0u;
    {
        const unsigned bits = __float_as_uint(value) >> 16;
        const unsigned pat = bits * 0x00010001u, msk = bits == 0u ? 0x7FFF7FFFu : 0xFFFFFFFFu;    // zero: either sign
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            u16x2 miss = {0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                miss += __builtin_elementwise_min(halves((q[i][e] ^ pat) & msk), (u16x2)((unsigned short)1));
            mine[i >> 2] |= (8u - (unsigned)(miss[0] + miss[1])) << (8 * (i & 3));
        }
    }
    if ((mine[0] | mine[1] | mine[2] | mine[3]) != 0u) {
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            const unsigned n = (mine[i >> 2] >> (8 * (i & 3))) & 255u;
            if (n) atomicAdd(&sh.slot_tot[i], n);
        }
    }
    __syncthreads();
    unsigned left = (unsigned)sh.j;
    int slot = 0;
#pragma unroll 1
    while (slot < SLOTS - 1 && left >= sh.slot_tot[slot]) left -= sh.slot_tot[slot++];
    unsigned n_here = 0;
    u32x4 here = ninf;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
        if (i == slot) {
            n_here = (mine[i >> 2] >> (8 * (i & 3))) & 255u;
            here = q[i];
        }
    const unsigned incl = wave_scan(n_here, lane);
    if (lane == 63) sh.wave_tot[wave] = incl;
    __syncthreads();
    unsigned before = incl - n_here;
#pragma unroll 1
    for (int w = 0; w < wave; ++w) before += sh.wave_tot[w];
    if (left >= before && left < before + n_here) {
        unsigned skip = left - before;
        int found = 0;
#pragma unroll
        for (int e = 7; e >= 0; --e) {
            // entries are scanned downwards: the (n_here - 1 - skip)-th match from the end
            const float v = (e & 1) ? bf16hi(here[e >> 1]) : bf16lo(here[e >> 1]);
            if (v == value) {
                if (n_here - 1u == skip) found = e;
                --n_here;
            }
        }
        sh.token = (tid + slot * THREADS) * 8 - off + found;
    }
    __syncthreads();

    if constexpr (EPI) {
        // ---- generate.py:103-123 on the row's temperature-1 softmax, from the histogram ----
        const llada_remask_args& r = a.r;
        const int token = sh.token;
        s_sum = wave_total(s_sum);
        if (lane == 0) sh.conf[wave] = s_sum;
        __syncthreads();
        double S = 0.0;
#pragma unroll
        for (int w = 0; w < NWV; ++w) S += sh.conf[w];
        if (r.remasking == LLADA_REMASK_LOW_CONFIDENCE || r.remasking == LLADA_REMASK_HIGH_CONFIDENCE) {
            const double dl = value == m ? 0.0 : (double)value - (double)m;
            const float pf = token == excl_conf ? 0.f : (float)(exp(dl) / S);
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
            for (int win = 0; win < (regular ? 1 : 4); ++win) {
                if (!regular) count_window(win);
                const int c_lo = regular ? 0 : win * (WINDOW / 64), c_hi = regular ? n_chunks : c_lo + WINDOW / 64;
                for (int c = c_lo + wave; c < c_hi; c += NWV) {
                    const unsigned n = key_count(sh, c * 64 + lane, regular);
                    if (n == 0u) continue;
                    const float v = key_value(c * 64 + lane, regular);
                    es += seen(n, v) * term(v == m ? 0.0 : (double)v - (double)m);
                }
            }
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
template <bool EPI>
__global__ void __launch_bounds__(THREADS) sample_rows_kernel(const SampleArgs a) {
    __shared__ Shared sh;
    const int row = blockIdx.x;
    const int tid = threadIdx.x;
    int pos = row, b = row, col = 0;
    if constexpr (EPI) {
        pos = a.r.row_pos ? a.r.row_pos[row] : row;
        b = pos / a.r.L;
        col = pos - b * a.r.L;
        if (a.r.x[pos] != a.r.mask_id || col >= a.r.block_end) return;      // the defaults stand (uniform)
    }
    const double T = a.s.row_temperature ? (double)a.s.row_temperature[b] : a.s.temperature;
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
    const int ex_conf = EPI && (a.r.flags & LLADA_FLAG_CONF_EOS_EOT_INF) && a.r.eot_id != ex_all ? a.r.eot_id : -1;
    float conf = 0.f;
    sample_row<EPI>(a, sh, lc, lu, T, top_k, top_p, min_p, u, ex_all, ex_conf, conf);
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

int check_sampling(const char* who, const llada_sampling* s) {
    LLADA_CHECK_ARG(s != nullptr, "%s: null sampling parameters", who);
    LLADA_CHECK_ARG(s->row_temperature || (s->temperature >= 0.0 && s->temperature <= 1.0e30), "%s: temperature %g", who, s->temperature);
    LLADA_CHECK_ARG(s->row_top_k || s->top_k >= 0, "%s: top_k %d", who, s->top_k);
    LLADA_CHECK_ARG(s->row_top_p || (s->top_p > 0.0 && s->top_p <= 1.0), "%s: top_p %g is outside (0, 1]", who, s->top_p);
    LLADA_CHECK_ARG(s->row_min_p || (s->min_p >= 0.0 && s->min_p <= 1.0), "%s: min_p %g is outside [0, 1]", who, s->min_p);
    return LLADA_OK;
}

}  // namespace

extern "C" int llada_sample_rows(const void* logits, const void* uncond_logits, int64_t row_stride, double cfg_scale,
                                 int32_t n_rows, int32_t vocab, const llada_sampling* sampling, uint64_t seed, uint32_t step,
                                 uint32_t row_offset, int64_t* tokens, float* probs, void* stream) {
    LLADA_CHECK_ARG(logits && tokens && n_rows > 0 && vocab > 0, "sample_rows: bad argument");
    LLADA_CHECK_ARG(row_stride >= vocab || n_rows == 1, "sample_rows: rows overlap (stride %lld, vocab %d)", (long long)row_stride, vocab);
    LLADA_CHECK_ARG((((uintptr_t)logits | (uintptr_t)uncond_logits) & 1) == 0, "sample_rows: misaligned logits");
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
    hipLaunchKernelGGL(sample_rows_kernel<false>, dim3(n_rows), dim3(THREADS), 0, (hipStream_t)stream, a);
    LLADA_CHECK_LAUNCH("sample_rows_kernel");
    return LLADA_OK;
}

extern "C" int llada_remask_scores_sampled(const llada_remask_args* args, const llada_sampling* sampling, void* stream) {
    LLADA_CHECK_ARG(args != nullptr, "remask_scores_sampled: null args");
    const llada_remask_args& r = *args;
    LLADA_CHECK_ARG(r.logits && r.x && r.x0 && r.confidence, "remask_scores_sampled: null tensor");
    LLADA_CHECK_ARG(r.n_rows > 0 && r.B > 0 && r.L > 0 && r.vocab > 0, "remask_scores_sampled: bad shape");
    LLADA_CHECK_ARG(r.row_pos != nullptr || r.n_rows == (int64_t)r.B * r.L, "remask_scores_sampled: row_pos is required unless n_rows == B*L");
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
    hipLaunchKernelGGL(sample_rows_kernel<true>, dim3(r.n_rows), dim3(THREADS), 0, st, a);
    LLADA_CHECK_LAUNCH("sample_rows_kernel");
    return LLADA_OK;
}
