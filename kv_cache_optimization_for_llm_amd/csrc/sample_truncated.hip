// A token from the best of a row: the first k in the order of the logits, of those the shortest run that has the share p of their
// weight, of those the ones of at least min_p of the best one's weight.
//
//     order   logit descending, among equal ones the lower id first; -inf and NaN are not in it
//     w_i     exp((l_i - max l) / T)
//     first   the k first of the order (k <= 0 or k >= all: all of them), S_k their weight
//     second  the shortest beginning of these with a weight of at least p S_k (p >= 1: all; at least one token)
//     third   of these the ones with w_i >= min_p, and the best ones in any case (min_p <= 0: all)
//     token   with S what is left: the first id, by ids, at which the weights up to it exceed u S
//
// Which tokens stay hangs on long sums next to a border, so weights are whole numbers: W_i = 2^s w_i, rounded (within 0.75), s = 46 for a
// vocabulary of up to 2^16 and one less for every doubling, from an exponential in 64 bits.  Sums of them are exact and the same in
// any order: atomics may add them up, and a row draws the same token whoever shares the launch with it.
//
// The order is one of 64-bit places, (the logit's bits, descending) above (the id): both cuts are a place, and what stays is what
// lies in front of it.
//
// Vocabularies of up to 262,144 take four launches, the first three of them with many workgroups a row, each of some steps of
// 1,024 tokens:
//   1. trunc_best_kernel     the best place of every workgroup's tokens; for a small k also of groups of 32 to 512
//   2. trunc_bins_kernel     bins by the distance from the best, 1/32 of a factor of two wide: how many tokens a bin has where
//                            the row asks for k, their weight where it asks for p alone
//   3. trunc_collect_kernel  finds the bin in which the cut lies and leaves a list of tokens: where k is asked for those of all bins up to
//                            it (p's cut is among them), else those of this bin, and the sums of what lies in front of it by 256 ids
//   4. trunc_pick_kernel     a workgroup a row: for a small k its list from the groups that can hold the k best (such rows pass 2 and 3 by);
//                            the cuts among the list's tokens, what stays by 256 ids, then the token among 256
// A list has room for 4,096 tokens.  A row with more in the bin of its cut (nearly equal logits), or with a larger k among
// them, is taken by the last kernel alone, as rows of larger vocabularies are by sample_truncated_kernel: a cut is found by counting,
// the places still in question are cut into 1,024 ranges, their numbers and weights added up in LDS, and the range in which the sum passes what is
// sought is the next turn's; the row is read again in every turn (out of LDS up to 16,384 tokens).
//
// us in a graph.  Vocabulary 128,256: 1 row of a p 21, of a k 17; 64 rows of p 0.9 49 (7.2 + 18 + 17 + 9.2 for the four kernels), of a k up to 50 24 (7.4 + 1.8 + 1.8 +
// 14.2: 33 MB are 6.4 us at a copy's rate); 256 rows of p 0.98 at a temperature of 2, which keep most of the vocabulary, 118 (21 + 34 + 59 + 10: the
// first reads 131 MB at 6.2 TB/s, the next two weigh every token); rows of nearly equal logits 410 to 480.  One launch, against four: 1,024 tokens 10 / 16
// to 25, 2,048 13 to 15 / 17 to 22, 4,096 16 to 21 / 17 to 29, 8,192 28 to 31 / 18 to 25.
#include "common.h"
#include "counter_uniform.h"
#include "wave_scan.h"

#include <algorithm>
#include <type_traits>

#define TR_THREADS 256
#define TR_WAVES (TR_THREADS / KVA_WAVE)
#define TR_NO_TOKEN (-1)
#define TR_DIGITS 1024
#define TR_PER (TR_DIGITS / TR_THREADS)
#define TR_BUCKETS 1024                 // ranges of ids, in which what stays is added up

struct TruncArgs {
    const float *logits;
    long long stride;
    int vocab, scale_bits;
    const float *inv_t;                 // <= 0: the best token; no number: the row is passed over
    const int *top_k;                   // absent: all of them
    const float *top_p, *min_p;
    const float *uniform;               // absent: the counter-based number of (seed, key, step)
    unsigned seed;
    const unsigned *key, *step;
    int *tokens, *host_tokens, *kept;
    float *logprob;
};

// What a row asks for.  Where a row's draw ends (`drawn`) all of it is loaded at once, one trip to memory in front of everything else; an
// absent array's place is taken by one that is there.  (us in a graph, loaded where used / at once: 1 row 21.4 / 20.8, 64 rows without cuts 28.6 / 27.3.
// The kernels that weigh whole rows gain nothing: 256 rows 117 / 120.)
struct TruncRow {
    float inv_t, p, min_p, u;
    int k;
    __device__ inline TruncRow(const TruncArgs &a, int row, bool drawn) {
        const float *ps = a.top_p != nullptr ? a.top_p : a.inv_t, *ms = a.min_p != nullptr ? a.min_p : a.inv_t;
        const int *ks = a.top_k != nullptr ? a.top_k : reinterpret_cast<const int *>(a.inv_t);
        inv_t = a.inv_t[row], p = ps[row], min_p = ms[row], k = ks[row], u = 0.f;
        if (drawn) {
            if (a.uniform != nullptr) u = a.uniform[row];
            else u = counter_uniform(a.seed, a.key[row], a.step[row]);
        }
        if (drawn) asm volatile("" : "+s"(inv_t), "+s"(p), "+s"(min_p), "+s"(k), "+v"(u));         // (else each is loaded where it is used first)
        p = a.top_p != nullptr ? p : 1.f;
        min_p = a.min_p != nullptr ? min_p : 0.f;
        k = a.top_k != nullptr ? k : 0;
    }
};

// descending logits as ascending 32-bit numbers; the two zeros are one (l + 0: -0 becomes 0)
__device__ inline unsigned tr_falling(float l) {
    const unsigned b = __float_as_uint(l + 0.f);
    return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ inline u64 tr_place(float l, int id) { return (u64)tr_falling(l) << 32 | (unsigned)id; }

// ... and back
__device__ inline float tr_logit(u64 place) {
    const unsigned k = (unsigned)(place >> 32);
    return __uint_as_float(k & 0x80000000u ? k : ~k & 0x7fffffffu);
}

typedef float tr_f32x4 __attribute__((ext_vector_type(4), aligned(4)));

// Four neighbouring logits from token t on; what lies behind the vocabulary is -inf.
__device__ inline void tr_load4(const float *rl, int t, int vocab, float (&l)[4]) {
    if (t + 3 < vocab) {
        const tr_f32x4 v = *reinterpret_cast<const tr_f32x4 *>(rl + t);
        l[0] = v.x, l[1] = v.y, l[2] = v.z, l[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) l[i] = t + i < vocab ? rl[t + i] : -INFINITY;
    }
}

// How a row weighs its logits.  With x = 128 (s - (best - l) / (T ln 2)) and m its nearest whole number, W = 2^(m / 128) 2^((x - m) / 128):
// the first from a table of 2^(j / 128) and an exponent, the second, 1 + q with |q| < 0.0028, by four terms of its series (1.2e-15 off).  W is
// then within 0.75 of 2^s w (0.72 the most of 2 million at s = 46: half of it is W's own rounding, a quarter x's).  With three terms every weight
// is up to 2.2e-12 of itself too low, 158 units of the best one's, for 1 % of the time of a launch that weighs whole rows (256 rows 116.7 / 118.1 us).
// A number below 2^51 and 1.5 2^52 (2^52) add up to one whose last bits are the number's whole part, rounded.  A logit that weighs
// less than 1/8, and one that is none, has the x of 1/8 and the weight 0.  What bounds the kernels that weigh a whole row is the
// number of instructions, 64-bit ones above all (some ten cycles each): a polynomial of eleven terms and an exponent instead of the table, 256 rows of
// 128,256: bins 38 us instead of 33, sums 63 instead of 59.
#define TR_TABLE 128
struct TruncWeights {
    double best, rate;                  // 128 / (T ln 2)
    int bits;
    const double *table;

    __device__ inline TruncWeights(float best_, float inv_t, int bits_, const double *table_) : best(best_), bits(bits_), table(table_) {
        // (a temperature of nothing has no infinite rate: 0 times it is 0)
        rate = fmin((double)inv_t, 1e300) * (TR_TABLE * 1.4426950408889634);
    }
    // x, at least that of a weight of 1/8
    __device__ inline double scaled(float l) const { return fmax(fma(best - (double)l, -rate, (double)TR_TABLE * bits), -3.0 * TR_TABLE); }
    __device__ inline u64 of(double x) const {
        const double shifted = x + 6755399441055744.0, y = x - (shifted - 6755399441055744.0);
        const int m = (int)(unsigned)__double_as_longlong(shifted);
        // (ln 2 / 128)^i / i!
        double q = fma(y, fma(y, 3.5830323054002512e-11, 2.646642144433097e-08), 1.4662262387640425e-05);
        q = y * fma(y, q, 0.0054152123481245725);
        const u64 from_table = (u64)__double_as_longlong(table[m & (TR_TABLE - 1)]);
        const double t = __longlong_as_double((long long)(from_table + ((u64)((unsigned)(m >> 7) << 20) << 32)));
        return (u64)__double_as_longlong(fma(t, q, t) + 4503599627370496.0) & 0xfffffffffffffull;
    }
    __device__ inline u64 of(float l) const { return of(scaled(l)); }
    __device__ inline u64 of(u64 place) const { return of(tr_logit(place)); }
    // Bins from the best logit down, 1/32 of an octave wide: what lies within half a 128th of the same four 128ths; the last one
    // takes all that weighs 1/8 and less.
    __device__ inline int last_bin() const { return TR_TABLE / 4 * (bits + 3); }
    __device__ inline int bin(double x) const {
        const int m = (int)(unsigned)__double_as_longlong(x + 6755399441055744.0);
        return (TR_TABLE * bits - m) >> 2;
    }
    // how far below the best one, in units of log2(weight)
    __device__ inline double octaves(float l) const { return (best - (double)l) * (rate / TR_TABLE); }
};
__device__ inline void tr_fill_table(double *table) {
    if (threadIdx.x < TR_TABLE) table[threadIdx.x] = exp2((double)threadIdx.x / TR_TABLE);
}

// Sum of numbers below 2^48 over the wavefront, in the last lane: 24 bits at a time, so that no step carries.
__device__ inline u64 tr_wave_sum48(u64 v) {
    const unsigned lo = wave_prefix((unsigned)v & 0xffffffu), hi = wave_prefix((unsigned)(v >> 24));
    return ((u64)hi << 24) + lo;
}
__device__ inline u64 tr_wave_min(u64 v) {
    return wave_last(wave_scan(v, ~0ull, [](u64 a, u64 b) { return a < b ? a : b; }));
}
__device__ inline u64 tr_wave_max(u64 v) {
    return wave_last(wave_scan(v, 0ull, [](u64 a, u64 b) { return a > b ? a : b; }));
}

#define TR_PAIRS 64                     // so many tokens are compared with one another

struct TruncShared {
    u64 sum[TR_DIGITS];
    unsigned count[TR_DIGITS];
    u64 bucket_sum[TR_BUCKETS];
    unsigned bucket_count[TR_BUCKETS];
    u64 part[2 * TR_WAVES];
    unsigned part_count[TR_WAVES];
    u64 place[TR_PAIRS], weight[TR_PAIRS];
    double table[TR_TABLE];
    u64 lo, hi, above;
    unsigned inside_count, gathered;
    int found;
};

// The smallest of all threads' numbers and the largest.
__device__ inline void tr_block_range(TruncShared &s, u64 &lo, u64 &hi) {
    lo = tr_wave_min(lo);
    hi = tr_wave_max(hi);
    __syncthreads();
    if (threadIdx.x % KVA_WAVE == 0) s.part[threadIdx.x / KVA_WAVE] = lo, s.part[TR_WAVES + threadIdx.x / KVA_WAVE] = hi;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TR_WAVES; ++w) lo = min(lo, s.part[w]), hi = max(hi, s.part[TR_WAVES + w]);
}

// Inclusive prefix sums of a number and a count a thread over the workgroup.
__device__ inline void tr_block_prefix(TruncShared &s, u64 &v, unsigned &c) {
    const int lane = threadIdx.x % KVA_WAVE, wave = threadIdx.x / KVA_WAVE;
    v = wave_prefix(v);
    c = wave_prefix(c);
    __syncthreads();
    if (lane == KVA_WAVE - 1) s.part[wave] = v, s.part_count[wave] = c;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TR_WAVES - 1; ++w)
        if (w < wave) v += s.part[w], c += s.part_count[w];
}

// The sums of the threads' four numbers and counts of an array of 1,024 each, up to and with the thread's.
struct FourSums {
    u64 v[TR_PER], upto;
    unsigned c[TR_PER], count;
};
__device__ inline FourSums tr_four(TruncShared &s, const u64 *sum, const unsigned *count) {
    FourSums r;
    r.upto = 0, r.count = 0;
#pragma unroll
    for (int i = 0; i < TR_PER; ++i) {
        r.v[i] = sum[threadIdx.x * TR_PER + i], r.c[i] = count[threadIdx.x * TR_PER + i];
        r.upto += r.v[i], r.count += r.c[i];
    }
    tr_block_prefix(s, r.upto, r.count);
    return r;
}

// Up to 64 tokens, their places in s.place: how many of them and what weight (beside `front`) lies up to each of them, itself
// included.  Four threads a token, which all get it.
struct PairSums {
    bool on;
    u64 place, own, upto;
    unsigned rank;
};
template <typename WEIGHT>
__device__ inline PairSums tr_pairs(TruncShared &s, int n, u64 front, WEIGHT weight) {
    const int tid = threadIdx.x, j = tid / 4;
    if (tid < n) s.weight[tid] = weight(s.place[tid]);
    __syncthreads();
    PairSums r{j < n, j < n ? s.place[j] : 0, j < n ? s.weight[j] : 0, 0, 0};
#pragma unroll 4
    for (int i = tid % 4; i < n; i += 4) {
        const bool in = s.place[i] <= r.place;
        r.upto += in ? s.weight[i] : 0;
        r.rank += in ? 1 : 0;
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
        r.upto += __shfl_xor(r.upto, off, KVA_WAVE);
        r.rank += __shfl_xor(r.rank, off, KVA_WAVE);
    }
    r.upto += front;
    return r;
}
// The place of the need-th of them, and the weight up to it.
__device__ inline u64 tr_pair_by_count(TruncShared &s, const PairSums &r, unsigned need, u64 &upto) {
    if (r.on && r.rank == need) s.above = r.place, s.hi = r.upto;       // (the threads of one token, the same)
    __syncthreads();
    upto = s.hi;
    return s.above;
}
// The place at which the weight reaches `need`.
__device__ inline u64 tr_pair_by_weight(TruncShared &s, const PairSums &r, u64 need) {
    if (r.on && r.upto - r.own < need && need <= r.upto) s.lo = r.place;
    __syncthreads();
    return s.lo;
}

// What a row leaves: its token, how many stayed, its log-probability.
struct TruncResult {
    int token, kept;
    float logprob;
    __device__ inline void store(const TruncArgs &a, int row) const {
        a.tokens[row] = token;
        if (a.host_tokens != nullptr) a.host_tokens[row] = token;
        if (a.kept != nullptr) a.kept[row] = kept;
        if (a.logprob != nullptr) a.logprob[row] = logprob;
    }
};

// A row that no weights decide: without a token, greedy, or without finite weights.  `at`: its best place (all ones: none)
__device__ inline bool tr_decided(u64 at, float best, float inv_t, TruncResult &r) {
    const bool none = at == ~0ull;
    if (!none && inv_t > 0.f && best < INFINITY) return false;
    if (none || inv_t > 0.f) r = TruncResult{TR_NO_TOKEN, 0, -INFINITY};
    else r = TruncResult{(int)(unsigned)at, 1, 0.f};
    return true;
}

// The weight that p's cut has to reach, of `total`.
__device__ inline u64 tr_share(float p, u64 total) {
    const double share = ceil((double)p * (double)total);
    return share >= 1.0 ? min((u64)share, total) : 1ull;
}

// The x of TruncWeights that a token needs to stay (the best ones stay in any case).
__device__ inline double tr_least(const TruncRow &row, int bits) {
    return row.min_p > 0.f ? TR_TABLE * (bits + fmin(log2((double)row.min_p), 0.0)) : -INFINITY;
}

__device__ inline u64 tr_target(float u, u64 all) {
    const u64 target = u > 0.f ? (u64)(fmin((double)u, 1.0) * (double)all) : 0ull;
    return min(target, all - 1);
}

// Of the places that each(f) hands to f(place), from .. to: the one at which their number (by_count) or weight, with
// `front` in front of them, reaches `need`.  There is one.  By count `upto` gets the weight up to it.
template <typename EACH, typename WEIGHT>
__device__ inline u64 tr_cut(TruncShared &s, u64 from, u64 to, bool by_count, u64 front, u64 need, u64 &upto, EACH each, WEIGHT weight) {
    const int tid = threadIdx.x;
    u64 front_weight = by_count ? 0 : front;
    while (true) {
        const u64 span = to - from;
        const int shift = span < TR_DIGITS ? 0 : 64 - __clzll((long long)span) - 10;
#pragma unroll
        for (int i = 0; i < TR_PER; ++i) s.sum[tid + i * TR_THREADS] = 0, s.count[tid + i * TR_THREADS] = 0;
        if (tid == 0) s.gathered = 0;
        __syncthreads();
        each([&](u64 at) {
            if (at < from || at > to) return;
            const int digit = (int)((at - from) >> shift);
            atomicAdd(&s.sum[digit], weight(at));
            atomicAdd(&s.count[digit], 1u);
        });
        __syncthreads();
        const FourSums sums = tr_four(s, s.sum, s.count);
        u64 run = sums.upto;
        unsigned seen = sums.count;
#pragma unroll
        for (int i = TR_PER - 1; i >= 0; --i) {
            const u64 reach = front + (by_count ? (u64)seen : run), behind = reach - (by_count ? (u64)sums.c[i] : sums.v[i]);
            run -= sums.v[i], seen -= sums.c[i];
            if (behind < need && need <= reach) {       // (one range of them all)
                s.found = tid * TR_PER + i;
                s.above = behind;
                s.lo = front_weight + run;
                s.hi = front_weight + run + sums.v[i];
                s.inside_count = sums.c[i];
            }
        }
        __syncthreads();
        const int digit = s.found;
        const unsigned inside = s.inside_count;
        front = s.above;
        front_weight = s.lo;
        upto = s.hi;
        __syncthreads();
        from += (u64)digit << shift;
        if (shift == 0) return from;
        to = min(to, from + ((1ull << shift) - 1));
        if (inside > TR_PAIRS) continue;
        each([&](u64 at) {
            if (at >= from && at <= to) s.place[atomicAdd(&s.gathered, 1u)] = at;
        });
        __syncthreads();
        const PairSums r = tr_pairs(s, inside, front_weight, weight);
        const u64 at = by_count ? tr_pair_by_count(s, r, (unsigned)(need - front), upto) : tr_pair_by_weight(s, r, need);
        __syncthreads();
        return at;
    }
}

// Four neighbouring tokens: the weight of those that stay up to `last`, and how many they are.
__device__ inline void tr_stay4(const float (&l)[4], int t, const TruncWeights &weigh, u64 last, double least, u64 (&w)[4], unsigned &count) {
    count = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double x = weigh.scaled(l[i]);
        const bool stays = l[i] > -INFINITY && tr_place(l[i], t + i) <= last && x >= least;
        w[i] = stays ? weigh.of(x) : 0;
        count += stays ? 1 : 0;
    }
}

// The token of a row, from what stays by ranges of `per` ids (a multiple of 256), in s.bucket_sum and s.bucket_count.
__device__ inline void tr_draw(const TruncArgs &a, TruncShared &s, const float *rl, int row, float u, int per, const TruncWeights &weigh, u64 last, double least) {
    const int tid = threadIdx.x, lane = tid % KVA_WAVE;
    const FourSums sums = tr_four(s, s.bucket_sum, s.bucket_count);
    if (tid == TR_THREADS - 1) s.hi = sums.upto, s.inside_count = sums.count;
    __syncthreads();
    const u64 all = s.hi, target = tr_target(u, all);
    u64 run = sums.upto;
#pragma unroll
    for (int i = TR_PER - 1; i >= 0; --i) {
        run -= sums.v[i];
        if (run <= target && target < run + sums.v[i]) s.found = tid * TR_PER + i, s.above = run;
    }
    __syncthreads();
    if (tid >= KVA_WAVE) return;
    run = s.above;
    for (int t0 = s.found * per; t0 < a.vocab; t0 += 4 * KVA_WAVE) {
        const int t = t0 + 4 * lane;
        float l[4];
        u64 w[4];
        unsigned unused;
        tr_load4(rl, t, a.vocab, l);
        tr_stay4(l, t, weigh, last, least, w, unused);
        const u64 mine = w[0] + w[1] + w[2] + w[3], upto = wave_prefix(mine), whole = wave_last(upto);
        if (target >= run + whole) {            // (the same in all lanes; a range's sum is its tokens')
            run += whole;
            continue;
        }
        u64 at = run + upto - mine;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (at <= target && target < at + w[i])
                TruncResult{t + i, (int)s.inside_count, (float)(-0.6931471805599453 * (weigh.octaves(l[i]) + log2((double)all) - (double)weigh.bits))}.store(a, row);
            at += w[i];
        }
        return;
    }
}

// A row (`rl`: its logits) by one workgroup that reads it in every turn; s.table is filled, or will be with the next barrier.
__device__ inline void trunc_whole_row(const TruncArgs &a, TruncShared &s, const float *rl, int row, const TruncRow &of) {
    const int tid = threadIdx.x, lane = tid % KVA_WAVE, wave = tid / KVA_WAVE, vocab = a.vocab, bits = a.scale_bits;
    const float inv_t = of.inv_t, p = of.p;
    const int k = of.k;
    auto each = [&](auto f) {
        float l[4];
        tr_load4(rl, 4 * tid, vocab, l);
        for (int t = 4 * tid; t < vocab; t += 4 * TR_THREADS) {
            float next[4];
            tr_load4(rl, t + 4 * TR_THREADS, vocab, next);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (l[i] > -INFINITY) f(tr_place(l[i], t + i));
                l[i] = next[i];
            }
        }
    };
    // the best place and the last one
    u64 lo = ~0ull, hi = 0;
    unsigned valid = 0;
    each([&](u64 at) {
        lo = min(lo, at);
        hi = max(hi, at);
        ++valid;
    });
    u64 none = 0;
    tr_block_prefix(s, none, valid);
    if (tid == TR_THREADS - 1) s.inside_count = valid;
    tr_block_range(s, lo, hi);
    valid = s.inside_count;
    const float best = valid ? tr_logit(lo) : 0.f;
    TruncResult r;
    if (tr_decided(lo, best, inv_t, r)) {
        if (tid == 0) r.store(a, row);
        return;
    }
    const TruncWeights weigh(best, inv_t, bits, s.table);
    const double least = tr_least(of, bits);
    auto weight = [&](u64 at) { return weigh.of(at); };
    u64 last = hi, total = 0;               // the last place that stays, the weight up to it
    __syncthreads();
    if (k > 0 && (unsigned)k < valid) last = tr_cut(s, lo, hi, true, 0, (u64)k, total, each, weight);
    if (p < 1.f) {
        if (total == 0) {
            u64 sum = 0;
            unsigned unused = 0;
            each([&](u64 at) { sum += weight(at); });
            tr_block_prefix(s, sum, unused);
            if (tid == TR_THREADS - 1) s.hi = sum;
            __syncthreads();
            total = s.hi;
            __syncthreads();
        }
        last = tr_cut(s, lo, last, false, 0, tr_share(p, total), total, each, weight);
    }
    // what stays, a wavefront a range of ids
    const int per = (vocab + TR_BUCKETS * 4 * KVA_WAVE - 1) / (TR_BUCKETS * 4 * KVA_WAVE) * (4 * KVA_WAVE);
#pragma unroll
    for (int i = 0; i < TR_BUCKETS / TR_THREADS; ++i) s.bucket_sum[tid + i * TR_THREADS] = 0, s.bucket_count[tid + i * TR_THREADS] = 0;
    __syncthreads();
    for (int b = wave; b * per < vocab; b += TR_WAVES) {
        u64 sum = 0;
        unsigned count = 0;
        float l[4];
        tr_load4(rl, b * per + 4 * lane, vocab, l);
        for (int t0 = b * per; t0 < min(vocab, (b + 1) * per); t0 += 4 * KVA_WAVE) {
            float next[4];
            u64 w[4];
            unsigned n;
            tr_load4(rl, t0 + 4 * KVA_WAVE + 4 * lane, vocab, next);
            tr_stay4(l, t0 + 4 * lane, weigh, last, least, w, n);
            sum += tr_wave_sum48(w[0] + w[1] + w[2] + w[3]);
            count += n;
#pragma unroll
            for (int i = 0; i < 4; ++i) l[i] = next[i];
        }
        count = wave_prefix(count);
        if (lane == KVA_WAVE - 1) s.bucket_sum[b] = sum, s.bucket_count[b] = count;
    }
    __syncthreads();
    tr_draw(a, s, rl, row, of.u, per, weigh, last, least);
}

// grid (rows).  HELD: the row stands in LDS.
#define TR_HELD_VOCAB 16384
template <bool HELD>
__global__ void __launch_bounds__(TR_THREADS)
sample_truncated_kernel(TruncArgs a) {
    __shared__ TruncShared s;
    __shared__ __attribute__((aligned(16))) float held[HELD ? TR_HELD_VOCAB : 4];
    const TruncRow of(a, blockIdx.x, true);
    if (isnan(of.inv_t)) return;
    tr_fill_table(s.table);             // (the first barrier comes before its first use)
    const float *rl = a.logits + blockIdx.x * a.stride;
    if (HELD) {
        for (int t = 4 * threadIdx.x; t < a.vocab; t += 4 * TR_THREADS) {
            float l[4];
            tr_load4(rl, t, a.vocab, l);
            *reinterpret_cast<float4 *>(held + t) = make_float4(l[0], l[1], l[2], l[3]);       // (each thread its own: no barrier yet)
        }
    }
    trunc_whole_row(a, s, HELD ? held : rl, blockIdx.x, of);
}

// ---------------------------------------------------------------- many workgroups a row
#define TR_BINS 2048                    // (TruncWeights::last_bin is below 1,600)
#define TR_LIST 4096
#define TR_STEP 1024                    // tokens a workgroup takes at a time: 256 threads, 4 neighbouring tokens each
#define TR_BUCKET 256                   // ... and a wavefront of them
#define TR_SPLIT_THREADS 256
#define TR_SPLIT_WAVES (TR_SPLIT_THREADS / KVA_WAVE)
#define TR_WAVE_LIST 1024
#define TR_MAX_PARTS 64
#define TR_FEW_MOST 1024
#define TR_FEW_MOST_OF_FEW_ROWS 256
#define TR_FEW_ROWS 3
#define TR_FEW_STEPS 4096
#define TR_GROUPS 64                    // groups a part
#define TR_MAX_VOCAB (TR_BUCKET * TR_BUCKETS)

struct TruncSpace {                     // of all rows
    u64 *best;                          // [parts]
    u64 *tops;                          // [parts * 64]: the best place of every group, four neighbouring threads' tokens of a part
    u64 *bins;                          // [TR_BINS]
    u64 *sought;                        // [2]: the weight in front of the cut's bin, and the one the cut has to reach
    u64 *sums;                          // [buckets]: what stays for certain, by ids
    unsigned *counts;                   // [buckets]
    u64 *list;                          // [TR_LIST]: places
    int *listed;                        // [1]: tokens that asked for a place in the list
    int parts, part_tokens, buckets;
    int few;                            // the largest k that is found by the groups' best tokens
};

// What a row's cut is found by: nothing, the number of tokens up to a bin, their weight, or the best tokens of the groups.  The last is for a
// small k, as long as one workgroup reads the k groups it leaves sooner than many read the row twice more: up to 1,024, half of the groups, and
// 4,096 steps of theirs; of three rows, which have the chip to themselves, up to 256.  us in a graph by groups / by bins, k of all of a launch's rows up
// to ...: 1 row of 128,256 (2 steps a group), 600 28 / 24; 4 rows, 600 29 / 31, 1,000 35 / 31; 16 rows, 1,000 36 / 67; 37 rows of 50,021 (2 steps), 400
// 26 / 52, 1,000 44 / 57; 64 rows of 128,256 (8 steps), 100 28 / 51, 400 45 / 62; 256 rows of 128,256 (32 steps), 100 56 / 84.  A launch with both
// kinds pays for both: these with k up to 250 100 / 85.
enum { TR_ALL = 0, TR_COUNT = 1, TR_WEIGHT = 2, TR_FEW = 3 };
__device__ inline int tr_mode(const TruncArgs &a, const TruncSpace &sp, const TruncRow &row) {
    if (row.k > 0 && row.k < a.vocab) return row.k <= sp.few ? TR_FEW : TR_COUNT;
    return row.p < 1.f ? TR_WEIGHT : TR_ALL;
}

// The four tokens of a thread in the step that begins at t0 (the same in all threads: a whole step needs no test a token).
__device__ inline void tr_load_step(const float *rl, int t0, int vocab, float (&l)[4]) {
    const int t = t0 + 4 * threadIdx.x;
    if (t0 + TR_STEP <= vocab) {
        const tr_f32x4 v = *reinterpret_cast<const tr_f32x4 *>(rl + t);
        l[0] = v.x, l[1] = v.y, l[2] = v.z, l[3] = v.w;
    } else {
        tr_load4(rl, t, vocab, l);
    }
}

// The best place of a row, from its parts' (every wavefront for itself): asked for first, found later.
static_assert(TR_MAX_PARTS <= KVA_WAVE, "a lane a part");
__device__ inline u64 tr_part_best(const TruncSpace &sp, int row) {
    const int part = threadIdx.x % KVA_WAVE;
    return part < sp.parts ? sp.best[(size_t)row * sp.parts + part] : ~0ull;
}

// grid (parts, rows)
__global__ void __launch_bounds__(TR_SPLIT_THREADS)
trunc_best_kernel(TruncArgs a, TruncSpace sp) {
    __shared__ u64 of_wave[TR_SPLIT_WAVES];
    const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    const float *rl = a.logits + row * a.stride;
    float l[4], top = -INFINITY;
    tr_load_step(rl, part * sp.part_tokens, a.vocab, l);
    const TruncRow of(a, row, false);
    if (isnan(of.inv_t)) return;
    // (the next launches add to these)
    const int per = (TR_BINS + sp.parts - 1) / sp.parts;
    for (int i = part * per + tid; i < min(TR_BINS, (part + 1) * per); i += TR_SPLIT_THREADS) sp.bins[(size_t)row * TR_BINS + i] = 0;
    if (part == 0 && tid == 0) sp.listed[row] = 0;
    const int end = min(a.vocab, (part + 1) * sp.part_tokens), lane = tid % KVA_WAVE, wave = tid / KVA_WAVE;
    int id = 0;
    for (int t0 = part * sp.part_tokens; t0 < end; t0 += TR_STEP) {
        const int t = t0 + 4 * tid;
        float next[4];
        tr_load_step(rl, t0 + TR_STEP, a.vocab, next);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (l[i] > top) top = l[i], id = t + i;     // (ascending ids: the first of equal ones)
#pragma unroll
        for (int i = 0; i < 4; ++i) l[i] = next[i];
    }
    u64 at = top > -INFINITY ? tr_place(top, id) : ~0ull;
    if (tr_mode(a, sp, of) == TR_FEW) {
        u64 of = min(at, (u64)__shfl_xor(at, 1, KVA_WAVE));
        of = min(of, (u64)__shfl_xor(of, 2, KVA_WAVE));
        if (tid % 4 == 0) sp.tops[((size_t)row * sp.parts + part) * TR_GROUPS + tid / 4] = of;
    }
    at = tr_wave_min(at);
    if (lane == 0) of_wave[wave] = at;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < TR_SPLIT_WAVES; ++w) at = min(at, of_wave[w]);
        sp.best[(size_t)row * sp.parts + part] = at;
    }
}

// grid (parts, rows).  Two sets of bins, a lane's by its number: most of a row's tokens lie in some tens of bins, and additions to the
// same one wait for each other.
#define TR_SETS 2
__global__ void __launch_bounds__(TR_SPLIT_THREADS)
trunc_bins_kernel(TruncArgs a, TruncSpace sp) {
    __shared__ u64 bins[TR_BINS * TR_SETS];
    __shared__ double table[TR_TABLE];
    const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, bits = a.scale_bits;
    const TruncRow of(a, row, false);
    const float inv_t = of.inv_t;
    const int mode = tr_mode(a, sp, of);
    if (!(inv_t > 0.f) || mode == TR_ALL || mode == TR_FEW) return;
    const float *rl = a.logits + row * a.stride;
    const int end = min(a.vocab, (part + 1) * sp.part_tokens);
    const u64 part_best = tr_part_best(sp, row);
    float l[4];
    tr_load_step(rl, part * sp.part_tokens, a.vocab, l);
    for (int i = tid; i < TR_BINS * TR_SETS; i += TR_SPLIT_THREADS) bins[i] = 0;
    tr_fill_table(table);
    const u64 at = tr_wave_min(part_best);
    if (at == ~0ull) return;
    const float best = tr_logit(at);
    const TruncWeights weigh(best, inv_t, bits, table);
    __syncthreads();
    u64 *mine = bins + tid % TR_SETS;
    auto run = [&](auto counting) {
        for (int t0 = part * sp.part_tokens; t0 < end; t0 += TR_STEP) {
            float next[4];
            tr_load_step(rl, t0 + TR_STEP, a.vocab, next);
            double x[4];
            u64 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = weigh.scaled(l[i]);
                // (what is not in the order weighs nothing)
                w[i] = counting ? (l[i] > -INFINITY ? 1 : 0) : weigh.of(x[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (w[i] != 0) atomicAdd(mine + weigh.bin(x[i]) * TR_SETS, w[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) l[i] = next[i];
        }
    };
    if (mode == TR_COUNT) run(std::true_type{});
    else run(std::false_type{});
    __syncthreads();
    for (int i = tid; i < TR_BINS; i += TR_SPLIT_THREADS) {
        u64 v = 0;
#pragma unroll
        for (int j = 0; j < TR_SETS; ++j) v += bins[i * TR_SETS + j];
        if (v != 0) atomicAdd(&sp.bins[(size_t)row * TR_BINS + i], v);
    }
}

// grid (parts, rows)
__global__ void __launch_bounds__(TR_SPLIT_THREADS)
trunc_collect_kernel(TruncArgs a, TruncSpace sp) {
    constexpr int PER = TR_BINS / TR_SPLIT_THREADS;
    __shared__ u64 of_wave[TR_SPLIT_WAVES];
    // (a wavefront has a list of its own, and counts it itself)
    __shared__ int found[TR_SPLIT_WAVES][TR_WAVE_LIST], cut_bin;
    __shared__ u64 sums[TR_BUCKETS];
    __shared__ unsigned short counts[TR_BUCKETS];
    __shared__ double table[TR_TABLE];
    const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid % KVA_WAVE, wave = tid / KVA_WAVE, bits = a.scale_bits;
    const TruncRow of(a, row, false);
    const float inv_t = of.inv_t;
    const int mode = tr_mode(a, sp, of);
    if (!(inv_t > 0.f) || mode == TR_FEW) return;
    const float *rl = a.logits + row * a.stride;
    const int end = min(a.vocab, (part + 1) * sp.part_tokens);
    int t0 = part * sp.part_tokens;
    const u64 part_best = tr_part_best(sp, row);
    float l[4];
    tr_load_step(rl, t0, a.vocab, l);
    u64 v[PER] = {};
    if (mode != TR_ALL) {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = sp.bins[(size_t)row * TR_BINS + tid * PER + i];
    }
    tr_fill_table(table);
    const u64 at = tr_wave_min(part_best);
    if (at == ~0ull) return;
    const float best = tr_logit(at);
    if (!(best < INFINITY)) return;
    int cut = TR_BINS;                      // the bin in which the cut lies; past the last: everything stays
    if (mode != TR_ALL) {
        u64 mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) mine += v[i];
        u64 upto = wave_prefix(mine);
        if (lane == KVA_WAVE - 1) of_wave[wave] = upto;
        if (tid == 0) cut_bin = TR_BINS - 1;            // (fewer tokens than k: all of them)
        __syncthreads();
        u64 total = 0;
#pragma unroll
        for (int w = 0; w < TR_SPLIT_WAVES; ++w) {
            if (w < wave) upto += of_wave[w];
            total += of_wave[w];
        }
        const u64 need = mode == TR_COUNT ? (u64)of.k : tr_share(of.p, total);
        u64 run = upto - mine;
        if (run < need && need <= upto) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (run < need && need <= run + v[i]) {
                    cut_bin = tid * PER + i;
                    if (part == 0) sp.sought[2 * row] = run, sp.sought[2 * row + 1] = need;
                }
                run += v[i];
            }
        }
    }
    __syncthreads();
    if (mode != TR_ALL) cut = cut_bin;
    const TruncWeights weigh(best, inv_t, bits, table);
    const double least = tr_least(of, bits);
    // (below this no logit is in the cut's bin: a bin and a bit more, rounded down)
    const double reach = weigh.best - (4.0 * cut + 8.0) / weigh.rate;
    const float nothing = mode == TR_ALL || cut >= weigh.last_bin() ? -INFINITY : (float)(reach - 1e-6 * fabs(reach));
    int listed = 0;
    auto run = [&](auto counting) {
        for (; t0 < end; t0 += TR_STEP) {
            float next[4];
            tr_load_step(rl, t0 + TR_STEP, a.vocab, next);
            u64 sum = 0;
            unsigned count = 0;
            bool asks[4] = {}, some = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) some |= l[i] >= nothing;
            if (__any(some)) {
                // (no branch around a weight: the four run side by side)
                double x[4];
                int bin[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = weigh.scaled(l[i]);
                    bin[i] = l[i] > -INFINITY ? weigh.bin(x[i]) : TR_BINS + 1;
                    asks[i] = counting ? bin[i] <= cut : bin[i] == cut;
                }
                if (!counting) {
                    u64 w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = weigh.of(x[i]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool stays = bin[i] < cut && x[i] >= least;
                        sum += stays ? w[i] : 0;
                        count += (unsigned)__popcll(__ballot(stays));
                    }
                    sum = tr_wave_sum48(sum);
                }
                if (__any(asks[0] || asks[1] || asks[2] || asks[3])) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const unsigned long long votes = __ballot(asks[i]);
                        const int to = listed + (int)__popcll(votes & ((1ull << lane) - 1));
                        if (asks[i] && to < TR_WAVE_LIST) found[wave][to] = t0 + 4 * tid + i;
                        listed += (int)__popcll(votes);
                    }
                }
            }
            if (!counting && lane == KVA_WAVE - 1) {
                // 256 ids of this wavefront
                sums[(t0 - part * sp.part_tokens) / TR_BUCKET + wave] = sum;
                counts[(t0 - part * sp.part_tokens) / TR_BUCKET + wave] = (unsigned short)count;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) l[i] = next[i];
        }
    };
    if (mode == TR_COUNT) run(std::true_type{});
    else run(std::false_type{});
    if (listed > 0) {
        // (one list too long is as a row's too long)
        const int n = min(listed, TR_WAVE_LIST);
        int base = 0;
        if (lane == 0) base = atomicAdd(&sp.listed[row], listed > TR_WAVE_LIST ? TR_LIST + 1 : listed);
        base = __builtin_amdgcn_readfirstlane(base);
        for (int i = lane; i < min(n, TR_LIST - base); i += KVA_WAVE) {
            const int id = found[wave][i];
            sp.list[(size_t)row * TR_LIST + base + i] = tr_place(rl[id], id);
        }
    }
    if (mode == TR_COUNT) return;
    __syncthreads();
    const int first = part * sp.part_tokens / TR_BUCKET, many = min(sp.buckets - first, sp.part_tokens / TR_BUCKET);
    for (int i = tid; i < many; i += TR_SPLIT_THREADS) {
        sp.sums[(size_t)row * sp.buckets + first + i] = sums[i];
        sp.counts[(size_t)row * sp.buckets + first + i] = counts[i];
    }
}

// grid (rows).  A chain of short steps with a barrier between them; four wavefronts, one a SIMD, so that a step of all lanes (a prefix
// sum over 1,024 numbers, say) costs its instructions once.
__global__ void __launch_bounds__(TR_THREADS)
trunc_pick_kernel(TruncArgs a, TruncSpace sp) {
    constexpr int TOPS = TR_MAX_PARTS * TR_GROUPS / TR_THREADS;
    __shared__ TruncShared s;
    __shared__ u64 place[TR_LIST];
    __shared__ unsigned short group_of[TR_MAX_PARTS * TR_GROUPS];
    __shared__ int asked, groups_in;
    const int row = blockIdx.x, tid = threadIdx.x, bits = a.scale_bits, vocab = a.vocab;
    const float *rl = a.logits + row * a.stride;
    const TruncRow of(a, row, true);
    const float inv_t = of.inv_t, p = of.p;
    if (isnan(inv_t)) return;
    const int mode = tr_mode(a, sp, of), groups = sp.parts * TR_GROUPS;
    // everything that hangs on nothing else is asked for at once
    const u64 part_best = tr_part_best(sp, row);
    const bool drawn = inv_t > 0.f, sums = drawn && (mode == TR_ALL || mode == TR_WEIGHT);
    const u64 front = mode == TR_WEIGHT && drawn ? sp.sought[2 * row] : 0, sought = mode == TR_WEIGHT && drawn ? sp.sought[2 * row + 1] : 0;
    int n = drawn ? sp.listed[row] : 0;
    const u64 *list = sp.list + (size_t)row * TR_LIST, place0 = list[tid];
    u64 tops[TOPS];
    if (mode == TR_FEW) {
#pragma unroll
        for (int i = 0; i < TOPS; ++i)
            tops[i] = tid + i * TR_THREADS < groups ? sp.tops[(size_t)row * groups + tid + i * TR_THREADS] : ~0ull;
    }
    tr_fill_table(s.table);
#pragma unroll
    for (int i = 0; i < TR_BUCKETS / TR_THREADS; ++i) {
        const int b = tid + i * TR_THREADS;
        const bool on = sums && b < sp.buckets;
        s.bucket_sum[b] = on ? sp.sums[(size_t)row * sp.buckets + b] : 0;
        s.bucket_count[b] = on ? sp.counts[(size_t)row * sp.buckets + b] : 0;
    }
    const u64 first = tr_wave_min(part_best);
    const float best = first == ~0ull ? 0.f : tr_logit(first);
    TruncResult r;
    if (tr_decided(first, best, inv_t, r)) {
        if (tid == 0) r.store(a, row);
        return;
    }
    const TruncWeights weigh(best, inv_t, bits, s.table);
    const double least = tr_least(of, bits);
    const unsigned k = mode == TR_FEW || mode == TR_COUNT ? (unsigned)of.k : 0;
    u64 last = ~0ull, total = 0;            // the last place that stays
    auto weight = [&](u64 at) { return weigh.of(at); };
    if (mode == TR_FEW) {
        // The k-th best of the groups' best tokens is no better than the k-th best token: what is sought lies among the tokens that are
        // no worse than it, and those in the groups that have such a token.  "No worse" goes by 1,024 steps between the best of them
        // and the last, or what weighs nothing: the k-th is soon found among them.
        u64 from = ~0ull, to = 0;
#pragma unroll
        for (int i = 0; i < TOPS; ++i)
            if (tops[i] != ~0ull) from = min(from, tops[i]), to = max(to, tops[i]);
#pragma unroll
        for (int i = 0; i < TR_PER; ++i) s.sum[tid + i * TR_THREADS] = 0, s.count[tid + i * TR_THREADS] = 0;
        if (tid == 0) asked = groups_in = 0, s.found = TR_DIGITS;
        tr_block_range(s, from, to);
        const float range = fminf(best - tr_logit(to), (float)fmin((double)TR_TABLE * (bits + 3) / weigh.rate, 3e38));
        const float scale = range > 0.f ? (TR_DIGITS - 1) / range : 0.f;
        auto step_of = [&](float l) { return (int)fminf((best - l) * scale, TR_DIGITS - 1.f); };
#pragma unroll
        for (int i = 0; i < TOPS; ++i)
            if (tops[i] != ~0ull) atomicAdd(&s.count[step_of(tr_logit(tops[i]))], 1u);
        __syncthreads();
        const FourSums by = tr_four(s, s.sum, s.count);
        unsigned seen = by.count;
#pragma unroll
        for (int i = TR_PER - 1; i >= 0; --i) {
            if (seen - by.c[i] < k && k <= seen) s.found = tid * TR_PER + i;
            seen -= by.c[i];
        }
        __syncthreads();
        const int reach = s.found;          // (fewer than k: all of them)
#pragma unroll
        for (int i = 0; i < TOPS; ++i)
            if (tops[i] != ~0ull && step_of(tr_logit(tops[i])) <= reach) group_of[atomicAdd(&groups_in, 1)] = (unsigned short)(tid + i * TR_THREADS);
        __syncthreads();
        // Four threads a group and step: its 16 tokens.  A wavefront is alone on its SIMD, so what counts is the length of the chain: all of a
        // round's hits are places taken by one addition, and none of it branches but the taking (37 rows of 50,021 and k up to 400: 27 us,
        // 31 with an addition a token).
        const int steps = sp.part_tokens / TR_STEP, in = groups_in * steps, lane = tid % KVA_WAVE;
        // (j / steps is the high half of j (2^32 / steps, rounded up): j is below 2^15)
        const unsigned inverse = steps > 1 ? (unsigned)((0x100000000ull + steps - 1) / steps) : 0;
        const float limit = reach < TR_DIGITS - 1 ? reach + 1.f : NAN;          // (of the last step on: all of them)
        constexpr int AHEAD = 4;            // loads on their way
        for (int base = 0; base < in; base += AHEAD * TR_THREADS / 4) {
            tr_f32x4 l[AHEAD];
            int from_id[AHEAD];
            unsigned hit[AHEAD], hits = 0;
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int j = base + tid / 4 + u * TR_THREADS / 4, at = min(j, in - 1), which = steps > 1 ? (int)__umulhi((unsigned)at, inverse) : at;
                const int group = group_of[which];
                const int t = j < in ? group / TR_GROUPS * sp.part_tokens + (at - which * steps) * TR_STEP + group % TR_GROUPS * 16 + tid % 4 * 4 : vocab;
                from_id[u] = min(t, vocab - 4);
                hit[u] = 15u << min(t - from_id[u], 4);         // (a load that would end behind the row begins in front of its tokens)
                l[u] = *reinterpret_cast<const tr_f32x4 *>(rl + from_id[u]);
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                unsigned in_reach = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) in_reach |= l[u][i] > -INFINITY && !((best - l[u][i]) * scale >= limit) ? 1u << i : 0;
                hit[u] &= in_reach;
                hits += __popc(hit[u]);
            }
            const unsigned upto = wave_prefix(hits);
            int slot = 0;
            if (lane == KVA_WAVE - 1 && upto > 0) slot = atomicAdd(&asked, (int)upto);
            slot = __builtin_amdgcn_readlane(slot, KVA_WAVE - 1) + (int)(upto - hits);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                while (hit[u] != 0) {
                    const int i = __ffs(hit[u]) - 1;
                    hit[u] &= hit[u] - 1;
                    const u64 at = tr_place(i < 2 ? (i == 0 ? l[u][0] : l[u][1]) : (i == 2 ? l[u][2] : l[u][3]), from_id[u] + i);
                    if (slot < TR_LIST) place[slot] = at;
                    if (slot < TR_PAIRS) s.place[slot] = at;
                    ++slot;
                }
        }
        __syncthreads();
        n = asked;
    }
    if (n > TR_LIST) {
        __syncthreads();
        trunc_whole_row(a, s, rl, row, of);
        return;
    }
    if (mode != TR_FEW) {
        if (tid < n) place[tid] = place0;
        if (tid < min(n, TR_PAIRS)) s.place[tid] = place0;
#pragma unroll 4
        for (int i = tid + TR_THREADS; i < n; i += TR_THREADS) place[i] = list[i];
    }
    __syncthreads();
    if (mode != TR_ALL) {
        const u64 need = mode == TR_WEIGHT ? sought : (u64)min(k, (unsigned)n);
        const bool by_count = mode != TR_WEIGHT;
        if (n <= TR_PAIRS) {
            const PairSums pairs = tr_pairs(s, n, front, weight);
            if (by_count) {
                last = tr_pair_by_count(s, pairs, (unsigned)need, total);
                if (p < 1.f) last = tr_pair_by_weight(s, pairs, tr_share(p, total));
            } else {
                last = tr_pair_by_weight(s, pairs, need);
            }
        } else {
            u64 from = ~0ull, to = 0;
            for (int i = tid; i < n; i += TR_THREADS) from = min(from, place[i]), to = max(to, place[i]);
            tr_block_range(s, from, to);
            auto each = [&](auto f) {
                for (int i = tid; i < n; i += TR_THREADS) f(place[i]);
            };
            last = tr_cut(s, from, to, by_count, front, need, total, each, weight);
            if (by_count && p < 1.f) last = tr_cut(s, from, last, false, 0, tr_share(p, total), total, each, weight);
        }
    }
    // the list's tokens that stay, beside what lies in front of them
    for (int i = tid; i < n; i += TR_THREADS) {
        const u64 at = place[i];
        const double x = weigh.scaled(tr_logit(at));
        if (at > last || x < least) continue;
        atomicAdd(&s.bucket_sum[(unsigned)at / TR_BUCKET], weigh.of(x));
        atomicAdd(&s.bucket_count[(unsigned)at / TR_BUCKET], 1u);
    }
    __syncthreads();
    tr_draw(a, s, rl, row, of.u, TR_BUCKET, weigh, last, least);
}

// How many workgroups a row gets in the first three launches, and their tokens.
static int trunc_parts(int rows, int vocab, int *part_tokens) {
    const int steps = (vocab + TR_STEP - 1) / TR_STEP;
    int parts = (1024 + rows - 1) / rows;
    parts = parts < 1 ? 1 : parts > TR_MAX_PARTS ? TR_MAX_PARTS : parts;
    parts = parts > steps ? steps : parts;
    *part_tokens = (steps + parts - 1) / parts * TR_STEP;
    return (vocab + *part_tokens - 1) / *part_tokens;
}

static bool trunc_split(int vocab) { return vocab > 4096 && vocab <= TR_MAX_VOCAB; }

extern "C" long long kva_sample_truncated_workspace_bytes(int rows, int vocab) {
    if (rows <= 0 || !trunc_split(vocab)) return 0;
    int part_tokens;
    const long long parts = trunc_parts(rows, vocab, &part_tokens), buckets = (vocab + TR_BUCKET - 1) / TR_BUCKET;
    return rows * (8 * (parts + TR_BINS + parts * TR_GROUPS + 2 + TR_LIST + buckets) + 4 * (buckets + 1));
}

// address [10], the host's: of the tokens, inverse temperatures, top_k, top_p, min_p, uniform numbers, keys, steps, kept and logprob (0: absent)
extern "C" int kva_sample_truncated(const long long *address, const float *logits, long long stride, int rows, int vocab, unsigned seed,
                                    int *host_tokens, void *workspace, hipStream_t stream) {
    int *tokens = (int *)address[0], *kept = (int *)address[8];
    const int *top_k = (const int *)address[2];
    const unsigned *key = (const unsigned *)address[6], *step = (const unsigned *)address[7];
    const float *inv_t = (const float *)address[1], *top_p = (const float *)address[3], *min_p = (const float *)address[4],
                *uniform = (const float *)address[5];
    float *logprob = (float *)address[9];
    int *host_mapped = nullptr;
    if (host_tokens != nullptr) {
        void *dev = nullptr;
        const hipError_t e = hipHostGetDevicePointer(&dev, host_tokens, 0);
        if (e != hipSuccess) (void)hipGetLastError();
        KVA_REQUIRE(e == hipSuccess && dev != nullptr, "sample_truncated: host_tokens is not pinned host memory mapped for the device (%s)",
                    hipGetErrorString(e));
        host_mapped = (int *)dev;
    }
    KVA_REQUIRE(rows >= 0 && rows <= 65535 && vocab > 0 && vocab <= 1 << 24, "sample_truncated: bad sizes rows=%d vocab=%d", rows, vocab);
    KVA_REQUIRE((inv_t != nullptr && tokens != nullptr) || rows == 0, "sample_truncated: a temperature and a place for a token per row are needed");
    KVA_REQUIRE(uniform != nullptr || (key != nullptr && step != nullptr) || rows == 0, "sample_truncated: random numbers or keys and steps are needed");
    if (rows == 0) return KVA_OK;
    int log_vocab = 0;
    while ((1 << log_vocab) < vocab) ++log_vocab;
    const int bits = log_vocab > 16 ? 62 - log_vocab : 46;
    const TruncArgs a{logits, stride, vocab, bits, inv_t, top_k, top_p, min_p, uniform, seed, key, step, tokens, host_mapped, kept, logprob};
    if (!trunc_split(vocab)) {
        if (vocab <= TR_HELD_VOCAB) hipLaunchKernelGGL(sample_truncated_kernel<true>, dim3(rows), dim3(TR_THREADS), 0, stream, a);
        else hipLaunchKernelGGL(sample_truncated_kernel<false>, dim3(rows), dim3(TR_THREADS), 0, stream, a);
        KVA_CHECK_LAUNCH("sample_truncated");
        return KVA_OK;
    }
    KVA_REQUIRE(workspace != nullptr && (uintptr_t)workspace % 8 == 0, "sample_truncated: a workspace of kva_sample_truncated_workspace_bytes is needed");
    TruncSpace sp;
    sp.parts = trunc_parts(rows, vocab, &sp.part_tokens);
    sp.buckets = (vocab + TR_BUCKET - 1) / TR_BUCKET;
    sp.few = std::min({rows <= TR_FEW_ROWS ? TR_FEW_MOST_OF_FEW_ROWS : TR_FEW_MOST, sp.parts * TR_GROUPS / 2, TR_FEW_STEPS / (sp.part_tokens / TR_STEP)});
    sp.best = (u64 *)workspace;
    sp.bins = sp.best + (size_t)rows * sp.parts;
    sp.tops = sp.bins + (size_t)rows * TR_BINS;
    sp.sought = sp.tops + (size_t)rows * sp.parts * TR_GROUPS;
    sp.sums = sp.sought + (size_t)rows * 2;
    sp.list = sp.sums + (size_t)rows * sp.buckets;
    sp.counts = (unsigned *)(sp.list + (size_t)rows * TR_LIST);
    sp.listed = (int *)(sp.counts + (size_t)rows * sp.buckets);
    const dim3 grid(sp.parts, rows), block(TR_SPLIT_THREADS);
    hipLaunchKernelGGL(trunc_best_kernel, grid, block, 0, stream, a, sp);
    hipLaunchKernelGGL(trunc_bins_kernel, grid, block, 0, stream, a, sp);
    hipLaunchKernelGGL(trunc_collect_kernel, grid, block, 0, stream, a, sp);
    hipLaunchKernelGGL(trunc_pick_kernel, dim3(rows), dim3(TR_THREADS), 0, stream, a, sp);
    KVA_CHECK_LAUNCH("sample_truncated");
    return KVA_OK;
}
