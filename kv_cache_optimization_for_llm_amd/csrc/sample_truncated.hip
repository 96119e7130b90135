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
// Which tokens stay hangs on long sums next to a border, so weights are whole numbers: W_i = round(2^s w_i), s = 46 for a
// vocabulary of up to 2^16 and one less for every doubling, from an exponential in 64 bits.  Sums of them are exact and the same in
// any order: atomics may add them up, and a row draws the same token whoever shares the launch with it.
//
// The order is one of 64-bit places, (the logit's bits, descending) above (the id): both cuts are a place, and what stays is what
// lies in front of it.  A cut is found by counting: the places still in question are cut into 1,024 ranges, their numbers and
// weights added up in LDS, and the range in which the sum passes what is sought is the next turn's.
//
// sample_truncated_kernel: a workgroup a row, which reads the row again in every turn.
#include "common.h"
#include "counter_uniform.h"

#define TR_THREADS 1024
#define TR_WAVES (TR_THREADS / KVA_WAVE)
#define TR_NO_TOKEN (-1)
#define TR_DIGITS 1024

typedef unsigned long long u64;

struct TruncArgs {
    const float *logits;
    long long stride;
    int vocab, scale_bits;
    const float *inv_t;                 // <= 0: the best token
    const int *top_k;                   // absent: all of them
    const float *top_p, *min_p;
    const float *uniform;               // absent: the counter-based number of (seed, key, step)
    unsigned seed;
    const unsigned *key, *step;
    int *tokens, *host_tokens, *kept;
    float *logprob;
};

// descending logits as ascending 32-bit numbers; the two zeros are one (l + 0: -0 becomes 0)
__device__ inline unsigned tr_falling(float l) {
    const unsigned b = __float_as_uint(l + 0.f);
    return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ inline u64 tr_place(float l, int id) { return (u64)tr_falling(l) << 32 | (unsigned)id; }

// how far below the best one a logit lies, in units of log2(weight)
__device__ inline double tr_octaves(float best, float l, double octaves_per_unit) {
    const double d = (double)best - (double)l;
    return d == 0.0 ? 0.0 : d * octaves_per_unit;
}
// round(2^bits 2^-octaves)
__device__ inline u64 tr_weight(double octaves, int bits) {
    return octaves < bits + 1.0 ? (u64)__double2ll_rn(exp2((double)bits - octaves)) : 0ull;
}

__device__ inline u64 tr_wave_prefix(u64 v) {
    const int lane = threadIdx.x % KVA_WAVE;
#pragma unroll
    for (int off = 1; off < KVA_WAVE; off <<= 1) {
        const u64 below = __shfl_up(v, off, KVA_WAVE);
        if (lane >= off) v += below;
    }
    return v;
}

struct TruncShared {
    u64 sum[TR_DIGITS];
    unsigned count[TR_DIGITS];
    u64 part[TR_WAVES];
    unsigned part_count[TR_WAVES];
    u64 lo, hi, above;
    unsigned above_count, inside_count;
    int found;
};

// The smallest of all threads' numbers and the largest.
__device__ inline void tr_block_range(TruncShared &s, u64 &lo, u64 &hi) {
#pragma unroll
    for (int off = KVA_WAVE / 2; off > 0; off >>= 1) {
        const u64 a = __shfl_xor(lo, off, KVA_WAVE), b = __shfl_xor(hi, off, KVA_WAVE);
        lo = min(lo, a);
        hi = max(hi, b);
    }
    __syncthreads();
    if (threadIdx.x % KVA_WAVE == 0) s.sum[threadIdx.x / KVA_WAVE] = lo, s.part[threadIdx.x / KVA_WAVE] = hi;
    __syncthreads();
    lo = s.sum[0], hi = s.part[0];
    for (int w = 1; w < TR_WAVES; ++w) lo = min(lo, s.sum[w]), hi = max(hi, s.part[w]);
    __syncthreads();
}

// Inclusive prefix sums of a number and a count a thread over the workgroup.
__device__ inline void tr_block_prefix(TruncShared &s, u64 &v, unsigned &c) {
    const int lane = threadIdx.x % KVA_WAVE, wave = threadIdx.x / KVA_WAVE;
    v = tr_wave_prefix(v);
#pragma unroll
    for (int off = 1; off < KVA_WAVE; off <<= 1) {
        const unsigned below = __shfl_up(c, off, KVA_WAVE);
        if (lane >= off) c += below;
    }
    __syncthreads();
    if (lane == KVA_WAVE - 1) s.part[wave] = v, s.part_count[wave] = c;
    __syncthreads();
    for (int w = 0; w < wave; ++w) v += s.part[w], c += s.part_count[w];
}

// grid (rows)
__global__ void __launch_bounds__(TR_THREADS)
sample_truncated_kernel(TruncArgs a) {
    __shared__ TruncShared s;
    const int row = blockIdx.x, tid = threadIdx.x, vocab = a.vocab, bits = a.scale_bits;
    const float *rl = a.logits + row * a.stride;
    const float inv_t = a.inv_t[row];
    const bool sampled = inv_t > 0.f;
    // the best place and the last one
    u64 lo = ~0ull, hi = 0;
    unsigned valid = 0;
    for (int t = tid; t < vocab; t += TR_THREADS) {
        const float l = rl[t];
        if (!(l > -INFINITY)) continue;
        const u64 at = tr_place(l, t);
        lo = min(lo, at);
        hi = max(hi, at);
        ++valid;
    }
    {
        u64 none = 0;
        tr_block_prefix(s, none, valid);
        if (tid == TR_THREADS - 1) s.inside_count = valid;
        tr_block_range(s, lo, hi);
        valid = s.inside_count;
    }
    const int best_id = (int)(unsigned)lo;
    const float best = valid ? rl[best_id] : 0.f;
    int token = valid ? best_id : TR_NO_TOKEN, kept = valid ? 1 : 0;
    float logprob = valid ? 0.f : -INFINITY;
    if (sampled && valid && best == INFINITY) token = TR_NO_TOKEN, kept = 0, logprob = -INFINITY;
    if (sampled && token >= 0) {
        const double rate = (double)inv_t * 1.4426950408889634;
        // The place of the order's n-th token (by_count), or of the first at which the weights reach `need`, of those up to
        // `hi`; `before` gets the weights in front of it, `weight` its own.  There is one.
        auto cut = [&](u64 from, u64 to, bool by_count, u64 need, u64 &upto) {
            u64 front = 0;                      // numbers or weights in front of `from`, and the weights alone
            u64 front_weight = 0;
            while (true) {
                const u64 span = to - from;
                const int shift = span < TR_DIGITS ? 0 : 64 - __clzll((long long)span) - 10;
                s.sum[tid] = 0;
                s.count[tid] = 0;
                __syncthreads();
                for (int t = tid; t < vocab; t += TR_THREADS) {
                    const float l = rl[t];
                    if (!(l > -INFINITY)) continue;
                    const u64 at = tr_place(l, t);
                    if (at < from || at > to) continue;
                    const int digit = (int)((at - from) >> shift);
                    atomicAdd(&s.sum[digit], tr_weight(tr_octaves(best, l, rate), bits));
                    atomicAdd(&s.count[digit], 1u);
                }
                __syncthreads();
                const u64 mine = s.sum[tid];
                const unsigned n = s.count[tid];
                u64 sum = mine;
                unsigned count = n;
                tr_block_prefix(s, sum, count);
                const u64 reach = front + (by_count ? (u64)count : sum), behind = reach - (by_count ? (u64)n : mine);
                if (behind < need && need <= reach) {           // (one thread's range)
                    s.found = tid;
                    s.above = behind;
                    s.lo = front_weight + sum - mine;
                    s.hi = front_weight + sum;
                }
                __syncthreads();
                const int digit = s.found;
                if (shift == 0) {
                    upto = s.hi;
                    const u64 at = from + (u64)digit;
                    __syncthreads();
                    return at;
                }
                front = s.above;
                front_weight = s.lo;
                from += (u64)digit << shift;
                to = min(to, from + ((1ull << shift) - 1));
                __syncthreads();
            }
        };
        u64 last = hi, total = 0;               // the last place that stays, the weight up to it
        const int k = a.top_k != nullptr ? a.top_k[row] : 0;
        const float p = a.top_p != nullptr ? a.top_p[row] : 1.f;
        const double least = a.min_p != nullptr ? (double)a.min_p[row] : 0.0;
        if (k > 0 && (unsigned)k < valid) last = cut(lo, hi, true, (u64)k, total);
        if (p < 1.f) {
            if (total == 0) {
                u64 sum = 0;
                unsigned none = 0;
                for (int t = tid; t < vocab; t += TR_THREADS)
                    if (rl[t] > -INFINITY) sum += tr_weight(tr_octaves(best, rl[t], rate), bits);
                tr_block_prefix(s, sum, none);
                if (tid == TR_THREADS - 1) s.hi = sum;
                __syncthreads();
                total = s.hi;
                __syncthreads();
            }
            const double share = ceil((double)p * (double)total);
            const u64 need = share >= 1.0 ? min((u64)share, total) : 1ull;
            last = cut(lo, last, false, need, total);
        }
        // what stays, by ids: ranges of ids first, then the tokens of one
        const int per = (vocab + TR_THREADS - 1) / TR_THREADS;
        auto stays = [&](float l, int t, u64 &weight) {
            weight = 0;
            if (!(l > -INFINITY) || tr_place(l, t) > last) return false;
            const double octaves = tr_octaves(best, l, rate);
            weight = tr_weight(octaves, bits);
            if (least > 0.0 && octaves > 0.0 && !(exp2(-octaves) >= least)) {
                weight = 0;
                return false;
            }
            return true;
        };
        u64 sum = 0;
        unsigned count = 0;
        for (int t = tid * per; t < min(vocab, (tid + 1) * per); ++t) {
            u64 w;
            if (stays(rl[t], t, w)) ++count;
            sum += w;
        }
        const u64 mine = sum;
        tr_block_prefix(s, sum, count);
        if (tid == TR_THREADS - 1) s.hi = sum, s.inside_count = count;
        __syncthreads();
        const u64 all = s.hi;
        kept = (int)s.inside_count;
        const float u = a.uniform != nullptr ? a.uniform[row] : counter_uniform(a.seed, a.key[row], a.step[row]);
        u64 target = u > 0.f ? (u64)(fmin((double)u, 1.0) * (double)all) : 0ull;
        target = min(target, all - 1);
        if (sum - mine <= target && target < sum) {
            u64 run = sum - mine, w = 0;
            int t = tid * per;
            for (;; ++t) {
                stays(rl[t], t, w);
                run += w;
                if (target < run) break;
            }
            s.found = t;
        }
        __syncthreads();
        token = s.found;
        logprob = (float)(-0.6931471805599453 * (tr_octaves(best, rl[token], rate) + log2((double)all) - (double)bits));
    }
    if (tid == 0) {
        a.tokens[row] = token;
        if (a.host_tokens != nullptr) a.host_tokens[row] = token;
        if (a.kept != nullptr) a.kept[row] = kept;
        if (a.logprob != nullptr) a.logprob[row] = logprob;
    }
}

extern "C" int kva_sample_truncated(int *tokens, const float *logits, long long stride, int rows, int vocab, const float *inv_t,
                                    const int *top_k, const float *top_p, const float *min_p, const float *uniform, unsigned seed,
                                    const unsigned *key, const unsigned *step, int *kept, float *logprob, int *host_tokens,
                                    hipStream_t stream) {
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
    KVA_REQUIRE(inv_t != nullptr || rows == 0, "sample_truncated: a temperature per row is needed");
    KVA_REQUIRE(uniform != nullptr || (key != nullptr && step != nullptr) || rows == 0, "sample_truncated: random numbers or keys and steps are needed");
    if (rows == 0) return KVA_OK;
    int log_vocab = 0;
    while ((1 << log_vocab) < vocab) ++log_vocab;
    const int bits = log_vocab > 16 ? 62 - log_vocab : 46;
    const TruncArgs a{logits, stride, vocab, bits, inv_t, top_k, top_p, min_p, uniform, seed, key, step, tokens, host_mapped, kept, logprob};
    hipLaunchKernelGGL(sample_truncated_kernel, dim3(rows), dim3(TR_THREADS), 0, stream, a);
    KVA_CHECK_LAUNCH("sample_truncated");
    return KVA_OK;
}
