// What a request asks of its logits before a token is taken from them.  With l the logit of a token, m whether the request's row of
// marks has it, c how often the request has said it:
//
//     m:            l <- l > 0 ? l / repetition : l * repetition
//     m and c > 0:  l <- l - (frequency c + presence)
//     biases:       l <- l + b, for every one of the row's list that names the token, in the list's order
//     grammar:      l <- -inf where the token's bit is not set, whatever the logit was
//
// One pass: the logits and a byte of marks a token come in 4 tokens a thread and load, a count is looked up only where the mark is
// set, a grammar is a bit a token.  A row's biases are a list in no order: every workgroup picks out those of its own tokens,
// 256 at a time, in the list's order, and the threads that hold the tokens add them.  What is computed is 32-bit throughout.
//
// What bounds it: memory.  A workgroup takes 1,024 tokens, which is as many loads on their way as there are (2,048 / 4,096 a workgroup:
// one row of 128,256 5.1 / 7.4 us instead of 4.0, 256 rows with marks and counts 82 / 95 instead of 76).  Where the rows, what they
// become and their marks are more than the memory-side cache's 256 MiB, all of it passes the caches by: 256 rows 59 to 63 us (4.7 TB/s) instead of
// 76, and 109 instead of 110 with a draw behind it; 192 rows (210 MiB) 41 instead of 43, but 86 instead of 79 with the draw, which then finds nothing kept.
// us in a graph: 1 row with everything 4.0, 64 rows with everything 18.1 (74 MB, 4.1 TB/s).
#include "common.h"

#define AL_THREADS 256
#define AL_WAVES (AL_THREADS / KVA_WAVE)
#define AL_TILE (4 * AL_THREADS)

typedef float al_f32x4 __attribute__((ext_vector_type(4), aligned(4)));         // (rows start at any multiple of their type)
typedef uint16_t al_u16x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint8_t al_u8x4 __attribute__((ext_vector_type(4), aligned(1)));

struct AdjustArgs {
    const void *logits;
    float *out;
    long long in_stride, out_stride;        // elements from a row to the next
    int vocab;
    const int *row_seat;                    // -1: no marks
    int seats;
    const unsigned char *marks;             // [seats, vocab]
    const int *counts;                      // [seats, vocab]
    const float *repetition, *presence, *frequency;
    const int *bias_start, *bias_token;     // [rows + 1], [biases]
    const float *bias_value;
    int biases;
    const int *allowed_row;                 // -1: everything is allowed
    const unsigned *allowed;                // [grammars, words]
    int grammars, words;
};

// grid (tiles, rows); a tile is 1,024 tokens, four neighbouring ones a thread
template <typename T, bool STREAMED>
__global__ void __launch_bounds__(AL_THREADS)
adjust_logits_kernel(AdjustArgs a) {
    __shared__ int hit_token[AL_THREADS];
    __shared__ float hit_value[AL_THREADS];
    __shared__ int hits_of[AL_WAVES];
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid % KVA_WAVE, wave = tid / KVA_WAVE, vocab = a.vocab;
    const int tile0 = blockIdx.x * AL_TILE, tile1 = min(vocab, tile0 + AL_TILE), t = tile0 + 4 * tid;
    const T *in = reinterpret_cast<const T *>(a.logits) + row * a.in_stride;
    float l[4];
    if (t + 3 < vocab) {
        if constexpr (sizeof(T) == 4) {
            const al_f32x4 *p = reinterpret_cast<const al_f32x4 *>(in + t);
            const al_f32x4 v = STREAMED ? __builtin_nontemporal_load(p) : *p;
            l[0] = v.x, l[1] = v.y, l[2] = v.z, l[3] = v.w;
        } else {
            const al_u16x4 *p = reinterpret_cast<const al_u16x4 *>(in + t);
            const al_u16x4 v = STREAMED ? __builtin_nontemporal_load(p) : *p;
            l[0] = bf16_bits_to_float(v.x), l[1] = bf16_bits_to_float(v.y);
            l[2] = bf16_bits_to_float(v.z), l[3] = bf16_bits_to_float(v.w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) l[i] = t + i < vocab ? to_float(in[t + i]) : 0.f;
    }
    // a row that names a seat or a grammar that is not there gets no token at all
    bool lost = false;
    if (a.row_seat != nullptr) {
        const int seat = a.row_seat[row];
        if (seat >= a.seats || seat < -1) lost = true;
        else if (seat >= 0) {
            const unsigned char *marks = a.marks + (size_t)seat * vocab;
            const int *counts = a.counts != nullptr ? a.counts + (size_t)seat * vocab : nullptr;
            const float rep = a.repetition != nullptr ? a.repetition[row] : 1.f;
            const float pres = a.presence != nullptr ? a.presence[row] : 0.f, freq = a.frequency != nullptr ? a.frequency[row] : 0.f;
            unsigned m = 0;
            if (t + 3 < vocab) {
                const al_u8x4 *p = reinterpret_cast<const al_u8x4 *>(marks + t);
                const al_u8x4 v = STREAMED ? __builtin_nontemporal_load(p) : *p;
                m = (v.x != 0) | (v.y != 0) << 1 | (v.z != 0) << 2 | (v.w != 0) << 3;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t + i < vocab && marks[t + i] != 0) m |= 1u << i;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!(m >> i & 1)) continue;
                float x = l[i];
                if (rep != 1.f) x = x > 0.f ? x / rep : x * rep;
                if (counts != nullptr) {
                    const int c = counts[t + i];
                    if (c > 0) x -= fmaf(freq, (float)c, pres);
                }
                l[i] = x;
            }
        }
    }
    if (a.bias_start != nullptr) {
        const int from = max(0, a.bias_start[row]), to = min(a.biases, a.bias_start[row + 1]);
        for (int base = from; base < to; base += AL_THREADS) {
            const int i = base + tid;
            const int token = i < to ? a.bias_token[i] : -1;
            const bool mine = token >= tile0 && token < tile1;
            const unsigned long long votes = __ballot(mine);
            if (lane == 0) hits_of[wave] = __popcll(votes);
            __syncthreads();
            int before = 0, hits = 0;
#pragma unroll
            for (int w = 0; w < AL_WAVES; ++w) {
                if (w < wave) before += hits_of[w];
                hits += hits_of[w];
            }
            if (mine) {
                const int at = before + __popcll(votes & ((1ull << lane) - 1));
                hit_token[at] = token;
                hit_value[at] = a.bias_value[i];
            }
            __syncthreads();
            for (int h = 0; h < hits; ++h) {
                const int rel = hit_token[h] - tile0;
                if (rel >> 2 != tid) continue;
                const int which = rel & 3;
                const float b = hit_value[h];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j == which) l[j] += b;
            }
            __syncthreads();
        }
    }
    const unsigned *allowed = nullptr;
    if (a.allowed_row != nullptr) {
        const int g = a.allowed_row[row];
        if (g >= a.grammars || g < -1) lost = true;
        else if (g >= 0) allowed = a.allowed + (size_t)g * a.words;
    }
    if (t >= vocab) return;
    float *out = a.out + row * a.out_stride;
    unsigned bits = 15;
    if (allowed != nullptr) bits = allowed[t / 32] >> t % 32;
    if (lost) bits = 0;
    al_f32x4 v;
    v.x = bits & 1 ? l[0] : -INFINITY;
    v.y = bits & 2 ? l[1] : -INFINITY;
    v.z = bits & 4 ? l[2] : -INFINITY;
    v.w = bits & 8 ? l[3] : -INFINITY;
    al_f32x4 *to = reinterpret_cast<al_f32x4 *>(out + t);
    if (t + 3 < vocab) {
        if (STREAMED) __builtin_nontemporal_store(v, to);
        else *to = v;
    } else
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (t + i < vocab) out[t + i] = v[i];
}

// address [11], the host's: of row_seat, marks, counts, repetition, presence, frequency, the biases' starts, tokens and values, allowed_row
// and allowed (0: absent)
extern "C" int kva_adjust_logits(const long long *address, float *out, long long out_stride, const void *logits, int dtype, long long in_stride,
                                 int rows, int vocab, int seats, int biases, int grammars, hipStream_t stream) {
    const int *row_seat = (const int *)address[0], *counts = (const int *)address[2], *bias_start = (const int *)address[6],
              *bias_token = (const int *)address[7], *allowed_row = (const int *)address[9];
    const unsigned char *marks = (const unsigned char *)address[1];
    const float *repetition = (const float *)address[3], *presence = (const float *)address[4], *frequency = (const float *)address[5],
                *bias_value = (const float *)address[8];
    const unsigned *allowed = (const unsigned *)address[10];
    KVA_REQUIRE(dtype == KVA_F32 || dtype == KVA_BF16, "adjust_logits: dtype %d", dtype);
    KVA_REQUIRE(rows >= 0 && rows <= 65535 && vocab > 0 && vocab < 1 << 30, "adjust_logits: bad sizes rows=%d vocab=%d", rows, vocab);
    KVA_REQUIRE(row_seat == nullptr || (marks != nullptr && seats > 0), "adjust_logits: seats without marks");
    KVA_REQUIRE(allowed_row == nullptr || (allowed != nullptr && grammars > 0), "adjust_logits: grammars are missing");
    KVA_REQUIRE(marks != nullptr || (counts == nullptr && repetition == nullptr), "adjust_logits: counts and repetition need marks");
    if (rows == 0) return KVA_OK;
    KVA_REQUIRE((marks == nullptr) == (row_seat == nullptr) && (allowed == nullptr) == (allowed_row == nullptr),
                "adjust_logits: marks and seats, grammars and the rows' numbers of them go together");
    KVA_REQUIRE(biases >= 0 && biases <= INT_MAX - AL_THREADS, "adjust_logits: %d biases", biases);
    KVA_REQUIRE(biases == 0 || (bias_start != nullptr && bias_token != nullptr && bias_value != nullptr), "adjust_logits: a part of the biases is missing");
    const AdjustArgs a{logits, out, in_stride, out_stride, vocab, row_seat, seats, marks, counts, repetition, presence, frequency, bias_start,
                       bias_token, bias_value, biases, allowed_row, allowed, grammars, (vocab + 31) / 32};
    const long long touched = (long long)rows * vocab * ((dtype == KVA_F32 ? 4 : 2) + 4 + (row_seat != nullptr ? 1 : 0));
    const bool streamed = touched > 256ll << 20;
    const dim3 grid((vocab + AL_TILE - 1) / AL_TILE, rows), block(AL_THREADS);
    const auto kernel = dtype == KVA_F32 ? (streamed ? adjust_logits_kernel<float, true> : adjust_logits_kernel<float, false>)
                                         : (streamed ? adjust_logits_kernel<bf16_t, true> : adjust_logits_kernel<bf16_t, false>);
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, a);
    KVA_CHECK_LAUNCH("adjust_logits");
    return KVA_OK;
}

// counts[seat][token] += 1 and marks[seat][token] = 1; additions of whole numbers, so any order gives the same
__global__ void __launch_bounds__(256)
count_tokens_kernel(unsigned char *__restrict__ marks, int *__restrict__ counts, int seats, int vocab, const int *__restrict__ of,
                    const int *__restrict__ tokens, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int seat = of[i], token = tokens[i];
    if (seat < 0 || seat >= seats || token < 0 || token >= vocab) return;
    const size_t at = (size_t)seat * vocab + token;
    marks[at] = 1;
    if (counts != nullptr) atomicAdd(counts + at, 1);
}

extern "C" int kva_count_tokens(unsigned char *marks, int *counts, int seats, int vocab, const int *of, const int *tokens, int n,
                                hipStream_t stream) {
    KVA_REQUIRE(n >= 0 && n <= INT_MAX - 255 && seats > 0 && vocab > 0, "count_tokens: bad sizes seats=%d vocab=%d tokens=%d", seats, vocab, n);
    if (n == 0) return KVA_OK;
    KVA_REQUIRE(marks != nullptr && of != nullptr && tokens != nullptr, "count_tokens: marks, seats and tokens are needed");
    hipLaunchKernelGGL(count_tokens_kernel, dim3((n + 255) / 256), dim3(256), 0, stream, marks, counts, seats, vocab, of, tokens, n);
    KVA_CHECK_LAUNCH("count_tokens");
    return KVA_OK;
}
