// What stands in front of a step's layers, made on the device from what the step's requests are: the pages that a request's
// block table gains, and for every token of the step its position, its seat and its place in every group of the cache.
//
//     needs    n_e = max(0, ceil(length_e / page) - held_e),  o_e = n_0 + ... + n_(e-1)
//     tables   table[seat_e][held_e + j] = pages[o_e + j],  j < n_e
//     tokens   q_e = l_0 + ... + l_(e-1); token t of entry e (q_e <= t < q_(e+1)) has position x = start_e + t - q_e and
//              slot table[seat_e][x / page] * page + x % page
//
// Every workgroup adds up the entries in front of its own itself instead of waiting for another launch's prefix sums: some
// thousand numbers out of L2 are a trip to memory and a tree of additions.  Sums are 64 bits wide.
#include "common.h"

#define ST_THREADS 256
#define ST_MAX_ENTRIES 4096
#define ST_MAX_GROUPS 8

// Inclusive prefix sum over the 64 lanes.
__device__ inline long long st_wave_prefix(long long v) {
    const int lane = threadIdx.x % KVA_WAVE;
#pragma unroll
    for (int off = 1; off < KVA_WAVE; off <<= 1) {
        const long long below = __shfl_up(v, off, KVA_WAVE);
        if (lane >= off) v += below;
    }
    return v;
}

// Sum over the workgroup, all threads get it.
__device__ inline long long st_block_sum(long long v, long long *scratch) {
    v = st_wave_prefix(v);
    __syncthreads();
    if (threadIdx.x % KVA_WAVE == KVA_WAVE - 1) scratch[threadIdx.x / KVA_WAVE] = v;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < ST_THREADS / KVA_WAVE; ++w) total += scratch[w];
    return total;
}

struct GrowArgs {
    int *table;
    const int *seats, *held, *lengths, *pages;
    int *offsets;               // [entries + 1]
    int entries, rows, blocks, page_size, num_pages;
};

// pages that entry e takes; none where its seat or its blocks lie outside the table
__device__ inline long long grow_need(const GrowArgs &a, int e) {
    const int seat = a.seats[e], held = a.held[e];
    const long long want = ((long long)a.lengths[e] + a.page_size - 1) / a.page_size;
    if (seat < 0 || seat >= a.rows || held < 0 || want > a.blocks || want <= held) return 0;
    return want - held;
}

// grid (entries, segments of the table's row)
__global__ void __launch_bounds__(ST_THREADS)
grow_tables_kernel(GrowArgs a, int segment) {
    __shared__ long long scratch[ST_THREADS / KVA_WAVE];
    const int e = blockIdx.x;
    const long long need = grow_need(a, e);
    // (the last entry's workgroup leaves the total; the others of an entry that takes nothing have only its offset to write)
    const int from = blockIdx.y * segment, to = (int)min((long long)from + segment, need);
    if (blockIdx.y > 0 && from >= to) return;
    long long before = 0;
    for (int i = threadIdx.x; i < e; i += ST_THREADS) before += grow_need(a, i);
    before = st_block_sum(before, scratch);
    if (blockIdx.y == 0 && threadIdx.x == 0) {
        a.offsets[e] = (int)min(before, (long long)INT_MAX);
        if (e == a.entries - 1) a.offsets[e + 1] = (int)min(before + need, (long long)INT_MAX);
    }
    if (before + need > a.num_pages) return;            // not all of its pages are there: it takes none
    const int *src = a.pages + before;
    int *dst = a.table + (size_t)a.seats[e] * a.blocks + a.held[e];
    for (int j = from + threadIdx.x; j < to; j += ST_THREADS) dst[j] = src[j];
}

extern "C" int kva_grow_tables(int *table, int rows, int blocks, const int *seats, const int *held, const int *lengths, int entries,
                               int page_size, const int *pages, int num_pages, int *offsets, hipStream_t stream) {
    KVA_REQUIRE(entries >= 0 && entries <= ST_MAX_ENTRIES, "grow_tables: %d requests are not in 0..%d", entries, ST_MAX_ENTRIES);
    KVA_REQUIRE(rows > 0 && blocks > 0 && page_size > 0 && num_pages >= 0, "grow_tables: bad sizes rows=%d blocks=%d page_size=%d pages=%d", rows,
                blocks, page_size, num_pages);
    if (entries == 0) return KVA_OK;
    const int segment = 2048;
    hipLaunchKernelGGL(grow_tables_kernel, dim3(entries, (blocks + segment - 1) / segment), dim3(ST_THREADS), 0, stream,
                       GrowArgs{table, seats, held, lengths, pages, offsets, entries, rows, blocks, page_size, num_pages}, segment);
    KVA_CHECK_LAUNCH("grow_tables");
    return KVA_OK;
}

struct RowsArgs {
    const int *lengths, *starts, *seats;
    int *q_start, *positions, *tok_seat;
    int entries, tokens, page_size, groups;
    const int *table[ST_MAX_GROUPS];
    int *slots[ST_MAX_GROUPS];
    int rows[ST_MAX_GROUPS], blocks[ST_MAX_GROUPS];
};

// grid (tokens / 1,024): four neighbouring tokens a thread
__global__ void __launch_bounds__(ST_THREADS)
step_rows_kernel(RowsArgs a) {
    __shared__ int first[ST_MAX_ENTRIES + 1];           // first[e]: the entry's first token (no larger than INT_MAX)
    __shared__ long long scratch[ST_THREADS / KVA_WAVE];
    const int tid = threadIdx.x, wave = tid / KVA_WAVE;
    long long run = 0;
    for (int base = 0; base < a.entries; base += ST_THREADS) {
        const int e = base + tid;
        const long long mine = e < a.entries ? max(0, a.lengths[e]) : 0;
        const long long upto = st_wave_prefix(mine);
        __syncthreads();
        if (tid % KVA_WAVE == KVA_WAVE - 1) scratch[wave] = upto;
        __syncthreads();
        long long below = run;
#pragma unroll
        for (int w = 0; w < ST_THREADS / KVA_WAVE; ++w) {
            if (w < wave) below += scratch[w];
            run += scratch[w];
        }
        if (e < a.entries) first[e] = (int)min(below + upto - mine, (long long)INT_MAX);
    }
    if (tid == 0) first[a.entries] = (int)min(run, (long long)INT_MAX);
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = tid; e <= a.entries; e += ST_THREADS) a.q_start[e] = first[e];
    const int end = min(first[a.entries], a.tokens);    // what lies behind the last entry is left as it is
    const long long t0 = (long long)blockIdx.x * (4 * ST_THREADS) + 4 * tid;
    if (t0 >= end) return;
    // the entry that t0 belongs to: the last whose first token is not behind it
    int lo = 0, hi = a.entries;                         // first[lo] <= t0 < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= t0) lo = mid;
        else hi = mid;
    }
    const int n = (int)min(4ll, end - t0);
    int seat[4];
    long long pos[4];
    int e = lo, start = a.starts[e], s = a.seats[e];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = (int)t0 + min(i, n - 1);
        if (t >= first[e + 1]) {
            do ++e;
            while (t >= first[e + 1]);                  // (t < end: an entry that holds it comes)
            start = a.starts[e];
            s = a.seats[e];
        }
        seat[i] = s;
        pos[i] = (long long)start + (t - first[e]);
    }
    auto store = [&](int *out, const int (&v)[4]) {
        if (n == 4 && ((uintptr_t)out & 15) == 0) {
            *reinterpret_cast<int4 *>(out + t0) = make_int4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < n) out[t0 + i] = v[i];
        }
    };
    const int where[4] = {(int)pos[0], (int)pos[1], (int)pos[2], (int)pos[3]};
    store(a.positions, where);
    store(a.tok_seat, seat);
    for (int g = 0; g < a.groups; ++g) {
        int slot[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long block = pos[i] / a.page_size;
            slot[i] = -1;
            if (i < n && pos[i] >= 0 && block < a.blocks[g] && seat[i] >= 0 && seat[i] < a.rows[g]) {
                const long long page = a.table[g][(size_t)seat[i] * a.blocks[g] + block];
                const long long place = page * a.page_size + (pos[i] - block * a.page_size);
                if (page >= 0 && place <= INT_MAX) slot[i] = (int)place;
            }
        }
        store(a.slots[g], slot);
    }
}

// group [groups][4], the host's: a table's address, its rows and blocks, and the address of the group's slots
extern "C" int kva_step_rows(const int *lengths, const int *starts, const int *seats, int entries, const long long *group, int groups,
                             int page_size, int tokens, int *q_start, int *positions, int *tok_seat, hipStream_t stream) {
    KVA_REQUIRE(entries >= 0 && entries <= ST_MAX_ENTRIES, "step_rows: %d entries are not in 0..%d", entries, ST_MAX_ENTRIES);
    KVA_REQUIRE(groups >= 0 && groups <= ST_MAX_GROUPS, "step_rows: %d groups are not in 0..%d", groups, ST_MAX_GROUPS);
    KVA_REQUIRE(tokens >= 0 && page_size > 0, "step_rows: bad sizes tokens=%d page_size=%d", tokens, page_size);
    RowsArgs a{lengths, starts, seats, q_start, positions, tok_seat, entries, tokens, page_size, groups, {}, {}, {}, {}};
    for (int g = 0; g < groups; ++g, group += 4) {
        KVA_REQUIRE(group[1] > 0 && group[2] > 0 && group[1] <= INT_MAX && group[2] <= INT_MAX, "step_rows: table %d is %lld x %lld", g, group[1], group[2]);
        a.table[g] = (const int *)group[0];
        a.rows[g] = (int)group[1];
        a.blocks[g] = (int)group[2];
        a.slots[g] = (int *)group[3];
    }
    const int grid = max(1, (int)(((long long)tokens + 4 * ST_THREADS - 1) / (4 * ST_THREADS)));
    hipLaunchKernelGGL(step_rows_kernel, dim3(grid), dim3(ST_THREADS), 0, stream, a);
    KVA_CHECK_LAUNCH("step_rows");
    return KVA_OK;
}
