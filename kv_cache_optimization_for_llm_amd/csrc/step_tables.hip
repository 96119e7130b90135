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
#include "wave_scan.h"

#define ST_THREADS 256
#define ST_MAX_ENTRIES 4096
#define ST_MAX_GROUPS 8
#define ST_STAGED 256

typedef int st_i32x4 __attribute__((ext_vector_type(4), aligned(4)));

// Sum over the workgroup, all threads get it.
__device__ inline u64 st_block_sum(u64 v, u64 *scratch) {
    v = wave_prefix(v);
    __syncthreads();
    if (threadIdx.x % KVA_WAVE == KVA_WAVE - 1) scratch[threadIdx.x / KVA_WAVE] = v;
    __syncthreads();
    u64 total = 0;
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

// grid (entries).  1,024 requests of up to 4,096 pages (8 MB written): 6.9 us in a graph, 7.9 with four workgroups a request of 2,048 blocks
// each, 64 requests of a page each 3.2: a trip to memory for the needs, one for the pages.
__global__ void __launch_bounds__(ST_THREADS)
grow_tables_kernel(GrowArgs a) {
    __shared__ u64 scratch[ST_THREADS / KVA_WAVE];
    const int e = blockIdx.x;
    const long long need = grow_need(a, e);
    u64 sum = 0;
    for (int i = threadIdx.x; i < e; i += ST_THREADS) sum += grow_need(a, i);
    const long long before = st_block_sum(sum, scratch);
    if (threadIdx.x == 0) {
        a.offsets[e] = (int)min(before, (long long)INT_MAX);
        if (e == a.entries - 1) a.offsets[e + 1] = (int)min(before + need, (long long)INT_MAX);
    }
    if (before + need > a.num_pages) return;            // not all of its pages are there: it takes none
    const int *src = a.pages + before;
    int *dst = a.table + (size_t)a.seats[e] * a.blocks + a.held[e];
    for (long long j = 4 * threadIdx.x; j < need; j += 4 * ST_THREADS) {
        if (j + 3 < need) *reinterpret_cast<st_i32x4 *>(dst + j) = *reinterpret_cast<const st_i32x4 *>(src + j);
        else
            for (long long i = j; i < need; ++i) dst[i] = src[i];
    }
}

// address [6], the host's: of the table, seats, held, lengths, pages and offsets
extern "C" int kva_grow_tables(const long long *address, int rows, int blocks, int entries, int page_size, int num_pages, hipStream_t stream) {
    int *table = (int *)address[0], *offsets = (int *)address[5];
    const int *seats = (const int *)address[1], *held = (const int *)address[2], *lengths = (const int *)address[3], *pages = (const int *)address[4];
    KVA_REQUIRE(entries >= 0 && entries <= ST_MAX_ENTRIES, "grow_tables: %d requests are not in 0..%d", entries, ST_MAX_ENTRIES);
    KVA_REQUIRE(rows > 0 && blocks > 0 && page_size > 0 && num_pages >= 0, "grow_tables: bad sizes rows=%d blocks=%d page_size=%d pages=%d", rows,
                blocks, page_size, num_pages);
    if (entries == 0) return KVA_OK;
    KVA_REQUIRE(table != nullptr && seats != nullptr && held != nullptr && lengths != nullptr && offsets != nullptr && (pages != nullptr || num_pages == 0),
                "grow_tables: a seat, held blocks and a length per request, and a row of pages are needed");
    hipLaunchKernelGGL(grow_tables_kernel, dim3(entries), dim3(ST_THREADS), 0, stream,
                       GrowArgs{table, seats, held, lengths, pages, offsets, entries, rows, blocks, page_size, num_pages});
    KVA_CHECK_LAUNCH("grow_tables");
    return KVA_OK;
}

struct RowsArgs {
    const int *lengths, *starts, *seats;
    int *q_start, *positions, *tok_seat;
    int entries, tokens, page_size, page_shift, groups; // page_shift: of a power of two, else -1
    const int *table[ST_MAX_GROUPS];
    int *slots[ST_MAX_GROUPS];
    int rows[ST_MAX_GROUPS], blocks[ST_MAX_GROUPS];
};

// grid (tokens / 1,024): four neighbouring tokens a thread.  Up to 256 entries' starts and seats come to LDS with their lengths, one
// trip to memory less on the way from the lengths to the slots; of 1,024 entries that is more than every workgroup saves (2^20 tokens
// 11.0 us against 10.3).  us in a graph: 64 entries of a token, two groups 5.0 (5.9 with a loop over the groups, a trip to memory each, and divisions of
// 64 bits), 2^20 tokens of 1,024 entries, three groups 10.3 (13.8): 20 MB written, and 64 bytes of a table read for every page of 16 tokens.
template <int ENTRIES, int GROUPS>
__global__ void __launch_bounds__(ST_THREADS)
step_rows_kernel(RowsArgs a) {
    constexpr bool STAGED = ENTRIES <= ST_STAGED;
    __shared__ int first[ENTRIES + 1];                  // first[e]: the entry's first token (no larger than INT_MAX)
    __shared__ int start_of[STAGED ? ENTRIES : 1], seat_of[STAGED ? ENTRIES : 1];
    __shared__ u64 scratch[ST_THREADS / KVA_WAVE];
    const int tid = threadIdx.x, wave = tid / KVA_WAVE;
    u64 run = 0;
    for (int base = 0; base < a.entries; base += 4 * ST_THREADS) {
        int n[4];
        u64 mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = base + 4 * tid + i;
            n[i] = e < a.entries ? max(0, a.lengths[e]) : 0;
            mine += n[i];
            if (STAGED && e < a.entries) start_of[e] = a.starts[e], seat_of[e] = a.seats[e];
        }
        const u64 upto = wave_prefix(mine);
        __syncthreads();
        if (tid % KVA_WAVE == KVA_WAVE - 1) scratch[wave] = upto;
        __syncthreads();
        u64 at = run + upto - mine;
#pragma unroll
        for (int w = 0; w < ST_THREADS / KVA_WAVE; ++w) {
            if (w < wave) at += scratch[w];
            run += scratch[w];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = base + 4 * tid + i;
            if (e < a.entries) first[e] = (int)min(at, (u64)INT_MAX);
            at += n[i];
        }
    }
    if (tid == 0) first[a.entries] = (int)min(run, (u64)INT_MAX);
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
    unsigned pos[4];                                    // (past 2^31: the kernels that read positions take them as they are)
    int e = lo, start = STAGED ? start_of[e] : a.starts[e], s = STAGED ? seat_of[e] : a.seats[e];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = (int)t0 + min(i, n - 1);
        if (t >= first[e + 1]) {
            do ++e;
            while (t >= first[e + 1]);                  // (t < end: an entry that holds it comes)
            start = STAGED ? start_of[e] : a.starts[e];
            s = STAGED ? seat_of[e] : a.seats[e];
        }
        seat[i] = s;
        pos[i] = (unsigned)start + (unsigned)(t - first[e]);
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
    unsigned block[4], row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        block[i] = a.page_shift >= 0 ? pos[i] >> a.page_shift : pos[i] / (unsigned)a.page_size;
        row[i] = pos[i] - block[i] * (unsigned)a.page_size;
    }
    // (all groups' pages are asked for before the first is used)
    int page[GROUPS][4];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        if (g >= a.groups) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool there = i < n && pos[i] <= INT_MAX && block[i] < (unsigned)a.blocks[g] && (unsigned)seat[i] < (unsigned)a.rows[g];
            page[g][i] = there ? a.table[g][(size_t)seat[i] * a.blocks[g] + block[i]] : -1;
        }
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        if (g >= a.groups) break;
        int slot[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned long long place = (unsigned long long)(unsigned)page[g][i] * (unsigned)a.page_size + row[i];
            slot[i] = page[g][i] >= 0 && place <= INT_MAX ? (int)place : -1;
        }
        store(a.slots[g], slot);
    }
}

// address [6 + 2 groups], the host's: of lengths, starts, seats, q_start, positions and tok_seat, then of a group's table and slots each; size
// [groups][2], the host's: a table's rows and blocks
extern "C" int kva_step_rows(const long long *address, const long long *size, int entries, int groups, int page_size, int tokens, hipStream_t stream) {
    KVA_REQUIRE(entries >= 0 && entries <= ST_MAX_ENTRIES, "step_rows: %d entries are not in 0..%d", entries, ST_MAX_ENTRIES);
    KVA_REQUIRE(groups >= 0 && groups <= ST_MAX_GROUPS, "step_rows: %d groups are not in 0..%d", groups, ST_MAX_GROUPS);
    KVA_REQUIRE(tokens >= 0 && page_size > 0, "step_rows: bad sizes tokens=%d page_size=%d", tokens, page_size);
    const int shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
    RowsArgs a{(const int *)address[0], (const int *)address[1], (const int *)address[2], (int *)address[3], (int *)address[4], (int *)address[5],
               entries, tokens, page_size, shift, groups, {}, {}, {}, {}};
    KVA_REQUIRE(a.q_start != nullptr && (entries == 0 || (a.lengths != nullptr && a.starts != nullptr && a.seats != nullptr)) &&
                    (tokens == 0 || (a.positions != nullptr && a.tok_seat != nullptr)),
                "step_rows: a length, a start and a seat per entry, and places for what is made of them are needed");
    for (int g = 0; g < groups; ++g) {
        const long long rows = size[2 * g], blocks = size[2 * g + 1];
        KVA_REQUIRE(rows > 0 && blocks > 0 && rows <= INT_MAX && blocks <= INT_MAX, "step_rows: table %d is %lld x %lld", g, rows, blocks);
        a.table[g] = (const int *)address[6 + 2 * g];
        a.slots[g] = (int *)address[7 + 2 * g];
        KVA_REQUIRE(a.table[g] != nullptr && (tokens == 0 || a.slots[g] != nullptr), "step_rows: table %d or its slots are missing", g);
        a.rows[g] = (int)rows;
        a.blocks[g] = (int)blocks;
    }
    const int grid = max(1, (int)(((long long)tokens + 4 * ST_THREADS - 1) / (4 * ST_THREADS)));
    const bool staged = entries <= ST_STAGED, few = groups <= 2;
    const auto kernel = staged ? (few ? step_rows_kernel<ST_STAGED, 2> : step_rows_kernel<ST_STAGED, ST_MAX_GROUPS>)
                               : (few ? step_rows_kernel<ST_MAX_ENTRIES, 2> : step_rows_kernel<ST_MAX_ENTRIES, ST_MAX_GROUPS>);
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(ST_THREADS), 0, stream, a);
    KVA_CHECK_LAUNCH("step_rows");
    return KVA_OK;
}
