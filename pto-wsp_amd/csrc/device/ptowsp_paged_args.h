// Kernel arguments of the paged-cache operators (ptowsp_paged.h), shared by
// the host library and the kernels.  Strides are in elements.
#pragma once

namespace ptowsp {

constexpr int kPlanRows = 1024;     // rows of a workgroup of paged_plan's second launch
constexpr int kAttendThreads = 256, kAttendTile = 128;  // a workgroup of paged_attention, and tokens of its tile
constexpr int kSpanInts = 8;        // AttendArgs::spans of a workgroup
constexpr int kUnitInts = 4;        // AttendArgs::units of an entry
constexpr int kUnitHead = 4;        // AttendArgs::units before the entries

struct PlanArgs {
    const int* lengths;
    const int* counts;
    const int* free_pages;
    const int* used;
    int* table;
    int* new_lengths;
    int* new_used;
    int* starts;
    int* slots;
    long long s_lengths, s_counts, s_free, s_table, s_table_col, s_new_lengths, s_starts, s_slots;
    long long batch, width, nfree, rows;
    int page;
    int* err;      // 4: the plan does not fit (nothing is written), 5: a page number out of range
    int* scratch;  // two-launch form: {ok, total}, then starts, lengths and first new page of each request
};

struct StoreArgs {
    const char* x[2];  // keys, values
    char* cache[2];
    float* scale[2];
    const int* slots;
    long long s_x[2][2];      // row, head
    long long s_cache[2][3];  // page, head, token
    long long s_scale[2][2];  // page, head
    long long s_slots;
    long long rows, pages;
    int heads;
    int* err;  // 6: a slot outside the cache (its rows are not stored)
};

struct AttendArgs {
    const char* q;
    const char* cache[2];
    const float* scale[2];
    const int* table;
    const int* lengths;
    const int* starts;
    char* out;
    float* lse;
    long long s_q[2], s_out[2], s_lse[2];  // row, head
    long long s_cache[2][3];               // page, head, token
    long long s_scale[2][2];               // page, head
    long long s_table, s_lengths, s_starts;
    long long batch, width, pages, rows;
    int heads;     // key heads
    int window;    // 0: none
    float factor;  // scale * log2(e)
    int* err;      // 7: starts, lengths or a page out of range
    int blocks;    // workgroups for few rows
    int* spans;    // per workgroup: where the unit that it leaves open is joined
    float* parts;  // partial results, two per workgroup
    // Prompts: the list of their units, and partial results of those that are cut.
    int* units;
    float* unit_parts;
    int room, counters;  // entries and counters that `units` has room for
    int cus;             // workgroups that run at once
    int few;       // requests of at most so many rows are left to the kernel for few rows
};

}  // namespace ptowsp
