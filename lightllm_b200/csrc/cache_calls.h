// What the calls of a cache that is drafted into and thinned out take (span_attention.cu, cache_rows.cu).  csrc/ops.py fills these structs
// member by member; a change takes the library's next version number.
#pragma once

// q, out [T, Hq, hd]; caches [num_slots, Hkv, hd]; span arrays [S]; table [S, max_pages]; scratch of llb_span_scratch_floats.
typedef struct LlbSpanCall {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    const int* span_row;
    const int* span_len;
    const int* span_pos;
    const int* table;
    float* scratch;
    int* error_flag;
    int dtype, S, T, max_pages, page_size, num_slots, Hq, Hkv, hd;
    float scale;
} LlbSpanCall;

// mask [T, words].
typedef struct LlbTreeAttention {
    LlbSpanCall span;
    const unsigned long long* mask;
    int words, unused;
} LlbTreeAttention;

// Causal; mass_in (may be null) and mass [Hkv, num_slots], may be the same; a request's rows beyond max_len are left out.
typedef struct LlbAttentionMass {
    LlbSpanCall span;
    const float* mass_in;
    float* mass;
    int max_len, unused;
} LlbAttentionMass;

// tokens, parents, targets [T]; caches [L, num_slots, row_bytes]; path [S, width], count [S], next [S].
typedef struct LlbTreeCommit {
    const int* tokens;
    const int* parents;
    const int* targets;
    void* k;
    void* v;
    const int* span_row;
    const int* span_len;
    const int* span_pos;
    const int* table;
    int* path;
    int* count;
    int* next;
    int S, T, L, max_pages, page_size, num_slots, row_bytes, width;
} LlbTreeCommit;

// caches [L, num_slots, Hkv, head_bytes]; mass, positions and their outputs [L, Hkv, num_slots] (the outputs may be the inputs).
typedef struct LlbCacheEvict {
    void* k;
    void* v;
    const float* mass;
    const int* positions;
    float* mass_out;
    int* positions_out;
    const int* lengths;
    const int* ends;
    const int* table;
    int S, L, Hkv, max_pages, page_size, num_slots, head_bytes, budget, first, latest;
} LlbCacheEvict;
