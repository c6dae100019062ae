// attn_kv.h -- launch records and device helpers of the paged key-value cache's kernels (attn_kv.hip: append,
// evict; attn_decode.hip: attention of one new token; attn_plan.hip: pages and slots of a step; attn_rope.hip:
// rotary positions, packed rows into the cache; attn_chunk.hip: attention of several new tokens).
//
// Layout: a page holds `page` tokens of every kv head in 32 x 32 blocks of 16-bit values,
//   K [num_pages][Hkv][page/32][D/32][32 tokens][32 dims]
//   V [num_pages][Hkv][page/32][D/32][32 dims][32 tokens]
// so that the 32 tokens of a tile are 64*D contiguous bytes in either, K in the order in which S^T = K Q^T reads
// its A operand and V, transposed, in the order in which O^T = V^T P^T does: a decoding wave loads both straight
// from HBM into MFMA operand registers, 1024 contiguous bytes an instruction, without LDS or lane exchanges.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "tkm_attn.h"

namespace tkm {

struct AppendArgs {
    tkm_attn_kv kv;
    const void* qkv;
    int S, Hq;
    const int32_t* start;   // NULL: kv.len, advanced in place
    const int32_t* n_new;   // NULL: S rows each
    void* stream;
};

struct DecodeArgs {
    tkm_attn_kv kv;
    const void* q;
    long long q_stride;     // elements between two sequences' rows of q
    void* o;
    float* lse;             // or NULL
    int Hq;
    float scale;
    int add_weights;
    void* ws;
    void* stream;
};

struct EvictArgs {
    tkm_attn_kv src, dst;   // the same tables and lengths: in place
    int32_t* kept;
    int budget, sink, recent;
    void* stream;
};

struct RopeArgs {
    tkm_attn_rope rope;
    const void* in;
    long long in_stride;
    void* out;
    long long out_stride;
    const int32_t* pos;     // NULL: r % S
    int S, rows, Hq, Hkv, D, dtype, inverse, clear;     // clear: rows of negative positions become 0
    void* stream;
};

struct StoreArgs {
    tkm_attn_kv kv;
    const tkm_attn_rope* rope;    // or NULL
    const void* qkv;
    long long stride;
    void* q;                      // or NULL
    long long q_stride;
    const int32_t *seq, *pos;
    const int64_t* slot;
    int rows, Hq;
    void* stream;
};

struct PlanArgs {
    tkm_attn_kv kv;
    tkm_attn_pages pages;
    const int32_t *want, *start;  // start NULL: kv.len
    tkm_attn_plan plan;
    int rows;
    void* stream;
};

struct ChunkArgs {
    tkm_attn_kv kv;
    const void* q;
    long long q_stride;
    const int32_t *row_start, *n_new;
    int rows;
    void* o;
    float* lse;             // or NULL
    int Hq;
    float scale;
    int causal, window;
    void* ws;
    void* stream;
};

// Whether a call's launches stay below the 2^32 threads that HIP takes (of arguments that are valid otherwise).
inline bool launch_fits(double groups, int threads) { return groups * threads < 4294967296.0; }
bool append_fits(const tkm_attn_kv& kv, int S);
bool decode_fits(const tkm_attn_kv& kv, int Hq, int add_weights);
bool evict_fits(const tkm_attn_kv& src, const tkm_attn_kv& dst, int budget);
bool rows_fit(const tkm_attn_kv* kv, int rows);
bool chunk_fits(const tkm_attn_kv& kv, int rows, int Hq);

// Each launches on args.stream, of a call that fits, and returns 0, or -1 when a launch failed (what depends on it is
// then not launched).
int launch_append(const AppendArgs& a);
int launch_decode(const DecodeArgs& a);
int launch_evict(const EvictArgs& a);
int launch_rope(const RopeArgs& a);
int launch_store(const StoreArgs& a);
int launch_plan(const PlanArgs& a);
int launch_chunk(const ChunkArgs& a);
size_t chunk_workspace(const tkm_attn_kv& kv, int rows, int Hq);
size_t decode_workspace(const tkm_attn_kv& kv, int Hq, int add_weights);
// Tiles of 32 tokens times kv-head groups that a decoding call may meet (int range is checked against this).
double decode_tiles_most(const tkm_attn_kv& kv, int Hq);

}  // namespace tkm
