// attn_kv.h -- launch records and device helpers of the paged key-value cache's kernels (attn_kv.hip: append,
// evict; attn_decode.hip: attention of one new token).
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

// Whether a call's launches stay below the 2^32 threads that HIP takes (of arguments that are valid otherwise).
inline bool launch_fits(double groups, int threads) { return groups * threads < 4294967296.0; }
bool append_fits(const tkm_attn_kv& kv, int S);
bool decode_fits(const tkm_attn_kv& kv, int Hq, int add_weights);
bool evict_fits(const tkm_attn_kv& src, const tkm_attn_kv& dst, int budget);

// Each launches on args.stream, of a call that fits, and returns 0, or -1 when a launch failed (what depends on it is
// then not launched).
int launch_append(const AppendArgs& a);
int launch_decode(const DecodeArgs& a);
int launch_evict(const EvictArgs& a);
size_t decode_workspace(const tkm_attn_kv& kv, int Hq, int add_weights);
// Tiles of 32 tokens times kv-head groups that a decoding call may meet (int range is checked against this).
double decode_tiles_most(const tkm_attn_kv& kv, int Hq);

}  // namespace tkm
