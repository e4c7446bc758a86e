// fpa_serve.h -- parameter blocks and launchers of the serving operators: the paged cache, First Passage
// Attention of new tokens against it, the verification of drafted tokens.
//
// A page holds 64 positions of every head.  With page p of the pool and head h (ph = p * H + h):
//   k        [ph][64][D]   rows of positions, as the score product's row operand reads them
//   v        [ph][D][64]   transposed, so that the operand of V^T P^T (one feature, 16 consecutive positions)
//                          is contiguous too: no transpose and no LDS between HBM and the matrix cores
//   phi, psi [ph][64]      float32
//   phi_min  [ph]          min of phi over the page's written positions: the range minimum of a query far
//                          behind a key reads one value for every 64 positions in between
//   k_exp, v_exp [ph][64]  int8, e4m3 caches only: the row of a position is code * 2^exp
#pragma once

#include "fpa_params.h"

namespace fpa {

constexpr int PG = 64;                         // positions of a page
constexpr int EXP_MIN = -60, EXP_MAX = 60;     // exponents of e4m3 rows
enum { ST_F16 = 0, ST_F32 = 1, ST_E4M3 = 2 };  // FPA_F16, FPA_F32, FPA_E4M3

struct e4m3 {  // storage only
    uint8_t code;
};

struct Pages {
    void *k, *v;
    float *phi, *psi, *phi_min;
    int8_t *k_exp, *v_exp;
    int64_t n;  // pages of the pool
    int H;
};

// Append (k, v, phi, psi in) and read (out) move positions start[b] + i, i < counts[b] (N without counts).
struct MoveParams {
    Pages c;
    const void *k; S3 sk;  // append: (B, H, N, D) with unit d stride
    const void *v; S3 sv;
    const float *phi; S3 sphi;
    const float *psi; S3 spsi;
    void *ko, *vo;         // read: (B, H, N, D), (B, H, N) contiguous
    float *phio, *psio;
    const int32_t *table; int64_t stable;
    const int32_t *start, *counts;
    int B, N, P, D;
};

struct AttendParams {
    Pages c;
    const void *q; S3 sq;  // (B, H, N, D)
    void *o; S3 so;
    const float *beta;
    const int32_t *table; int64_t stable;
    const int32_t *lengths;
    const int32_t *prefix;
    float *part, *ml;      // per part and row: O (D floats), then its running maximum and sum
    int32_t *counts;       // parts done of each (b, h), or (h, tile) with a prefix; 0 before and after every launch
    int B, N, P;
    int PL;                // positions of the shared prefix (0: none)
    int chunk, nchunk;     // pages of a part (set on the device), parts at most, of a sequence's own pages
    int least, slots;      // a part's pages are a multiple of `least`; workgroups that run at once
    int64_t own_groups;    // workgroups for the sequences' own pages
    int pchunk, npchunk;   // the same of the prefix (npchunk = 0: none)
    bool alone;            // a wave takes a sequence's own pages of a head by itself (nchunk = 1)
    float sc2;             // log2(e) / sqrt(D)
};

struct VerifyParams {
    const void *target; int64_t stb, stn;
    const void *draft; int64_t sdb, sdn;  // NULL: the drafts have no probabilities
    const int64_t *tokens; int64_t sxb;
    const float *accept_u; int64_t sub;
    const float *sample_u;
    int64_t *accepted, *out;
    double *sums;     // (B, 4 spans, 2): of each quarter of a span
    int32_t *counts;  // (B,): spans done; 0 before and after every launch
    int B, N, V;
    int span, spans;
};

hipError_t launch_append(const MoveParams &p, int dtype, int store, hipStream_t s);
hipError_t launch_read(const MoveParams &p, int dtype, int store, hipStream_t s);
hipError_t launch_attend(const AttendParams &p, int dtype, int store, int D, hipStream_t s);
// Whether a wave takes all own pages of a sequence and head.
bool attend_alone(int64_t B, int64_t H, int64_t N, int64_t pages, int D, int dtype, bool prefix);
int attend_rows(int64_t rows, int D, int dtype);  // rows of a tile of the prefix
int attend_waves(int D);  // of a workgroup
// Steps a page of the kernel, for a sequence's own N rows (sets = 0) or the prefix's tiles of 16 * sets rows.
int attend_steps(int D, int dtype, int store, int64_t N, bool prefix, int sets);
// Pages of the prefix's parts and their number.
void attend_parts(int64_t items, int64_t pages, int D, int steps, int64_t taken, int &chunk, int &nchunk);
// Sequences' own pages: least, slots, parts at most and workgroups (see AttendParams).
void attend_own(int64_t B, int64_t units, int64_t pages, int D, int steps, int page_bytes, bool prefix, int &least, int &slots, int &nchunk, int64_t &groups);
// Tokens of a span.
int verify_span(int64_t B, int64_t V);
hipError_t launch_verify(const VerifyParams &p, int dtype, hipStream_t s);

}  // namespace fpa
