// How the calls of the sequence operators are cut: which form of a kernel, by rules on sizes and types alone.  Host code without HIP.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "../../include/turboae_hip.h"

namespace tae {
namespace seq {

inline size_t dtype_bytes(int32_t t) { return t == TAE_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int32_t t) { return t >= TAE_DTYPE_F32 && t <= TAE_DTYPE_BF16; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- selective_scan
// How a call is cut: lanes for a channel, each with per_lane states, and pieces along the positions.
struct ScanPlan {
    int lanes = 0, per_lane = 1, groups = 1, pieces = 1, piece_len = 0;       // lanes = 0: few positions, by scan_step_kernel or scan_short_kernel
    size_t steps_bytes = 0, bytes = 0;
};

constexpr int kScanThreads = 256, kLaneWaves = 8;         // of a workgroup; waves of one of scan_lane_kernel
constexpr int kPieceUnit = 64;                   // pieces are whole tiles

// The ways to share a channel's states (4, 8, 16, 32 or 64 with those filled up) among lanes: by scan_short_kernel (lanes = 0, four states
// each), by scan_lane_kernel with one lane, else by selective_scan_kernel.  ns: what a wave takes for a position, with other waves on its
// SIMD; alone: the number of waves whose time one by itself takes; start: us before a round of waves is under way, which up to 64
// positions do not hide.  Fitted to lengths from 2 to 8192 and 128 to 204800 channels of all sequences together, in bf16 with gate.  What is
// taken is not always the best: up to 15 % behind it in the list, which gives whole calls at the best number of pieces.
//     us, pieces in (); batch x len x channels x states      1 lane      4 lanes     8 lanes     16 lanes    taken
//     1 x 4096 x 4096 x 16                                   149 (32)                144 (16)    169 (5)     1 lane (32)
//     8 x 2048 x 1024 x 16                                   147 (16)                136 (8)     128 (1)     16 lanes (1)
//     1 x 2048 x 512 x 16                                     78 (32)                 24 (32)     27 (16)    8 lanes (32)
//     64 x 256 x 256 x 16                                     85 (4)                  30 (1)      38 (1)     8 lanes (1)
//     500 x 100 x 200 x 16                                    68 (1)                  65 (1)      86 (1)     1 lane (1)
//     500 x 100 x 200 x 16, fp32, no gate                     61 (1)                  63 (1)      81 (1)     1 lane (1)
//     2 x 2048 x 2048 x 32                                                           127 (8)     125 (1)     16 lanes (1)
//     20 x 400 x 600 x 8                                                              34 (1)                 8 lanes (1)
//     40 x 569 x 416 x 4                                                  62 (1)                             4 lanes (9), 68
//     8 x 512 x 256 x 64                                                                          51 (1)     16 lanes (4), 59
//     78 x 3961 x 16 x 8                                                              71 (16)                8 lanes (31), 71
// Sequences are counted with all of their positions, whatever `lengths` holds.
struct ScanForm {
    int lanes, per_lane;
    double ns, alone, start;
};
constexpr ScanForm kForms[] = {{0, 4, 232, 1.45, 1}, {0, 8, 180, 1.85, 1}, {0, 16, 152, 2.2, 1}, {0, 32, 130, 2.6, 1}, {0, 64, 138, 2.45, 1},
                              {4, 1, 71, 1.15, 2}, {8, 1, 31, 1.7, 1}, {1, 16, 300, 1.8, 6}, {8, 2, 49, 1.45, 1}, {16, 1, 31, 1.5, 1.3}, {8, 4, 75, 1.5, 2},
                              {16, 2, 45, 1.25, 2.5}, {16, 4, 96, 1.1, 4}};

// Few channels leave SIMDs empty: then fewer states for each lane, or pieces along the positions, which cost a pass for their ends (0.6 of the
// main one) and a launch that joins them (8 us).  The choice is the cheapest by these numbers and the waves that a SIMD (1024 of them) runs.
inline bool plan_scan(const tae_scan_args* p, ScanPlan* out) {
    if (p->batch < 1 || p->len < 1 || p->channels < 1 || p->states < 1 || p->states > 64 || !dtype_ok(p->dtype)) return false;
    if (p->len == 1) return true;
    int padded = 4;
    while (padded < p->states) padded *= 2;
    double least = 0.0;
    for (const ScanForm& f : kForms) {
        const int share = f.lanes ? f.lanes : padded / 4;
        if (f.per_lane * (f.lanes ? f.lanes : 1) != padded || (!f.lanes && p->len > 32)) continue;        // few positions: 32 at the most
        const int64_t groups = ceil_div(p->channels, f.lanes == 1 ? 64 : kScanThreads / share);
        for (int64_t pieces = 1; pieces <= (f.lanes ? 64 : 1); ++pieces) {
            const int64_t piece_len = ceil_div(ceil_div(p->len, pieces), kPieceUnit) * kPieceUnit;
            if (ceil_div(p->len, piece_len) < pieces) continue;
            auto time = [&](int64_t n) {
                const double cus = ceil_div(n * p->batch * groups, f.lanes == 1 ? kLaneWaves : 1) / 256.0;         // workgroups for each
                const double all = f.lanes == 1 ? 2.0 * std::ceil(cus) : cus < 4.0 ? std::ceil(cus) : cus;          // waves for a SIMD of the fullest
                return std::max(all, f.alone) * std::min<int64_t>(piece_len, p->len) * f.ns * 1e-3 + (p->len <= 64 ? f.start * std::max(all, 1.0) : 0.0);
            };
            const double cost = time(pieces) + (pieces > 1 ? 0.6 * time(pieces - 1) + 8.0 : 0.0);
            if (least == 0.0 || cost < least) {
                least = cost;
                out->lanes = f.lanes;
                out->per_lane = f.per_lane;
                out->groups = (int)groups;
                out->pieces = (int)pieces;
                out->piece_len = (int)piece_len;
            }
        }
    }
    if (out->pieces > 1) {
        out->steps_bytes = ((size_t)p->batch * out->pieces * p->channels * 4 + 255) / 256 * 256;
        out->bytes = out->steps_bytes + (size_t)p->batch * (out->pieces + 1) * p->channels * p->states * 4;
    }
    return true;
}

// One position and few: lanes that share a channel, V adjacent states each.
inline int state_lanes(int states, int V) {
    int lanes = 1;
    while (lanes * V < states) lanes *= 2;
    return lanes;
}

// One position: four sequences for each workgroup, so that A is read once for them, as long as two workgroups for each CU remain.
inline int step_sequences(int batch, int channels, int states, int V) { return batch >= 4 && (int64_t)channels * states / V * batch >= 4 * 512 * kScanThreads ? 4 : 1; }

// ---- int8_linear
// How the rows of a product are dealt out: all in one launch (int8_rows_kernel), 16 NF x 16 MF outputs for a workgroup (int8_few_kernel), tiles
// (int8_linear_kernel; two: two workgroups for a CU).
enum class Int8Form { rows, few16, few32, few64, tiles128, tiles128_two, tiles256 };

// Whether int8_rows_kernel takes a call: its rows fit the registers of a workgroup (and so LDS, 16 bytes off multiples of 64 so that the rows
// meet all banks), and the workgroups that repeat the quantising are few.
constexpr int kRowsGroups = 4;                   // groups of 16 bytes that a lane holds
constexpr int64_t kRowsBlocks = 512;
inline int rows_share(const tae_int8_args* p) { return p->rows == 1 ? 8 : p->rows == 2 ? 4 : p->rows <= 4 ? 2 : 1; }
inline bool int8_in_one(const tae_int8_args* p) {
    const int64_t across = 64 * 16 / (int64_t)dtype_bytes(p->dtype) * rows_share(p);
    return p->rows <= 8 && p->inputs <= across * kRowsGroups && ceil_div(p->outputs, 16) <= kRowsBlocks;
}

// Which form.  Up to 256 tiles of 128 x 128 the cheapest by what whole calls measured in bf16, in us, kk = inputs / 4096 and r rounds of 256
// workgroups (1 at least):
//     few, 16 x 16 a workgroup   5.2 + 1.2 kk + r max(3.5, 3.7 kk)        few, 64 x 32   6.0 + 1.2 kk + r max(4.2, 11.4 kk)
//     few, 32 x 32               5.2 + 1.2 kk + r max(3.0, 7.2 kk)        tiles          8.0 + 15.6 kk
// off by a tenth at most from 512 to 16384 inputs, 64 to 16384 outputs and 16 to 512 rows.  Among them, with 4096 outputs:
//     4096 inputs, rows    16   32   64  128  256  512          16384 inputs, rows   16   32   64  128  256  512
//     16 x 16              10   14   22   38   69  131                               27   42   71  127  236  458
//     32 x 32              12   14   14   22   36   66                               38   41   42   70  126  239
//     64 x 32              14   16   18   19   30   53                               43   48   56   57  100  185
//     tiles                22   23   22   23   24   26                               71   71   71   71   72   76
// More tiles:
//     4096 inputs and outputs, rows                        1024  2048  3000  4096          8000 rows, 4000 outputs, inputs  200  500 1000 2000
//     128 x 128, four buffers                                30    51    72    98                                            41   53   70  107
//     the same, two buffers, two workgroups for a CU         34    46    67    91                                            35   47   63   96
//     256 x 256                                                    57    63    83                                            57   65   78  101
inline Int8Form int8_form(const tae_int8_args* p) {
    if (int8_in_one(p)) return Int8Form::rows;
    const int64_t m = p->rows, n = p->outputs;
    const int64_t large = ceil_div(m, 256) * ceil_div(n, 256), small = ceil_div(m, 128) * ceil_div(n, 128);
    if (large >= 192 && p->inputs >= 4096) return Int8Form::tiles256;
    if (small > 256) return Int8Form::tiles128_two;
    const double kk = p->inputs / 4096.0;
    auto rounds = [&](int rows, int outputs) { return std::max(1.0, ceil_div(m, rows) * ceil_div(n, outputs) / 256.0); };
    const double by16 = 5.2 + 1.2 * kk + rounds(16, 16) * std::max(3.5, 3.7 * kk), by32 = 5.2 + 1.2 * kk + rounds(32, 32) * std::max(3.0, 7.2 * kk);
    const double by64 = 6.0 + 1.2 * kk + rounds(64, 32) * std::max(4.2, 11.4 * kk), tiles = 8.0 + 15.6 * kk, least = std::min({by16, by32, by64, tiles});
    return least == by16 ? Int8Form::few16 : least == by32 ? Int8Form::few32 : least == by64 ? Int8Form::few64 : Int8Form::tiles128;
}

inline bool int8_sizes(const tae_int8_args* p) {
    return p->rows >= 1 && p->inputs >= 1 && p->inputs <= 131072 && p->outputs >= 1 && p->rows <= (1 << 30) && p->outputs <= (1 << 30);
}

// ---- token_logprobs
struct LogprobsPlan {
    int lanes = 64, ept = 32, parts = 1, part_len = 0;
    size_t stats_bytes = 0, bytes = 0;
};

// aligned_rows: every row starts on a 16-byte boundary.  An unaligned part that is read in granules of 16 bytes reaches into one more; rows of
// up to 64 are read by single elements and do not.  (Nor are those of up to 512 with alternatives, but an unaligned one of 505 to 512 is no
// worse off in granules: 20000 x 508 in bf16 with one alternative 16 us, by single elements 23; x 511 in fp32 with eight 23 and 20.)
inline bool plan_logprobs(const tae_logprobs_args* p, bool aligned_rows, LogprobsPlan* s) {
    if (p->rows < 1 || p->vocab < 1 || p->vocab > (1 << 21) || p->top < 0 || p->top > 32 || p->top > p->vocab || !dtype_ok(p->dtype)) return false;
    const int V = 16 / (int)dtype_bytes(p->dtype);
    const int spare = aligned_rows ? 0 : V;
    auto parts_of = [&](int lanes, int ept, int most) {
        s->lanes = lanes;
        s->ept = ept;
        s->parts = (int)ceil_div(p->vocab, most);
        s->part_len = (int)std::min<int64_t>(most, ceil_div(ceil_div(p->vocab, s->parts), 8) * 8);
        s->parts = (int)ceil_div(p->vocab, s->part_len);
    };
    // the fewest lanes that hold a row; long rows in parts, smaller ones where few rows would leave SIMDs empty
    const int64_t elements = (int64_t)p->rows * p->vocab;
    if (p->vocab <= 64) parts_of(8, 8, 64);
    else if (p->vocab <= 512 - spare) parts_of(64, 8, 512 - spare);     // with alternatives single elements: all lanes have some, and so a close bound of them
    else if (p->vocab <= 2048 - spare || (elements < (int64_t)2048 * 2048 && p->vocab <= (1 << 18))) parts_of(64, 32, 2048 - spare);
    else if (p->vocab <= 8192 - spare || (elements < (int64_t)1024 * 8192 && p->vocab <= (1 << 20))) parts_of(256, 32, 8192 - spare);
    else parts_of(256, 64, 16384 - spare);
    if (s->parts > 1) {
        s->stats_bytes = (size_t)p->rows * s->parts * 16;
        s->bytes = s->stats_bytes + (size_t)p->rows * s->parts * p->top * 8;
    }
    return true;
}

}  // namespace seq
}  // namespace tae
