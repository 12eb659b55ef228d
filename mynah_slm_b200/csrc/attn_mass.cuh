// How the sums of attention weights are cut into units of work (attn_mass.cu, attn_mass_tcgen05.cu): a unit is some key tiles of
// one sequence against some of its row tiles, for one kv head. A step of many rows (prompts) has one key tile a unit and is cut
// over its rows too; in one whose sequences have a single row tile each (decode steps, short pieces) a unit takes several key
// tiles. Both counts are such that all units together are about `target`, worked out on the device from the step's own lengths.
#pragma once
#include "attn_rows.cuh"

struct MassArgs {
    RowsArgs r;
    int keys, rows;                   // cached rows a key tile, packed rows a row tile
    int by_keys;                      // 1: no sequence of the step has more than one row tile
    int target;                       // units to aim at over all kv heads; 0: a key tile a unit, rows are never cut
    int score_rows;                   // > 0: the attention keeps its scores, of so many rows a kv head at most
};

struct MassUnit {
    int b, kt0, kt1;                  // key tiles [kt0, kt1)
    int piece, pieces, rt;            // row tiles [piece * rt, (piece + 1) * rt) of the sequence's
    int unit0;
    SeqShape s;
};

__device__ __forceinline__ int mass_ktiles(const SeqShape& s, const MassArgs& a) { return s.n_q > 0 ? (s.kvl + a.keys - 1) / a.keys : 0; }
__device__ __forceinline__ int mass_rtiles(const SeqShape& s, const MassArgs& a) { return a.r.by_tile.div(s.n_q * a.r.G + a.rows - 1); }

// Finds unit `flat`, like find_row_unit: a sequence's units lie together, key tiles ascending (the first keys have the most rows
// above them), a key tile's pieces one after the other.
__device__ __forceinline__ bool find_mass_unit(const int* __restrict__ cu_q, const int* __restrict__ kv_len, const PageTable& pt, const MassArgs& a, int flat,
                                               MassUnit& u, int* status) {
    __shared__ int found_s[3];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        int each = a.by_keys ? 1 : 1 << 28;                // key tiles a unit, or row tiles
        if (a.target > 0) {
            long long work = 0;
            for (int b0 = 0; b0 < a.r.B; b0 += 32) {
                if (b0 + lane < a.r.B) {
                    const SeqShape s = seq_shape(cu_q, kv_len, pt, b0 + lane, a.r, status);
                    work += (long long)mass_ktiles(s, a) * mass_rtiles(s, a);
                }
            }
            work = warp_sum_ll(work);
            each = (int)max(1ll, (work * a.r.KV + a.target - 1) / a.target);
        }
        int fb = -1, base = 0, first = 0;
        for (int b0 = 0; b0 < a.r.B && fb < 0; b0 += 32) {
            int n = 0;
            if (b0 + lane < a.r.B) {
                const SeqShape s = seq_shape(cu_q, kv_len, pt, b0 + lane, a.r, status);
                const int kt = mass_ktiles(s, a);
                n = a.by_keys ? (kt + each - 1) / each : kt * ((mass_rtiles(s, a) + each - 1) / each);
            }
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const int excl = incl - n;
            const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && flat >= base + excl && flat < base + incl);
            if (hit != 0u) {
                const int src = __ffs(hit) - 1;
                fb = b0 + src;
                first = base + __shfl_sync(0xffffffffu, excl, src);
            }
            base += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) {
            found_s[0] = fb;
            found_s[1] = first;
            found_s[2] = each;
        }
    }
    __syncthreads();
    u.b = found_s[0];
    if (u.b < 0) return false;
    u.unit0 = found_s[1];
    const int each = found_s[2], at = flat - u.unit0;
    u.s = seq_shape(cu_q, kv_len, pt, u.b, a.r, status);
    if (a.by_keys) {
        u.rt = 1 << 28;
        u.piece = 0;
        u.pieces = 1;
        u.kt0 = at * each;
        u.kt1 = min(u.kt0 + each, mass_ktiles(u.s, a));
    } else {
        u.rt = each;
        u.pieces = (mass_rtiles(u.s, a) + each - 1) / each;
        u.kt0 = at / u.pieces;
        u.kt1 = u.kt0 + 1;
        u.piece = at % u.pieces;
    }
    return true;
}

// The first row tile with a token that sees the key tile's first key.
__device__ __forceinline__ int mass_first_tile(const MassUnit& u, const MassArgs& a) {
    const int tok = max(0, u.kt0 * a.keys - (u.s.kvl - u.s.n_q));
    return tok * a.r.G / a.rows;
}

// Where a key's sum lies, or -1.
__device__ __forceinline__ long long mass_at(const PageTable& pt, int b, int key, int KV, int g) {
    const int page = page_of(pt, b, key);
    return page < 0 ? -1 : ((long long)page * KV + g) * PAGE_TOKENS + key % PAGE_TOKENS;
}

// Most units (of one kv head) for `n_ids` pages of all sequences.
static inline long long mass_units_max(const MassArgs& a, int n_ids) {
    const long long cut = a.target > 0 ? ceil_div(a.target, a.r.KV) : 0;
    if (a.by_keys && a.target > 0) return cut + a.r.B;
    return ceil_div_ll((long long)n_ids * PAGE_TOKENS, a.keys) + a.r.B + cut;
}

bool mass_tcgen05_takes(int dtype, int H, int KV, int HD);
int launch_mass_tcgen05(const void* q, const void* k, const float* lse, float* mass, float* part, const int* cu_q, const int* kv_len,
                        PageTable pt, const MassArgs& a, int n_ids, int* status, cudaStream_t stream);
