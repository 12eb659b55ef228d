// How the sums of attention weights are cut into units of work (attn_mass.cu, attn_mass_tcgen05.cu): a unit is some key tiles of
// one sequence against some of its row tiles, for one kv head. A step of many rows (prompts) has one key tile a unit and is cut
// over its rows too; in one whose sequences have a single row tile each (decode steps, short pieces) a unit takes several key
// tiles. On the tensor cores both counts are such that all units together are about `target`, worked out on the device from the
// step's own lengths. On the general kernel a unit is one key tile, and a sequence's row tiles are cut into `own_pieces` at most by
// their own number alone: a sum's bits are then the same whatever else is in the step (row_units.cuh).
#pragma once
#include "attn_rows.cuh"

struct MassArgs {
    RowsArgs r;
    int keys, rows;                   // cached rows a key tile, packed rows a row tile
    int by_keys;                      // 1: no sequence of the step has more than one row tile
    int target;                       // units to aim at over all kv heads; 0: a key tile a unit, rows cut by the sequence alone
    int own_pieces;                   // target 0: pieces of a sequence's row tiles at most
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

// Row tiles a piece: `each` of the step, or by the sequence alone.
__device__ __forceinline__ int mass_piece(const SeqShape& s, const MassArgs& a, int each) {
    return a.target > 0 ? each : max(1, quotient(mass_rtiles(s, a) + a.own_pieces - 1, a.own_pieces));
}

// Finds unit `flat`: a sequence's units lie together, key tiles ascending (the first keys have the most rows above them), a key
// tile's pieces one after the other.
__device__ __forceinline__ bool find_mass_unit(const int* __restrict__ cu_q, const int* __restrict__ kv_len, const PageTable& pt, const MassArgs& a, int flat,
                                               MassUnit& u, int* status) {
    __shared__ int found_s[3];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        int each = 1;                                      // key tiles a unit, or row tiles
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
                const int rt = mass_piece(s, a, each);
                n = a.by_keys ? (kt + each - 1) / each : kt * quotient(mass_rtiles(s, a) + rt - 1, rt);
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
        u.rt = mass_piece(u.s, a, each);
        u.pieces = quotient(mass_rtiles(u.s, a) + u.rt - 1, u.rt);
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
    const long long cut = a.target > 0 ? ceil_div(a.target, a.r.KV) : 0, most = ceil_div_ll((long long)n_ids * PAGE_TOKENS, a.keys) + a.r.B;
    if (a.target > 0) return a.by_keys ? cut + a.r.B : most + cut;
    const long long tiles = ceil_div_ll((long long)a.r.most_q * a.r.G, a.rows);        // of the longest sequence
    return most * (a.by_keys ? 1 : tiles < a.own_pieces ? tiles : a.own_pieces);
}

bool mass_tcgen05_takes(int dtype, int H, int KV, int HD);
int launch_mass_tcgen05(const void* q, const void* k, const float* lse, float* mass, float* part, const int* cu_q, const int* kv_len,
                        PageTable pt, const MassArgs& a, int n_ids, int* status, cudaStream_t stream);
