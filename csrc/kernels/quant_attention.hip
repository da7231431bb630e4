// quant_attention.hip — attention over a paged cache in 8 or 4 bits (chronos_quant_kv.h), for one token of each sequence, several, or prompts, and for groups
// of sequences whose first pages are the same.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  over the keys j <= position of i; token i of a sequence is at ctx - len + i.
//
// Rows are (token, query head) pairs of one key head; a workgroup takes a tile of 16 NQT rows, of one sequence, one key head and one piece of the keys.  Its four
// waves take steps of 32 keys in turn, each with a running reference and sum, and are joined through LDS; pieces of the keys are joined by a second launch.  S^T = K Q^T
// and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16: with the keys as rows of the first product a lane holds the scores of its own query row, and the probabilities are
// the second one's operand as they are.  Codes go from memory to registers and become bfloat16 there, which is exact (eight bits, and e2m1 times a power of two):
//   * K: the dimensions of a product may be taken in any order that queries and keys share, so a lane takes its row's bytes 16 at a time;
//   * V: the operand wants eight keys of one dimension, the page has the dimensions of one key.  Row m of product dt is dimension m D / 16 + dt: a lane then needs the
//     same D / 16 neighbouring bytes of its eight keys, for all products, and no exchange between lanes.
// int8: a key's scale multiplies its scores, a value's the probabilities.  These are then rounded to float16 (2^-11): in bfloat16 the largest probability of a row, 1 times a scale, would
// be off by up to 2^-8 where without scales it is exact (.0025 of the output's size in place of .0017, of which its own rounding is .0016).  Each row's sums have a reference
// that keeps its products in float16's range, the largest at 2^7 to 2^15; what is 2^-32 of the largest and less may get lost.  That holds for value scales of 2^-83 to 2^101: probabilities are
// float32 and go up to 2^90, so that they can be summed, and no lower than 2^-126, so beside smaller or larger scales less than 2^-32 gets lost, and all at 2^-115.
// mxfp4: the conversion takes the scale, so a key's 32-dimension blocks have scales of their own that no probability can carry, and only bfloat16 has room for them: probabilities are bfloat16
// (2^-8).  The sum that divides is of the rounded ones: what all of a row's large probabilities are off by in common then cancels, and an average of equal values is that value.  2 x 128 rows
// of 64 heads on 16k shared keys: .0019 of the output's size, no number off by more than .0083, 189 us; with a sum of the unrounded .0020, .0119, 186 us.  The output's rounding alone is .00165 and .0078.
//
// The reference that a row's probabilities are 2^(score - ref) of only moves when a score is far over it (2^8; int8: as float16 allows): rescaling the sums costs as much as all
// else that a step does to them, and while it stays no lane needs to know of another.  mxfp4: where values are so large that 2^8 times as much, over 2^30 keys, would pass float32's
// range (E over 213, numbers over 2^86), the scores stay as far below the reference as it takes (most_over).  Averages are joined with weights that add up to one, or 2^-8 of them.
//
// What no sum may take: keys behind the position, behind the context, on pages that the table does not have (numbers outside 0 .. pages - 1 are left out): their
// scores are -inf and their probabilities zero by selection, not by product; their values cannot be NaN either (a value scale of NaN acts on the probabilities of
// rows that see it).  Rows without any key are zeros.
#include <limits.h>

#include "chronos_lds.h"
#include "chronos_quant_kv.h"

namespace chronos {
namespace qkv {

struct AttnArgs {
    const uint16_t* q;
    int64_t q_stride;         // elements between tokens
    Cache cache;
    const int32_t* bt;        // [B, width]
    int64_t bt_stride;
    int width;
    const int32_t* q_start;   // [B + 1] or nullptr: token i is sequence i
    const int32_t* ctx_len;   // [B]
    const int32_t* group_start;   // [groups + 1] or nullptr
    const int32_t* prefix_len;    // [groups]
    int B, T, groups, hq;
    float scale_log2;
    uint16_t* out;            // [T, hq, D]
    float* part_o;            // [slots, T * hq, D]
    float* part_l;            // [slots, T * hq]: base-2 logarithm of the sum of probabilities, -inf: no keys; part_o is what they average to
    int slots, splits, slot0;
    int page_shift;           // pages of a power of two tokens; -1: others
    bool last;                // the sequences' own keys, after what their groups share, in one piece: joins both and writes the output
    bool longest;             // tiles by the number of their keys, most first (find_longest)
};

namespace {

// ---- which rows a workgroup has -----------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int first_row(const AttnArgs& a, int seq) {   // token where sequence seq begins; tokens behind the last sequence are its follower's
    if (seq <= 0) return 0;
    if (seq > a.B) return a.T;
    if (!a.q_start) return min(seq, a.T);
    return min(max(a.q_start[seq], 0), a.T);
}
__device__ __forceinline__ int first_seq(const AttnArgs& a, int group) { return min(max(a.group_start[group], 0), a.B); }

struct Tile {
    int item;       // sequence or group; a.B: the tokens behind the last sequence
    int tok0, toks;   // the item's tokens
    int at;         // the tile's first row among the item's toks * G
    __device__ __forceinline__ void same() {   // they are the same in all lanes, and the compiler may know
        item = __builtin_amdgcn_readfirstlane(item);
        tok0 = __builtin_amdgcn_readfirstlane(tok0);
        toks = __builtin_amdgcn_readfirstlane(toks);
        at = __builtin_amdgcn_readfirstlane(at);
    }
};
// Tile `index` of the items' tiles of `rows` rows, in order.  Every wave finds it by itself: 64 items at a time, their tiles counted up across the lanes.
template <bool GROUPS> __device__ __forceinline__ bool find_tile(const AttnArgs& a, int index, int G, int rows, int lane, Tile& out) {
    if (!GROUPS && !a.q_start) {
        const int per = (G + rows - 1) / rows, t = index / per;
        if (t >= a.T) return false;
        out = Tile{min(t, a.B), t, 1, (index - t * per) * rows};
        return true;
    }
    const int items = GROUPS ? a.groups : a.B + 1;
    int before = 0;
    for (int i0 = 0; i0 < items; i0 += 64) {
        const int i = i0 + lane;
        int t0 = 0, t1 = 0;
        if (i < items) {
            t0 = first_row(a, GROUPS ? first_seq(a, i) : i);
            t1 = first_row(a, GROUPS ? first_seq(a, i + 1) : i + 1);
        }
        const int n = max(t1 - t0, 0) * G, tiles = (n + rows - 1) / rows;
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o, 64);
            if (lane >= o) upto += v;
        }
        const int total = __builtin_amdgcn_readlane(upto, 63);
        if (index < before + total) {
            const int l = __builtin_ctzll(__ballot(before + upto > index));
            out.item = i0 + l;
            out.tok0 = __builtin_amdgcn_readlane(t0, l);
            out.toks = __builtin_amdgcn_readlane(t1, l) - out.tok0;
            out.at = (index - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(tiles, l))) * rows;
            return true;
        }
        before += total;
    }
    return false;
}
// Tile `index` of up to 255 sequences' tiles, those with most keys first (within 32): where tiles are more than the card holds at a time, a prompt's last ones, which are
// its longest, are not what all others wait for.  Every wave finds it by itself, halving the range of lengths: count() tiles have more than 32 `level` keys.
__device__ __forceinline__ bool find_longest(const AttnArgs& a, int index, int G, int rows, int lane, Tile& out) {
    constexpr int CH = 4;
    int t0[CH], n[CH], ctx[CH], most = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int seq = i * 64 + lane;
        t0[i] = seq <= a.B ? first_row(a, seq) : a.T;
        n[i] = seq <= a.B ? max(first_row(a, seq + 1) - t0[i], 0) : 0;
        ctx[i] = seq < a.B ? (int)min((int64_t)max(a.ctx_len[seq], 0), (int64_t)a.width * a.cache.page) : 0;
        most = max(most, ctx[i]);
    }
    const int shift = __builtin_ctz(rows);   // a power of two
    auto of = [&](int i, int level) {   // tiles of item i * 64 + lane with more than 32 level keys: its last ones
        const int tiles = (n[i] * G + rows - 1) >> shift, more = level * 32 - ctx[i] + n[i];
        return level < 0 ? tiles : ctx[i] <= level * 32 ? 0 : tiles - min(more > 0 ? (more * G) >> shift : 0, max(tiles - 1, 0));
    };
    auto count = [&](int level) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i * 64 <= a.B) c += of(i, level);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) c += __shfl_xor(c, o, 64);
        return __builtin_amdgcn_readfirstlane(c);
    };
    if (index >= count(-1)) return false;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o, 64));
    int low = -1, high = __builtin_amdgcn_readfirstlane(most) / 32 + 1;   // count(low) > index >= count(high)
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (count(mid) > index) low = mid;
        else high = mid;
    }
    int before = count(high);   // the tile is one of those with more than 32 low keys and no more than 32 high
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if (i * 64 > a.B) break;
        const int some = of(i, low), here = some - of(i, high);
        int upto = here;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o, 64);
            if (lane >= o) upto += v;
        }
        const int total = __builtin_amdgcn_readlane(upto, 63);
        if (index < before + total) {
            const int l = __builtin_ctzll(__ballot(before + upto > index));
            out.item = i * 64 + l;
            out.tok0 = __builtin_amdgcn_readlane(t0[i], l);
            out.toks = __builtin_amdgcn_readlane(n[i], l);
            const int tiles = (out.toks * G + rows - 1) >> shift;
            out.at = (tiles - __builtin_amdgcn_readlane(some, l) + index - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(here, l))) << shift;
            return true;
        }
        before += total;
    }
    return false;
}
// whole pages of the prefix that sequence seq shares with its group (0: none), and the group
__device__ __forceinline__ int shared_keys(const AttnArgs& a, int group) {
    const int64_t n = min((int64_t)max(a.prefix_len[group], 0), (int64_t)a.width * a.cache.page);
    return (int)(n - n % a.cache.page);
}
__device__ __forceinline__ int shared_of(const AttnArgs& a, int seq, int lane) {
    int g = -1;   // groups that begin at or before seq, less one
    for (int i0 = 0; i0 <= a.groups; i0 += 64) {
        const int i = i0 + lane;
        g += __popcll(__ballot(i <= a.groups && first_seq(a, min(i, a.groups)) <= seq));
    }
    return g >= 0 && g < a.groups ? shared_keys(a, g) : -1;
}

// What a workgroup's item is: its sequence (of a group: the one whose table is read), context and the keys that the launch has of it
template <bool GROUPS> struct Item {
    int seq, ctx, k0;
    __device__ __forceinline__ Item(const AttnArgs& a, const Tile& t, int lane) : seq(t.item), ctx(0), k0(0) {
        if constexpr (GROUPS) {
            seq = min(first_seq(a, t.item), a.B - 1);
        } else {
            if (seq < a.B) {
                ctx = __builtin_amdgcn_readfirstlane((int)min((int64_t)max(a.ctx_len[seq], 0), (int64_t)a.width * a.cache.page));
                if (a.group_start) k0 = __builtin_amdgcn_readfirstlane(shared_of(a, seq, lane));
            } else {
                k0 = -1;
                seq = 0;
            }
        }
    }
    // the last position that token t sees
    __device__ __forceinline__ int sees(const AttnArgs& a, const Tile& tile, int t) const {
        if constexpr (!GROUPS) return ctx - tile.toks + (t - tile.tok0);
        int s0 = first_seq(a, tile.item), s1 = first_seq(a, tile.item + 1) - 1;   // the token's sequence: the last that begins at or before it
        if (a.q_start) {
            while (s0 < s1) {
                const int mid = (s0 + s1 + 1) >> 1;
                if (first_row(a, mid) <= t) s0 = mid;
                else s1 = mid - 1;
            }
        } else {
            s0 = t;
        }
        return min(max(a.ctx_len[s0], 0), a.width * a.cache.page) - first_row(a, s0 + 1) + t;
    }
    // keys [k0, the end) of rows that see up to `last`; a piece of them
    __device__ __forceinline__ void piece(const AttnArgs& a, const Tile& tile, int last, int split, int unit, int& from, int& to) const {
        int k1;
        if constexpr (GROUPS) k1 = min(shared_keys(a, tile.item), last + 1);
        else k1 = min(ctx, last + 1);
        const int b = max(k0, 0), n = max(k1 - b, 0);
        const int chunk = max(((n + a.splits - 1) / a.splits + unit - 1) / unit * unit, unit);
        from = (int)min((int64_t)b + (int64_t)split * chunk, (int64_t)INT_MAX - 1024);
        to = min(k1, from + chunk);
    }
    // rows of a sequence outside all groups: nothing is written to the slots of what groups share, so the first piece marks them empty
    __device__ __forceinline__ void mark(const AttnArgs& a, const Tile& tile, int rows, int h, int G, int threads) const {
        if constexpr (!GROUPS)
            if (k0 < 0 && a.slot0 > 0)
                for (int i = threadIdx.x; i < rows * a.slot0; i += threads) {
                    const int R = tile.at + i % rows;
                    if (R < tile.toks * G)
                        a.part_l[(int64_t)(i / rows) * a.T * a.hq + (int64_t)(tile.tok0 + R / G) * a.hq + h * G + R % G] = -INFINITY;
                }
    }
};

// ---- codes to operands --------------------------------------------------------------------------------------------------------------------------------
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int KIND, int D> struct Step {   // 32 keys of one wave
    static constexpr int KW = row_bytes<KIND, D>() / 16;   // words of K a lane has of a key: a quarter of the row
    static constexpr int VW = row_bytes<KIND, D>() >= 64 ? row_bytes<KIND, D>() / 64 : 1;   // words of V a lane has of a key: a sixteenth of the row
    uint32_t k[2][KW], v[8][VW];
    f32x4 ks[2], vs[2];      // int8: scales of keys 16 g + 4 h4 + i
    uint32_t ke[2], ve[8];   // mxfp4: E of the lane's key and block; words of all blocks' E of its eight keys
    int blk[2];              // pages, -1: not there
};
// Pages of 32 keys' two halves: asked for a step ahead, known when they are used (the wait for them is then over)
struct Pages {
    int raw;   // of the first half in the lower lanes, of the second in the upper ones
    __device__ __forceinline__ void ask(const AttnArgs& a, const int32_t* bt, int t0, int end, int lane) {
        const int at = t0 + (lane >> 5) * 16;
        raw = -1;
        if (at < end) raw = bt[a.page_shift >= 0 ? at >> a.page_shift : at / a.cache.page];
    }
    // the page, -1: not there; its row
    __device__ __forceinline__ int blk(const AttnArgs& a, int g) const {
        const int b = __builtin_amdgcn_readlane(raw, 32 * g);
        return b < a.cache.pages ? max(b, -1) : -1;
    }
    static __device__ __forceinline__ int off(const AttnArgs& a, int at) { return a.page_shift >= 0 ? at & (a.cache.page - 1) : at % a.cache.page; }
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <bool ONCE, typename T> __device__ __forceinline__ T take(const uint8_t* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
    else return *reinterpret_cast<const T*>(p);
}
template <int KIND, int D, bool ONCE> __device__ __forceinline__ void load_step(const AttnArgs& a, const Pages& p, int t0, int h, int lane, Step<KIND, D>& s) {
    constexpr int RB = row_bytes<KIND, D>();
    const int r = lane & 15, h4 = lane >> 4;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        s.blk[g] = p.blk(a, g);
        const int64_t row = ((int64_t)max(s.blk[g], 0) * a.cache.heads + h) * a.cache.page + Pages::off(a, t0 + 16 * g);   // of 16, all of one page
        const uint8_t* kp = a.cache.k + (row + r) * RB;
        if constexpr (KIND == kInt8) {
#pragma unroll
            for (int u = 0; u < D / 64; ++u) {
                const u32x4 x = take<ONCE, u32x4>(kp + 64 * u + 16 * h4);
                s.k[g][4 * u] = x.x, s.k[g][4 * u + 1] = x.y, s.k[g][4 * u + 2] = x.z, s.k[g][4 * u + 3] = x.w;
            }
            s.ks[g] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(a.cache.ks) + row + 4 * h4);
            s.vs[g] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(a.cache.vs) + row + 4 * h4);
        } else {
            if constexpr (D == 128) {
                const u32x4 x = take<ONCE, u32x4>(kp + 16 * h4);
                s.k[g][0] = x.x, s.k[g][1] = x.y, s.k[g][2] = x.z, s.k[g][3] = x.w;
            } else {
                const u32x2 x = take<ONCE, u32x2>(kp + 8 * h4);
                s.k[g][0] = x.x, s.k[g][1] = x.y;
            }
            s.ke[g] = *(reinterpret_cast<const uint8_t*>(a.cache.ks) + (row + r) * (D / 32) + h4 * (D / 32) / 4);
            const uint8_t* ve = reinterpret_cast<const uint8_t*>(a.cache.vs) + (row + 4 * h4) * (D / 32);
            if constexpr (D == 128) {
                const uint4 x = *reinterpret_cast<const uint4*>(ve);
                s.ve[4 * g] = x.x, s.ve[4 * g + 1] = x.y, s.ve[4 * g + 2] = x.z, s.ve[4 * g + 3] = x.w;
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(ve);
                s.ve[4 * g] = w.x & 0xffff, s.ve[4 * g + 1] = w.x >> 16, s.ve[4 * g + 2] = w.y & 0xffff, s.ve[4 * g + 3] = w.y >> 16;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint8_t* vp = a.cache.v + (row + 4 * h4 + i) * RB + (RB / 16) * r;
            if constexpr (RB == 128) {
                const u32x2 x = take<ONCE, u32x2>(vp);
                s.v[4 * g + i][0] = x.x, s.v[4 * g + i][1] = x.y;
            } else if constexpr (RB == 64) {
                s.v[4 * g + i][0] = take<ONCE, uint32_t>(vp);
            } else {
                s.v[4 * g + i][0] = take<ONCE, uint16_t>(vp);
            }
        }
    }
}

__device__ __forceinline__ bf16x8 eight(uint32_t a, uint32_t b) {
    bf16x8 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        o[j] = (__bf16)code8(a, j);
        o[4 + j] = (__bf16)code8(b, j);
    }
    return o;
}
// K operand of product c: key r, dimensions key_dim(c, h4) .. + 7
template <int KIND, int D> __device__ __forceinline__ int key_dim(int c, int h4) { return KIND == kInt8 ? 64 * (c >> 1) + 16 * h4 + 8 * (c & 1) : D / 4 * h4 + 8 * c; }
template <int KIND, int D> __device__ __forceinline__ bf16x8 key_operand(const Step<KIND, D>& s, int g, int c) {
    if constexpr (KIND == kInt8) {
        return eight(s.k[g][2 * c], s.k[g][2 * c + 1]);
    } else {
        bf16x2 b[4];
        codes4(s.k[g][c], unit4(s.ke[g]), b);
        return bf16x8{b[0][0], b[0][1], b[1][0], b[1][1], b[2][0], b[2][1], b[3][0], b[3][1]};
    }
}
// V operands: dimension r D / 16 + dt, keys 4 h4 .. + 3 and 16 + 4 h4 .. + 3.
// int8: float16 of the code / 512, two keys at a time: the byte, its top bit turned, is a denormal float16 of u 2^-24, u = code + 128; one fused multiply-add (with 2^15 and -1/4) makes
// code / 512 of it, exactly.
constexpr float kCodeUnit = 1.f / 512.f;
__device__ __forceinline__ uint32_t pair8(uint32_t first, uint32_t second, int i) {   // words with their top bits turned; byte i of both
    const uint32_t u = __builtin_amdgcn_perm(second, first, 0x0c040c00u + 0x00010001u * (uint32_t)i);
    const f16x2 x = __builtin_bit_cast(f16x2, u);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x, f16x2{(_Float16)32768.f, (_Float16)32768.f}, f16x2{(_Float16)-0.25f, (_Float16)-0.25f}));
}
// Two operands of V at a time, of neighbouring dimensions 2 k and 2 k + 1 of the lane's D / 16: eight 16-bit numbers each
template <int KIND, int D> struct Values {
    const uint32_t (&v)[8][Step<KIND, D>::VW];   // int8: with the codes' top bits turned
    float scale[8];                              // mxfp4
    __device__ __forceinline__ Values(Step<KIND, D>& s, int r) : v(s.v) {
        if constexpr (KIND == kInt8) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int x = 0; x < Step<KIND, D>::VW; ++x) s.v[j][x] ^= 0x80808080u;
        } else {
            const int sh = 8 * (r * (D / 16) / 32);
#pragma unroll
            for (int j = 0; j < 8; ++j) scale[j] = __uint_as_float(((s.ve[j] >> sh) & 255) << 23);
        }
    }
    __device__ __forceinline__ uint32_t two(int j, int k) const {   // bfloat16 of codes 2 k and 2 k + 1
        const uint32_t w = v[j][0];
        return __builtin_bit_cast(uint32_t, k == 0   ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale[j], 0)
                                            : k == 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale[j], 1)
                                            : k == 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale[j], 2)
                                                     : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale[j], 3));
    }
    __device__ __forceinline__ void pair(int k, uint4 (&o)[2]) const {
        uint32_t w[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (KIND == kInt8) {
#pragma unroll
                for (int e = 0; e < 2; ++e) w[e][j] = pair8(v[2 * j][(2 * k + e) >> 2], v[2 * j + 1][(2 * k + e) >> 2], (2 * k + e) & 3);
            } else {
                const uint32_t a = two(2 * j, k), b = two(2 * j + 1, k);
                w[0][j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
                w[1][j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            }
        }
        o[0] = uint4{w[0][0], w[0][1], w[0][2], w[0][3]};
        o[1] = uint4{w[1][0], w[1][1], w[1][2], w[1][3]};
    }
    static __device__ __forceinline__ f32x4 mul(const uint4& v, const uint4& p, f32x4 acc) {
        if constexpr (KIND == kInt8) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, v), __builtin_bit_cast(f16x8, p), acc, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, p), acc, 0, 0, 0);
    }
};
// Two probabilities (int8: times their scales) to 16 bits
template <int KIND> __device__ __forceinline__ uint32_t round2(float a, float b) {
    if constexpr (KIND == kInt8) return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
    else return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

// mxfp4: l and two rounded probabilities
__device__ __forceinline__ float sum2(uint32_t p, float l) { return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p), bf16x2{(__bf16)1.f, (__bf16)1.f}, l, false); }

// mxfp4: how far scores over the reference may be beside values of exponents up to E (bytes of the cache, 252 at most).  A value is less than 2^(E - 124), so 2^30 products stay within 2^127.
__device__ __forceinline__ float most_over(uint32_t E) { return fminf(8.f, 221.f - (float)E); }
// A row's reference moves: to `up` over base, the highest score so far or (int8) what its probabilities times scales allow; never down, once there is one.  x are the
// scores over base, and then over the new one; returns what sums so far are to be multiplied by.
template <int N> __device__ __forceinline__ float moved_ref(float& ref, float base, float mx, float up, float (&x)[N]) {
    const float to = ref == -INFINITY ? (mx == -INFINITY ? -INFINITY : base + up) : base + fmaxf(up, 0.f);
    const float d = base - (to == -INFINITY ? 0.f : to), f = ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(d);
    ref = to;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += d;
    return f;
}

// ---- the tile -----------------------------------------------------------------------------------------------------------------------------------------
// GROUPS: the items are groups of sequences, the keys those that each shares; otherwise sequences, their keys behind what they share.
// ONCE: the codes are marked as read once.
// Bound by the codes' bytes where keys are many (two sequences of 128k, 64 query heads, mxfp4: 285 MB in 57 to 59 us, 4.9 TB/s; the join behind it 5), by the chain of loads (length, page, codes)
// and, where keys are few, by that chain once a step, since a wave asks for a step's codes when the one before is done, and by the waves' join (a sequence of 140 keys, two steps of one wave: 6.7 us).
template <int KIND, int D, int NQT, bool GROUPS, bool ONCE>
__global__ void __launch_bounds__(256, NQT == 1 ? (KIND == kInt8 && D == 128 ? 3 : 4) : 2) quant_rows_kernel(const AttnArgs a) {
    constexpr int ROWS = 16 * NQT, NC = D / 32, ND = D / 16;
    __shared__ __attribute__((aligned(16))) f32x4 so[3][ND][64];
    __shared__ float sl[3][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, h4 = lane >> 4;
    const int heads = a.cache.heads, G = a.hq / heads;
    const int h = blockIdx.x % heads;
    const int split = blockIdx.y;
    Tile tile;
    if (!find_tile<GROUPS>(a, blockIdx.x / heads, G, ROWS, lane, tile)) return;
    tile.same();
    // keys from the first on, if no piece is cut: the wave's first pages do not wait for the context's length
    Pages pg{-1};
    const bool guess = !GROUPS && a.splits == 1 && !a.group_start && tile.item < a.B;
    if (guess) pg.ask(a, a.bt + (int64_t)tile.item * a.bt_stride, w * 32, a.width * a.cache.page, lane);
    // the rows of this lane: the last position each sees, and its queries
    const Item<GROUPS> item(a, tile, lane);
    if (split == 0 && !a.last) item.mark(a, tile, ROWS, h, G, 256);
    int rpos[NQT];
    bf16x8 qf[NQT][NC];
    int first = INT_MAX, last = -1;   // the last position that all rows of the tile see, and that any does
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
        const int R = tile.at + 16 * qt + r;
        const bool valid = R < tile.toks * G;
        const int t = tile.tok0 + (valid ? R / G : 0), hd = h * G + R % G;
        rpos[qt] = valid ? item.sees(a, tile, t) : INT_MAX;   // what the rows behind the tile's make is not written
        if constexpr (GROUPS) {
            last = max(last, valid ? rpos[qt] : -1);
            first = min(first, rpos[qt]);
        }
        const uint16_t* qp = a.q + t * a.q_stride + (int64_t)hd * D;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            bf16x8 v = *reinterpret_cast<const bf16x8*>(qp + key_dim<KIND, D>(c, h4));
            if (!valid) v = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
            qf[qt][c] = v;
        }
    }
    if constexpr (GROUPS) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            first = min(first, __shfl_xor(first, o, 64));
            last = max(last, __shfl_xor(last, o, 64));
        }
        first = __builtin_amdgcn_readfirstlane(first);
        last = __builtin_amdgcn_readfirstlane(last);
    } else {   // the tile's first token's, and its last's
        first = __builtin_amdgcn_readfirstlane(item.ctx - tile.toks + tile.at / G);
        last = __builtin_amdgcn_readfirstlane(item.ctx - tile.toks + min(tile.toks - 1, (tile.at + ROWS - 1) / G));
    }
    int ks, ke;
    item.piece(a, tile, last, split, 128, ks, ke);
    const int32_t* bt = a.bt + (int64_t)item.seq * a.bt_stride;
    float ref[NQT], l[NQT];   // sums are of 2^(score - ref)
    f32x4 o[NQT][ND];
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
        ref[qt] = -INFINITY;
        l[qt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[qt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    auto compute = [&](int t0, Step<KIND, D>& s) {
        f32x4 sc[NQT][2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
#pragma unroll
            for (int qt = 0; qt < NQT; ++qt) sc[qt][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const bf16x8 kf = key_operand<KIND, D>(s, g, c);
#pragma unroll
                for (int qt = 0; qt < NQT; ++qt) sc[qt][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[qt][c], sc[qt][g], 0, 0, 0);
            }
        }
        // Values that are NaN, by their scales: 4-bit ones from 253 on (192 and more, which is 2^65, is looked for in all keys at once), float ones that are
        // not finite (or negative).  They count as zeros and their keys' scores as NaN.
        uint32_t nan = 0, top = 0;   // of this lane's keys, bit j; int8: the largest scale's bits
        float over = 8.f;            // mxfp4: most_over of this lane's keys
        if constexpr (KIND == kFp4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) top |= s.ve[j] & (s.ve[j] << 1) & 0x80808080u;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(s.vs[j >> 2][j & 3]));
        }
        const bool odd = __ballot(KIND == kFp4 ? top != 0 : top >= 0x7f800000u) != 0;
        if (odd) {
            if constexpr (KIND == kFp4) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int b = 0; b < D / 32; ++b) {
                        const uint32_t E = (s.ve[j] >> (8 * b)) & 255;
                        if (E > 252) {
                            nan |= 1u << j;
                            s.ve[j] &= ~(255u << (8 * b));
                        } else {
                            over = fminf(over, most_over(E));
                        }
                    }
            } else {
                top = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t v = __float_as_uint(s.vs[j >> 2][j & 3]);
                    if (v >= 0x7f800000u) nan |= 1u << j, v = 0;
                    top = max(top, v);
                    s.vs[j >> 2][j & 3] = __uint_as_float(v);
                }
            }
        }
        const bool part = odd || t0 + 32 > ke || t0 + 31 > first || s.blk[0] < 0 || s.blk[1] < 0;   // some row does not see some key
        // scores over the reference may be so high: int8, times the lane's scales, as float16 holds
        const float most = KIND == kInt8 ? fminf(15.f - __log2f(__uint_as_float(top)), 100.f) : over;
        uint4 pw[NQT];
#pragma unroll
        for (int qt = 0; qt < NQT; ++qt) {
            const float base = ref[qt] == -INFINITY ? 0.f : ref[qt];
            float x[8], mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float mul = KIND == kInt8 ? s.ks[j >> 2][j & 3] * a.scale_log2 : a.scale_log2;
                x[j] = __builtin_fmaf(sc[qt][j >> 2][j & 3], mul, -base);
            }
            if (part) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = t0 + 16 * (j >> 2) + 4 * h4 + (j & 3);
                    const bool seen = s.blk[j >> 2] >= 0 && key < ke && key <= rpos[qt];
                    x[j] = !seen ? -INFINITY : nan >> j & 1 ? __builtin_nanf("") : x[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) mx = fmaxf(mx, x[j]);
            if (__builtin_expect(__ballot(mx > (ref[qt] == -INFINITY ? -INFINITY : most)) != 0, false)) {
                float up = rows_max(mx - fminf(most, 0.f));   // mxfp4
                mx = rows_max(mx);
                if constexpr (KIND == kInt8) {
                    up = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 8; ++j) up = fmaxf(up, x[j] + __log2f(s.vs[j >> 2][j & 3]));
                    up = fmaxf(rows_max(up) - 7.f, mx - 90.f);
                }
                const float f = moved_ref(ref[qt], base, mx, up, x);
                l[qt] *= f;
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) o[qt][dt] *= f;
            }
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = __builtin_amdgcn_exp2f(x[j]);
                if constexpr (KIND == kInt8) {
                    l[qt] += p[j];
                    p[j] *= s.vs[j >> 2][j & 3];
                }
            }
            pw[qt] = uint4{round2<KIND>(p[0], p[1]), round2<KIND>(p[2], p[3]), round2<KIND>(p[4], p[5]), round2<KIND>(p[6], p[7])};
            if constexpr (KIND == kFp4) l[qt] = sum2(pw[qt].w, sum2(pw[qt].z, sum2(pw[qt].y, sum2(pw[qt].x, l[qt]))));
        }
        const Values<KIND, D> val(s, r);
#pragma unroll
        for (int k = 0; k < ND / 2; ++k) {
            uint4 v[2];
            val.pair(k, v);
#pragma unroll
            for (int qt = 0; qt < NQT; ++qt)
#pragma unroll
                for (int e = 0; e < 2; ++e) o[qt][2 * k + e] = val.mul(v[e], pw[qt], o[qt][2 * k + e]);
        }
    };

    {
        int t0 = ks + w * 32;
        if (!guess) pg.ask(a, bt, t0, ke, lane);
        for (; t0 < ke; t0 += 128) {
            Step<KIND, D> s;
            load_step<KIND, D, ONCE>(a, pg, t0, h, lane, s);
            pg.ask(a, bt, t0 + 128, ke, lane);
            compute(t0, s);
        }
    }
    // ---- the waves' averages: those of 16 rows to the wave that has them to write ------------------------------------------------------------------------
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
        const float all = rows_sum(l[qt]), inv = all == 0.f ? 0.f : (KIND == kInt8 ? 1.f / kCodeUnit : 1.f) / all;
        float lse = all == 0.f ? -INFINITY : ref[qt] + __log2f(all);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[qt][dt] *= inv;
        const int R = tile.at + 16 * qt + r;
        const bool live = R < tile.toks * G;
        const int64_t row = (int64_t)(tile.tok0 + R / G) * a.hq + h * G + R % G;
        if constexpr (!GROUPS) {
            if (a.last && item.k0 >= 0 && live) {   // the pieces of the group's keys, in turn over the waves; a wave's average of a piece and its own
                for (int s = w; s < a.slot0; s += 4) {
                    const int64_t at = (int64_t)s * a.T * a.hq + row;
                    const float other = a.part_l[at];
                    if (other == -INFINITY) continue;
                    f32x4 x[4][ND / 4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int c = 0; c < ND / 4; ++c) x[i][c] = *reinterpret_cast<const f32x4*>(a.part_o + at * D + (4 * h4 + i) * ND + 4 * c);
                    const float mx = fmaxf(lse, other);
                    float f = __builtin_amdgcn_exp2f(lse - mx), g = __builtin_amdgcn_exp2f(other - mx);
                    const float both = 1.f / (f + g);
                    lse = mx + __log2f(f + g);
                    f *= both, g *= both;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int dt = 0; dt < ND; ++dt) o[qt][dt][i] = o[qt][dt][i] * f + x[i][dt >> 2][dt & 3] * g;
                }
            }
        }
        const int owner = qt & 3;
        const int place = w < owner ? w : w - 1;
        if (qt) __syncthreads();
        if (w != owner) {
            sl[place][lane] = lse;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) so[place][dt][lane] = o[qt][dt];
        }
        __syncthreads();
        if (w == owner) {
            float mx = lse;
#pragma unroll
            for (int p = 0; p < 3; ++p) mx = fmaxf(mx, sl[p][lane]);
            const float base = mx == -INFINITY ? 0.f : mx;
            float f = __builtin_amdgcn_exp2f(lse - base), g[3], sum = f;
#pragma unroll
            for (int p = 0; p < 3; ++p) sum += g[p] = __builtin_amdgcn_exp2f(sl[p][lane] - base);
            const float one = sum == 0.f ? 0.f : 1.f / sum;
            f *= one;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) o[qt][dt] *= f;
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                g[p] *= one;
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) o[qt][dt] += so[p][dt][lane] * g[p];
            }
            if (live && (a.slots == 1 || a.last)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint16_t* dst = a.out + row * D + (4 * h4 + i) * ND;
                    uint16_t v[ND];
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt) v[dt] = f2bf(o[qt][dt][i]);
                    if constexpr (ND == 8) *reinterpret_cast<u16x8*>(dst) = u16x8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
                    else *reinterpret_cast<u16x4*>(dst) = u16x4{v[0], v[1], v[2], v[3]};
                }
            } else if (live) {
                const int64_t at = (int64_t)(a.slot0 + split) * a.T * a.hq + row;
                if (h4 == 0) a.part_l[at] = sum == 0.f ? -INFINITY : base + __log2f(sum);
                if (sum != 0.f) {   // nothing there is not read either
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int dt = 0; dt < ND; dt += 4)
                            *reinterpret_cast<f32x4*>(a.part_o + at * D + (4 * h4 + i) * ND + dt) =
                                f32x4{o[qt][dt][i], o[qt][dt + 1][i], o[qt][dt + 2][i], o[qt][dt + 3][i]};
                }
            }
        }
    }
}

// ---- many rows: keys through LDS -------------------------------------------------------------------------------------------------------------------------
// Tiles of 32 WAVES rows, 32 a wave, for rows that are many (prompts, the rows of a group): there the products and the probabilities bound it, and codes become operands
// once for all waves.  A step is 16 WAVES keys: half of the waves turn its keys into bfloat16 [key][D] in LDS, the others its values into [D][key], from registers that were
// loaded a step earlier, into the buffer that is not being read; one barrier a step.  16 bytes behind every row keep its readers, 16 bytes a lane and a row
// each, out of each other's banks.  v_mfma_f32_32x32x16: a lane has 16 of 32 keys of one row, and the probabilities are the second product's operand as they are, its values' keys in the same order
// (4 h + (j & 3) + 8 (j >> 2) of 16).
// Two prompts of 1950 tokens and two of 330 on up to 3296 keys, 32 query heads, int8, 113 GFLOP: 175 us, 650 TFLOP/s, matrix cores busy 31 % of the time and vector ALUs 48 %; 2 x 128 sequences of 64 query heads on 16k
// shared keys, mxfp4, 137 GFLOP: 158 to 164 us, 850 TFLOP/s, 37 % and 41 % (profiles/quant_kv_counters.txt).  One after the other for the most part: priorities of waves, half of them a step's part
// late, products a part late beside the next probabilities (which spills), and reads from LDS further ahead all gain nothing or lose.
template <int KIND, int D, int WAVES> struct TileStep {
    static constexpr int KT = 16 * WAVES, KS = 2 * D + 16, VS = 2 * KT + 16;   // bytes from key to key, and from dimension to dimension
    alignas(16) uint8_t k[KT * KS];
    alignas(16) uint8_t v[D * VS];
    alignas(16) float km[KT], vm[KT];   // int8: scales of keys, times scale_log2, and values; 0 where a key is not there
    uint32_t there[KT / 32], nan[KT / 32];
    float top[KT / 32];                 // int8: base-2 logarithm of the largest of vm; mxfp4: most_over of the values
};

// 32 keys' codes on their way into LDS, by one wave: keys or values
template <int KIND, int D> struct Fetch {
    static constexpr int RB = row_bytes<KIND, D>(), NP = RB * 32 / 1024;   // pieces of 1 KiB
    static constexpr int VW = Step<KIND, D>::VW;
    uint32_t w[8 * VW > 4 * NP ? 8 * VW : 4 * NP];   // keys: 4 words of each piece; values: VW of each key
    uint32_t e[KIND == kFp4 ? 8 : 1];                // mxfp4: E of the pieces' blocks, or the words of the eight keys' values
    uint32_t scale;                                  // keys' waves, int8: lane i < 32: of key i, i >= 32: its value's; mxfp4: the word of key i's value
    int blk0, blk1, t0;                              // pages of the first 16 keys and of the others, -1: not there; the first key

    static __device__ __forceinline__ int64_t row_of(const AttnArgs& a, int blk, int at, int h) {
        return ((int64_t)max(blk, 0) * a.cache.heads + h) * a.cache.page + Pages::off(a, at);
    }
    __device__ __forceinline__ void keys(const AttnArgs& a, const Pages& pg, int at, int h, int lane) {
        t0 = at;
        blk0 = pg.blk(a, 0), blk1 = pg.blk(a, 1);
        const int64_t row0 = row_of(a, blk0, at, h), row1 = row_of(a, blk1, at + 16, h);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            constexpr int KP = 1024 / RB;   // keys of a piece
            const int key = p * KP + lane / (RB / 16);
            const int64_t row = (NP == 1 ? key < 16 : p * KP < 16) ? row0 + key : row1 + key - 16;
            const uint4 x = *reinterpret_cast<const uint4*>(a.cache.k + row * RB + (lane % (RB / 16)) * 16);
            w[4 * p] = x.x, w[4 * p + 1] = x.y, w[4 * p + 2] = x.z, w[4 * p + 3] = x.w;
            if constexpr (KIND == kFp4) e[p] = *(reinterpret_cast<const uint8_t*>(a.cache.ks) + row * (D / 32) + lane % (RB / 16));
        }
        const int key = lane & 31;
        const int64_t row = key < 16 ? row0 + key : row1 + key - 16;
        if constexpr (KIND == kInt8) scale = reinterpret_cast<const uint32_t*>(lane < 32 ? a.cache.ks : a.cache.vs)[row];
        else if constexpr (D == 128) scale = reinterpret_cast<const uint32_t*>(a.cache.vs)[row];
        else scale = reinterpret_cast<const uint16_t*>(a.cache.vs)[row];
    }
    __device__ __forceinline__ void values(const AttnArgs& a, const Pages& pg, int at, int h, int lane) {
        t0 = at;
        blk0 = pg.blk(a, 0), blk1 = pg.blk(a, 1);
        const int r = lane & 15, h2 = lane >> 4 & 1;
        const int64_t row = (lane < 32 ? row_of(a, blk0, at, h) : row_of(a, blk1, at + 16, h)) + 4 * h2;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint8_t* vp = a.cache.v + (row + (j & 3) + 8 * (j >> 2)) * RB + (RB / 16) * r;
            if constexpr (RB == 128) {
                const uint2 x = *reinterpret_cast<const uint2*>(vp);
                w[VW * j] = x.x, w[VW * j + 1] = x.y;
            } else if constexpr (RB == 64) {
                w[VW * j] = *reinterpret_cast<const uint32_t*>(vp);
            } else {
                w[VW * j] = *reinterpret_cast<const uint16_t*>(vp);
            }
        }
        if constexpr (KIND == kFp4) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const uint8_t* ep = reinterpret_cast<const uint8_t*>(a.cache.vs) + (row + 8 * g) * (D / 32);
                if constexpr (D == 128) {
                    const uint4 x = *reinterpret_cast<const uint4*>(ep);
                    e[4 * g] = x.x, e[4 * g + 1] = x.y, e[4 * g + 2] = x.z, e[4 * g + 3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(ep);
                    e[4 * g] = x.x & 0xffff, e[4 * g + 1] = x.x >> 16, e[4 * g + 2] = x.y & 0xffff, e[4 * g + 3] = x.y >> 16;
                }
            }
        }
    }
    // keys 32 i .. of the step
    template <int WAVES> __device__ __forceinline__ void put_keys(TileStep<KIND, D, WAVES>& s, int i, int end, float scale_log2, int lane) const {
        const uint32_t in = t0 >= end ? 0u : end - t0 >= 32 ? ~0u : (1u << (end - t0)) - 1u;
        const uint32_t there = in & ((blk0 >= 0 ? 0xffffu : 0u) | (blk1 >= 0 ? 0xffff0000u : 0u));
        const int key = lane & 31;
        const bool here = there >> key & 1;
        if constexpr (KIND == kInt8) {
            float x = here ? __uint_as_float(scale) : 0.f;
            const bool bad = lane >= 32 && !(x >= 0.f && x < INFINITY);
            if (bad) x = 0.f;
            if (lane < 32) s.km[32 * i + key] = x * scale_log2;
            else s.vm[32 * i + key] = x;
            const float top = wave_max(lane < 32 ? 0.f : x);
            const uint32_t nan = (uint32_t)(__ballot(bad) >> 32);
            if (lane == 0) s.top[i] = __log2f(top), s.there[i] = there, s.nan[i] = nan;
        } else {
            bool bad = false;
#pragma unroll
            for (int b = 0; b < D / 32; ++b) bad |= (scale >> (8 * b) & 255) > 252;
            const uint32_t nan = (uint32_t)__ballot(bad && here && lane < 32);
            float over = 8.f;
            if (__ballot(scale & (scale << 1) & 0x80808080u)) {   // values from 2^65 on (D = 64: `scale` has two bytes)
#pragma unroll
                for (int b = 0; b < D / 32; ++b) {
                    const uint32_t E = scale >> (8 * b) & 255;
                    if (here && E <= 252) over = fminf(over, most_over(E));
                }
                over = -wave_max(-over);
            }
            if (lane == 0) s.there[i] = there, s.nan[i] = nan, s.top[i] = over;
        }
        constexpr int KP = 1024 / RB;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int at = 32 * i + p * KP + lane / (RB / 16), part = lane % (RB / 16);
            if constexpr (KIND == kInt8) {
#pragma unroll
                for (int x = 0; x < 2; ++x) *reinterpret_cast<bf16x8*>(s.k + at * s.KS + (2 * part + x) * 16) = eight(w[4 * p + 2 * x], w[4 * p + 2 * x + 1]);
            } else {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    bf16x2 b[4];
                    codes4(w[4 * p + x], unit4(e[p]), b);
                    *reinterpret_cast<bf16x8*>(s.k + at * s.KS + (4 * part + x) * 16) = bf16x8{b[0][0], b[0][1], b[1][0], b[1][1], b[2][0], b[2][1], b[3][0], b[3][1]};
                }
            }
        }
    }
    template <int WAVES> __device__ __forceinline__ void put_values(TileStep<KIND, D, WAVES>& s, int i, int lane) const {
        const int r = lane & 15;
        Step<KIND, D> st;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int x = 0; x < VW; ++x) st.v[j][x] = w[VW * j + x];
            if constexpr (KIND == kFp4) {
                const uint32_t one = e[j] >> (8 * (r * (D / 16) / 32)) & 255;
                st.ve[j] = (one > 252 ? 0 : one) << (8 * (r * (D / 16) / 32));
            }
        }
        const Values<KIND, D> val(st, r);
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            uint4 o[2];
            val.pair(k, o);
#pragma unroll
            for (int x = 0; x < 2; ++x) *reinterpret_cast<uint4*>(s.v + (16 * (2 * k + x) + r) * s.VS + (4 * i + (lane >> 4)) * 16) = o[x];
        }
    }
};

template <int KIND, int D, int WAVES, bool GROUPS>
__global__ void __launch_bounds__(64 * WAVES, 2) quant_tile_kernel(const AttnArgs a) {
    constexpr int ROWS = 32 * WAVES, KT = 16 * WAVES, NC = D / 16, NT = D / 32;
    typedef TileStep<KIND, D, WAVES> TS;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    TS* steps = reinterpret_cast<TS*>(lds);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, h2 = lane >> 5;
    const int heads = a.cache.heads, G = a.hq / heads;
    const int h = blockIdx.x % heads, split = blockIdx.y;
    Tile tile;
    if (!GROUPS && a.longest) {
        if (!find_longest(a, blockIdx.x / heads, G, ROWS, lane, tile)) return;
    } else if (!find_tile<GROUPS>(a, blockIdx.x / heads, G, ROWS, lane, tile)) {
        return;
    }
    tile.same();
    const Item<GROUPS> item(a, tile, lane);
    if (split == 0) item.mark(a, tile, ROWS, h, G, 64 * WAVES);

    // The keys come first: nothing of the rows is needed to fetch them.  A group's rows see all that it shares, unless a context ends in it: then some are masked.
    int ks, ke;
    item.piece(a, tile, GROUPS ? INT_MAX - 1 : item.ctx - tile.toks + min(tile.toks - 1, (tile.at + ROWS - 1) / G), split, KT, ks, ke);
    ks = __builtin_amdgcn_readfirstlane(ks);
    ke = __builtin_amdgcn_readfirstlane(ke);
    const int32_t* bt = a.bt + (int64_t)item.seq * a.bt_stride;
    const bool of_keys = w < WAVES / 2;
    const int part = of_keys ? w : w - WAVES / 2;   // of the step's keys
    Fetch<KIND, D> f;
    Pages pg;
    pg.ask(a, bt, ks + 32 * part, ke, lane);
    auto fetch = [&](int at) {   // the step's codes, and the next one's pages
        if (of_keys) f.keys(a, pg, at + 32 * part, h, lane);
        else f.values(a, pg, at + 32 * part, h, lane);
        pg.ask(a, bt, at + KT + 32 * part, ke, lane);
    };
    auto store = [&](TS& s) {
        if (of_keys) f.template put_keys<WAVES>(s, part, ke, a.scale_log2, lane);
        else f.template put_values<WAVES>(s, part, lane);
    };
    if (ks < ke) fetch(ks);

    const int R = tile.at + 32 * w + r, live_rows = tile.toks * G;
    const bool valid = R < live_rows;
    const int t = tile.tok0 + (valid ? R / G : 0);
    const int rpos = valid ? item.sees(a, tile, t) : -1;
    bf16x8 qf[NC];
    {
        const uint16_t* qp = a.q + t * a.q_stride + (int64_t)(h * G + R % G) * D + 8 * h2;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            qf[c] = *reinterpret_cast<const bf16x8*>(qp + 16 * c);
            if (!valid) qf[c] = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
        }
    }
    int first = valid ? rpos : INT_MAX, last = rpos;   // of the wave's rows
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        first = min(first, __shfl_xor(first, o, 64));
        last = max(last, __shfl_xor(last, o, 64));
    }
    first = __builtin_amdgcn_readfirstlane(first);
    last = __builtin_amdgcn_readfirstlane(last);

    float ref = -INFINITY, l = 0.f;   // sums are of 2^(score - ref)
    f32x16 o[NT];
#pragma unroll
    for (int T = 0; T < NT; ++T)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[T][i] = 0.f;

    auto scores = [&](const TS& s, int sub) {
        f32x16 sc;
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(s.k + (32 * sub + r) * TS::KS + (2 * c + h2) * 16), qf[c], sc, 0, 0, 0);
        return sc;
    };
    // 32 keys from t0 on, the step's sub-th, whose scores are made; makes the next ones' beside the probabilities
    f32x16 sc;
    auto compute = [&](const TS& s, int sub, int t0) {
        const float base = ref == -INFINITY ? 0.f : ref;
        float x[16], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const f32x4 km = KIND == kInt8 ? *reinterpret_cast<const f32x4*>(s.km + 32 * sub + 4 * h2 + 2 * i) : f32x4{a.scale_log2, a.scale_log2, a.scale_log2, a.scale_log2};
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i + e] = __builtin_fmaf(sc[i + e], km[e], -base);
        }
        const uint32_t there = __builtin_amdgcn_readfirstlane(s.there[sub]), nans = __builtin_amdgcn_readfirstlane(s.nan[sub]);
        if (t0 + 31 > first || (~there | nans)) {   // some row does not see some key, or a key's value is NaN
            const uint32_t row = rpos < t0 ? 0u : rpos - t0 >= 31 ? ~0u : (2u << (rpos - t0)) - 1u;
            const uint32_t seen = (there & row) >> (4 * h2), nan = nans >> (4 * h2);
#pragma unroll
            for (int i = 0; i < 16; ++i) {   // key 4 h2 + (i & 3) + 8 (i >> 2)
                const uint32_t bit = 1u << ((i & 3) + 8 * (i >> 2));
                x[i] = !(seen & bit) ? -INFINITY : nan & bit ? __builtin_nanf("") : x[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[i]);
        // scores over the reference may be so high: int8, times the largest scale, as float16 holds
        const float most = KIND == kInt8 ? fminf(15.f - s.top[sub], 100.f) : s.top[sub];
        if (__builtin_expect(__ballot(mx > (ref == -INFINITY ? -INFINITY : most)) != 0, false)) {
            mx = lanes_xor32(mx, LaneMax{});
            float up = mx - fminf(most, 0.f);   // mxfp4
            if constexpr (KIND == kInt8) {
                up = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) up = fmaxf(up, x[i] + __log2f(s.vm[32 * sub + 4 * h2 + (i & 3) + 8 * (i >> 2)]));
                up = fmaxf(lanes_xor32(up, LaneMax{}) - 7.f, mx - 90.f);
            }
            const float f = moved_ref(ref, base, mx, up, x);
            l *= f;
#pragma unroll
            for (int T = 0; T < NT; ++T) o[T] *= f;
        }
        if (sub + 1 < KT / 32) sc = scores(s, sub + 1);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {   // 16 keys: probabilities, and their part of the sums
            uint32_t pw[4];
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(x[8 * kk + j + e]);
                    if constexpr (KIND == kInt8) l += p[e];
                }
                if constexpr (KIND == kInt8) {
                    const f32x4 vm = *reinterpret_cast<const f32x4*>(s.vm + 32 * sub + 16 * kk + 4 * h2 + 2 * j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] *= vm[e];
                }
                pw[j >> 1] = round2<KIND>(p[0], p[1]);
                pw[(j >> 1) + 1] = round2<KIND>(p[2], p[3]);
                if constexpr (KIND == kFp4) l = sum2(pw[(j >> 1) + 1], sum2(pw[j >> 1], l));
            }
            const uint4 p{pw[0], pw[1], pw[2], pw[3]};
#pragma unroll
            for (int T = 0; T < NT; ++T) {
                const uint4 v = *reinterpret_cast<const uint4*>(s.v + (32 * T + r) * TS::VS + (4 * sub + 2 * kk + h2) * 16);
                if constexpr (KIND == kInt8) o[T] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v), __builtin_bit_cast(f16x8, p), o[T], 0, 0, 0);
                else o[T] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, p), o[T], 0, 0, 0);
            }
        }
    };

    if (ks < ke) {
        store(steps[0]);
        __syncthreads();
        int b = 0;
        for (int t0 = ks; t0 < ke; t0 += KT, b ^= 1) {
            const bool more = t0 + KT < ke;
            if (more) fetch(t0 + KT);
            if (t0 <= last) {
                sc = scores(steps[b], 0);
#pragma unroll
                for (int sub = 0; sub < KT / 32; ++sub) {
                    const int at = t0 + 32 * sub;
                    if (at > last || at >= ke) break;   // no row of the wave sees these
                    compute(steps[b], sub, at);
                }
            }
            if (more) store(steps[b ^ 1]);
            __syncthreads();
        }
    }

    // Sums to memory, by way of LDS (the wave's rows in its own part): 16 bytes a lane, a row's in neighbouring lanes.  Row 32 T + (i & 3) + 8 (i >> 2) + 4 h2 of V is
    // dimension D / 16 (row % 16) + row / 16: a lane has D / 16 neighbouring dimensions at a time.
    l = lanes_xor32(l, LaneSum{});
    const bool direct = a.slots == 1;
    const float mul = l == 0.f ? 0.f : (KIND == kInt8 ? 1.f / kCodeUnit : 1.f) / l;
    if (!direct && h2 == 0 && valid) a.part_l[(int64_t)(a.slot0 + split) * a.T * a.hq + (int64_t)t * a.hq + h * G + R % G] = l == 0.f ? -INFINITY : ref + __log2f(l);
    constexpr int OS = D + 4;   // floats from row to row
    float* mine = reinterpret_cast<float*>(lds) + w * 16 * OS;
#pragma unroll
    for (int half = 0; half < 2; ++half) {   // 16 rows at a time
        if ((r >> 4) == half) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float* dst = mine + (r & 15) * OS + ((i & 3) + 8 * (i >> 2) + 4 * h2) * (D / 16);
#pragma unroll
                for (int T = 0; T < NT; T += 2) *reinterpret_cast<f32x4*>(dst + 2 * T) = f32x4{o[T][i], o[T][i + 8], o[T + 1][i], o[T + 1][i + 8]} * mul;
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // of this wave alone
        constexpr int PER = D / 8;   // lanes of a row, eight dimensions each
#pragma unroll
        for (int i = 0; i < 16 * PER / 64; ++i) {
            const int at = (i * 64 + lane) / PER, c = lane % PER, Rr = tile.at + 32 * w + 16 * half + at;
            if (Rr >= live_rows) continue;
            const int64_t row = (int64_t)(tile.tok0 + Rr / G) * a.hq + h * G + Rr % G;
            const f32x4 x = *reinterpret_cast<const f32x4*>(mine + at * OS + 8 * c), y = *reinterpret_cast<const f32x4*>(mine + at * OS + 8 * c + 4);
            if (direct) {
                *reinterpret_cast<u16x8*>(a.out + row * D + 8 * c) = u16x8{f2bf(x[0]), f2bf(x[1]), f2bf(x[2]), f2bf(x[3]), f2bf(y[0]), f2bf(y[1]), f2bf(y[2]), f2bf(y[3])};
            } else {
                float* dst = a.part_o + ((int64_t)(a.slot0 + split) * a.T * a.hq + row) * D + 8 * c;
                *reinterpret_cast<f32x4*>(dst) = x;
                *reinterpret_cast<f32x4*>(dst + 4) = y;
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// Rows of the pieces' averages o_s, of sums 2^(l_s): out = sum_s 2^(l_s - m) o_s / sum_s 2^(l_s - m).  D / 4 lanes have a row, `per` such groups share its pieces and are
// joined through LDS.  Weights are 2^-8 of what they are: those of up to 128 pieces then add up to no more than a half, so that averages near the end of float32's range keep within it.
// The sums of up to D / 4 pieces are read at once, a lane each, and handed round; what the pieces hold does not wait for them.
template <int D>
__global__ void __launch_bounds__(256) quant_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_l, uint16_t* __restrict__ out, int64_t rows,
                                                         int slots, int per) {
    constexpr int L = D / 4, GR = 256 / L;
    __shared__ f32x4 so[GR][L];
    __shared__ float sl[GR], sm[GR];
    const int c = threadIdx.x % L, gr = threadIdx.x / L;
    const int64_t at = (int64_t)blockIdx.x * (GR / per) + gr / per, row = at < rows ? at : rows - 1;
    float mx = -INFINITY, sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = gr % per; s0 < slots; s0 += per * L) {   // pieces s0, s0 + per, ..: lane c has the c-th
        const int n = min(L, (slots - s0 + per - 1) / per);
        const float mine = c < n ? part_l[(int64_t)(s0 + per * c) * rows + row] : -INFINITY;
        const bool there = !(mine == -INFINITY);
        float top = mine;
#pragma unroll
        for (int k = 1; k < L; k <<= 1) top = fmaxf(top, __shfl_xor(top, k, L));
        top = fmaxf(top, mx);
        const float base = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f(mx - base);
        mx = top;
        o *= old;
        const float w = there ? __builtin_amdgcn_exp2f(mine - base) : 0.f;
        float all = w;
#pragma unroll
        for (int k = 1; k < L; k <<= 1) all += __shfl_xor(all, k, L);
        sum = sum * old + all;
        const float* p = part_o + (s0 * rows + row) * D + 4 * c;
        const uint64_t used = __ballot(there) >> (threadIdx.x & 63 & ~(L - 1)) & ((1ull << L) - 1);
        const int upto = n <= 8 ? n : used ? 64 - __builtin_clzll(used) : 0;   // behind the last that there is nothing is read; a few do not wait to be known
#pragma unroll 4
        for (int i = 0; i < upto; ++i, p += per * rows * D) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(p);
            const float f = __shfl(w, i, L) * 0x1p-8f;
            const bool on = __shfl((int)there, i, L);   // what an empty piece has there was never written
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] += on ? x[j] * f : 0.f;
        }
    }
    if (per > 1) {
        so[gr][c] = o;
        if (c == 0) sl[gr] = sum, sm[gr] = mx;
        __syncthreads();
        if (gr % per) return;
        for (int i = 1; i < per; ++i) mx = fmaxf(mx, sm[gr + i]);
        const float base = mx == -INFINITY ? 0.f : mx;
        sum = 0.f;
        o = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < per; ++i) {
            const float f = __builtin_amdgcn_exp2f(sm[gr + i] - base);
            o += so[gr + i][c] * f;
            sum += sl[gr + i] * f;
        }
    }
    if (at >= rows) return;
    const float inv = sum == 0.f ? 0.f : 0x1p8f / sum;
    *reinterpret_cast<u16x4*>(out + row * D + 4 * c) = u16x4{f2bf(o[0] * inv), f2bf(o[1] * inv), f2bf(o[2] * inv), f2bf(o[3] * inv)};
}

template <int KIND, int D, bool GROUPS> void launch_rows(int rows, const AttnArgs& a, int64_t tiles, hipStream_t st) {
    // Marked as read once from 192 MiB of codes on (by the table's width).  Where caches are many, a layer each, that gains 3 to 7 % (int8, 64 sequences of 2048, 256 MiB: 52 and 48 us;
    // mxfp4, two of 128k: 63 and 60); where the last cache (256 MB) still holds this one from the call before, it loses (64 of 2048: 45 and 49; mxfp4, 80 of 2048, 160 MiB: 35 and 39), and so
    // smaller ones are not.
    const bool once = !a.group_start && (int64_t)a.B * a.width * a.cache.page * a.cache.heads * row_bytes<KIND, D>() * 2 >= (int64_t)192 << 20;
    const dim3 g((unsigned)(tiles * a.cache.heads), a.splits), b(256);
    if (rows == 16) {
        if (!GROUPS && once) hipLaunchKernelGGL((quant_rows_kernel<KIND, D, 1, GROUPS, !GROUPS>), g, b, 0, st, a);
        else hipLaunchKernelGGL((quant_rows_kernel<KIND, D, 1, GROUPS, false>), g, b, 0, st, a);
    } else if (rows == 32) {
        hipLaunchKernelGGL((quant_rows_kernel<KIND, D, 2, GROUPS, false>), g, b, 0, st, a);
    } else if (rows == 128) {
        if constexpr (GROUPS) {
            constexpr int lds = 2 * sizeof(TileStep<KIND, D, 4>);
            lds_limit<quant_tile_kernel<KIND, D, 4, true>>(lds);
            hipLaunchKernelGGL((quant_tile_kernel<KIND, D, 4, true>), g, b, lds, st, a);
        }
    } else {
        constexpr int lds = 2 * sizeof(TileStep<KIND, D, 8>);
        lds_limit<quant_tile_kernel<KIND, D, 8, GROUPS>>(lds);
        hipLaunchKernelGGL((quant_tile_kernel<KIND, D, 8, GROUPS>), g, dim3(512), lds, st, a);
    }
}
template <bool GROUPS> void launch_rows_of(int kind, int D, int rows, const AttnArgs& a, int64_t tiles, hipStream_t st) {
    if (kind == kInt8 && D == 64) launch_rows<kInt8, 64, GROUPS>(rows, a, tiles, st);
    else if (kind == kInt8) launch_rows<kInt8, 128, GROUPS>(rows, a, tiles, st);
    else if (D == 64) launch_rows<kFp4, 64, GROUPS>(rows, a, tiles, st);
    else launch_rows<kFp4, 128, GROUPS>(rows, a, tiles, st);
}

// workgroups of a launch with tiles of `tile` rows, without pieces, if the items' rows are alike
int64_t workgroups(int64_t rows, int64_t items, int heads, int tile) {
    const int64_t tiles = (rows + tile - 1) / tile;
    return (tiles > items ? tiles : items) * heads;
}
// Rows of a tile, by the rows that an item has on average and the workgroups that this makes.  Small tiles read the keys more often, and large ones leave CUs idle and rows
// empty.  16 / 32 / 128 / 256 rows, each with the pieces that suit it best, 32 query and 8 key heads of 128, int8: 8 sequences of 64 rows on 2000 keys 25 / 27 / 33 / 33 us, 32 of 64 on 2000
// 65 / 46 / 69 / 76, 32 of 128 on 2000 112 / 82 / 96 / 77, 32 of 128 on 500 41 / 33 / 34 / 31, 4 of 512 on 500 24 / 18 / 27 / 28.  What a group shares (4 rows a sequence and key head):
// 16 sequences on 2048 keys 20 / 21 / 24 / 24, 64 on 8192 53 / 38 / 50 / 45, 128 on 16384 139 / 107 / 92 / 112, two groups of those 259 / 194 / 149 / 130.
int tile_of(int64_t rows, int64_t items, int heads, int64_t keys, bool own) {
    const int64_t per = items > 0 ? rows / items : rows;
    if (per <= 16) return 16;
    // 1 x 128 rows on 16000 keys: 43 us in 16 pieces with 16 rows, 34 with 32; 2 x 64 sequences of 8 rows on 8192, one key head: 37 and 30
    if (workgroups(rows, items, heads, 16) <= (own ? 256 : 64) && (own ? per <= 64 || keys < 4096 : per <= 128)) return 16;
    if (per >= 112 && workgroups(rows, items, heads, 256) >= (own ? 128 : 32)) return 256;
    return !own && per >= 192 && workgroups(rows, items, heads, 256) >= 16 ? 128 : 32;
}

}  // namespace

// What a call needs beside its tensors: rows of tiles, pieces of the keys.  keys: at most so many an item, by the table's width.
AttnPlan quant_attention_plan(int T, int B, bool single, int groups, int hq, int heads, int64_t keys) {
    AttnPlan p{};
    const int64_t rows = (int64_t)T * (hq / heads);
    auto side = [&](int64_t items, bool own, int& tile, int64_t& tiles, int& splits) {
        tile = tile_of(rows, items, heads, keys, own);
        tiles = rows / tile + items + 1;
        const int64_t wgs = workgroups(rows, items, heads, tile), full = tile == 256 ? 256 : 512;   // a workgroup a CU, or two
        int64_t s = full / wgs, least = 256;
        if (own) {
            const int64_t busy = rows > 16 * items ? 160 : 224;
            // Pieces take a launch to join.  int8, 32 query and 8 key heads of 128, us in 1 / 2 / 4 / 8 / 16 pieces (mixed: lengths of a quarter of the keys to all):
            //   few workgroups, as many pieces as fill the card: 1 x 2048 keys 21 / 16 / 12 / 11 / 11, 12 x 2048 23 / 18 / 17 / 17 / 20, 12 x 4096 42 / 28 / 25 / 24 / 27;
            //   none for short keys: 4 x 768 10.7 / 11.5 / 11.3 / 11.2 / 11.4, 12 x 768 10.8 / 11.2 / 12.4 / 12.2 / 14, and over that 4 x 1280 15 / 13 / 11 / 11 / 11.5; with more than 96
            //   workgroups 27 x 1280 17 / 20 / 21 / 23 / 28, 13 x 1280 16 / 15 / 15 / 16 / 18, and over that 13 x 2048 23 / 19 / 17 / 20 / 21;
            //   768 / workgroups from there to `busy`: 13 x 4096 42 / 28 / 25 / 28 / 27, 20 x 2048 24 / 24 / 23 / 23 / 27, mixed 23 / 22 / 20 / 21 / 25;
            //   from `busy` on none: 27 x 2048 25 / 26 / 28 / 29 / 34, mixed 23 / 21 / 22 / 24 / 29, 28 x 2048 25 / 26 / 28 / 30 / 34, mixed 24 / 24 / 25 / 27 / 32; in tiles of 32 rows, which do more with
            //   a key, sooner: 4 x 64 rows on 2000 31 / 34 / 40 / 55, 8 x 64 45 / 56 / 70 / 99;
            //   but for contexts that may be long, of which one may be far longer than the others: 28 x 4096 52 / 49 / 51 / 52 / 60, mixed 51 / 44 / 40 / 40 / 47, 63 x 4096 91 / 98 / 103 / 114 /
            //   129, mixed 89 / 93 / 78 / 82 / 93;
            //   tiles of 256, a workgroup a CU: 1 x 1024 rows on 4096 146 / 100 / 110 in 1 / 2 / 4, 1 x 2048 on 4096 157 / 160 / 197; 20 x 32 on 2000, which get two, 72 / 87 / 84.
            // For the most keys of a piece: 1 x 65536 in 8 / 16 / 32 / 64 81 / 46 / 30 / 31, 2 x 131072 186 / 108 / 97 / 101, 64 x 16384 in 1 / 2 / 4 / 8 352 / 359 / 358 / 370, mixed 316 / 306 / 301 / 290.
            if (tile == 256) s = (full + wgs / 2) / wgs;
            else if (wgs > 96) s = wgs < busy ? 768 / wgs : keys >= 4096 ? 1024 / wgs : 1;
            const int64_t longest = wgs < full ? 4096 : 16 * wgs;   // of a piece; the more there is beside it the longer one may take
            if (tile < 256 && keys / longest > s) s = keys / longest;
            if (keys <= (wgs > 96 ? 1280 : 768)) s = 1;
            // What sequences have of their own behind a shared prefix is taken to be short: in 1 / 4 / 8 / 16 pieces 64 sequences of 120 keys behind 2048 26 / 36 / 45 / 60 us, 16 of 1000 28 / 25 / 27 /
            // 30.  Where it is long, this loses: 8 of 4000 53 / 30 / 29 / 30, two of 18000 (64 query heads) 175 / 59 / 39 / 30.
            if (groups > 0) least = 32768;
        } else if (tile <= 32) {
            least = 4 * tile;   // 9 sequences on 480 shared keys: 13.5 us in pieces of 64, 17 in ones of 256
            const int64_t most = keys / 512 > 16 ? keys / 512 : 16;   // those behind wait for the sums: 16 sequences on 2048, one key head, in 16 pieces 16 us, in 32 18
            s = s < most ? s : most;
        }
        s = s < (keys + least - 1) / least ? s : (keys + least - 1) / least;
        splits = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
    };
    side(B, true, p.own_rows, p.own_tiles, p.own_splits);
    // one token of each sequence: tiles are counted without a look at where sequences begin
    if (single) p.own_tiles = (int64_t)T * ((hq / heads + p.own_rows - 1) / p.own_rows);
    if (groups > 0) side(groups, false, p.group_rows, p.group_tiles, p.group_splits);
    p.slots = p.own_splits + p.group_splits;
    p.last = groups > 0 && p.own_rows <= 32 && p.own_splits == 1;
    // A tile of 256 rows has a CU for itself.  Prompts of up to 2048 tokens behind up to 2048 of context, two of them: 163 us so, 218 in order; 16 of up to 256: 64 and 66.
    p.longest = !single && groups == 0 && B < 256 && p.own_rows == 256 && p.own_tiles * heads > 256;
    return p;
}

void launch_quant_attention(int kind, int D, const AttnPlan& p, const uint16_t* q, int64_t q_stride, const Cache& cache, const int32_t* bt, int64_t bt_stride, int width,
                            const int32_t* q_start, const int32_t* ctx_len, const int32_t* group_start, const int32_t* prefix_len, int B, int T, int groups, int hq,
                            float scale, uint16_t* out, float* part_o, float* part_l, hipStream_t st) {
    if (T == 0) return;
    AttnArgs a{q, q_stride, cache, bt, bt_stride, width, q_start, ctx_len, groups ? group_start : nullptr, prefix_len, B, T, groups, hq, scale * 1.4426950408889634f,
               out, part_o, part_l, p.slots, 0, 0,
               (cache.page & (cache.page - 1)) ? -1 : __builtin_ctz(cache.page), false, false};
    if (groups) {
        a.splits = p.group_splits;
        a.slot0 = 0;
        launch_rows_of<true>(kind, D, p.group_rows, a, p.group_tiles, st);
    }
    a.splits = p.own_splits;
    a.slot0 = p.group_splits;
    a.last = p.last;
    a.longest = p.longest;
    launch_rows_of<false>(kind, D, p.own_rows, a, p.own_tiles, st);
    if (p.slots > 1 && !a.last) {
        const int64_t rows = (int64_t)T * hq;
        const int gr = 256 / (D / 4);
        int per = 1;   // lanes' groups of a row: the rows fill the card with one, or there are pieces to share
        while (per < gr && per * 2 <= p.slots && rows * per < 2048 * gr) per *= 2;
        const dim3 g((unsigned)((rows + gr / per - 1) / (gr / per))), b(256);
        if (D == 64) hipLaunchKernelGGL(quant_join_kernel<64>, g, b, 0, st, part_o, part_l, out, rows, p.slots, per);
        else hipLaunchKernelGGL(quant_join_kernel<128>, g, b, 0, st, part_o, part_l, out, rows, p.slots, per);
    }
}

}  // namespace qkv
}  // namespace chronos
