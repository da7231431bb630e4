// quant_attention.hip — attention over a paged cache in 8 or 4 bits (chronos_quant_kv.h), for one token of each sequence, several, or prompts, and for groups
// of sequences whose first pages are the same.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  over the keys j <= position of i; token i of a sequence is at ctx - len + i.
//
// Rows are (token, query head) pairs of one key head; a workgroup takes a tile of 16 NQT rows, of one sequence, one key head and one piece of the keys.  Its four
// waves take steps of 32 keys in turn, each with a running maximum and sum, and are joined through LDS; pieces of the keys are joined by a second launch.  S^T = K Q^T
// and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16: with the keys as rows of the first product a lane holds the scores of its own query row, and the probabilities are
// the second one's operand as they are.  Codes go from memory to registers and become bfloat16 there, which is exact (eight bits, and e2m1 times a power of two):
//   * K: the dimensions of a product may be taken in any order that queries and keys share, so a lane takes its row's bytes 16 at a time;
//   * V: the operand wants eight keys of one dimension, the page has the dimensions of one key.  Row m of product dt is dimension m D / 16 + dt: a lane then needs the
//     same D / 16 neighbouring bytes of its eight keys, for all products, and no exchange between lanes.
// int8: a key's scale multiplies its scores, a value's the probabilities, in float32 before they are rounded to bfloat16 (2^-9, as everywhere in this library:
// rows average many of them and the output has the same step).  mxfp4: the conversion takes the scale.
//
// What no sum may take: keys behind the position, behind the context, on pages that the table does not have (numbers outside 0 .. pages - 1 are left out): their
// scores are -inf and their probabilities zero by selection, not by product; their values cannot be NaN either (a value scale of NaN acts on the probabilities of
// rows that see it).  Rows without any key are zeros.
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
    float2* part_ml;          // [slots, T * hq]: maximum (base 2) and sum
    int slots, splits, slot0;
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

// ---- codes to operands --------------------------------------------------------------------------------------------------------------------------------
template <int KIND, int D> struct Step {   // 32 keys of one wave
    static constexpr int KW = row_bytes<KIND, D>() / 16;   // words of K a lane has of a key: a quarter of the row
    static constexpr int VW = row_bytes<KIND, D>() >= 64 ? row_bytes<KIND, D>() / 64 : 1;   // words of V a lane has of a key: a sixteenth of the row
    uint32_t k[2][KW], v[8][VW];
    f32x4 ks[2], vs[2];      // int8: scales of keys 16 g + 4 h4 + i
    uint32_t ke[2], ve[8];   // mxfp4: E of the lane's key and block; words of all blocks' E of its eight keys
    bool ok[2];              // the page is there
};

template <int KIND, int D> __device__ __forceinline__ void load_step(const AttnArgs& a, const int32_t* bt, int h, int t0, int end, int lane, Step<KIND, D>& s) {
    constexpr int RB = row_bytes<KIND, D>();
    using S = Step<KIND, D>;
    const int r = lane & 15, h4 = lane >> 4;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int tg = t0 + 16 * g;
        const bool in = tg < end;
        const int at = in ? tg : t0;
        int blk = __builtin_amdgcn_readfirstlane(bt[at / a.cache.page]);
        s.ok[g] = in && blk >= 0 && blk < a.cache.pages;
        if (!s.ok[g]) blk = 0;
        const int64_t row = ((int64_t)blk * a.cache.heads + h) * a.cache.page + at % a.cache.page;   // of 16, all of one page
        const uint8_t* kp = a.cache.k + (row + r) * RB;
        if constexpr (KIND == kInt8) {
#pragma unroll
            for (int u = 0; u < D / 64; ++u) {
                const uint4 x = *reinterpret_cast<const uint4*>(kp + 64 * u + 16 * h4);
                s.k[g][4 * u] = x.x, s.k[g][4 * u + 1] = x.y, s.k[g][4 * u + 2] = x.z, s.k[g][4 * u + 3] = x.w;
            }
            s.ks[g] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(a.cache.ks) + row + 4 * h4);
            s.vs[g] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(a.cache.vs) + row + 4 * h4);
        } else {
            if constexpr (D == 128) {
                const uint4 x = *reinterpret_cast<const uint4*>(kp + 16 * h4);
                s.k[g][0] = x.x, s.k[g][1] = x.y, s.k[g][2] = x.z, s.k[g][3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(kp + 8 * h4);
                s.k[g][0] = x.x, s.k[g][1] = x.y;
            }
            const uint8_t* ke = reinterpret_cast<const uint8_t*>(a.cache.ks) + (row + r) * (D / 32) + h4 * (D / 32) / 4;
            s.ke[g] = *ke;
            const uint8_t* ve = reinterpret_cast<const uint8_t*>(a.cache.vs) + (row + 4 * h4) * (D / 32);
            if constexpr (D == 128) {
                const uint4 x = *reinterpret_cast<const uint4*>(ve);
                s.ve[4 * g] = x.x, s.ve[4 * g + 1] = x.y, s.ve[4 * g + 2] = x.z, s.ve[4 * g + 3] = x.w;
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(ve);
                s.ve[4 * g] = w.x & 0xffff;
                s.ve[4 * g + 1] = w.x >> 16;
                s.ve[4 * g + 2] = w.y & 0xffff;
                s.ve[4 * g + 3] = w.y >> 16;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint8_t* vp = a.cache.v + (row + 4 * h4 + i) * RB + (RB / 16) * r;
            if constexpr (RB == 128) {
                const uint2 x = *reinterpret_cast<const uint2*>(vp);
                s.v[4 * g + i][0] = x.x, s.v[4 * g + i][1] = x.y;
            } else if constexpr (RB == 64) {
                s.v[4 * g + i][0] = *reinterpret_cast<const uint32_t*>(vp);
            } else {
                s.v[4 * g + i][0] = *reinterpret_cast<const uint16_t*>(vp);
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
        codes4(s.k[g][c], __uint_as_float(s.ke[g] << 23), b);
        return bf16x8{b[0][0], b[0][1], b[1][0], b[1][1], b[2][0], b[2][1], b[3][0], b[3][1]};
    }
}
// V operands of all products: dimension r D / 16 + dt, keys 4 h4 .. + 3 and 16 + 4 h4 .. + 3
template <int KIND, int D> __device__ __forceinline__ void value_operands(const Step<KIND, D>& s, int r, bf16x8 (&o)[D / 16]) {
    if constexpr (KIND == kInt8) {
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
            for (int j = 0; j < 8; ++j) o[dt][j] = (__bf16)code8(s.v[j][dt >> 2], dt & 3);
    } else {
        const int sh = 8 * (r * (D / 16) / 32);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float scale = __uint_as_float(((s.ve[j] >> sh) & 255) << 23);
            bf16x2 b[4];
            codes4(s.v[j][0], scale, b);
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) o[dt][j] = b[dt >> 1][dt & 1];
        }
    }
}

// ---- the tile -----------------------------------------------------------------------------------------------------------------------------------------
// GROUPS: the items are groups of sequences, the keys those that each shares; otherwise sequences, their keys behind what they share.
template <int KIND, int D, int NQT, bool GROUPS>
__global__ void __launch_bounds__(256, NQT <= 2 ? 2 : 1) quant_rows_kernel(const AttnArgs a) {
    constexpr int ROWS = 16 * NQT, NC = D / 32, ND = D / 16;
    __shared__ __attribute__((aligned(16))) f32x4 so[3][ND][64];
    __shared__ float sm[3][64], sl[3][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, h4 = lane >> 4;
    const int heads = a.cache.heads, G = a.hq / heads;
    const int h = blockIdx.x % heads, split = blockIdx.y;
    Tile tile;
    if (!find_tile<GROUPS>(a, blockIdx.x / heads, G, ROWS, lane, tile)) return;

    // the rows of this lane: the last position each sees, and its queries
    int rpos[NQT];
    bf16x8 qf[NQT][NC];
    int last = -1;   // the last position that any row of the tile sees
    int own0 = 0, seq = tile.item, ctx = 0;   // own0: keys that the sequence shares with its group, which are not this launch's
    if constexpr (!GROUPS) {
        if (seq < a.B) {
            ctx = (int)min((int64_t)max(a.ctx_len[seq], 0), (int64_t)a.width * a.cache.page);
            if (a.group_start) own0 = shared_of(a, seq, lane);
        } else {
            own0 = -1;
        }
        if (own0 < 0 && a.slot0 > 0 && split == 0) {   // no group: nothing was written to the first slots
            for (int i = threadIdx.x; i < ROWS * a.slot0; i += 256) {
                const int R = tile.at + i % ROWS;
                if (R < tile.toks * G)
                    a.part_ml[(int64_t)(i / ROWS) * a.T * a.hq + (int64_t)(tile.tok0 + R / G) * a.hq + h * G + R % G] = float2{-INFINITY, 0.f};
            }
        }
        own0 = max(own0, 0);
    }
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
        const int R = tile.at + 16 * qt + r;
        const bool valid = R < tile.toks * G;
        const int t = tile.tok0 + (valid ? R / G : 0), hd = h * G + R % G;
        rpos[qt] = -1;
        if (valid) {
            if constexpr (GROUPS) {   // the token's sequence: the last that begins at or before it
                int s0 = first_seq(a, tile.item), s1 = first_seq(a, tile.item + 1) - 1;
                if (a.q_start) {
                    while (s0 < s1) {
                        const int mid = (s0 + s1 + 1) >> 1;
                        if (first_row(a, mid) <= t) s0 = mid;
                        else s1 = mid - 1;
                    }
                } else {
                    s0 = t;
                }
                rpos[qt] = min(a.ctx_len[s0], a.width * a.cache.page) - first_row(a, s0 + 1) + t;
            } else {
                rpos[qt] = ctx - tile.toks + (t - tile.tok0);
            }
        }
        last = max(last, rpos[qt]);
        const uint16_t* qp = a.q + t * a.q_stride + (int64_t)hd * D;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            bf16x8 v = *reinterpret_cast<const bf16x8*>(qp + key_dim<KIND, D>(c, h4));
            if (!valid) v = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
            qf[qt][c] = v;
        }
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) last = max(last, __shfl_xor(last, o, 64));
    last = __builtin_amdgcn_readfirstlane(last);
    int k0, k1;   // this tile's keys
    if constexpr (GROUPS) {
        k0 = 0;
        k1 = min(shared_keys(a, tile.item), last + 1);
        seq = min(first_seq(a, tile.item), a.B - 1);
    } else {
        k0 = min(own0, ctx);
        k1 = min(ctx, last + 1);
    }
    const int n = max(k1 - k0, 0);
    int chunk = (n + a.splits - 1) / a.splits;
    chunk = max((chunk + 127) & ~127, 128);
    const int ks = k0 + split * chunk, ke = min(k1, ks + chunk);
    const int32_t* bt = a.bt + (int64_t)(seq < a.B ? seq : 0) * a.bt_stride;

    float m[NQT], l[NQT];
    f32x4 o[NQT][ND];
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
        m[qt] = -INFINITY;
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
        uint32_t nan = 0;   // keys of this lane whose values are NaN, bit 4 g + i
        if constexpr (KIND == kFp4) {
            uint32_t big = 0;   // E of 192 and more does not come from numbers: looked for in all keys at once
#pragma unroll
            for (int j = 0; j < 8; ++j) big |= s.ve[j] & (s.ve[j] << 1);
            if (__ballot((big & 0x80808080u) != 0)) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int b = 0; b < D / 32; ++b)
                        if (((s.ve[j] >> (8 * b)) & 255) > 252) {
                            nan |= 1u << j;
                            s.ve[j] &= ~(255u << (8 * b));
                        }
            }
        }
        float kmul[2][4];
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) kmul[g][i] = KIND == kInt8 ? s.ks[g][i] * a.scale_log2 : a.scale_log2;
        bf16x8 vf[ND];
        value_operands<KIND, D>(s, r, vf);
#pragma unroll
        for (int qt = 0; qt < NQT; ++qt) {
            float mx = -INFINITY;
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = t0 + 16 * g + 4 * h4 + i;
                    const bool seen = s.ok[g] && tok < ke && tok <= rpos[qt];
                    const float v = seen ? sc[qt][g][i] * kmul[g][i] : -INFINITY;
                    sc[qt][g][i] = v;
                    mx = fmaxf(mx, v);
                }
            mx = fmaxf(m[qt], rows_max(mx));
            const float base = mx == -INFINITY ? 0.f : mx;
            const float alpha = __builtin_amdgcn_exp2f(m[qt] - base);
            m[qt] = mx;
            float ps = 0.f;
            bf16x8 pf;
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float p = __builtin_amdgcn_exp2f(sc[qt][g][i] - base);
                    const bool seen = s.ok[g] && t0 + 16 * g + 4 * h4 + i < ke && t0 + 16 * g + 4 * h4 + i <= rpos[qt];
                    if constexpr (KIND == kFp4) {
                        if (nan >> (4 * g + i) & 1) p = seen ? __builtin_nanf("") : 0.f;
                    }
                    ps += p;
                    if constexpr (KIND == kInt8) p = seen ? p * s.vs[g][i] : 0.f;
                    pf[4 * g + i] = (__bf16)p;
                }
            l[qt] = l[qt] * alpha + ps;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
                o[qt][dt] *= alpha;
                o[qt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[dt], pf, o[qt][dt], 0, 0, 0);
            }
        }
    };

    {   // two steps of the wave under way
        Step<KIND, D> A, B;
        int t0 = ks + w * 32;
        if (t0 < ke) load_step<KIND, D>(a, bt, h, t0, ke, lane, A);
        for (; t0 < ke; t0 += 256) {
            if (t0 + 128 < ke) load_step<KIND, D>(a, bt, h, t0 + 128, ke, lane, B);
            compute(t0, A);
            if (t0 + 128 >= ke) break;
            if (t0 + 256 < ke) load_step<KIND, D>(a, bt, h, t0 + 256, ke, lane, A);
            compute(t0 + 128, B);
        }
    }

    // ---- the waves' sums: those of 16 rows to the wave that has them to write ----------------------------------------------------------------------------
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
        l[qt] = rows_sum(l[qt]);
        const int owner = qt & 3;
        const int place = w < owner ? w : w - 1;
        if (qt) __syncthreads();
        if (w != owner) {
            sm[place][lane] = m[qt];
            sl[place][lane] = l[qt];
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) so[place][dt][lane] = o[qt][dt];
        }
        __syncthreads();
        if (w == owner) {
            float mx = m[qt];
#pragma unroll
            for (int p = 0; p < 3; ++p) mx = fmaxf(mx, sm[p][lane]);
            const float base = mx == -INFINITY ? 0.f : mx;
            float f = __builtin_amdgcn_exp2f(m[qt] - base), sum = l[qt] * f;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) o[qt][dt] *= f;
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                f = __builtin_amdgcn_exp2f(sm[p][lane] - base);
                sum += sl[p][lane] * f;
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) o[qt][dt] += so[p][dt][lane] * f;
            }
            const int R = tile.at + 16 * qt + r;
            const bool live = R < tile.toks * G;
            const int64_t row = (int64_t)(tile.tok0 + R / G) * a.hq + h * G + R % G;
            if (live && a.slots == 1) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint16_t* dst = a.out + row * D + (4 * h4 + i) * ND;
                    uint16_t v[ND];
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt) v[dt] = f2bf(o[qt][dt][i] * inv);
                    if constexpr (ND == 8) *reinterpret_cast<u16x8*>(dst) = u16x8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
                    else *reinterpret_cast<u16x4*>(dst) = u16x4{v[0], v[1], v[2], v[3]};
                }
            } else if (live) {
                const int64_t at = (int64_t)(a.slot0 + split) * a.T * a.hq + row;
                if (h4 == 0) a.part_ml[at] = float2{mx, sum};
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

// Rows of the pieces' sums: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  D / 4 lanes have a row, `per` such groups share its pieces and are joined through
// LDS.  The maxima and sums of up to D / 4 pieces are read at once, a lane each, and handed round; what the pieces hold does not wait for them.
template <int D>
__global__ void __launch_bounds__(256) quant_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, uint16_t* __restrict__ out, int64_t rows,
                                                         int slots, int per) {
    constexpr int L = D / 4, GR = 256 / L;
    __shared__ f32x4 so[GR][L];
    __shared__ float sl[GR], sm[GR];
    const int c = threadIdx.x % L, gr = threadIdx.x / L;
    const int64_t at = (int64_t)blockIdx.x * (GR / per) + gr / per, row = at < rows ? at : rows - 1;
    float mx = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = gr % per; s0 < slots; s0 += per * L) {   // pieces s0, s0 + per, ..: lane c has the c-th
        const int n = min(L, (slots - s0 + per - 1) / per), mine = s0 + per * c;
        const float2 ml = c < n ? part_ml[mine * rows + row] : float2{-INFINITY, 0.f};
        const bool there = ml.y != 0.f;
        float top = there ? ml.x : -INFINITY;
#pragma unroll
        for (int k = 1; k < L; k <<= 1) top = fmaxf(top, __shfl_xor(top, k, L));
        top = fmaxf(top, mx);
        const float base = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f(mx - base);
        mx = top;
        l *= old;
        o *= old;
        const float w = there ? __builtin_amdgcn_exp2f(ml.x - base) : 0.f;
        float sum = there ? ml.y * w : 0.f;
#pragma unroll
        for (int k = 1; k < L; k <<= 1) sum += __shfl_xor(sum, k, L);
        l += sum;
        const float* p = part_o + (s0 * rows + row) * D + 4 * c;
#pragma unroll 4
        for (int i = 0; i < n; ++i, p += per * rows * D) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(p);
            const float f = __shfl(w, i, L);
            const bool on = __shfl((int)there, i, L);   // what an empty piece has there was never written
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] += on ? x[j] * f : 0.f;
        }
    }
    if (per > 1) {
        so[gr][c] = o;
        if (c == 0) sl[gr] = l, sm[gr] = mx;
        __syncthreads();
        if (gr % per) return;
        for (int i = 1; i < per; ++i) mx = fmaxf(mx, sm[gr + i]);
        const float base = mx == -INFINITY ? 0.f : mx;
        l = 0.f;
        o = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < per; ++i) {
            const float f = __builtin_amdgcn_exp2f(sm[gr + i] - base);
            o += so[gr + i][c] * f;
            l += sl[gr + i] * f;
        }
    }
    if (at >= rows) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<u16x4*>(out + row * D + 4 * c) = u16x4{f2bf(o[0] * inv), f2bf(o[1] * inv), f2bf(o[2] * inv), f2bf(o[3] * inv)};
}

template <int KIND, int D, bool GROUPS> void launch_rows(int nqt, const AttnArgs& a, int64_t tiles, hipStream_t st) {
    const dim3 g((unsigned)(tiles * a.cache.heads), a.splits), b(256);
    if (nqt == 1) hipLaunchKernelGGL((quant_rows_kernel<KIND, D, 1, GROUPS>), g, b, 0, st, a);
    else if (nqt == 2) hipLaunchKernelGGL((quant_rows_kernel<KIND, D, 2, GROUPS>), g, b, 0, st, a);
    else hipLaunchKernelGGL((quant_rows_kernel<KIND, D, 4, GROUPS>), g, b, 0, st, a);
}
template <bool GROUPS> void launch_rows_of(int kind, int D, int nqt, const AttnArgs& a, int64_t tiles, hipStream_t st) {
    if (kind == kInt8 && D == 64) launch_rows<kInt8, 64, GROUPS>(nqt, a, tiles, st);
    else if (kind == kInt8) launch_rows<kInt8, 128, GROUPS>(nqt, a, tiles, st);
    else if (D == 64) launch_rows<kFp4, 64, GROUPS>(nqt, a, tiles, st);
    else launch_rows<kFp4, 128, GROUPS>(nqt, a, tiles, st);
}

// Rows of a tile, by the rows that an item has on average
int tiles_of(int64_t rows, int64_t items) {
    const int64_t per = items > 0 ? rows / items : rows;
    return per <= 16 ? 1 : per <= 32 ? 2 : 4;
}

}  // namespace

// What a call needs beside its tensors: rows of tiles, pieces of the keys.  keys: at most so many an item, by the table's width.
AttnPlan quant_attention_plan(int T, int B, int groups, int hq, int heads, int64_t keys) {
    AttnPlan p{};
    const int64_t rows = (int64_t)T * (hq / heads);
    auto side = [&](int64_t items, int& nqt, int64_t& tiles, int& splits) {
        nqt = tiles_of(rows, items);
        tiles = rows / (16 * nqt) + items + 1;
        const int64_t wgs = ((rows + 16 * nqt - 1) / (16 * nqt) > items ? (rows + 16 * nqt - 1) / (16 * nqt) : items) * heads;
        int64_t s = (1024 + wgs - 1) / wgs;
        s = s < (keys + 255) / 256 ? s : (keys + 255) / 256;
        splits = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
    };
    side(B, p.own_nqt, p.own_tiles, p.own_splits);
    if (groups > 0) side(groups, p.group_nqt, p.group_tiles, p.group_splits);
    p.slots = p.own_splits + p.group_splits;
    return p;
}

void launch_quant_attention(int kind, int D, const AttnPlan& p, const uint16_t* q, int64_t q_stride, const Cache& cache, const int32_t* bt, int64_t bt_stride, int width,
                            const int32_t* q_start, const int32_t* ctx_len, const int32_t* group_start, const int32_t* prefix_len, int B, int T, int groups, int hq,
                            float scale, uint16_t* out, float* part_o, float* part_ml, hipStream_t st) {
    if (T == 0) return;
    AttnArgs a{q, q_stride, cache, bt, bt_stride, width, q_start, ctx_len, groups ? group_start : nullptr, prefix_len, B, T, groups, hq, scale * 1.4426950408889634f,
               out, part_o, reinterpret_cast<float2*>(part_ml), p.slots, 0, 0};
    if (groups) {
        a.splits = p.group_splits;
        a.slot0 = 0;
        launch_rows_of<true>(kind, D, p.group_nqt, a, p.group_tiles, st);
    }
    a.splits = p.own_splits;
    a.slot0 = p.group_splits;
    // one token of each sequence: tiles are counted without a look at where sequences begin
    const int64_t tiles = q_start ? p.own_tiles : (int64_t)T * ((hq / cache.heads + 16 * p.own_nqt - 1) / (16 * p.own_nqt));
    launch_rows_of<false>(kind, D, p.own_nqt, a, tiles, st);
    if (p.slots > 1) {
        const int64_t rows = (int64_t)T * hq;
        const int gr = 256 / (D / 4);
        int per = 1;   // lanes' groups of a row: the rows fill the card with one, or there are pieces to share
        while (per < gr && per * 2 <= p.slots && rows * per < 2048 * gr) per *= 2;
        const dim3 g((unsigned)((rows + gr / per - 1) / (gr / per))), b(256);
        if (D == 64) hipLaunchKernelGGL(quant_join_kernel<64>, g, b, 0, st, part_o, reinterpret_cast<const float2*>(part_ml), out, rows, p.slots, per);
        else hipLaunchKernelGGL(quant_join_kernel<128>, g, b, 0, st, part_o, reinterpret_cast<const float2*>(part_ml), out, rows, p.slots, per);
    }
}

}  // namespace qkv
}  // namespace chronos
