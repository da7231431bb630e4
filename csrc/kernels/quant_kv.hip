// quant_kv.hip — a key/value cache in 8 or 4 bits (chronos_quant_kv.h has its layout): written from a projection's rows in one pass, and read back.
//
// norm_rope_kv_quant.  qkv[T, (Hq + 2 Hkv) D], per head row x:
//   y = x / sqrt(mean(x^2) + eps) * w     queries and keys that have weights
//   y1' = y1 c - y2 s, y2' = y2 c + y1 s  queries and keys, the first R dimensions in two halves, c, s = cos_sin[pos, : R / 2], cos_sin[pos, R / 2 :]
//   q = y' in bfloat16; k = y', v = x in the cache's codes and scales, at block_table[tok_seq, pos / page], row pos % page.
// It reads T (Hq + 2 Hkv) D 2 bytes and writes T Hq D 2 and the rows' codes: bytes are what bounds it.  D / 8 lanes a head row, 16 bytes a lane; a lane's rotation
// partner is D / 16 lanes away or none, and its eight numbers are read a second time (they are in the cache) where an exchange would go through LDS.  Keys and values
// go by double up to their codes: a key next to a border between two codes then takes the code of the formula, whatever the order of sums, and it costs nothing beside
// the bytes.  The queries, most of the rows, are float32, in a power of two's units where their squares would pass its range (all rows in double: 237 us for 16384 tokens of 64 + 16 heads of 128 in int8, against 133, 645 MB at 4.8 TB/s).
#include "chronos_quant_kv.h"

namespace chronos {
namespace qkv {
namespace {

// over n neighbouring lanes, n = 4, 8 or 16, all of them active
template <int CTRL> __device__ __forceinline__ double dpp(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int n, typename Op> __device__ __forceinline__ double group_all(double v, Op&& op) {
    v = op(v, dpp<0xb1>(v));                      // quad_perm 1 0 3 2
    v = op(v, dpp<0x4e>(v));                      // quad_perm 2 3 0 1
    if constexpr (n > 4) v = op(v, dpp<0x141>(v));   // row_half_mirror
    if constexpr (n > 8) v = op(v, dpp<0x140>(v));   // row_mirror
    return v;
}
struct Sum { __device__ double operator()(double a, double b) const { return a + b; } };
struct Max { __device__ double operator()(double a, double b) const { return fmax(a, b); } };

__device__ __forceinline__ void ld8(const uint16_t* p, float (&v)[8]) {
    const u16x8 r = *reinterpret_cast<const u16x8*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = bf2f(r[j]);
}

// Eight numbers of a row into its codes; lane c of the row's D / 8 (all active).  `there`: the row has a place.
template <int KIND, int D> __device__ __forceinline__ void put(const double (&y)[8], int c, bool there, uint8_t* codes, void* scales, int64_t row) {
    constexpr double kInf = __builtin_huge_val();
    double top = 0.;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmax(top, fabs(y[j]) < kInf ? fabs(y[j]) : kInf);   // NaN counts as an infinity
    if constexpr (KIND == kInt8) {
        top = group_all<D / 8>(top, Max{});
        const bool whole = top < kInf;
        const float s = whole ? (float)(top / 127.) : __builtin_nanf("");
        const double inv = s > 0.f ? 1. / (double)s : 0.;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int n = whole ? min(max((int)rint(y[j] * inv), -127), 127) : 0;   // past 127 where the scale is denormal
            w[j >> 2] |= (uint32_t)(n & 255) << (8 * (j & 3));
        }
        if (!there) return;
        *reinterpret_cast<uint2*>(codes + row * D + 8 * c) = uint2{w[0], w[1]};
        if (c == 0) reinterpret_cast<float*>(scales)[row] = s;
    } else {
        top = group_all<4>(top, Max{});
        const bool whole = group_all<D / 8>(top, Max{}) < kInf;
        // top = m 2^p, 1 <= m < 2: at most 7 2^e = 1.75 2^(e + 2) with e = p - 2, or p - 1 where m is over 1.75
        const uint64_t u = __builtin_bit_cast(uint64_t, top);
        int e = (int)(u >> 52) - 1023 - 2 + ((u & 0xfffffffffffffull) > 0xc000000000000ull);
        e = min(max(e, -126), 125);
        const double inv = __builtin_bit_cast(double, (uint64_t)(1023 - e) << 52);
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double a = fabs(y[j]) * inv;
            // codes are 1/2 apart up to 2, 1 up to 4, 2 up to 6
            const double n = rint(a * (a < 2. ? 2. : a < 4. ? 1. : .5));
            const int code = min((int)fmin(n, 16.) + (a < 2. ? 0 : a < 4. ? 2 : 4), 7);
            w |= (uint32_t)(code | (y[j] < 0. ? 8 : 0)) << (4 * j);
        }
        if (!there) return;
        *reinterpret_cast<uint32_t*>(codes + row * (D / 2) + 4 * c) = whole ? w : 0;
        if ((c & 3) == 0) reinterpret_cast<uint8_t*>(scales)[row * (D / 32) + (c >> 2)] = whole ? (uint8_t)(e + 127) : 255;
    }
}

struct Place {
    int64_t row;   // first of page * heads + head rows of the token's slot, head 0; a head further is `page` rows on
    bool there;
};
__device__ __forceinline__ Place place(const Cache& c, const int32_t* bt, int64_t bt_stride, int seqs, int width, int seq, int p) {
    Place r{0, false};
    if (p < 0 || seq < 0 || seq >= seqs || p / c.page >= width) return r;
    const int blk = bt[seq * bt_stride + p / c.page];
    if (blk < 0 || blk >= c.pages) return r;
    r.row = (int64_t)blk * c.heads * c.page + p % c.page;
    r.there = true;
    return r;
}

// A block has 256 / (D / 8) * N neighbouring query heads of a token (the place, the angles and the weights serve all of them, the rows' loads are under way together),
// or 256 / (D / 8) of its key and value heads: `parts` blocks a token, the first q_parts with queries.
template <int KIND, int D, int N>
__global__ void __launch_bounds__(256) norm_rope_kv_quant_kernel(
    const uint16_t* __restrict__ qkv, int64_t qkv_stride, const int32_t* __restrict__ pos, const int32_t* __restrict__ tok_seq,
    const int32_t* __restrict__ bt, int64_t bt_stride, int seqs, int width, const float* __restrict__ cos_sin, int R, int P,
    const uint16_t* __restrict__ q_norm, const uint16_t* __restrict__ k_norm, double eps, uint16_t* __restrict__ q_out, Cache cache, int hq, int q_parts, int parts) {
    constexpr int L = D / 8, S = 256 / L;   // lanes of a head row, head rows side by side
    const int64_t t = blockIdx.x / parts;
    const int part = blockIdx.x % parts, c = threadIdx.x % L;
    const int H = R / 16;   // chunks of eight dimensions in a half of the rotation
    const bool turns = c < 2 * H;
    const int other = c < H ? c + H : turns ? c - H : c;   // the lane's partner's; its numbers count for nothing where there is none
    const uint16_t* src = qkv + t * qkv_stride;
    const int p = pos[t], seq = tok_seq[t];
    const u16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
    float cs[8], sn[8];
    auto angles = [&](bool there) {
        const float* row = cos_sin + (int64_t)(there ? p : 0) * R + 8 * (c < H ? c : turns ? c - H : 0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cs[j] = row[j];
            sn[j] = row[R / 2 + j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cs[j] = turns ? cs[j] : 1.f;
            sn[j] = c < H ? -sn[j] : sn[j];
        }
    };
    // a row's numbers are inv * (x cs w + x' sn w'), x' and w' the partner's
    if (part < q_parts) {
        const int head0 = part * (S * N) + threadIdx.x / L;
        u16x8 xr[N], xp[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint16_t* row = src + (int64_t)min(head0 + S * i, hq - 1) * D;
            xr[i] = *reinterpret_cast<const u16x8*>(row + 8 * c);
            xp[i] = *reinterpret_cast<const u16x8*>(row + 8 * other);
        }
        float w[8], wo[8];
        if (q_norm) {
            ld8(q_norm + 8 * c, w);
            ld8(q_norm + 8 * other, wo);
        }
        const bool there = place(cache, bt, bt_stride, seqs, width, seq, p).there && p < P;
        angles(there);
        if (q_norm) {
#pragma unroll
            for (int j = 0; j < 8; ++j) cs[j] *= w[j], sn[j] *= wo[j];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            u16x8 po = turns ? xp[i] : zero;
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = bf2f(xr[i][j]);
            float f = 1.f;
            if (q_norm) {
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
                float m = group_sum(ss, L) * (1.f / D) + (float)eps;
                if (!(m > 0x1p-100f && m < 0x1p100f)) {   // squares at the ends of float32's range: the row times a power of two, eps times its square
                    const float by = m < 1.f ? 0x1p80f : 0x1p-80f;
                    ss = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        x[j] *= by;
                        po[j] = f2bf(bf2f(po[j]) * by);
                        ss += x[j] * x[j];
                    }
                    m = group_sum(ss, L) * (1.f / D) + (float)(eps * by * by);
                }
                f = rsqrtf(m);
            }
            u16x8 o;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = f2bf(f * (x[j] * cs[j] + bf2f(po[j]) * sn[j]));
            if (head0 + S * i < hq) *reinterpret_cast<u16x8*>(q_out + (t * hq + head0 + S * i) * D + 8 * c) = there ? o : zero;
        }
        return;
    }
    const int at = (part - q_parts) * S + threadIdx.x / L, head = min(at, 2 * cache.heads - 1);
    const uint16_t* row = src + (int64_t)(hq + head) * D;
    const bool key = head < cache.heads;
    const u16x8 xr = *reinterpret_cast<const u16x8*>(row + 8 * c), xp = *reinterpret_cast<const u16x8*>(row + 8 * other);
    Place pl = place(cache, bt, bt_stride, seqs, width, seq, p);
    pl.there = pl.there && p < P;
    double y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = bf2f(xr[j]);
    if (key) {
        const u16x8 po = turns ? xp : zero;
        angles(pl.there);
        double inv = 1.;
        float w[8], wo[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 1.f, wo[j] = 1.f;
        if (k_norm) {
            ld8(k_norm + 8 * c, w);
            ld8(k_norm + 8 * other, wo);
            double ss = 0.;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += y[j] * y[j];
            inv = 1. / sqrt(group_all<L>(ss, Sum{}) * (1. / D) + eps);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = inv * (y[j] * cs[j] * w[j] + (double)bf2f(po[j]) * sn[j] * wo[j]);
    }
    pl.row += (int64_t)(key ? head : head - cache.heads) * cache.page;
    put<KIND, D>(y, c, pl.there && at == head, key ? cache.k : cache.v, key ? cache.ks : cache.vs, pl.row);
}

// k, v [T, Hkv, D] in bfloat16 of tokens of the cache; zeros where a token has no place.  Reads the codes, writes 4 T Hkv D bytes, which bound it: 128k tokens of 8 heads of 128 in 4 bits, 680 MB,
// 156 us, 4.4 TB/s, what a copy reaches.  N head rows a lane,
// their places, then their codes under way together.
template <int KIND, int D, int N>
__global__ void __launch_bounds__(256) quant_kv_read_kernel(const int32_t* __restrict__ pos, const int32_t* __restrict__ tok_seq, const int32_t* __restrict__ bt,
                                                            int64_t bt_stride, int seqs, int width, Cache cache, uint16_t* __restrict__ k,
                                                            uint16_t* __restrict__ v, int64_t T) {
    constexpr int L = D / 8, S = 256 / L, W = KIND == kInt8 ? 2 : 1;
    const int c = threadIdx.x % L;
    const int64_t first = (int64_t)blockIdx.x * (S * N) + threadIdx.x / L, most = T * cache.heads;
    int64_t row[N];
    bool there[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int64_t at = first + S * i, unit = at < most ? at : most - 1, t = unit / cache.heads;
        const Place pl = place(cache, bt, bt_stride, seqs, width, tok_seq[t], pos[t]);
        there[i] = pl.there;
        row[i] = pl.row + (unit - t * cache.heads) * cache.page;   // a row of the cache in any case
    }
    uint32_t w[2][N][W], e[2][N];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const uint8_t* codes = kv ? cache.v : cache.k;
        const void* scales = kv ? cache.vs : cache.ks;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (KIND == kInt8) {
                const uint2 x = *reinterpret_cast<const uint2*>(codes + row[i] * D + 8 * c);
                w[kv][i][0] = x.x, w[kv][i][1] = x.y;
                e[kv][i] = reinterpret_cast<const uint32_t*>(scales)[row[i]];
            } else {
                w[kv][i][0] = *reinterpret_cast<const uint32_t*>(codes + row[i] * (D / 2) + 4 * c);
                e[kv][i] = reinterpret_cast<const uint8_t*>(scales)[row[i] * (D / 32) + (c >> 2)];
            }
        }
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (first + S * i >= most) break;
            u16x8 o;
            if constexpr (KIND == kInt8) {
                const float s = __uint_as_float(e[kv][i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = f2bf(code8(w[kv][i][j >> 2], j & 3) * s);
            } else {
                bf16x2 b[4];
                codes4(w[kv][i][0], unit4(e[kv][i]), b);
                o = __builtin_bit_cast(u16x8, (bf16x8{b[0][0], b[0][1], b[1][0], b[1][1], b[2][0], b[2][1], b[3][0], b[3][1]}));
                if (e[kv][i] > 252) o = u16x8{0x7fc0, 0x7fc0, 0x7fc0, 0x7fc0, 0x7fc0, 0x7fc0, 0x7fc0, 0x7fc0};
            }
            if (!there[i]) o = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
            *reinterpret_cast<u16x8*>((kv ? v : k) + (first + S * i) * D + 8 * c) = o;
        }
}

}  // namespace

void launch_norm_rope_kv_quant(int kind, int D, const uint16_t* qkv, int64_t qkv_stride, const int32_t* pos, const int32_t* tok_seq, const int32_t* bt,
                               int64_t bt_stride, int seqs, int width, const float* cos_sin, int R, int P, const uint16_t* q_norm, const uint16_t* k_norm, double eps,
                               uint16_t* q_out, const Cache& cache, int64_t T, int hq, hipStream_t st) {
    if (T == 0) return;
    const int side = 256 / (D / 8);
    // four head rows a lane where the card is full all the same: 16384 tokens of 64 query heads 132 us, one row a lane 177; 4096 tokens 33 and 39; 1024 of 32 heads alike
    const bool four = T * ((hq + 4 * side - 1) / (4 * side)) >= 1024;
    const int q_parts = (hq + (four ? 4 : 1) * side - 1) / ((four ? 4 : 1) * side), parts = q_parts + (2 * cache.heads + side - 1) / side;
    const dim3 b(256);
    // a launch has fewer than 2^32 threads
    const int64_t most = (1 << 23) / parts > 0 ? (1 << 23) / parts : 1;
    for (int64_t t = 0; t < T; t += most) {
        const dim3 g((unsigned)((T - t < most ? T - t : most) * parts));
#define CHRONOS_QKV(K, DD, N)                                                                                                                                        \
    if (kind == K && D == DD && four == (N == 4))                                                                                                                    \
        hipLaunchKernelGGL((norm_rope_kv_quant_kernel<K, DD, N>), g, b, 0, st, qkv + t * qkv_stride, qkv_stride, pos + t, tok_seq + t, bt, bt_stride, seqs, width,   \
                           cos_sin, R, P, q_norm, k_norm, eps, q_out + t * hq * D, cache, hq, q_parts, parts);
        CHRONOS_QKV(kInt8, 64, 1) CHRONOS_QKV(kInt8, 128, 1) CHRONOS_QKV(kFp4, 64, 1) CHRONOS_QKV(kFp4, 128, 1)
        CHRONOS_QKV(kInt8, 64, 4) CHRONOS_QKV(kInt8, 128, 4) CHRONOS_QKV(kFp4, 64, 4) CHRONOS_QKV(kFp4, 128, 4)
    }
#undef CHRONOS_QKV
}

void launch_quant_kv_read(int kind, int D, const int32_t* pos, const int32_t* tok_seq, const int32_t* bt, int64_t bt_stride, int seqs, int width, const Cache& cache,
                          uint16_t* k, uint16_t* v, int64_t T, hipStream_t st) {
    if (T == 0) return;
    const int64_t units = T * cache.heads, side = 256 / (D / 8);
    const bool four = units >= 1 << 19;   // 128k tokens of 8 heads in 4 bits 157 us, one row a lane 168; 32k alike; 8k 10.4 and 9.2
    const dim3 g((unsigned)((units + (four ? 4 : 1) * side - 1) / ((four ? 4 : 1) * side))), b(256);
#define CHRONOS_QKV(K, DD, N)                    \
    if (kind == K && D == DD && four == (N == 4)) \
        hipLaunchKernelGGL((quant_kv_read_kernel<K, DD, N>), g, b, 0, st, pos, tok_seq, bt, bt_stride, seqs, width, cache, k, v, T);
    CHRONOS_QKV(kInt8, 64, 1) CHRONOS_QKV(kInt8, 128, 1) CHRONOS_QKV(kFp4, 64, 1) CHRONOS_QKV(kFp4, 128, 1)
    CHRONOS_QKV(kInt8, 64, 4) CHRONOS_QKV(kInt8, 128, 4) CHRONOS_QKV(kFp4, 64, 4) CHRONOS_QKV(kFp4, 128, 4)
#undef CHRONOS_QKV
}

}  // namespace qkv
}  // namespace chronos
