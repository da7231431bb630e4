// chronos_quant_kv.h — the layout of a key/value cache held in 8 or 4 bits, shared by the kernels that write it, read it back and attend to it
// (quant_kv.hip, quant_attention.hip) and by their host checks.
//
//   int8:   k, v [pages, heads, page, D] signed codes, -127 .. 127; ks, vs float32 [pages, heads, page].  A number is code * scale of its token and head,
//           scale = max|x| / 127 rounded to float32.
//   mxfp4:  k, v [pages, heads, page, D / 2] bytes of two e2m1 codes, the even dimension's in the lower half; ks, vs [pages, heads, page, D / 32] bytes E.
//           A number is its code's value (0 .5 1 1.5 2 3 4 6, the top bit the sign) times 2^(E - 127), one E per 32 dimensions: the smallest with
//           max|x| <= 7 2^(E - 127), in 1 .. 252 (larger maxima are cut off at 6 2^125).  Up to 7 and not to 6, as 6 is the nearest code up to there: over normal
//           values the error is .112 of their size, .115 with 6 or 8 in its place.
//   A row (token, head) that holds an infinity or a NaN is held as NaN as a whole: scale NaN, E = 255 in all its blocks.  253 and 254, which no write makes, are read as 255
//   is: six of their units pass float32's range.
//   Attention keeps its accuracy for values between 2^-76 and 2^108 in int8, and up to the end of the range in mxfp4; smaller ones are written and read back as ever, but attention may
//   give zeros for them.  Scores have to be numbers of float32.
#pragma once
#include "chronos_hip.h"

namespace chronos {
namespace qkv {

enum { kInt8 = 0, kFp4 = 1 };

struct Cache {
    uint8_t *k, *v;
    void *ks, *vs;
    int pages, heads, page;
};

// How a call of the attention is cut up (quant_attention.hip): rows of a tile, tiles and pieces of the keys, for the sequences' own keys and for those that
// groups share; slots of partial sums, 1: none; whether the launch over the own keys joins the groups' pieces itself, and whether it takes the tiles with most keys first
struct AttnPlan {
    int own_rows, own_splits, group_rows, group_splits, slots;
    int64_t own_tiles, group_tiles;
    bool last, longest;
};

template <int KIND, int D> constexpr int row_bytes() { return KIND == kInt8 ? D : D / 2; }
template <int KIND, int D> constexpr int scale_bytes() { return KIND == kInt8 ? 4 : D / 32; }

// a signed byte of a word, as a float
__device__ __forceinline__ float code8(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// the power of two that E stands for
__device__ __forceinline__ float unit4(uint32_t E) { return __uint_as_float((E > 252 ? 255 : E) << 23); }

// bfloat16 of the eight e2m1 codes of a word, times a power of two (exact)
__device__ __forceinline__ void codes4(uint32_t w, float scale, bf16x2 (&v)[4]) {
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
}

}  // namespace qkv
}  // namespace chronos
