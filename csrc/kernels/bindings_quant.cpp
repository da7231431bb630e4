// bindings_quant.cpp — the operators of a key/value cache in 8 or 4 bits (quant_kv.hip, quant_attention.hip) as torch.ops.chronos.*.  As in bindings.cpp everything
// that a kernel takes for granted of its tensors is checked here, launches go to the current stream of the tensors' device, and scratch comes from torch's allocator
// with every call.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <algorithm>
#include <tuple>
#include <vector>

#include "chronos_quant_kv.h"

namespace chronos {
namespace qkv {
void launch_norm_rope_kv_quant(int, int, const uint16_t*, int64_t, const int32_t*, const int32_t*, const int32_t*, int64_t, int, int, const float*, int, int,
                               const uint16_t*, const uint16_t*, double, uint16_t*, const Cache&, int64_t, int, hipStream_t);
void launch_quant_kv_read(int, int, const int32_t*, const int32_t*, const int32_t*, int64_t, int, int, const Cache&, uint16_t*, uint16_t*, int64_t, hipStream_t);
AttnPlan quant_attention_plan(int, int, bool, int, int, int, int64_t);
void launch_quant_attention(int, int, const AttnPlan&, const uint16_t*, int64_t, const Cache&, const int32_t*, int64_t, int, const int32_t*, const int32_t*,
                            const int32_t*, const int32_t*, int, int, int, int, float, uint16_t*, float*, float*, hipStream_t);
}  // namespace qkv
}  // namespace chronos

namespace {

using at::Tensor;
using chronos::qkv::Cache;
constexpr int64_t kMost = 1ll << 30;   // tokens, pages, table entries: the kernels count them in int

#define CHK(c, ...) TORCH_CHECK((c), "chronos: ", __VA_ARGS__)

inline hipStream_t cur_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
inline const uint16_t* bf(const Tensor& t) { return reinterpret_cast<const uint16_t*>(t.data_ptr()); }
inline uint16_t* bfm(const Tensor& t) { return reinterpret_cast<uint16_t*>(t.data_ptr()); }

void on(const Tensor& t, const Tensor& like, const char* n) { CHK(t.is_cuda() && t.device() == like.device(), n, " must be on ", like.device()); }
const int32_t* ints(const Tensor& t, const Tensor& like, int64_t least, const char* n) {
    on(t, like, n);
    CHK(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous(), n, " must be a contiguous int32 vector");
    CHK(t.numel() >= least, n, " needs ", least, " entries, has ", t.numel());
    return t.data_ptr<int32_t>();
}

struct Held {
    int kind, D;
    Cache c;
};
Held held(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
    CHK(k.is_cuda(), "the cache must be on a GPU");
    for (const auto& p : {std::make_pair(&v, "v"), std::make_pair(&ks, "ks"), std::make_pair(&vs, "vs")}) on(*p.first, k, p.second);
    const bool int8 = k.scalar_type() == at::kChar;
    CHK(int8 || k.scalar_type() == at::kByte, "k must be int8 codes or uint8 pairs of e2m1 codes");
    CHK(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), "k and v must be [pages, heads, page, row] of one type");
    const int64_t D = int8 ? k.size(3) : 2 * k.size(3);
    CHK(D == 64 || D == 128, "heads of 64 or 128 dimensions, not ", D);
    CHK(k.size(2) > 0 && k.size(2) % 16 == 0, "pages of a multiple of 16 tokens, not ", k.size(2));
    CHK(k.size(0) > 0 && k.size(1) > 0 && k.size(0) < kMost && k.size(1) < 65536 && k.size(2) < kMost, "the cache has no pages or heads, or too many");
    for (const Tensor* s : {&ks, &vs}) {
        CHK(s->scalar_type() == (int8 ? at::kFloat : at::kByte), "scales must be float32 (int8 codes) or uint8 (e2m1 codes)");
        CHK(s->dim() == (int8 ? 3 : 4) && s->size(0) == k.size(0) && s->size(1) == k.size(1) && s->size(2) == k.size(2) && (int8 || s->size(3) == D / 32),
            "scales must be [pages, heads, page] (int8 codes) or [pages, heads, page, D / 32] (e2m1 codes)");
    }
    for (const Tensor* s : {&k, &v, &ks, &vs}) CHK(s->is_contiguous() && (uintptr_t)s->data_ptr() % 16 == 0, "k, v, ks and vs must be contiguous, from a multiple of 16 bytes");
    return Held{int8 ? 0 : 1, (int)D,
                Cache{(uint8_t*)k.data_ptr(), (uint8_t*)v.data_ptr(), ks.data_ptr(), vs.data_ptr(), (int)k.size(0), (int)k.size(1), (int)k.size(2)}};
}
void table(const Tensor& t, const Tensor& like) {
    on(t, like, "block_table");
    CHK(t.scalar_type() == at::kInt && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1), "block_table must be int32 [sequences, pages] with neighbouring pages side by side");
    CHK(t.size(0) < kMost && t.size(1) < kMost, "block_table is too large");
}

Tensor norm_rope_kv_quant(const Tensor& qkv, const Tensor& pos, const Tensor& tok_seq, const Tensor& block_table, const Tensor& cos_sin, const Tensor& k, const Tensor& v,
                          const Tensor& ks, const Tensor& vs, int64_t hq, const c10::optional<Tensor>& q_norm, const c10::optional<Tensor>& k_norm, double eps) {
    const Held c = held(k, v, ks, vs);
    const int64_t D = c.D, heads = c.c.heads;
    on(qkv, k, "qkv");
    CHK(qkv.scalar_type() == at::kBFloat16 && qkv.dim() == 2, "qkv must be bfloat16 [T, (hq + 2 hkv) D]");
    CHK(hq >= 0 && hq < 65536 && qkv.size(1) == (hq + 2 * heads) * D, "qkv must be [T, (hq + 2 hkv) D] = [T, ", (hq + 2 * heads) * D, "], has rows of ", qkv.size(1));
    CHK(qkv.size(0) < kMost, "too many tokens");
    const int64_t T = qkv.size(0);
    CHK(pos.dim() == 1 && pos.numel() == T && tok_seq.dim() == 1 && tok_seq.numel() == T, "pos and tok_seq need an entry per token");
    const int32_t *pp = ints(pos, k, T, "pos"), *sp = ints(tok_seq, k, T, "tok_seq");
    table(block_table, k);
    on(cos_sin, k, "cos_sin");
    const int64_t R = cos_sin.dim() == 2 ? cos_sin.size(1) : -1;
    CHK(cos_sin.scalar_type() == at::kFloat && R >= 16 && R % 16 == 0 && R <= D, "cos_sin must be float32 [positions, R], R a multiple of 16 up to D");
    CHK(cos_sin.is_contiguous() && (uintptr_t)cos_sin.data_ptr() % 16 == 0 && cos_sin.size(0) < kMost, "cos_sin must be contiguous, from a multiple of 16 bytes");
    CHK(cos_sin.size(0) > 0 || T == 0, "cos_sin has no positions");
    CHK(eps >= 0., "eps must not be negative");
    c10::hip::HIPGuardMasqueradingAsCUDA g(k.device());
    // rows and weights that the kernel cannot take 16 bytes at a time are laid out anew
    auto flat = [](const Tensor& t) { return t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous); };
    const bool rows = T == 0 || (qkv.stride(1) == 1 && qkv.stride(0) % 8 == 0 && qkv.stride(0) >= 0 && (uintptr_t)qkv.data_ptr() % 16 == 0);
    const Tensor x = rows ? qkv : qkv.clone(at::MemoryFormat::Contiguous);
    Tensor wn[2];
    const c10::optional<Tensor>* given[2] = {&q_norm, &k_norm};
    for (int i = 0; i < 2; ++i)
        if (given[i]->has_value()) {
            const Tensor& t = **given[i];
            on(t, k, i ? "k_norm" : "q_norm");
            CHK(t.scalar_type() == at::kBFloat16 && t.dim() == 1 && t.numel() == D, i ? "k_norm" : "q_norm", " must be bfloat16 [D]");
            wn[i] = flat(t);
        }
    auto out = at::empty({T, hq, D}, qkv.options());
    chronos::qkv::launch_norm_rope_kv_quant(c.kind, c.D, bf(x), x.stride(0), pp, sp, block_table.data_ptr<int32_t>(), block_table.stride(0), (int)block_table.size(0),
                                            (int)block_table.size(1), cos_sin.data_ptr<float>(), (int)R, (int)cos_sin.size(0), wn[0].defined() ? bf(wn[0]) : nullptr,
                                            wn[1].defined() ? bf(wn[1]) : nullptr, eps, bfm(out), c.c, T, (int)hq, cur_stream());
    return out;
}

std::tuple<Tensor, Tensor> quant_kv_read(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& block_table, const Tensor& pos,
                                         const Tensor& tok_seq) {
    const Held c = held(k, v, ks, vs);
    CHK(pos.dim() == 1 && tok_seq.dim() == 1 && tok_seq.numel() == pos.numel() && pos.numel() < kMost, "pos and tok_seq need an entry per token");
    const int64_t T = pos.numel();
    const int32_t *pp = ints(pos, k, T, "pos"), *sp = ints(tok_seq, k, T, "tok_seq");
    table(block_table, k);
    c10::hip::HIPGuardMasqueradingAsCUDA g(k.device());
    auto ko = at::empty({T, c.c.heads, c.D}, k.options().dtype(at::kBFloat16)), vo = at::empty_like(ko);
    chronos::qkv::launch_quant_kv_read(c.kind, c.D, pp, sp, block_table.data_ptr<int32_t>(), block_table.stride(0), (int)block_table.size(0), (int)block_table.size(1), c.c,
                                       bfm(ko), bfm(vo), T, cur_stream());
    return {ko, vo};
}

Tensor quant_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& block_table, const Tensor& ctx_len,
                       const c10::optional<Tensor>& q_start, const c10::optional<Tensor>& group_start, const c10::optional<Tensor>& prefix_len, double scale, int64_t max_ctx) {
    const Held c = held(k, v, ks, vs);
    const int64_t D = c.D, heads = c.c.heads;
    on(q, k, "q");
    CHK(q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.size(2) == D, "q must be bfloat16 [T, hq, ", D, "]");
    const int64_t T = q.size(0), hq = q.size(1);
    CHK(hq > 0 && hq < 65536 && hq % heads == 0, "q heads (", hq, ") must be a multiple of the cache's (", heads, ")");
    CHK(T < kMost && T * hq < kMost, "too many tokens");
    table(block_table, k);
    const int64_t B = ctx_len.numel();
    const int32_t* cp = ints(ctx_len, k, 0, "ctx_len");
    CHK(block_table.size(0) >= B, "block_table needs a row per sequence");
    const int32_t* qs = nullptr;
    if (q_start.has_value()) qs = ints(*q_start, k, B + 1, "q_start");
    else CHK(T >= B, "without q_start every sequence has a token: q needs ", B, " rows, has ", T);
    CHK(group_start.has_value() == prefix_len.has_value(), "group_start and prefix_len go together");
    int64_t groups = 0;
    const int32_t *gs = nullptr, *pl = nullptr;
    if (group_start.has_value()) {
        groups = prefix_len->numel();
        pl = ints(*prefix_len, k, 0, "prefix_len");
        gs = ints(*group_start, k, groups + 1, "group_start");
        CHK(groups < kMost, "too many groups");
    }
    const int64_t keys = block_table.size(1) * c.c.page;
    CHK(keys < kMost, "block_table is too wide");
    c10::hip::HIPGuardMasqueradingAsCUDA g(k.device());
    if (T == 0 || B == 0 || keys == 0) return at::zeros({T, hq, D}, q.options());
    const auto p = chronos::qkv::quant_attention_plan((int)T, (int)B, qs == nullptr, (int)groups, (int)hq, (int)heads, max_ctx > 0 && max_ctx < keys ? max_ctx : keys);
    // a launch has fewer than 2^32 threads: up to 512 a tile and head, and 32 a row of the one that joins
    CHK(std::max(p.own_tiles, p.group_tiles) * heads < (1 << 23) && T * hq < (1 << 27), "too many tokens or sequences for one call");
    auto out = at::empty({T, hq, D}, q.options());
    const bool rows = q.stride(2) == 1 && q.stride(1) == D && q.stride(0) % 8 == 0 && q.stride(0) >= 0 && (uintptr_t)q.data_ptr() % 16 == 0;
    const Tensor x = rows ? q : q.clone(at::MemoryFormat::Contiguous);
    Tensor po, pm;
    if (p.slots > 1) {
        po = at::empty({p.slots, T * hq, D}, q.options().dtype(at::kFloat));
        pm = at::empty({p.slots, T * hq}, q.options().dtype(at::kFloat));
    }
    chronos::qkv::launch_quant_attention(c.kind, c.D, p, bf(x), x.stride(0), c.c, block_table.data_ptr<int32_t>(), block_table.stride(0), (int)block_table.size(1), qs, cp,
                                         gs, pl, (int)B, (int)T, (int)groups, (int)hq, (float)scale, bfm(out), p.slots > 1 ? po.data_ptr<float>() : nullptr,
                                         p.slots > 1 ? pm.data_ptr<float>() : nullptr, cur_stream());
    return out;
}

// How quant_attention cuts a call up: rows of a tile of the sequences' own keys, pieces of those keys, rows and pieces of what groups share, and whether the own keys' launch joins the groups'
// pieces and whether it takes its longest tiles first.  single: no q_start; keys: the table's width in keys, or max_ctx.
std::vector<int64_t> quant_attention_plan(int64_t T, int64_t B, bool single, int64_t groups, int64_t hq, int64_t heads, int64_t keys) {
    CHK(T > 0 && T < kMost && B > 0 && B < kMost && groups >= 0 && groups < kMost && keys > 0 && keys < kMost, "a plan needs tokens, sequences and keys");
    CHK(heads > 0 && hq > 0 && hq < 65536 && hq % heads == 0, "q heads (", hq, ") must be a multiple of the cache's (", heads, ")");
    const auto p = chronos::qkv::quant_attention_plan((int)T, (int)B, single, (int)groups, (int)hq, (int)heads, keys);
    return {p.own_rows, p.own_splits, p.group_rows, p.group_splits, p.last, p.longest};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(chronos, m) {
    m.def("norm_rope_kv_quant(Tensor qkv, Tensor pos, Tensor tok_seq, Tensor block_table, Tensor cos_sin, Tensor(a!) k, Tensor(b!) v, Tensor(c!) ks, Tensor(d!) vs, "
          "int hq, Tensor? q_norm, Tensor? k_norm, float eps) -> Tensor");
    m.def("quant_kv_read(Tensor k, Tensor v, Tensor ks, Tensor vs, Tensor block_table, Tensor pos, Tensor tok_seq) -> (Tensor, Tensor)");
    m.def("quant_attention(Tensor q, Tensor k, Tensor v, Tensor ks, Tensor vs, Tensor block_table, Tensor ctx_len, Tensor? q_start, Tensor? group_start, "
          "Tensor? prefix_len, float scale, int max_ctx=-1) -> Tensor");
    m.def("quant_attention_plan(int T, int B, bool single, int groups, int hq, int heads, int keys) -> int[]", &quant_attention_plan);
}

TORCH_LIBRARY_IMPL(chronos, CUDA, m) {
    m.impl("norm_rope_kv_quant", &norm_rope_kv_quant);
    m.impl("quant_kv_read", &quant_kv_read);
    m.impl("quant_attention", &quant_attention);
}
