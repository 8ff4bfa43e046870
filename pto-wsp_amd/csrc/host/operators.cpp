#include "operators_shared.hpp"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <map>
#include <stdexcept>

#include "../device/ptowsp_paged_args.h"

namespace ptowsp {

namespace {

constexpr int kPlanThreads = 1024, kPlanBatch = 4096;  // one workgroup's threads and requests

const std::vector<Spec>& specs() {
    static const std::vector<Spec> all = {
        {"paged_plan",
         {{"lengths", kIndex, 1, false, false}, {"counts", kIndex, 1, false, false}, {"page_table", kIndex, 2, true, false},
          {"free_pages", kIndex, 1, false, false}, {"used", kIndex, 1, false, false}, {"new_lengths", kIndex, 1, true, false},
          {"new_used", kIndex, 1, true, false}, {"starts", kIndex, 1, true, false}, {"slots", kIndex, 1, true, false}}},
        {"paged_store",
         {{"k", kReal, 3, false, false}, {"v", kReal, 3, false, false}, {"slots", kIndex, 1, false, false},
          {"k_cache", kCode, 4, true, false}, {"v_cache", kCode, 4, true, false}, {"k_scale", kScale, 2, true, false},
          {"v_scale", kScale, 2, true, false}}},
        {"paged_attention",
         {{"q", kReal, 3, false, false}, {"k_cache", kCode, 4, false, false}, {"v_cache", kCode, 4, false, false},
          {"k_scale", kScale, 2, false, false}, {"v_scale", kScale, 2, false, false}, {"page_table", kIndex, 2, false, false},
          {"lengths", kIndex, 1, false, false}, {"starts", kIndex, 1, false, false}, {"out", kReal, 3, true, false},
          {"lse", kScale, 2, true, true}}},
        {"paged_prefix_attention",
         {{"q", kReal, 3, false, false}, {"k_cache", kCode, 4, false, false}, {"v_cache", kCode, 4, false, false},
          {"k_scale", kScale, 2, false, false}, {"v_scale", kScale, 2, false, false}, {"page_table", kIndex, 2, false, false},
          {"lengths", kIndex, 1, false, false}, {"starts", kIndex, 1, false, false}, {"prefix_table", kIndex, 2, false, false},
          {"prefix_lengths", kIndex, 1, false, false}, {"members", kIndex, 1, false, false}, {"out", kReal, 3, true, false},
          {"lse", kScale, 2, true, true}}}};
    return all;
}

const Spec& spec_of(const Node& n) {
    for (const std::vector<Spec>* all : {&specs(), &block_specs()})
        for (const Spec& s : *all)
            if (n.op == s.op) return s;
    throw CompileError("unknown operator '" + n.op + "'");
}

Shapes shapes_of(const Module& m, const Node& n) {
    const Spec& spec = spec_of(n);
    Shapes r{n, spec, {}, {}};
    size_t next = 0;
    for (const Param& p : spec.params) {
        if (next >= n.tensor_args.size() || n.tensor_args[next].param != p.name) {
            if (!p.optional) refuse(n, std::string("missing operand ") + p.name);
            r.shape.push_back({});
            r.dtype.push_back(DType::F32);
            continue;
        }
        const TensorArg& t = n.tensor_args[next++];
        const TensorInfo& ti = m.tensors[t.tid];
        if (t.idx.size() > ti.shape.size()) refuse(n, std::string("too many indices into ") + p.name);
        std::vector<int64_t> s(ti.shape.begin() + static_cast<std::ptrdiff_t>(t.idx.size()), ti.shape.end());
        if (static_cast<int>(s.size()) != p.rank)
            refuse(n, std::string(p.name) + " has the shape " + shape_text(s) + ", rank " + std::to_string(p.rank) + " is needed");
        const DType d = ti.dtype;
        const bool ok = p.group == kIndex       ? d == DType::I32
                        : p.group == kScale     ? d == DType::F32
                        : p.group == kCode      ? d == DType::I8 || d == DType::F8E4M3
                        : p.group == kE4M3Code  ? d == DType::F8E4M3
                                                : d == DType::BF16 || d == DType::F16 || d == DType::F32;
        if (!ok) refuse(n, std::string(p.name) + " has the unsupported type " + dtype_name(d));
        r.shape.push_back(std::move(s));
        r.dtype.push_back(d);
    }
    if (next != n.tensor_args.size()) refuse(n, "unknown operand " + n.tensor_args[next].param);
    return r;
}

// The cache's tensors agree with each other: [P, H, page, D] and [P, H].
void check_cache(const Shapes& s) {
    const auto& c = s.of("k_cache");
    const int64_t P = c[0], H = c[1], page = c[2], D = c[3];
    s.want("v_cache", c);
    s.same_type("k_cache", "v_cache");
    s.want("k_scale", {P, H});
    s.want("v_scale", {P, H});
    if (P < 1 || P > (int64_t(1) << 31) - 1) refuse(s.n, "a cache of " + std::to_string(P) + " pages");
    if (H < 1 || H > 65536) refuse(s.n, std::to_string(H) + " key heads");
    if (page < 1 || page > 4096) refuse(s.n, "pages of " + std::to_string(page) + " tokens (1 to 4096 are supported)");
    if (D < 16 || D > 256 || D % 16) refuse(s.n, "head size " + std::to_string(D) + " (a multiple of 16 up to 256 is needed)");
}

std::string entry_source(const std::string& entries) { return "#include \"ptowsp_paged.h\"\n" + entries; }

// ---- paged_plan ----
// One workgroup does it all while its LDS holds the requests' sums and the
// rows are few; otherwise one sums and as many as needed write the rows.  64
// requests, one launch or two: 1024 rows 6.6 us and 12.9, 6144 rows 11.7 and 12.6,
// 8192 rows 14.2 and 12.6.
constexpr int64_t kPlanOneRows = 6144;

std::string plan_source() {
    const std::string t = std::to_string(kPlanThreads);
    return entry_source("extern \"C\" __global__ __launch_bounds__(" + t + ") void ptowsp_paged_plan(ptowsp::PlanArgs A) { ptowsp::plan_one<" + t + ", " +
                        std::to_string(kPlanBatch) + ">(A); }\n"
                        "extern \"C\" __global__ __launch_bounds__(" + t + ") void ptowsp_paged_plan_sums(ptowsp::PlanArgs A) { ptowsp::plan_sums<" + t +
                        ">(A); }\n"
                        "extern \"C\" __global__ __launch_bounds__(256) void ptowsp_paged_plan_rows(ptowsp::PlanArgs A) { ptowsp::plan_rows<256>(A); }\n");
}

void run_plan(const Node& n, const std::vector<Operand>& o, const OperatorRun& run) {
    static const std::string source = plan_source();
    PlanArgs A{};
    auto ints = [&](size_t i) { return reinterpret_cast<int*>(o[i].ptr); };
    A.lengths = ints(0), A.s_lengths = o[0].stride[0];
    A.counts = ints(1), A.s_counts = o[1].stride[0];
    A.table = ints(2), A.s_table = o[2].stride[0], A.s_table_col = o[2].stride[1];
    A.free_pages = ints(3), A.s_free = o[3].stride[0];
    A.used = ints(4);
    A.new_lengths = ints(5), A.s_new_lengths = o[5].stride[0];
    A.new_used = ints(6);
    A.starts = ints(7), A.s_starts = o[7].stride[0];
    A.slots = ints(8), A.s_slots = o[8].stride[0];
    A.batch = o[0].shape[0], A.width = o[2].shape[1], A.nfree = o[3].shape[0], A.rows = o[8].shape[0];
    A.page = static_cast<int>(attr(n, "page_size"));
    A.err = run.err;
    if (A.batch <= kPlanBatch && A.rows <= kPlanOneRows) {
        run.launch(source, "ptowsp_paged_plan", 1, kPlanThreads, &A, sizeof A);
        return;
    }
    A.scratch = reinterpret_cast<int*>(run.scratch(sizeof(int) * static_cast<size_t>(2 + 3 * A.batch)));
    run.launch(source, "ptowsp_paged_plan_sums", 1, kPlanThreads, &A, sizeof A);
    if (A.rows > 0) run.launch(source, "ptowsp_paged_plan_rows", (A.rows + kPlanRows - 1) / kPlanRows, 256, &A, sizeof A);
}

// ---- the cache's operands ----
void cache_strides(const Node& n, const Operand& codes, const Operand& scales, long long (&s_cache)[3], long long (&s_scale)[2]) {
    const char* who = "the cache";
    if (codes.stride[3] != 1) stop(n, std::string(who) + "'s last dimension must have stride 1");
    for (int d = 0; d < 3; ++d)
        if (codes.stride[d] % 16) stop(n, std::string(who) + "'s strides must be multiples of 16");
    if (reinterpret_cast<uintptr_t>(codes.ptr) % 16) stop(n, std::string(who) + " must be aligned to 16 bytes");
    if (codes.shape[0] > 1 && (codes.stride[0] >> 32 || scales.stride[0] >> 32)) stop(n, std::string(who) + "'s pages lie too far apart");
    if (codes.stride[2] > (int64_t(1) << 26)) stop(n, std::string(who) + "'s tokens lie too far apart");
    for (int d = 0; d < 3; ++d) s_cache[d] = codes.stride[d];
    for (int d = 0; d < 2; ++d) s_scale[d] = scales.stride[d];
}

// Rows of 16-byte pieces: unit stride, aligned.
bool vectors(const Operand& x) {
    const int64_t piece = 16 / dtype_size(x.dtype);
    return x.stride[0] % piece == 0 && x.stride[1] % piece == 0 && reinterpret_cast<uintptr_t>(x.ptr) % 16 == 0;
}

// ---- paged_store ----
std::string store_source(int D, int page, int type, int code, bool vec, int chunk) {
    return entry_source("extern \"C\" __global__ __launch_bounds__(256) void ptowsp_paged_store(ptowsp::StoreArgs A) { ptowsp::store_rows<" +
                        std::to_string(D) + ", " + std::to_string(page) + ", " + std::to_string(type) + ", " + std::to_string(code) + ", " + flag(vec) +
                        ", " + std::to_string(chunk) + ">(A); }\n");
}

// Rows of a wave: one while the waves are few (every row of a decode step has
// a page of its own), a page's worth otherwise (a prompt's rows of a page go
// together, and waves without a first row end at once).  8 heads of 128 in bf16,
// one row a wave or a page's: 64 single tokens 5.2 us and 27.9, 1024 13.6 and 27.6,
// 4096 51.5 and 45.9; a prompt of 256 tokens 6.1 and 6.8, of 1024 10.4 and 7.2, of
// 2048 16.1 and 7.4.
int store_chunk(int64_t rows, int64_t heads, int64_t page) { return rows * heads * 2 <= 16384 ? 1 : static_cast<int>(std::min<int64_t>(page, 64)); }

void run_store(const Node& n, const std::vector<Operand>& o, const OperatorRun& run) {
    StoreArgs A{};
    const int64_t rows = o[0].shape[0], heads = o[3].shape[1], page = o[3].shape[2], D = o[3].shape[3];
    for (int i = 0; i < 2; ++i) {
        if (o[i].stride[2] != 1) stop(n, std::string(i ? "v" : "k") + "'s last dimension must have stride 1");
        A.x[i] = o[i].ptr;
        A.s_x[i][0] = o[i].stride[0], A.s_x[i][1] = o[i].stride[1];
        A.cache[i] = o[3 + i].ptr;
        A.scale[i] = reinterpret_cast<float*>(o[5 + i].ptr);
        cache_strides(n, o[3 + i], o[5 + i], A.s_cache[i], A.s_scale[i]);
    }
    A.slots = reinterpret_cast<const int*>(o[2].ptr);
    A.s_slots = o[2].stride[0];
    A.rows = rows, A.pages = o[3].shape[0];
    A.err = run.err;
    A.heads = static_cast<int>(heads);
    if (rows == 0) return;
    const int chunk = store_chunk(rows, heads, page);
    const int64_t waves = (rows + chunk - 1) / chunk * heads * 2, blocks = (waves + 3) / 4;
    if (blocks >= (int64_t(1) << 24)) stop(n, "too many rows for one call");
    const std::string source = store_source(static_cast<int>(D), static_cast<int>(page), type_id(o[0].dtype), code_id(o[3].dtype),
                                            vectors(o[0]) && vectors(o[1]), chunk);
    run.launch(source, "ptowsp_paged_store", blocks, 256, &A, sizeof A);
}

// ---- paged_attention ----
struct AttendShape {
    int D, page, G, NT, type, code;
    bool window, lse, vec;
    int part;  // 0: paged_attention; of paged_prefix_attention 1: own tokens, 2: prefixes
};
std::string attend_type(const AttendShape& s, int nt, bool prompt) {
    auto num = [](int v) { return std::to_string(v); };
    return "ptowsp::Attend<" + num(s.D) + ", " + num(s.page) + ", " + num(s.G) + ", " + num(nt) + ", " + num(s.type) + ", " + num(s.code) + ", " +
           flag(s.window) + ", " + flag(s.lse) + ", " + flag(s.vec) + ", " + flag(prompt) + (s.part ? ", " + num(s.part) : "") + ">";
}
// Waves on a SIMD that the registers allow: 32 requests over 4096 tokens of head
// size 256 take 101 us with one and 197, spilling, with two.
int attend_waves(int64_t D) { return D > 128 ? 1 : 2; }
// Prompts: 16 * nt query rows a wave, `waves` waves on a SIMD.
struct PromptShape {
    int nt, waves;
};
PromptShape prompt_shape(const AttendShape& s) {
    return s.type != 2 && s.D <= 128 && s.page % 16 == 0 ? PromptShape{2, 2} : PromptShape{1, attend_waves(s.D)};
}
std::string attend_source(const AttendShape& s, bool prompts) {
    const std::string t = attend_type(s, s.NT, false), w = std::to_string(attend_waves(s.D));
    auto entry = [](const char* bounds, const char* name, const std::string& body) {
        return std::string("extern \"C\" __global__ __launch_bounds__(") + bounds + ") void ptowsp_paged_attention" + name + "(ptowsp::AttendArgs A) { " + body + "; }\n";
    };
    const std::string bounds = "256, " + w;
    if (!prompts) return entry_source(entry(bounds.c_str(), "", "__shared__ " + t + "::Shared lds; " + t + "::run(A, blockIdx.x, lds)") + entry("256", "_join", t + "::join(A)"));
    const std::string u = attend_type(s, prompt_shape(s).nt, true);
    return entry_source(entry("1024", "_units", u + "::list_units<1024>(A)") + entry(bounds.c_str(), "_prompts", u + "::both<" + t + ">(A)") +
                        entry(bounds.c_str(), "_finish", u + "::finish<" + t + ">(A)"));
}

// Query rows of a request and key head up to which its keys are streamed by
// all compute units alike (the kernel for few rows), and beyond which rows
// share them; and query rows of a call up to which none are shared, since they
// give the prompt kernel too few workgroups.  Groups of 4 x 8 key heads of 128 in
// bf16, few rows or prompts: 64 requests of 8 tokens 39 us and 60, of 16 tokens (64
// rows) 66 and 63, of 32 tokens 120 and 69; one prompt of 256 tokens (8192 rows in
// the call) 43 and 58, of 1024 98 and 94; two of 64 tokens over 16384 99 and 145, of
// 128 169 and 148.
constexpr int kFewRows = 64;
constexpr int64_t kFewInAll = 8192;

// 16 query rows at a time, or 32 where many read the same keys and the registers
// suffice (not for float32: 32 query heads 54 us, with 32 at a time 87).  bf16, 16
// requests over 2048 tokens: 32 rows of a key head 34 us, with 32 at a time 39; 64
// rows 48 and 46 (two requests over 16384 tokens 43 and 62); 128 rows 82 and 58; 32
// query heads of single tokens over 4096 52 and 43.
int attend_nt(int64_t rows, int64_t batch, int64_t G, int64_t D, int type) {
    const int64_t each = G * std::max<int64_t>(1, (rows + batch - 1) / std::max<int64_t>(1, batch));
    return type != 2 && D <= 128 && (G > 16 || each > 64) ? 2 : 1;
}

// The kernels of a call: of q [rows, q_heads, D] over the cache's [heads, page, D].
struct AttendForm {
    AttendShape s;
    bool prompts;  // requests of more than `few` tokens go to the kernel for prompts
    int few;
};
AttendForm attend_form(const std::vector<int64_t>& q, const std::vector<int64_t>& cache, int64_t batch, DType type, DType code, bool window, bool lse, bool vec,
                       int part = 0) {
    const int64_t rows = q[0], D = q[2];
    AttendForm f;
    f.s = AttendShape{static_cast<int>(D), static_cast<int>(cache[2]), static_cast<int>(q[1] / cache[1]), 1, type_id(type), code_id(code), window, lse, vec, part};
    f.few = std::max(1, kFewRows / f.s.G);
    // Launched if there can be such a request while every other one has a token.
    f.prompts = part == 2 ? rows > f.few : rows - batch >= f.few && rows * q[1] > kFewInAll;
    f.s.NT = attend_nt(f.prompts ? batch : rows, batch, f.s.G, D, f.s.type);
    return f;
}

// The operands of attention that its calls have alike.
AttendArgs attend_args(const Node& n, const std::vector<Operand>& o, const Operand& out, const OperatorRun& run) {
    AttendArgs A{};
    const Operand& q = o[0];
    if (q.stride[2] != 1 || out.stride[2] != 1) stop(n, "q's and out's last dimensions must have stride 1");
    A.q = q.ptr, A.out = out.ptr;
    for (int d = 0; d < 2; ++d) A.s_q[d] = q.stride[d], A.s_out[d] = out.stride[d];
    for (int i = 0; i < 2; ++i) {
        A.cache[i] = o[1 + i].ptr;
        A.scale[i] = reinterpret_cast<const float*>(o[3 + i].ptr);
        cache_strides(n, o[1 + i], o[3 + i], A.s_cache[i], A.s_scale[i]);
    }
    if (o[5].shape[1] > 1 && o[5].stride[1] != 1) stop(n, "page_table's last dimension must have stride 1");
    A.table = reinterpret_cast<const int*>(o[5].ptr), A.s_table = o[5].stride[0];
    A.lengths = reinterpret_cast<const int*>(o[6].ptr), A.s_lengths = o[6].stride[0];
    A.starts = reinterpret_cast<const int*>(o[7].ptr), A.s_starts = o[7].stride[0];
    A.batch = o[6].shape[0], A.width = o[5].shape[1], A.pages = std::min<int64_t>(o[1].shape[0], int64_t(1) << 31), A.rows = q.shape[0];
    A.heads = static_cast<int>(o[1].shape[1]);
    A.factor = static_cast<float>(n.op_floats.at("scale") * 1.4426950408889634);
    A.err = run.err;
    return A;
}

size_t whole(int64_t bytes) { return (static_cast<size_t>(bytes) + 255) / 256 * 256; }

// The workspace that a form's kernels need, and its places in it.
struct AttendSpace {
    size_t spans, few, units, need;  // bytes before the partial results of few rows, the units, the units' partial results; in all
};
AttendSpace attend_space(const Node& n, const AttendForm& form, AttendArgs& A, int cus) {
    const AttendShape& s = form.s;
    A.few = form.prompts ? form.few : 0x7FFFFFFF;
    const int rb = 16 * s.NT, dp = (s.D + 63) / 64 * 64;
    const int64_t blocks = attend_waves(s.D) * static_cast<int64_t>(cus);
    A.blocks = static_cast<int>(blocks);
    AttendSpace r{};
    r.spans = whole(blocks * kSpanInts * 4);
    r.few = r.spans + whole(2 * blocks * rb * (2 + dp) * 4);
    r.units = r.need = r.few;
    if (form.prompts) {
        // Units, pieces and partial results as list_units makes them, at most.
        const PromptShape p = prompt_shape(s);
        const int prb = 16 * p.nt, c = s.G <= prb ? prb / s.G : 1, hs = s.G <= prb ? 1 : (s.G + prb - 1) / prb;
        A.cus = cus * p.waves;
        if (s.part == 2) {
            // Pieces of units in several, as line() makes them: A.cus, or twice what 4 / 3 of them share.
            A.room = 8 * A.cus / 3 + 1;
            r.need = r.units + whole(static_cast<int64_t>(A.room) * 4 * prb * (2 + dp) * 4);
            return r;
        }
        const int64_t entries = hs * (A.rows / (4 * c) + std::min<int64_t>(A.batch, A.rows / (A.few + 1))) + A.cus / A.heads + 1;
        if (entries * A.heads >= (int64_t(1) << 24)) stop(n, "too many rows for one call");
        A.room = static_cast<int>(entries), A.counters = 2 * A.cus;
        r.units += whole((kUnitHead + entries * (kUnitInts + A.heads) + A.counters + A.cus / A.heads + 1) * 4);
        r.need = r.units + whole(int64_t(2) * A.cus * 4 * prb * (2 + dp) * 4);
    }
    return r;
}
void attend_place(const AttendSpace& space, char* scratch, AttendArgs& A) {
    A.spans = reinterpret_cast<int*>(scratch);
    A.parts = reinterpret_cast<float*>(scratch + space.spans);
    A.units = reinterpret_cast<int*>(scratch + space.few);
    A.unit_parts = reinterpret_cast<float*>(scratch + space.units);
}
void attend_launch(const AttendForm& form, const AttendSpace& space, char* scratch, AttendArgs& A, const OperatorRun& run) {
    attend_place(space, scratch, A);
    const std::string source = attend_source(form.s, form.prompts);
    if (form.prompts) {
        run.launch(source, "ptowsp_paged_attention_units", 1, 1024, &A, sizeof A);
        run.launch(source, "ptowsp_paged_attention_prompts", static_cast<int64_t>(A.room) * A.heads + A.blocks, 256, &A, sizeof A);
        run.launch(source, "ptowsp_paged_attention_finish", A.blocks, 256, &A, sizeof A);
    } else {
        run.launch(source, "ptowsp_paged_attention", A.blocks, 256, &A, sizeof A);
        run.launch(source, "ptowsp_paged_attention_join", A.blocks, 256, &A, sizeof A);
    }
}

void run_attend(const Node& n, const std::vector<Operand>& o, const OperatorRun& run) {
    const Operand &q = o[0], &out = o[8];
    const bool lse = o.size() > 9 && o[9].shape.size() == 2;
    AttendArgs A = attend_args(n, o, out, run);
    if (lse) {
        A.lse = reinterpret_cast<float*>(o[9].ptr);
        for (int d = 0; d < 2; ++d) A.s_lse[d] = o[9].stride[d];
    }
    A.window = static_cast<int>(std::min<int64_t>(attr(n, "window"), 0x7FFFFFFF));
    if (A.rows == 0 || A.batch == 0) return;
    const AttendForm form = attend_form(q.shape, o[1].shape, A.batch, q.dtype, o[1].dtype, A.window > 0, lse, vectors(q) && vectors(out));
    const AttendSpace space = attend_space(n, form, A, run.cus);
    attend_launch(form, space, run.scratch(space.need), A, run);
}

// ---- paged_prefix_attention ----
// own: the requests' own tokens; shared: the groups' prefixes.
std::string prefix_source(const AttendForm& own, const AttendForm& shared, int type, bool lse) {
    const std::string w = std::to_string(attend_waves(own.s.D)), bounds = "256, " + w;
    const std::string lp = attend_type(shared.s, prompt_shape(shared.s).nt, true), fp = attend_type(shared.s, shared.s.NT, false);
    const std::string uo = attend_type(own.s, prompt_shape(own.s).nt, true), fo = attend_type(own.s, own.s.NT, false);
    auto entry_of = [](const std::string& bounds, const char* name, const char* args, const std::string& body) {
        return "extern \"C\" __global__ __launch_bounds__(" + bounds + ") void ptowsp_paged_prefix" + name + "(ptowsp::" + args + " A) { " + body + "; }\n";
    };
    std::string source = entry_source(entry_of(bounds, "_parts", "PrefixArgs", "ptowsp::prefix_parts<" + lp + ", " + fp + ", " + fo + ", " + uo + ", " + flag(shared.prompts) + ", " + flag(own.prompts) + ">(A)"));
    source += entry_of("256", "_merge", "PrefixArgs", "ptowsp::merge_parts<" + std::to_string(own.s.D) + ", " + fp + "::RB, " + lp + "::RB, " + fo + "::RB, " + std::to_string(type) + ", " + flag(lse) + ">(A)");
    if (own.prompts) source += entry_of("1024", "_units", "AttendArgs", uo + "::list_units<1024>(A)") + entry_of(bounds, "_finish", "AttendArgs", uo + "::finish<" + fo + ">(A)");
    return source;
}

void run_prefix(const Node& n, const std::vector<Operand>& o, const OperatorRun& run) {
    const Operand &q = o[0], &table = o[8], &lengths = o[9], &members = o[10], &out = o[11];
    const bool lse = o.size() > 12 && o[12].shape.size() == 2;
    PrefixArgs P{};
    AttendArgs &own = P.own, &shared = P.shared;
    own = attend_args(n, o, out, run);
    shared = own;
    if (table.shape[1] > 1 && table.stride[1] != 1) stop(n, "prefix_table's last dimension must have stride 1");
    shared.table = reinterpret_cast<const int*>(table.ptr), shared.s_table = table.stride[0], shared.width = table.shape[1];
    shared.lengths = reinterpret_cast<const int*>(lengths.ptr), shared.s_lengths = lengths.stride[0], shared.batch = table.shape[0];
    shared.members = reinterpret_cast<const int*>(members.ptr), shared.s_members = members.stride[0];
    shared.requests = static_cast<int>(own.batch);
    if (own.rows == 0 || own.batch == 0) return;
    const int64_t heads = q.shape[1], D = q.shape[2], all = own.rows * heads;
    const AttendForm mine = attend_form(q.shape, o[1].shape, own.batch, q.dtype, o[1].dtype, false, true, vectors(q), 1);
    const AttendForm theirs = attend_form(q.shape, o[1].shape, shared.batch, q.dtype, o[1].dtype, false, true, vectors(q), 2);
    const AttendSpace spaces[2] = {attend_space(n, mine, own, run.cus), attend_space(n, theirs, shared, run.cus)};
    // Both parts' results, [row, head, D], and their entries, [row, head, 4].
    const size_t part_bytes = whole(all * D * 4), entry_bytes = whole(all * 16);
    char* at = run.scratch(2 * (part_bytes + entry_bytes) + spaces[0].need + spaces[1].need);
    for (int i = 0; i < 2; ++i) {
        AttendArgs& A = i ? shared : own;
        A.out = at;
        A.s_out[0] = heads * D, A.s_out[1] = D;
        A.lse = reinterpret_cast<float*>(at + part_bytes);
        A.s_lse[0] = 4 * heads, A.s_lse[1] = 4;
        attend_place(spaces[i], at + part_bytes + entry_bytes, A);
        at += part_bytes + entry_bytes + spaces[i].need;
    }
    const int few_prefixes = shared.batch > 0 ? shared.blocks : 0;  // workgroups for prefixes of few rows
    const bool line = theirs.prompts && shared.batch > 0;
    if (line) {
        // Pieces, at most: line_limit() makes no more than A.cus of few units.
        const int prb = 16 * prompt_shape(theirs.s).nt, c = theirs.s.G <= prb ? prb / theirs.s.G : 1, hs = theirs.s.G <= prb ? 1 : (theirs.s.G + prb - 1) / prb;
        const int64_t units = hs * (own.rows / (4 * c) + std::min<int64_t>(shared.batch, own.rows / (shared.few + 1))) * shared.heads;
        if (units >= (int64_t(1) << 22)) stop(n, "too many rows for one call");
        P.lines = 2 * units <= shared.cus ? shared.cus : static_cast<int>(units) + shared.cus + shared.cus / 3;
    }
    P.q_heads = static_cast<int>(heads);
    P.out = out.ptr;
    for (int d = 0; d < 2; ++d) P.s_out[d] = out.stride[d];
    if (lse) {
        P.lse = reinterpret_cast<float*>(o[12].ptr);
        for (int d = 0; d < 2; ++d) P.s_lse[d] = o[12].stride[d];
    }
    const int lanes = D <= 64 ? 16 : D <= 128 ? 32 : 64;
    const int64_t groups = (all * lanes + 255) / 256;
    if (groups >= (int64_t(1) << 24)) stop(n, "too many rows for one call");
    AttendForm shared_form = theirs;
    shared_form.prompts = line;
    const std::string source = prefix_source(mine, shared_form, type_id(q.dtype), lse);
    if (mine.prompts) run.launch(source, "ptowsp_paged_prefix_units", 1, 1024, &own, sizeof own);
    const int64_t prompts = mine.prompts ? static_cast<int64_t>(own.room) * own.heads : 0;
    run.launch(source, "ptowsp_paged_prefix_parts", P.lines + few_prefixes + own.blocks + prompts, 256, &P, sizeof P);
    if (mine.prompts) run.launch(source, "ptowsp_paged_prefix_finish", own.blocks, 256, &own, sizeof own);
    run.launch(source, "ptowsp_paged_prefix_merge", groups, 256, &P, sizeof P);
}

// ---- operands that share memory ----
// Multiples x of `step` bytes, lo <= x <= hi.
struct Term {
    int64_t step, lo, hi;
};

// Whether base + the sum of the terms can lie between `above` and `below`, both
// exclusive.  Terms by descending step: each is left with the few multiples that
// the smaller ones can make up for.  Strides that leave it many run out of `tries`
// and count as a hit.
bool reaches(const std::vector<Term>& t, size_t k, int64_t base, int64_t above, int64_t below, int& tries) {
    if (--tries < 0) return true;
    if (k == t.size()) return base > above && base < below;
    int64_t least = 0, most = 0;  // of the terms behind this one
    for (size_t i = k + 1; i < t.size(); ++i) least += t[i].step * t[i].lo, most += t[i].step * t[i].hi;
    auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
    const int64_t lo = std::max(t[k].lo, floor_div(above - base - most, t[k].step) + 1);
    const int64_t hi = std::min(t[k].hi, -floor_div(-(below - base - least), t[k].step) - 1);
    for (int64_t x = lo; x <= hi; ++x)
        if (reaches(t, k + 1, base + t[k].step * x, above, below, tries)) return true;
    return false;
}
bool reaches(std::vector<Term> t, int64_t base, int64_t above, int64_t below) {
    std::sort(t.begin(), t.end(), [](const Term& a, const Term& b) { return a.step > b.step; });
    std::vector<Term> merged;
    for (const Term& x : t) {
        if (!merged.empty() && merged.back().step == x.step) merged.back().lo += x.lo, merged.back().hi += x.hi;
        else merged.push_back(x);
    }
    int tries = 1 << 16;
    return reaches(merged, 0, base, above, below, tries);
}

int64_t extent(const Operand& o) {  // bytes from the first element to the end of the last
    int64_t e = 1;
    for (size_t d = 0; d < o.shape.size(); ++d) {
        if (o.shape[d] == 0) return 0;
        e += (o.shape[d] - 1) * o.stride[d];
    }
    return e * dtype_size(o.dtype);
}

// Whether some byte belongs to an element of each.
bool meet(const Operand& a, const Operand& b) {
    const int64_t ea = extent(a), eb = extent(b), base = b.ptr - a.ptr;
    if (!ea || !eb || base >= ea || base <= -eb) return false;
    std::vector<Term> t;
    for (const Operand* o : {&a, &b})
        for (size_t d = 0; d < o->shape.size(); ++d)
            if (o->shape[d] > 1 && o->stride[d] > 0) {
                const int64_t step = o->stride[d] * dtype_size(o->dtype), n = o->shape[d] - 1;
                t.push_back(o == &a ? Term{step, -n, 0} : Term{step, 0, n});
            }
    return reaches(std::move(t), base, -static_cast<int64_t>(dtype_size(b.dtype)), dtype_size(a.dtype));
}

// Whether two elements of an operand share memory.
bool folds(const Operand& o) {
    std::vector<std::pair<int64_t, int64_t>> dims;  // stride, last index
    if (!extent(o)) return false;
    for (size_t d = 0; d < o.shape.size(); ++d)
        if (o.shape[d] > 1) dims.push_back({o.stride[d], o.shape[d] - 1});
    std::sort(dims.begin(), dims.end());
    int64_t reach = 0;
    bool nested = true;  // every dimension steps over the smaller ones
    for (const auto& [stride, last] : dims) {
        nested &= stride > reach;
        reach += stride * last;
    }
    for (size_t first = 0; !nested && first < dims.size(); ++first) {
        // Two that differ in dimension `first` and those of smaller strides.
        std::vector<Term> t{{dims[first].first, 1, dims[first].second}};
        for (size_t d = 0; d < first; ++d) t.push_back({dims[d].first, -dims[d].second, dims[d].second});
        if (reaches(std::move(t), 0, -1, 1)) return true;
    }
    return false;
}

}  // namespace

void check_operator(const Module& m, const Node& n) {
    const Shapes s = shapes_of(m, n);
    if (is_block_operator(n)) {
        check_block_operator(s);
    } else if (n.op == "paged_plan") {
        const int64_t B = s.of("lengths")[0], page = attr(n, "page_size");
        s.want("counts", {B});
        if (s.of("page_table")[0] != B) refuse(n, "page_table has " + std::to_string(s.of("page_table")[0]) + " rows for " + std::to_string(B) + " requests");
        s.want("new_lengths", {B});
        s.want("starts", {B + 1});
        s.want("used", {1});
        s.want("new_used", {1});
        if (page < 1 || page > 4096) refuse(n, "pages of " + std::to_string(page) + " tokens (1 to 4096 are supported)");
        if (B > (1 << 24) || s.of("slots")[0] > (int64_t(1) << 31) - 1) refuse(n, "too many requests or rows");
    } else if (n.op == "paged_store") {
        check_cache(s);
        const auto &k = s.of("k"), &c = s.of("k_cache");
        s.want("v", k);
        s.same_type("k", "v");
        s.want("slots", {k[0]});
        s.want("k", {k[0], c[1], c[3]});
        if (k[0] > (int64_t(1) << 31) - 1) refuse(n, "too many rows");
    } else {
        check_cache(s);
        const auto &q = s.of("q"), &c = s.of("k_cache");
        const int64_t B = s.of("lengths")[0];
        if (q[2] != c[3]) refuse(n, "q has the head size " + std::to_string(q[2]) + ", the cache " + std::to_string(c[3]));
        if (q[1] < c[1] || q[1] % c[1]) refuse(n, std::to_string(q[1]) + " query heads for " + std::to_string(c[1]) + " key heads");
        if (q[1] / c[1] > 1024) refuse(n, "more than 1024 query heads a key head");
        s.want("out", q);
        s.same_type("q", "out");
        if (s.of("page_table")[0] != B) refuse(n, "page_table has " + std::to_string(s.of("page_table")[0]) + " rows for " + std::to_string(B) + " requests");
        if (s.of("page_table")[1] > ((int64_t(1) << 31) - 4096) / c[2]) refuse(n, "the page table spans more than 2^31 tokens");
        s.want("starts", {B + 1});
        if (!s.of("lse").empty()) s.want("lse", {q[0], q[1]});
        if (q[0] > (int64_t(1) << 31) - 1 || B > (1 << 24)) refuse(n, "too many rows or requests");
        if (n.op == "paged_attention") {
            if (attr(n, "window") < 0) refuse(n, "a negative window");
        } else {
            const auto& p = s.of("prefix_table");
            s.want("prefix_lengths", {p[0]});
            s.want("members", {p[0] + 1});
            if (p[0] > (1 << 24)) refuse(n, "too many groups");
            if (p[1] > ((int64_t(1) << 31) - 4096) / c[2]) refuse(n, "the prefix table spans more than 2^31 tokens");
        }
        auto it = n.op_floats.find("scale");
        if (it == n.op_floats.end() || !std::isfinite(it->second)) refuse(n, "missing attribute scale");
    }
}

bool operator_writes(const Node& n, size_t operand) {
    const std::string& name = n.tensor_args[operand].param;
    for (const Param& p : spec_of(n).params)
        if (name == p.name) return p.written;
    return false;
}

void run_operator(const Node& n, const std::vector<Operand>& operands, const OperatorRun& run) {
    // Written operands: no two elements at one address, none where another operand
    // lies; of staged tensors the whole is copied back, so no two written ones have
    // host memory between each other.
    for (size_t i = 0; i < operands.size(); ++i) {
        const Operand& w = operands[i];
        if (!operator_writes(n, i) || !w.ptr) continue;
        const std::string& a = n.tensor_args[i].param;
        for (size_t d = 0; d < w.shape.size(); ++d)
            if (w.shape[d] > 1 && w.stride[d] == 0) stop(n, a + " is written and has stride 0");
        if (folds(w)) stop(n, a + " is written and has elements that share memory");
        for (size_t j = 0; j < operands.size(); ++j) {
            const Operand& o = operands[j];
            const std::string& b = n.tensor_args[j].param;
            if (i == j || !o.ptr) continue;
            if (w.tensor != o.tensor && w.host_bytes && o.host_bytes) {
                if (operator_writes(n, j) && w.host < o.host + o.host_bytes && o.host < w.host + w.host_bytes)
                    stop(n, a + " and " + b + " are written and share host memory (device memory may be shared row by row)");
                continue;
            }
            // Read by the thread that writes the same element, before it does.
            const bool in_place = (a == "new_lengths" && b == "lengths") || (a == "new_used" && b == "used") || (a == "q_out" && b == "q") ||
                                  (a == "k_out" && b == "k");
            bool same = in_place && o.ptr == w.ptr;
            for (size_t d = 0; same && d < w.shape.size(); ++d) same = w.shape[d] < 2 || o.stride[d] == w.stride[d];
            if (same) continue;
            if (o.ptr == w.ptr || (meet(w, o) && run.allocated(w.ptr, static_cast<size_t>(extent(w))) && run.allocated(o.ptr, static_cast<size_t>(extent(o)))))
                stop(n, a + " is written and lies where " + b + " does");
        }
    }
    if (is_block_operator(n)) run_block_operator(n, operands, run);
    else if (n.op == "paged_plan") run_plan(n, operands, run);
    else if (n.op == "paged_store") run_store(n, operands, run);
    else if (n.op == "paged_attention") run_attend(n, operands, run);
    else run_prefix(n, operands, run);
}

const char* operator_error(int flag) {
    switch (flag) {
        case 4: return "paged_plan: a negative length or count, or the page table, the free pages or the rows do not suffice (nothing was written)";
        case 5: return "paged_plan: a page number is negative or its slots exceed 32 bits (rows left out)";
        case 6: return "paged_store: a slot lies outside the cache (rows left out)";
        case 7: return "paged_attention: starts, a length or a page number is out of range";
        case 8: return "paged_norm_rotate: starts or a position is out of range (rows left out)";
        case 9: return "paged_prefix_attention: starts, members, a length or a page number is out of range";
    }
    return nullptr;
}

std::pair<std::string, std::string> operator_source(const Module& m, const Node& n) {
    const Shapes s = shapes_of(m, n);
    if (is_block_operator(n)) return block_operator_source(s);
    if (n.op == "paged_plan") return {plan_source(), "ptowsp_paged_plan"};
    const auto& c = s.of("k_cache");
    const int D = static_cast<int>(c[3]), page = static_cast<int>(c[2]), code = code_id(s.dtype[s.at("k_cache")]);
    if (n.op == "paged_store")
        return {store_source(D, page, type_id(s.dtype[0]), code, true, store_chunk(s.of("k")[0], c[1], c[2])), "ptowsp_paged_store"};
    if (n.op == "paged_prefix_attention") {
        const DType type = s.dtype[0], code_type = s.dtype[s.at("k_cache")];
        const int64_t groups = s.of("prefix_table")[0];
        AttendForm shared = attend_form(s.of("q"), c, groups, type, code_type, false, true, true, 2);
        shared.prompts = shared.prompts && groups > 0;
        return {prefix_source(attend_form(s.of("q"), c, s.of("lengths")[0], type, code_type, false, true, true, 1), shared, type_id(type), !s.of("lse").empty()),
                "ptowsp_paged_prefix_parts"};
    }
    const AttendForm f = attend_form(s.of("q"), c, s.of("lengths")[0], s.dtype[0], s.dtype[s.at("k_cache")], attr(n, "window") > 0, !s.of("lse").empty(), true);
    return {attend_source(f.s, f.prompts), f.prompts ? "ptowsp_paged_attention_prompts" : "ptowsp_paged_attention"};
}

}  // namespace ptowsp
