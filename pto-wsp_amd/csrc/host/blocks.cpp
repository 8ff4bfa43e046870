#include <algorithm>
#include <cmath>
#include <stdexcept>

#include "../device/ptowsp_blocks_args.h"
#include "operators_shared.hpp"

namespace ptowsp {

namespace {

int64_t parts(int64_t n, int64_t each) { return (n + each - 1) / each; }
int64_t scale_blocks(int64_t n) { return parts(n, kScaleBlock); }
std::string num(int64_t v) { return std::to_string(v); }

// The operand of a name, or null.
const Operand* find(const Node& n, const std::vector<Operand>& o, const char* name) {
    for (size_t i = 0; i < o.size(); ++i)
        if (n.tensor_args[i].param == name) return &o[i];
    return nullptr;
}
const Operand& get(const Node& n, const std::vector<Operand>& o, const char* name) {
    const Operand* x = find(n, o, name);
    if (!x) throw std::runtime_error(n.op + ": internal: no operand " + name);
    return *x;
}
// One whose elements of the last dimension lie one behind the other.
const Operand& dense(const Node& n, const std::vector<Operand>& o, const char* name) {
    const Operand& x = get(n, o, name);
    if (x.shape.back() > 1 && x.stride.back() != 1) stop(n, std::string(name) + "'s last dimension must have stride 1");
    return x;
}

std::string entry(const char* header, int threads, const std::string& name, const char* args, const std::string& body) {
    return std::string("#include \"") + header + "\"\nextern \"C\" __global__ __launch_bounds__(" + num(threads) + ") void " + name + "(ptowsp::" + args +
           " A) { " + body + "; }\n";
}

// ---- block_quantize ----
// Blocks of a row that 16 lanes take: one while there are few workgroups, two of 16-bit
// numbers where there are many.  bf16 of 4096 columns, one, two and four: 64 rows 3.2,
// 3.6 and 4.7 us; 1024 rows 4.9, 4.4 and 5.1; 16384 rows 35.5, 31.8 and 34.4; 8192 rows
// of float32 24.6, 25.0 and 26.2.
constexpr int64_t kFewBlocks = 16384;

struct QuantizeForm {
    std::string source;
    int64_t groups;  // workgroups of 256 threads
};
QuantizeForm quantize_form(int64_t M, int64_t K, int64_t rows, DType type) {
    const int64_t blocks = scale_blocks(K);
    const std::string t = num(type_id(type));
    std::string body = "ptowsp::quantize_squares<" + t + ">(A)";
    int64_t groups = scale_blocks(M) * blocks;
    if (rows == 1) {
        const int unroll = M * blocks > kFewBlocks && type != DType::F32 ? 2 : 1;
        groups = parts(M * blocks, 16 * unroll);
        body = "ptowsp::quantize_rows<" + t + ", " + num(unroll) + ">(A)";
    }
    return {entry("ptowsp_blocks.h", 256, "ptowsp_block_quantize", "QuantizeArgs", body), groups};
}

void run_quantize(const Node& n, const std::vector<Operand>& o, const OperatorRun& run) {
    const Operand &x = dense(n, o, "x"), &codes = dense(n, o, "codes"), &scales = get(n, o, "scales");
    QuantizeArgs A{};
    A.x = x.ptr, A.codes = codes.ptr, A.scales = reinterpret_cast<float*>(scales.ptr);
    A.s_x = x.stride[0], A.s_codes = codes.stride[0];
    for (int d = 0; d < 2; ++d) A.s_scales[d] = scales.stride[d];
    A.rows = x.shape[0], A.cols = x.shape[1];
    A.blocks = static_cast<unsigned>(scale_blocks(A.cols));
    A.many = static_cast<unsigned>(A.rows * A.blocks);
    if (A.rows == 0) return;
    const QuantizeForm f = quantize_form(A.rows, A.cols, attr(n, "rows"), x.dtype);
    run.launch(f.source, "ptowsp_block_quantize", f.groups, 256, &A, sizeof A);
}

// ---- block_matmul ----
// Tiles of results, and the us that a stage of K takes where a compute unit has one
// of them, and where it has as many as it holds.
struct MatmulTile {
    int bm, bn, wm, wn, ring, per_cu;
    double alone, shared;
};
// Fitted to 2900 timings of 42 shapes, from 1 x 82 x 128 to 8192 x 6144 x 4096, each
// with every tile and 1 to 8 splits of K, weights from memory, to bf16 and with rows that
// go straight to LDS: there the choice cost 4% over the fastest on average.  Scales were
// multiplied with each other then; their halves take every tile 1 to 5% longer.  64 rows of 6144 x 4096 take 12.5 us in tiles of 32 x
// 64, 16.5 in 64 x 64 and 60 in 256 x 256; 512 rows 47, 37 and 75, and 29 in 128 x
// 128; 8192 rows 341 in 128 x 128 and 224 in 256 x 256.
constexpr MatmulTile kTiles[] = {
    {16, 16, 1, 1, 0, 8, 0.13, 0.65},  // BlockStream
    {32, 64, 1, 4, 6, 2, 0.33, 0.45}, {64, 64, 2, 2, 4, 2, 0.41, 0.70}, {64, 128, 1, 4, 3, 2, 0.63, 0.95},
    {128, 128, 2, 2, 4, 1, 0.84, 0.94}, {256, 256, 4, 2, 2, 1, 2.3, 2.2},
};
constexpr int kStreamWaves = 4;
struct MatmulForm {
    std::string source;
    MatmulTile tile;
    int splits, threads;
    int64_t tiles_m, tiles_n;
};
MatmulForm matmul_form(int64_t M, int64_t N, int64_t K, DType type, bool direct, int cus) {
    const double stages = static_cast<double>(scale_blocks(K));
    MatmulForm f{};
    double best = 0.0;
    for (const MatmulTile& t : kTiles) {
        if (!t.ring && M > t.bm) continue;
        // Float32 results take twice the registers for codes; other addresses need some for pieces under way.
        if (t.bm == 256 && (type == DType::F32 || !direct)) continue;
        const double tiles = static_cast<double>(parts(M, t.bm)) * static_cast<double>(parts(N, t.bn));
        for (const int splits : {1, 2, 3, 4, 6, 8}) {
            if (splits > stages) break;
            const double each = tiles * splits / cus, room = t.per_cu;
            const double stage = each <= 1.0    ? t.alone * (0.6 + 0.4 * each)
                                 : each <= room ? t.alone + (t.shared - t.alone) * (each - 1.0) / (room - 1.0)
                                                : t.shared * 0.5 * (std::ceil(each / room) + each / room);
            double us = 3.4 + stage * (std::ceil(stages / splits) + 1.0);
            if (splits > 1) us += 3.7 + splits * 8.0 * static_cast<double>(M) * static_cast<double>(N) / 4.5e6;
            if (best > 0.0 && us >= best) continue;
            best = us;
            f.tile = t;
            f.splits = splits;
        }
    }
    f.tiles_m = parts(M, f.tile.bm), f.tiles_n = parts(N, f.tile.bn);
    const std::string out = num(type_id(type));
    std::string t;
    if (f.tile.ring) {
        f.threads = 64 * f.tile.wm * f.tile.wn;
        t = "ptowsp::BlockGemm<" + num(f.tile.bm) + ", " + num(f.tile.bn) + ", " + num(f.tile.wm) + ", " + num(f.tile.wn) + ", " + num(f.tile.ring) + ", " + flag(direct) +
            ", " + out + ">";
    } else {
        f.threads = 64 * kStreamWaves;
        t = "ptowsp::BlockStream<" + num(kStreamWaves) + ", " + std::string(flag(direct)) + ", " + out + ">";
    }
    f.source = entry("ptowsp_blocks.h", f.threads, "ptowsp_block_matmul", "MatmulArgs", "__shared__ " + t + "::Shared lds; " + t + "::run(A, lds)");
    if (f.splits > 1) f.source += "extern \"C\" __global__ __launch_bounds__(256) void ptowsp_block_matmul_join(ptowsp::MatmulArgs A) { ptowsp::join_splits<" + out + ">(A); }\n";
    return f;
}

// Whether rows can go straight to LDS: 16-byte pieces, offsets within a tile in 31 bits.
bool direct_rows(const Operand& x, const Operand& scale, int64_t K) {
    constexpr int64_t kMost = int64_t(1) << 31;
    return K % 16 == 0 && (x.shape[0] < 2 || x.stride[0] % 16 == 0) && reinterpret_cast<uintptr_t>(x.ptr) % 16 == 0 && 256 * x.stride[0] + K < kMost &&
           4 * (256 * scale.stride[0] + scale_blocks(K) * scale.stride[1]) < kMost;
}

void run_matmul(const Node& n, const std::vector<Operand>& o, const OperatorRun& run) {
    const Operand &a = dense(n, o, "a"), &b = dense(n, o, "b"), &out = dense(n, o, "out"), &as = get(n, o, "a_scale"), &bs = get(n, o, "b_scale");
    MatmulArgs A{};
    A.a = a.ptr, A.b = b.ptr, A.out = out.ptr;
    A.a_scale = reinterpret_cast<const float*>(as.ptr), A.b_scale = reinterpret_cast<const float*>(bs.ptr);
    A.s_a = a.stride[0], A.s_b = b.stride[0], A.s_out = out.stride[0];
    for (int d = 0; d < 2; ++d) A.s_as[d] = as.stride[d], A.s_bs[d] = bs.stride[d];
    A.M = a.shape[0], A.N = b.shape[0], A.K = a.shape[1];
    A.stages = static_cast<int>(scale_blocks(A.K));
    if (A.M == 0) return;
    const MatmulForm f = matmul_form(A.M, A.N, A.K, out.dtype, direct_rows(a, as, A.K) && direct_rows(b, bs, A.K), run.cus);
    if (f.tiles_m * f.tiles_n * f.splits >= (int64_t(1) << 22)) stop(n, "too many rows and columns for one call");
    A.tiles_m = static_cast<int>(f.tiles_m), A.tiles_n = static_cast<int>(f.tiles_n), A.splits = f.splits;
    if (f.splits > 1) A.parts = reinterpret_cast<float*>(run.scratch(static_cast<size_t>(f.splits * A.M * A.N) * 4));
    run.launch(f.source, "ptowsp_block_matmul", f.tiles_m * f.tiles_n * f.splits, f.threads, &A, sizeof A);
    if (f.splits > 1) run.launch(f.source, "ptowsp_block_matmul_join", parts(A.M * parts(A.N, 4), 256), 256, &A, sizeof A);
}

// ---- paged_norm_rotate ----
// Waves of a token: as many as its heads need at once while they are few, two where
// there are many tokens.  32 + 8 heads of 128 in bf16 (5 at once), one wave a token, two
// and five: 64 tokens 6.6, 5.2 and 3.9 us; 1024 tokens 8.0, 7.5 and 6.7; 16384 tokens
// 62.1, 60.3 and 68.6.
constexpr int64_t kFewWaves = 32768;

struct RotateForm {
    std::string source;
    int per_token;  // waves
};
RotateForm rotate_form(const std::vector<int64_t>& q, int64_t keys, int64_t R, DType type, DType weight, bool qn, bool kn, bool interleaved) {
    const int64_t D = q[2], P = R % 16 == 0 ? 8 : R % 8 == 0 ? 4 : R % 4 == 0 ? 2 : 1, groups = D / (2 * P);
    int64_t lanes = 1;
    while (lanes < groups && lanes < 64) lanes *= 2;
    const int64_t passes = parts(q[1] + keys, 64 / lanes);
    RotateForm f;
    f.per_token = static_cast<int>(q[0] * passes <= kFewWaves ? passes : std::min<int64_t>(passes, 2));
    const std::string t = "ptowsp::Rotate<" + num(D) + ", " + num(R) + ", " + num(type_id(type)) + ", " + num(type_id(weight)) + ", " + flag(qn) + ", " +
                          flag(kn) + ", " + flag(interleaved) + ">";
    f.source = entry("ptowsp_rotate.h", 256, "ptowsp_paged_norm_rotate", "RotateArgs",
                     "const long long wave = blockIdx.x * 4ll + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = wave / " + num(f.per_token) +
                         "; if (row < A.rows) " + t + "::run(A, row, static_cast<int>(wave - row * " + num(f.per_token) + "), " + num(f.per_token) + ")");
    return f;
}

void run_rotate(const Node& n, const std::vector<Operand>& o, const OperatorRun& run) {
    RotateArgs A{};
    const char* names[2][3] = {{"q", "q_out", "q_weight"}, {"k", "k_out", "k_weight"}};
    bool norm[2];
    DType weight = DType::F32;
    for (int i = 0; i < 2; ++i) {
        const Operand &x = dense(n, o, names[i][0]), &out = dense(n, o, names[i][1]);
        A.x[i] = x.ptr, A.out[i] = out.ptr, A.heads[i] = static_cast<int>(x.shape[1]);
        for (int d = 0; d < 2; ++d) A.s_x[i][d] = x.stride[d], A.s_out[i][d] = out.stride[d];
        norm[i] = find(n, o, names[i][2]) != nullptr;
        if (norm[i]) {
            const Operand& w = dense(n, o, names[i][2]);
            A.weight[i] = w.ptr;
            weight = w.dtype;
        }
    }
    const Operand &cos = dense(n, o, "cos"), &sin = dense(n, o, "sin"), &lengths = get(n, o, "lengths"), &starts = get(n, o, "starts");
    A.cos = reinterpret_cast<const float*>(cos.ptr), A.sin = reinterpret_cast<const float*>(sin.ptr);
    A.s_cos = cos.stride[0], A.s_sin = sin.stride[0], A.positions = cos.shape[0];
    A.lengths = reinterpret_cast<const int*>(lengths.ptr), A.s_lengths = lengths.stride[0];
    A.starts = reinterpret_cast<const int*>(starts.ptr), A.s_starts = starts.stride[0];
    if (const Operand* f = find(n, o, "offsets")) A.offsets = reinterpret_cast<const int*>(f->ptr), A.s_offsets = f->stride[0];
    const Operand& q = get(n, o, "q");
    A.rows = q.shape[0], A.batch = lengths.shape[0];
    A.eps = static_cast<float>(n.op_floats.at("eps"));
    A.err = run.err;
    if (A.rows == 0 || A.batch == 0) return;
    const RotateForm f = rotate_form(q.shape, A.heads[1], 2 * cos.shape[1], q.dtype, weight, norm[0], norm[1], attr(n, "interleaved") != 0);
    const int64_t groups = parts(A.rows * f.per_token, 4);
    if (groups >= (int64_t(1) << 24)) stop(n, "too many rows for one call");
    run.launch(f.source, "ptowsp_paged_norm_rotate", groups, 256, &A, sizeof A);
}

}  // namespace

const std::vector<Spec>& block_specs() {
    static const std::vector<Spec> all = {
        {"block_quantize", {{"x", kReal, 2, false, false}, {"codes", kE4M3Code, 2, true, false}, {"scales", kScale, 2, true, false}}},
        {"block_matmul",
         {{"a", kE4M3Code, 2, false, false}, {"a_scale", kScale, 2, false, false}, {"b", kE4M3Code, 2, false, false}, {"b_scale", kScale, 2, false, false},
          {"out", kReal, 2, true, false}}},
        {"paged_norm_rotate",
         {{"q", kReal, 3, false, false}, {"k", kReal, 3, false, false}, {"cos", kScale, 2, false, false}, {"sin", kScale, 2, false, false},
          {"lengths", kIndex, 1, false, false}, {"starts", kIndex, 1, false, false}, {"q_out", kReal, 3, true, false}, {"k_out", kReal, 3, true, false},
          {"q_weight", kReal, 1, false, true}, {"k_weight", kReal, 1, false, true}, {"offsets", kIndex, 1, false, true}}}};
    return all;
}

bool is_block_operator(const Node& n) {
    for (const Spec& s : block_specs())
        if (n.op == s.op) return true;
    return false;
}

void check_block_operator(const Shapes& s) {
    const Node& n = s.n;
    constexpr int64_t kMost = (int64_t(1) << 31) - 1;
    if (n.op == "block_quantize") {
        const auto& x = s.of("x");
        const int64_t rows = attr(n, "rows");
        if (rows != 1 && rows != kScaleBlock) refuse(n, "blocks of " + num(rows) + " rows (1 or " + num(kScaleBlock) + " are supported)");
        if (x[1] < 1) refuse(n, "x has no columns");
        s.want("codes", x);
        s.want("scales", {parts(x[0], rows), scale_blocks(x[1])});
        if (x[0] > kMost || x[1] > kMost || x[0] * scale_blocks(x[1]) > (int64_t(1) << 27) || parts(x[0], rows) * scale_blocks(x[1]) > (int64_t(1) << (rows == 1 ? 27 : 23)))
            refuse(n, "x has too many blocks for one call");
    } else if (n.op == "block_matmul") {
        const auto &a = s.of("a"), &b = s.of("b");
        if (a[1] != b[1]) refuse(n, "a has " + num(a[1]) + " columns, b " + num(b[1]));
        if (a[1] < 1 || b[0] < 1) refuse(n, "b is empty");
        s.want("a_scale", {a[0], scale_blocks(a[1])});
        s.want("b_scale", {scale_blocks(b[0]), scale_blocks(b[1])});
        s.want("out", {a[0], b[0]});
        if (a[0] > kMost || a[1] > kMost || b[0] > kMost) refuse(n, "too many rows or columns");
    } else {
        const auto &q = s.of("q"), &k = s.of("k"), &cos = s.of("cos");
        const int64_t B = s.of("lengths")[0], D = q[2];
        if (k[0] != q[0] || k[2] != D) refuse(n, "k has the shape " + shape_text(k) + ", q " + shape_text(q));
        s.same_type("q", "k");
        s.want("q_out", q);
        s.same_type("q", "q_out");
        s.want("k_out", k);
        s.same_type("k", "k_out");
        if (D < 16 || D > 256 || D % 16) refuse(n, "head size " + num(D) + " (a multiple of 16 up to 256 is needed)");
        if (q[1] < 1 || k[1] < 1 || q[1] > 65536 || k[1] > 65536) refuse(n, num(q[1]) + " query heads and " + num(k[1]) + " key heads");
        if (cos[0] < 1 || cos[1] < 1 || 2 * cos[1] > D) refuse(n, "cos has the shape " + shape_text(cos) + " for a head size of " + num(D));
        s.want("sin", cos);
        s.want("starts", {B + 1});
        if (!s.of("offsets").empty()) s.want("offsets", {B});
        const bool qw = !s.of("q_weight").empty(), kw = !s.of("k_weight").empty();
        if (qw) s.want("q_weight", {D});
        if (kw) s.want("k_weight", {D});
        if (qw && kw) s.same_type("q_weight", "k_weight");
        if (q[0] > kMost || B > (1 << 24)) refuse(n, "too many rows or requests");
        auto it = n.op_floats.find("eps");
        if (it == n.op_floats.end() || !std::isfinite(it->second) || it->second < 0.0) refuse(n, "eps must be a finite number that is not negative");
        attr(n, "interleaved");
    }
}

void run_block_operator(const Node& n, const std::vector<Operand>& operands, const OperatorRun& run) {
    if (n.op == "block_quantize") run_quantize(n, operands, run);
    else if (n.op == "block_matmul") run_matmul(n, operands, run);
    else run_rotate(n, operands, run);
}

std::pair<std::string, std::string> block_operator_source(const Shapes& s) {
    const Node& n = s.n;
    if (n.op == "block_quantize") return {quantize_form(s.of("x")[0], s.of("x")[1], attr(n, "rows"), s.dtype[s.at("x")]).source, "ptowsp_block_quantize"};
    // For the 256 compute units of the target.
    if (n.op == "block_matmul") return {matmul_form(s.of("a")[0], s.of("b")[0], s.of("a")[1], s.dtype[s.at("out")], s.of("a")[1] % 16 == 0, 256).source, "ptowsp_block_matmul"};
    const bool qn = !s.of("q_weight").empty(), kn = !s.of("k_weight").empty();
    return {rotate_form(s.of("q"), s.of("k")[1], 2 * s.of("cos")[1], s.dtype[s.at("q")], s.dtype[s.at(qn ? "q_weight" : "k_weight")], qn, kn,
                        attr(n, "interleaved") != 0)
                .source,
            "ptowsp_paged_norm_rotate"};
}

}  // namespace ptowsp
