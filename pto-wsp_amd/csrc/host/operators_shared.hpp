// What the operators' host files share: their operands' tables and checks.
#pragma once

#include <cstring>
#include <string>
#include <vector>

#include "operators.hpp"

namespace ptowsp {

enum Group { kIndex, kReal, kCode, kScale, kE4M3Code };  // I32; BF16, F16 or F32; I8 or F8E4M3; F32; F8E4M3

struct Param {
    const char* name;
    Group group;
    int rank;
    bool written;
    bool optional;
};

struct Spec {
    const char* op;
    std::vector<Param> params;
};

[[noreturn]] inline void refuse(const Node& n, const std::string& why) { throw CompileError(n.op + ": " + why); }
[[noreturn]] inline void stop(const Node& n, const std::string& why) { throw std::runtime_error(n.op + ": " + why); }

inline int64_t attr(const Node& n, const char* key) {
    auto it = n.op_ints.find(key);
    if (it == n.op_ints.end()) refuse(n, std::string("missing attribute ") + key);
    return it->second;
}

inline std::string shape_text(const std::vector<int64_t>& s) {
    std::string out = "[";
    for (size_t i = 0; i < s.size(); ++i) out += (i ? ", " : "") + std::to_string(s[i]);
    return out + "]";
}

// Operands in the order of the operator's parameters (null: left out).
struct Shapes {
    const Node& n;
    const Spec& spec;
    std::vector<std::vector<int64_t>> shape;
    std::vector<DType> dtype;
    size_t at(const char* name) const {
        for (size_t i = 0; i < spec.params.size(); ++i)
            if (!std::strcmp(spec.params[i].name, name)) return i;
        throw CompileError(std::string("internal: no operand ") + name);
    }
    const std::vector<int64_t>& of(const char* name) const { return shape[at(name)]; }
    void want(const char* name, const std::vector<int64_t>& s) const {
        if (of(name) != s) refuse(n, std::string(name) + " has the shape " + shape_text(of(name)) + ", " + shape_text(s) + " is needed");
    }
    void same_type(const char* a, const char* b) const {
        if (dtype[at(a)] != dtype[at(b)]) refuse(n, std::string(a) + " and " + b + " differ in type");
    }
};

inline int type_id(DType d) { return d == DType::BF16 ? 0 : d == DType::F16 ? 1 : 2; }
inline int code_id(DType d) { return d == DType::F8E4M3 ? 0 : 1; }
inline const char* flag(bool b) { return b ? "true" : "false"; }

// The operators over 8-bit blocks and paged_norm_rotate (blocks.cpp).
const std::vector<Spec>& block_specs();
bool is_block_operator(const Node& n);
void check_block_operator(const Shapes& s);
void run_block_operator(const Node& n, const std::vector<Operand>& operands, const OperatorRun& run);
std::pair<std::string, std::string> block_operator_source(const Shapes& s);

}  // namespace ptowsp
