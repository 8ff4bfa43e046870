// Operator steps of a workload (pto_wsp/paged.py): operands checked when a
// module is compiled, launches made when a run reaches the step.
#pragma once

#include <cstddef>
#include <cstdint>
#include <functional>
#include <string>
#include <vector>

#include "module.hpp"

namespace ptowsp {

// Throws CompileError where types, shapes or attributes of an operator step do not fit.
void check_operator(const Module& m, const Node& n);

// Whether the step writes the operand.
bool operator_writes(const Node& n, size_t operand);

// One operand at a run: the view's first element on the device.
struct Operand {
    char* ptr = nullptr;
    std::vector<int64_t> shape, stride;  // elements
    DType dtype = DType::F32;
    int tensor = 0;              // the tensor that it is a view of, and
    const char* host = nullptr;  // the host memory of a tensor that is staged
    size_t host_bytes = 0;
};

// What a step needs of the run around it.
struct OperatorRun {
    int cus = 1;         // compute units of the device
    int* err = nullptr;  // the kernels' error flag
    // Whether so many bytes lie in one allocation: operands whose memory the runtime
    // does not know are not compared.
    std::function<bool(const char*, size_t)> allocated;
    // Device scratch for the step: `need` bytes, any content.
    std::function<char*(size_t)> scratch;
    std::function<void(const std::string& source, const char* entry, int64_t blocks, int threads, const void* args, size_t bytes)> launch;
};

// Enqueues the step.  Throws std::runtime_error where strides, alignment or
// overlaps do not fit.
void run_operator(const Node& n, const std::vector<Operand>& operands, const OperatorRun& run);

// The message of an error flag that an operator's kernel raised, or null.
const char* operator_error(int flag);

// The source of the kernels that a run of the step launches, for operands laid out
// one behind the other, and its first entry (for builds without a GPU).
std::pair<std::string, std::string> operator_source(const Module& m, const Node& n);

}  // namespace ptowsp
