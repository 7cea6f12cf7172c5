// Argument checks of the operators' runs (ops.cu): host code without CUDA.
#pragma once

#include <cstdint>
#include <string>
#include <vector>

#include "../../include/rosenna.h"
#include "model_files.hpp"

namespace rosenna {

inline Status arg(const std::string &m) { return Status::Err(ROSENNA_ERR_ARG, m); }
inline Status shape(const std::string &m) { return Status::Err(ROSENNA_ERR_SHAPE, m); }
inline int64_t or_n(int64_t ld, int64_t n) { return ld ? ld : n; }

// An array of `rows` rows of n 4-byte values, `ld` apart.
struct Array {
    const char *name;
    const float *p;
    int64_t rows, ld;
    // first byte behind it
    intptr_t end(int64_t n) const { return reinterpret_cast<intptr_t>(p) + ((rows - 1) * ld + n) * 4; }
    bool empty(int64_t n) const { return !p || n <= 0 || rows <= 0; }
};

inline Status check_array(const Array &a, int64_t n, bool required) {
    if (!a.p) {
        if (required && n > 0 && a.rows > 0) return arg(std::string("null array ") + a.name);
        return Status::Ok();
    }
    if (reinterpret_cast<uintptr_t>(a.p) % sizeof(float)) return arg(std::string(a.name) + " is not aligned to its type");
    if (a.ld < n) return shape(std::string("ld of ") + a.name + " is smaller than n");
    if (a.ld > (int64_t)1 << 40 || (a.rows > 0 && a.ld > ((int64_t)1 << 60) / a.rows)) return shape(std::string("ld of ") + a.name + " is out of range");
    return Status::Ok();
}

// Whether two arrays of n columns share an element.  Column ranges of one array
// (equal ld) are told apart; otherwise the address ranges decide.
inline bool overlap(const Array &a, const Array &b, int64_t n) {
    if (a.empty(n) || b.empty(n)) return false;
    const intptr_t pa = reinterpret_cast<intptr_t>(a.p), pb = reinterpret_cast<intptr_t>(b.p);
    if (a.end(n) <= pb || b.end(n) <= pa) return false;
    if (a.ld == b.ld) {
        const int64_t off = (((pb - pa) / 4) % a.ld + a.ld) % a.ld;
        if (off >= n && off + n <= a.ld) return false;
    }
    return true;
}

// Every output against every input and the other outputs; `state_in` may be
// state_out itself.
inline Status check_overlaps(const std::vector<Array> &ins, const std::vector<Array> &outs, const Array &state_in, const Array &state_out,
                             int64_t n) {
    for (size_t i = 0; i < outs.size(); i++) {
        for (auto &a : ins)
            if (overlap(a, outs[i], n)) return arg(std::string(outs[i].name) + " overlaps " + a.name);
        for (size_t j = 0; j < i; j++)
            if (overlap(outs[j], outs[i], n)) return arg(std::string(outs[i].name) + " overlaps " + outs[j].name);
    }
    for (auto &o : outs)
        if (o.p != state_out.p && overlap(state_in, o, n)) return arg(std::string(o.name) + " overlaps " + state_in.name);
    const bool in_place = state_in.p && state_in.p == state_out.p && state_in.ld == state_out.ld;
    if (!in_place && overlap(state_in, state_out, n))
        return arg(std::string(state_out.name) + " overlaps " + state_in.name + " without being it");
    return Status::Ok();
}

// `rows`: the most features of an array (its rows for one step).
inline Status check_run(bool right_kind, int64_t n, int64_t T, int64_t rows) {
    if (!right_kind) return arg("not an operator of this kind");
    if (n < 0) return arg("negative batch size");
    if (T < 0) return arg("negative number of steps");
    // at most 2^38 elements an array, so that no product below overflows
    const int64_t limit = (int64_t)1 << 38, steps = T ? T : 1;
    if (n > limit || T >= (int64_t)1 << 28 || n > limit / steps || (rows > 0 && steps > limit / rows / (n ? n : 1)))
        return shape("batch or sequence too large");
    return Status::Ok();
}

inline Status check_workspace(const void *ws, int64_t bytes, int64_t need, bool required, const std::vector<Array> &arrays, int64_t n) {
    if (!ws) {
        if (required && need > 0) return arg("a workspace of " + std::to_string(need) + " bytes is needed");
        return Status::Ok();
    }
    if (bytes < need) return arg("the workspace has " + std::to_string(bytes) + " bytes; " + std::to_string(need) + " are needed");
    const intptr_t w = reinterpret_cast<intptr_t>(ws);
    if (w % 16) return arg("the workspace is not 16-byte aligned");
    for (auto &a : arrays)
        if (need > 0 && !a.empty(n) && reinterpret_cast<intptr_t>(a.p) < w + need && w < a.end(n))
            return arg(std::string("the workspace overlaps ") + a.name);
    return Status::Ok();
}

}  // namespace rosenna
