// overlap.hpp — whether a call's outputs share memory with its inputs or with each other.
#pragma once

#include <cstdint>
#include <initializer_list>
#include <string>

#include "ra_internal.hpp"

namespace ra {

struct Extent {
    const char* name;
    const void* at;  // NULL: not given
    unsigned __int128 bytes;
};

// `rows` rows of `dim` elements, ld apart.
inline Extent rows_of(const char* name, const void* at, int64_t rows, int64_t dim, int64_t ld, int64_t size) {
    return {name, at, rows > 0 ? ((unsigned __int128)(rows - 1) * (uint64_t)ld + (uint64_t)dim) * (uint64_t)size : 0};
}

inline bool overlap(const Extent& a, const Extent& b) {
    const auto from_a = reinterpret_cast<uintptr_t>(a.at), from_b = reinterpret_cast<uintptr_t>(b.at);
    return a.at && b.at && a.bytes && b.bytes && from_a < from_b + b.bytes && from_b < from_a + a.bytes;
}

inline ra_status refuse_overlap(const char* what, std::initializer_list<Extent> outputs, std::initializer_list<Extent> inputs) {
    for (auto o = outputs.begin(); o != outputs.end(); ++o) {
        for (auto p = outputs.begin(); p != o; ++p)
            if (overlap(*o, *p)) return fail(RA_ERR_INVALID_ARGUMENT, std::string(what) + ": " + o->name + " overlaps " + p->name);
        for (const Extent& i : inputs)
            if (overlap(*o, i)) return fail(RA_ERR_INVALID_ARGUMENT, std::string(what) + ": " + o->name + " overlaps " + i.name);
    }
    return RA_OK;
}

}  // namespace ra
