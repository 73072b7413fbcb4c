// Whether the results of a call lie apart from what it reads while it writes them.
#pragma once
#include <initializer_list>

#include "common.h"

namespace sp {

struct Memory {
    const char* name;
    const void* at;               // nullptr: not there
    int64_t bytes;
    bool meets(const Memory& o) const {
        if (at == nullptr || o.at == nullptr) return false;
        const uintptr_t a = (uintptr_t)at, b = (uintptr_t)o.at;
        return a < b ? b - a < (uintptr_t)bytes : a - b < (uintptr_t)o.bytes;
    }
};

// SP_ERR_ARG where one of `outs` overlaps another or one of `ins`.
inline int lie_apart(const char* fn, std::initializer_list<Memory> outs, std::initializer_list<Memory> ins) {
    for (const Memory* o = outs.begin(); o != outs.end(); ++o) {
        for (const Memory* p = outs.begin(); p != o; ++p)
            if (o->meets(*p)) return fail(SP_ERR_ARG, "%s: %s and %s overlap", fn, p->name, o->name);
        for (const Memory& i : ins)
            if (o->meets(i)) return fail(SP_ERR_ARG, "%s: %s and %s overlap", fn, o->name, i.name);
    }
    return SP_OK;
}

}  // namespace sp
