// Where the rows of a call's tensors lie: whether what one workgroup writes is what
// another reads.  Host code.
#pragma once
#include <algorithm>
#include <cstdint>

namespace crimpl {

namespace {

struct Rows {  // row (t, h), of `row` bytes, begins t * token + h * head bytes behind `at`
    uintptr_t at;
    uint64_t tokens, token, heads, head, row;
    Rows(const void* p, uint64_t tokens, uint64_t token, uint64_t heads, uint64_t head, uint64_t row)
        : at(reinterpret_cast<uintptr_t>(p)), tokens(tokens), token(tokens > 1 ? token : 0), heads(heads), head(heads > 1 ? head : 0),
          row(row)
    {
    }
    bool none() const { return !tokens || !heads || !row; }
    __int128 end() const
    {
        return static_cast<__int128>(at) + static_cast<__int128>(tokens - 1) * token + static_cast<__int128>(heads - 1) * head + row;
    }
};

// Whether a row meets another whose (token, head) lies (dt, dh) from its own in a tensor of the same
// strides that begins `apart` bytes behind: for any such pair but a row and itself.
inline bool rows_meet(const Rows& a, __int128 apart)
{
    typedef __int128 I;
    const I most = static_cast<I>(a.tokens) - 1, token = a.token, row = a.row;
    auto meets = [&](I from, I dt, bool itself) {
        const I x = from + dt * token;
        return dt >= -most && dt <= most && x < row && -x < row && !(itself && dt == 0);
    };
    for (I dh = 1 - static_cast<I>(a.heads); dh < static_cast<I>(a.heads); ++dh) {
        const I from = apart + dh * static_cast<I>(a.head);
        const bool itself = dh == 0 && apart == 0;
        if (token == 0) {
            if (meets(from, 0, itself) || (most > 0 && meets(from, 1, false))) return true;
            continue;
        }
        // the nearest ones: those around -from / token, or the last on that side
        const I near = std::min(most, std::max(-most, -from / token));
        for (I dt = near - 1; dt <= near + 1; ++dt)
            if (meets(from, dt, itself)) return true;
    }
    return false;
}

// Whether rows of one tensor lie over one another.
inline bool rows_overlap(const Rows& a)
{
    if (a.none()) return false;
    typedef __int128 I;
    const I tokens = a.tokens, heads = a.heads, token = a.token, head = a.head, row = a.row;
    if ((heads == 1 || head >= row) && (tokens == 1 || token >= (heads - 1) * head + row)) return false;
    if ((tokens == 1 || token >= row) && (heads == 1 || head >= (tokens - 1) * token + row)) return false;
    return rows_meet(a, 0);
}

// Whether rows that are written lie over rows that are read which are not the same ones: tensors that
// are the same, apart, or in between one another without meeting are fine.
inline bool rows_overwrite(const Rows& out, const Rows& in)
{
    if (out.none() || in.none()) return false;
    const bool alike = out.token == in.token && out.head == in.head;
    if (out.at == in.at && alike) return false;
    if (static_cast<__int128>(out.at) >= in.end() || static_cast<__int128>(in.at) >= out.end()) return false;
    return !alike || rows_meet(out, static_cast<__int128>(in.at) - static_cast<__int128>(out.at));
}

}  // namespace

}  // namespace crimpl
