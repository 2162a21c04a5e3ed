// End-to-end check of the operators for long and speculative answers as a C++ caller
// uses them: keys turned into a paged cache, weights of its tokens, an eviction by
// them with a pinned slot, the moves, and a verification of drafts.  Truth is
// computed here in double.  Prints "long_answers_check: OK" and exits 0 when every
// check passes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <stdexcept>
#include <vector>

#include <cu_roaring/cu_roaring.hpp>

#define HIP_OK(x)                                                                      \
    do {                                                                               \
        hipError_t e_ = (x);                                                           \
        if (e_ != hipSuccess) {                                                        \
            std::fprintf(stderr, "%s:%d %s\n", __FILE__, __LINE__, hipGetErrorString(e_)); \
            std::exit(2);                                                              \
        }                                                                              \
    } while (0)

static int g_fail = 0;
#define CHECK(c)                                                              \
    do {                                                                      \
        if (!(c)) {                                                           \
            std::fprintf(stderr, "CHECK failed %s:%d: %s\n", __FILE__, __LINE__, #c); \
            ++g_fail;                                                         \
        }                                                                     \
    } while (0)

template <class T>
struct Dev {
    T* p = nullptr;
    size_t n;
    explicit Dev(size_t n_) : n(n_) { HIP_OK(hipMalloc(reinterpret_cast<void**>(&p), (n ? n : 1) * sizeof(T))); }
    explicit Dev(const std::vector<T>& h) : Dev(h.size())
    {
        HIP_OK(hipMemcpy(p, h.data(), n * sizeof(T), hipMemcpyHostToDevice));
    }
    ~Dev() { (void)hipFree(p); }
    Dev(const Dev&) = delete;
    Dev& operator=(const Dev&) = delete;
    std::vector<T> host() const
    {
        std::vector<T> h(n);
        HIP_OK(hipMemcpy(h.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
        return h;
    }
};

static double up(uint16_t x)  // bf16
{
    const uint32_t b = static_cast<uint32_t>(x) << 16;
    float f;
    std::memcpy(&f, &b, 4);
    return f;
}

static uint16_t down(float f)
{
    uint32_t b;
    std::memcpy(&b, &f, 4);
    return static_cast<uint16_t>((b + 0x7FFFu + ((b >> 16) & 1u)) >> 16);
}

int main()
{
    using namespace cu_roaring;
    constexpr uint32_t PAGES = 8, PAGE = 16, HEADS = 4, KV = 2, DIM = 64, TOKENS = 50, COLS = 4, ROW = DIM * KV;
    std::mt19937 rng(5);
    std::normal_distribution<float> normal;
    auto random = [&](size_t n) {
        std::vector<uint16_t> x(n);
        for (auto& v : x) v = down(normal(rng));
        return x;
    };
    // the pages of one request, and its tokens' slots
    const std::vector<int32_t> pages = {6, 1, 4, 3};
    std::vector<int64_t> slots(TOKENS);
    std::vector<int32_t> positions(TOKENS);
    for (uint32_t i = 0; i < TOKENS; ++i) {
        slots[i] = pages[i / PAGE] * static_cast<int64_t>(PAGE) + i % PAGE;
        positions[i] = static_cast<int32_t>(100000 + i);
    }
    std::vector<double> freqs(DIM / 2);
    for (uint32_t i = 0; i < DIM / 2; ++i) freqs[i] = std::pow(10000.0, -2.0 * i / DIM);
    const auto q = random(TOKENS * HEADS * DIM), k = random(TOKENS * ROW), v = random(TOKENS * ROW);
    Dev<uint16_t> d_q(q), d_k(k), d_v(v), d_turned(q.size()), d_kc(PAGES * PAGE * ROW), d_vc(PAGES * PAGE * ROW);
    Dev<int64_t> d_slots(slots);
    Dev<int32_t> d_positions(positions), d_table(pages);
    Dev<double> d_freqs(freqs);
    const PagedCache cache{d_kc.p, d_vc.p, PAGE * ROW, ROW, DIM, PAGE * ROW, ROW, DIM, PAGES, PAGE, KV, DIM, CR_BF16};
    PagedRotaryArgs rotary{};
    rotary.q = d_q.p;
    rotary.q_token_stride = rotary.out_token_stride = HEADS * DIM;
    rotary.q_head_stride = rotary.out_head_stride = DIM;
    rotary.q_out = d_turned.p;
    rotary.k = d_k.p;
    rotary.v = d_v.p;
    rotary.k_token_stride = rotary.v_token_stride = ROW;
    rotary.k_head_stride = rotary.v_head_stride = DIM;
    rotary.d_positions = d_positions.p;
    rotary.d_freqs = d_freqs.p;
    rotary.d_slots = d_slots.p;
    rotary.n_tokens = TOKENS;
    rotary.n_heads = HEADS;
    rotary.rotated = DIM;
    rotary.magnitude = 1.0f;
    paged_rotary(rotary, cache);
    HIP_OK(hipDeviceSynchronize());
    const auto qt = d_turned.host(), kc = d_kc.host(), vc = d_vc.host();
    for (uint32_t t = 0; t < TOKENS; ++t)
        for (uint32_t i = 0; i < DIM / 2; ++i) {
            const double a = positions[t] * freqs[i], c = std::cos(a), s = std::sin(a);
            const double x = up(k[t * ROW + i]), y = up(k[t * ROW + i + DIM / 2]);
            const double got = up(kc[slots[t] * ROW + i]), bar = std::ldexp(std::fabs(x) + std::fabs(y), -8);
            CHECK(std::fabs(got - (x * c - y * s)) <= bar);
            CHECK(vc[slots[t] * ROW + i] == v[t * ROW + i]);
            const double u = up(q[t * HEADS * DIM + i]), w = up(q[t * HEADS * DIM + i + DIM / 2]);
            CHECK(std::fabs(up(qt[t * HEADS * DIM + i + DIM / 2]) - (w * c + u * s)) <=
                  std::ldexp(std::fabs(u) + std::fabs(w), -8));
        }

    // weights of all tokens by the last one's heads, with log-sums of zero
    const std::vector<int32_t> kv_len = {static_cast<int32_t>(TOKENS)}, one = {1}, first = {static_cast<int32_t>(TOKENS - 1)};
    Dev<int32_t> d_kv(kv_len), d_one(one), d_first(first);
    Dev<float> d_lse(std::vector<float>(TOKENS * HEADS, 0.0f)), d_weights(COLS * PAGE), d_weights_out(COLS * PAGE);
    PagedWeightsArgs weights{};
    weights.q = d_turned.p;
    weights.q_token_stride = HEADS * DIM;
    weights.q_head_stride = DIM;
    weights.lse = d_lse.p;
    weights.n_tokens = TOKENS;
    weights.n_heads = HEADS;
    weights.n_requests = 1;
    weights.d_starts = d_first.p;
    weights.d_new = d_one.p;
    weights.d_kv_len = d_kv.p;
    weights.d_table = d_table.p;
    weights.table_cols = COLS;
    weights.table_stride = COLS;
    weights.d_out = d_weights.p;
    weights.out_stride = COLS * PAGE;
    weights.scale = 0.125f;
    weights.causal = 1;
    paged_weights(weights, cache);
    HIP_OK(hipDeviceSynchronize());
    const auto w = d_weights.host();
    for (uint32_t i = 0; i < TOKENS; ++i) {
        double sum = 0;
        for (uint32_t h = 0; h < HEADS; ++h) {
            double s = 0;
            for (uint32_t d = 0; d < DIM; ++d)
                s += up(qt[((TOKENS - 1) * HEADS + h) * DIM + d]) * up(kc[slots[i] * ROW + h / 2 * DIM + d]);
            sum += std::exp(0.125 * s);
        }
        CHECK(std::fabs(w[i] - sum) < 1e-5 * sum);
    }

    // 20 of them stay: the pinned one, the newest two, the heaviest others
    const std::vector<int32_t> keep = {20};
    const uint32_t pin = static_cast<uint32_t>(slots[30]);
    GpuRoaring pinned = upload_from_ids(&pin, 1, PAGES * PAGE);
    Dev<int32_t> d_keep(keep), d_len(1), d_moves(COLS * PAGE), d_n(1), d_freed(COLS), d_counts(2);
    PagedEvictArgs evict{};
    evict.d_weights = d_weights.p;
    evict.weights_stride = evict.weights_out_stride = COLS * PAGE;
    evict.d_kv_len = d_kv.p;
    evict.d_keep = d_keep.p;
    evict.d_table = d_table.p;
    evict.table_cols = evict.table_stride = COLS;
    evict.page_size = PAGE;
    evict.n_pages = PAGES;
    evict.n_requests = 1;
    evict.recent = 2;
    evict.pinned = to_abi(&pinned);
    evict.d_weights_out = d_weights_out.p;
    evict.d_len = d_len.p;
    evict.d_moves = d_moves.p;
    evict.moves_cap = evict.moves_stride = COLS * PAGE / 2;
    evict.d_n_moves = d_n.p;
    evict.d_freed = d_freed.p;
    evict.freed_cap = COLS;
    evict.d_counts = d_counts.p;
    paged_evict(evict);
    paged_move(d_moves.p, COLS * PAGE / 2, COLS * PAGE / 2, d_n.p, 1, cache);
    HIP_OK(hipDeviceSynchronize());
    std::vector<uint32_t> order(TOKENS);
    for (uint32_t i = 0; i < TOKENS; ++i) order[i] = i;
    auto safe = [&](uint32_t i) { return i == 30 || i >= TOKENS - 2; };
    std::stable_sort(order.begin(), order.end(), [&](uint32_t a, uint32_t b) {
        return safe(a) != safe(b) ? safe(a) : !safe(a) && w[a] > w[b];
    });
    std::vector<bool> stays(TOKENS);
    for (int i = 0; i < 20; ++i) stays[order[i]] = true;
    std::vector<uint32_t> lies(20), movers;
    for (uint32_t i = 20; i < TOKENS; ++i)
        if (stays[i]) movers.push_back(i);
    const auto moves = d_moves.host(), n_moves = d_n.host(), counts = d_counts.host(), freed = d_freed.host();
    const auto moved = d_kc.host();
    const auto w_out = d_weights_out.host();
    size_t at = 0;
    for (uint32_t i = 0; i < 20; ++i) {
        lies[i] = stays[i] ? i : movers.at(at++);
        CHECK(w_out[i] == w[lies[i]]);
        for (uint32_t d = 0; d < ROW; ++d) CHECK(moved[slots[i] * ROW + d] == kc[slots[lies[i]] * ROW + d]);
    }
    CHECK(d_len.host()[0] == 20 && n_moves[0] == static_cast<int32_t>(movers.size()) && at == movers.size());
    CHECK(counts[0] == 2 && freed[0] == pages[2] && freed[1] == pages[3]);
    CHECK(counts[1] == n_moves[0] && moves[0] == slots[movers.at(0)]);
    gpu_roaring_free(pinned);

    // two drafts: the first is all that the model would say, the second can not be
    constexpr uint32_t VOCAB = 1000;
    std::vector<float> scores(3 * VOCAB, 0.0f);
    scores[7] = 100.0f;
    scores[VOCAB + 8] = -INFINITY;
    Dev<float> d_scores(scores), d_uniform(std::vector<float>{0.5f, 0.5f, 0.25f});
    Dev<int32_t> d_tokens(std::vector<int32_t>{0, 7, 8}), d_starts(std::vector<int32_t>{0, 3}), d_accepted(1), d_out(3);
    DraftVerifyArgs verify{};
    verify.d_scores = d_scores.p;
    verify.row_stride = VOCAB;
    verify.dtype = CR_F32;
    verify.n_rows = 3;
    verify.n_requests = 1;
    verify.vocab = VOCAB;
    verify.d_tokens = d_tokens.p;
    verify.d_starts = d_starts.p;
    verify.d_uniform = d_uniform.p;
    verify.temperature = 1.0f;
    verify.d_accepted = d_accepted.p;
    verify.d_out = d_out.p;
    verify.out_cols = verify.out_stride = 3;
    draft_verify(verify);
    HIP_OK(hipDeviceSynchronize());
    const auto out = d_out.host();
    // 999 tokens alike without token 8: a quarter of them lies before the 250th, which is token 250
    CHECK(d_accepted.host()[0] == 1 && out[0] == 7 && out[1] == 250 && out[2] == -1);

    bool threw = false;
    verify.temperature = 0.0f;
    try {
        draft_verify(verify);
    } catch (const std::runtime_error&) {
        threw = true;
    }
    CHECK(threw);
    if (g_fail) return 1;
    std::puts("long_answers_check: OK");
    return 0;
}
