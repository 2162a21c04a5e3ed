// End-to-end check of the operators for serving language models as a C++ caller
// uses them: two requests are planned into a paged cache whose free pages are a
// bitmap, their keys and values appended, attention taken with and without a
// filter, and beams selected and reordered.  Truth is computed here in double.
// Prints "serving_check: OK" and exits 0 when every check passes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
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
    explicit Dev(const std::vector<T>& h) : Dev(h.size()) { HIP_OK(hipMemcpy(p, h.data(), n * sizeof(T), hipMemcpyHostToDevice)); }
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

int main()
{
    using namespace cu_roaring;
    constexpr uint32_t PAGES = 64, PAGE = 16, HEADS = 4, KV = 2, DIM = 64, COLS = 8;
    const std::vector<int32_t> cached = {0, 0}, fresh = {70, 33};
    const uint32_t tokens = 103;
    std::vector<uint32_t> free_ids;
    for (uint32_t i = 0; i < PAGES; ++i)
        if (i % 3 != 1) free_ids.push_back(i);
    GpuRoaring free_pages = upload_from_ids(free_ids.data(), static_cast<uint32_t>(free_ids.size()), PAGES);

    // plan
    Dev<int32_t> d_cached(cached), d_new(fresh), table(2 * COLS), starts(3), kv_len(2), taken(16), counts(3);
    Dev<int64_t> slots(tokens);
    paged_plan(free_pages, PAGES, PAGE, d_cached.p, d_new.p, 2, table.p, COLS, COLS, slots.p, tokens, starts.p, kv_len.p,
               taken.p, 16, counts.p);
    const auto h_slots = slots.host();
    const auto h_counts = counts.host();
    CHECK(h_counts[0] == 103 && h_counts[1] == 8 && h_counts[2] == 0);
    for (uint32_t t = 0; t < tokens; ++t) {
        const uint32_t in = t < 70 ? t : t - 70, page = (t < 70 ? 0 : 5) + in / PAGE;
        CHECK(h_slots[t] == static_cast<int64_t>(free_ids[page]) * PAGE + in % PAGE);
    }

    // append, f16
    std::mt19937 rng(5);
    std::normal_distribution<float> normal;
    auto random = [&](size_t n) {
        std::vector<_Float16> v(n);
        for (auto& x : v) x = static_cast<_Float16>(normal(rng));
        return v;
    };
    const auto k = random(tokens * KV * DIM), v = random(tokens * KV * DIM), q = random(tokens * HEADS * DIM);
    Dev<_Float16> dk(k), dv(v), dq(q), kc(PAGES * PAGE * KV * DIM), vc(PAGES * PAGE * KV * DIM), out(tokens * HEADS * DIM);
    HIP_OK(hipMemset(kc.p, 0xFF, kc.n * 2));  // NaN where nothing was appended
    HIP_OK(hipMemset(vc.p, 0xFF, vc.n * 2));
    PagedCache cache{};
    cache.k = kc.p;
    cache.v = vc.p;
    cache.k_page_stride = cache.v_page_stride = PAGE * KV * DIM;
    cache.k_slot_stride = cache.v_slot_stride = KV * DIM;
    cache.k_head_stride = cache.v_head_stride = DIM;
    cache.n_pages = PAGES;
    cache.page_size = PAGE;
    cache.n_heads = KV;
    cache.head_dim = DIM;
    cache.dtype = CR_F16;
    paged_append(dk.p, dv.p, KV * DIM, DIM, KV * DIM, DIM, tokens, slots.p, cache);

    // attention, with every slot and with two of three
    std::vector<uint32_t> visible_ids;
    for (uint32_t i = 0; i < PAGES * PAGE; ++i)
        if (i % 3 != 0) visible_ids.push_back(i);
    GpuRoaring visible = upload_from_ids(visible_ids.data(), static_cast<uint32_t>(visible_ids.size()), PAGES * PAGE);
    Dev<int32_t> sel(2 * COLS * PAGE), sel_len(2), limits(tokens);
    paged_select(visible, PAGES, PAGE, table.p, COLS, COLS, starts.p, kv_len.p, 2, tokens, sel.p, COLS * PAGE, sel_len.p,
                 limits.p);
    Dev<float> lse(tokens * HEADS);
    for (const bool filtered : {false, true}) {
        PagedAttentionArgs a{};
        a.q = dq.p;
        a.out = out.p;
        a.q_token_stride = a.out_token_stride = HEADS * DIM;
        a.q_head_stride = a.out_head_stride = DIM;
        a.lse = lse.p;
        a.n_tokens = tokens;
        a.n_heads = HEADS;
        a.n_requests = 2;
        a.d_starts = starts.p;
        a.d_kv_len = kv_len.p;
        a.d_table = table.p;
        a.table_cols = a.table_stride = COLS;
        if (filtered) {
            a.d_sel = sel.p;
            a.sel_stride = COLS * PAGE;
            a.d_sel_len = sel_len.p;
            a.d_limits = limits.p;
        }
        a.scale = 0.125f;
        a.causal = 1;
        paged_attention(a, cache);
        HIP_OK(hipDeviceSynchronize());
        const auto h_out = out.host();
        const auto h_lse = lse.host();
        double worst = 0;
        for (uint32_t t = 0; t < tokens; ++t) {
            const uint32_t first = t < 70 ? 0 : 70;
            for (uint32_t h = 0; h < HEADS; ++h) {
                std::vector<double> p, o(DIM, 0.0);
                std::vector<uint32_t> seen;
                double sum = 0;
                for (uint32_t j = first; j <= t; ++j) {
                    if (filtered && h_slots[j] % 3 == 0) continue;
                    double s = 0;
                    for (uint32_t d = 0; d < DIM; ++d)
                        s += static_cast<double>(q[(t * HEADS + h) * DIM + d]) * static_cast<double>(k[(j * KV + h / 2) * DIM + d]);
                    p.push_back(std::exp(s * 0.125));
                    sum += p.back();
                    seen.push_back(j);
                }
                for (size_t i = 0; i < seen.size(); ++i)
                    for (uint32_t d = 0; d < DIM; ++d) o[d] += p[i] / sum * static_cast<double>(v[(seen[i] * KV + h / 2) * DIM + d]);
                for (uint32_t d = 0; d < DIM; ++d)
                    worst = std::max(worst, std::fabs(o[d] - static_cast<double>(h_out[(t * HEADS + h) * DIM + d])));
                if (seen.empty())
                    CHECK(std::isinf(h_lse[t * HEADS + h]));
                else
                    CHECK(std::fabs(std::log(sum) - h_lse[t * HEADS + h]) < 1e-4);
            }
        }
        CHECK(worst < 4e-3);  // values up to 4: two roundings of f16
    }

    // beams: the best tokens are allowed ones
    constexpr uint32_t W = 3, V = 500, K = 3;
    std::vector<float> scores(W * V), cum = {-1.0f, -2.0f, -0.5f};
    for (auto& x : scores) x = normal(rng);
    std::vector<uint32_t> tokens_allowed;
    for (uint32_t i = 0; i < V; i += 7) tokens_allowed.push_back(i);
    GpuRoaring allowed = upload_from_ids(tokens_allowed.data(), static_cast<uint32_t>(tokens_allowed.size()), V);
    Dev<float> d_scores(scores), d_cum(cum), best(K);
    Dev<int32_t> token(K), parent(K);
    beam_select(d_scores.p, CR_F32, 1, W, V, W * V, V, d_cum.p, nullptr, &allowed, nullptr, 0, K, best.p, token.p, parent.p);
    std::vector<int32_t> states = {10, 11, 20, 21, 30, 31};
    Dev<int32_t> d_states(states), moved(2 * K);
    beam_reorder(d_states.p, parent.p, 1, W, K, 8, 8, 8, nullptr, 0, moved.p);
    HIP_OK(hipDeviceSynchronize());
    const auto h_best = best.host();
    const auto h_token = token.host(), h_parent = parent.host(), h_moved = moved.host();
    std::vector<std::pair<float, uint32_t>> truth;
    for (uint32_t w = 0; w < W; ++w)
        for (uint32_t i = 0; i < V; i += 7) truth.push_back({-(cum[w] + scores[w * V + i]), w * V + i});
    std::sort(truth.begin(), truth.end());
    for (uint32_t i = 0; i < K; ++i) {
        CHECK(h_best[i] == -truth[i].first && static_cast<uint32_t>(h_parent[i]) * V + h_token[i] == truth[i].second);
        CHECK(h_moved[2 * i] == 10 * (h_parent[i] + 1) && h_moved[2 * i + 1] == 10 * (h_parent[i] + 1) + 1);
    }

    // refusals throw
    bool threw = false;
    try {
        paged_plan(free_pages, PAGES, 12, d_cached.p, d_new.p, 2, table.p, COLS, COLS, slots.p, tokens, starts.p, kv_len.p,
                   taken.p, 16, counts.p);
    } catch (const std::runtime_error&) {
        threw = true;
    }
    CHECK(threw);
    for (GpuRoaring* g : {&free_pages, &visible, &allowed}) gpu_roaring_free(*g);
    if (g_fail) return 1;
    std::puts("serving_check: OK");
    return 0;
}
