// Attention over a 4-bit cache: the checks of a call, the choice of the kernel, and what each key gained in weight.
#include "attention4.h"
#include "linear4.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace lb_a4;

struct Mass {
    const float* mass;
    float* total;
    const int32_t* rows;
    int64_t mass_stride, mass_head_stride, total_stride, total_head_stride;
    int n_mass;
};

// total = mass + the sum over a request's rows of 2^(score - log_sum), a thread a key.  The rows come in their order, so the sum does not depend on the launch.  The scores come from the attention
// kernel by way of memory, a row's 32-bit numbers a key, as a weight needs its row's whole sum: a launch, and 4 bytes a row and key each way (16 requests of 4,096 keys at most, with attention 29.8 us).
__global__ void __launch_bounds__(256)
attention4_mass_kernel(const Call c, const Mass w) {
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int seq = blockIdx.z, kvh = blockIdx.y, key = blockIdx.x * 256 + threadIdx.x;
    const Portion part = portion_of(c, seq);
    const int limit = min(c.max_keys, c.table_stride << c.pages.page_shift) - 1, newest = min(part.place + part.count - 1, limit);
    if (part.count <= 0 || key > newest) return;
    const int r = w.rows != nullptr ? w.rows[seq] : seq;
    if ((unsigned)r >= (unsigned)w.n_mass) return;
    const int64_t unit = ((int64_t)seq * c.pages.n_kv_head + kvh) * c.max_rows;
    const float* scores = c.scores + unit * c.score_keys + key;
    const float* log_sums = c.log_sums + unit;
    float sum = 0.0f;
    for (int token = 0; token < part.count; ++token) {
        const int place = min(part.place + token, limit);
        if (key > place || key < lb_first_visible(max(place, 0), c.window)) continue;
        for (int h = 0; h < c.per; ++h) {
            const int row = token * c.per + h;
            sum += exp2f(scores[(int64_t)row * c.score_keys] - log_sums[row]);
        }
    }
    const int64_t at = (int64_t)r * w.mass_stride + (int64_t)kvh * w.mass_head_stride + key;
    w.total[(int64_t)r * w.total_stride + (int64_t)kvh * w.total_head_stride + key] = w.mass[at] + sum;
}

constexpr int kMostMassTokens = 64;
thread_local int g_withhold_next = 0;            // this thread's next call's kernels leave barriers unsignalled (tests)

// How a call runs.
struct Plan {
    bool many;
    RowsPlan rows;
    TilesPlan tiles;
    int64_t scores, log_sums, partial, starts, bytes;       // offsets in the scratch memory
};

int check(const lb_attention4_args* args, Call* c, Plan* p) {
    LB_CHECK_ARG(args != nullptr, "attention4: no arguments");
    const lb_attention4_args& a = *args;
    if (int rc = lb_c4::pages_of(a.cache, "attention4", &c->pages)) return rc;
    LB_CHECK_ARG(a.n_head > 0 && a.n_head % a.cache->n_kv_head == 0, "attention4: %d heads over %d key/value heads", a.n_head, a.cache->n_kv_head);
    LB_CHECK_ARG(a.n_seq >= 0 && a.n_seq <= 65535 && a.n_tokens >= 0, "attention4: %d requests (up to 65535), %d tokens", a.n_seq, a.n_tokens);
    LB_CHECK_ARG(a.q_start != nullptr || a.n_tokens >= a.n_seq, "attention4: %d requests, %d tokens", a.n_seq, a.n_tokens);
    LB_CHECK_ARG(a.max_q_len > 0 && (a.q_start != nullptr || a.max_q_len == 1), "attention4: portions of up to %d tokens", a.max_q_len);
    LB_CHECK_ARG(a.max_keys > 0 && a.table_stride > 0 && (int64_t)a.table_stride * a.cache->page_size <= INT32_MAX, "attention4: up to %d keys, tables of %d pages", a.max_keys,
                 a.table_stride);
    const int64_t rows = (int64_t)a.max_q_len * (a.n_head / a.cache->n_kv_head);
    LB_CHECK_ARG(rows <= 1 << 22 && (rows + 7) / 8 * a.cache->n_kv_head <= 1 << 22 && a.cache->n_kv_head <= 65535, "attention4: %d tokens of %d heads are more than one launch takes", a.max_q_len,
                 a.n_head);
    LB_CHECK_ARG(a.total == nullptr || (a.mass != nullptr && a.max_q_len <= kMostMassTokens), "attention4: the keys' weights come from portions of up to %d tokens", kMostMassTokens);
    LB_CHECK_ARG(a.total == nullptr || (a.n_mass >= 0 && a.mass_stride >= 0 && a.mass_head_stride >= 0 && a.total_stride >= 0 && a.total_head_stride >= 0),
                 "attention4: weights of no size");
    const int keys = std::min(a.max_keys, a.table_stride * a.cache->page_size), n_sm = linear4_sm_count();
    c->q = static_cast<const __nv_bfloat16*>(a.q);
    c->q_start = a.q_start;
    c->last = a.last;
    c->table = a.block_table;
    c->out = static_cast<__nv_bfloat16*>(a.out);
    c->distance = a.distance;
    c->sink = a.sink;
    c->q_stride = a.q_stride;
    c->out_stride = a.out_stride;
    c->table_stride = a.table_stride;
    c->n_seq = a.n_seq;
    c->n_tokens = a.n_tokens;
    c->n_head = a.n_head;
    c->per = a.n_head / a.cache->n_kv_head;
    c->max_rows = (int)rows;
    c->score_keys = keys;
    c->max_keys = a.max_keys;
    c->window = a.window;
    c->scale = a.scale;
    c->soft_cap = a.soft_cap;
    c->withhold = 0;
    // What lies in the scratch memory: scores and divisors for the keys' weights, states, where requests' tiles start.
    auto up = [](int64_t n) { return (n + 15) / 16 * 16; };
    const int64_t units = (int64_t)a.n_seq * a.cache->n_kv_head;
    // (Under a window a request's rows see no more keys than it and the portion have, and what rounds them to tiles.)
    const int seen = a.window == 0 ? keys : (int)std::min<int64_t>(keys, std::abs((int64_t)a.window) + a.max_q_len + 2 * lb_c4::kBlockKeys);
    p->rows = rows_plan(a.n_seq, a.cache->n_kv_head, (int)rows, seen, a.cache->head_dim, n_sm);
    p->tiles = tiles_plan(a.n_seq, a.cache->n_kv_head, c->per, (int)rows, keys, a.window, a.cache->head_dim, n_sm);
    // The tcgen05 kernel takes a call where the estimates (rows_plan, tiles_plan), which are from both kernels' times on 84 calls of 1 to 128 tokens a request, say so: 8 requests on 2,048 keys, 32 heads
    // over 8: 8 tokens each 34 us on the kernel for few rows, 36 on this; 16 tokens 52 / 36; 1 request on 2,048 keys: 32 tokens 20 / 24, 128 tokens 51 / 32.
    p->many = a.total == nullptr && p->tiles.us < p->rows.us;
    // (The tcgen05 kernel takes 2^42 pairs of a query row and a key in some three seconds.  Under a window a tile of 256 rows walks that many keys, its rows' own and what rounds them.)
    const int64_t walked = a.window == 0 ? keys : std::min<int64_t>(keys, std::abs((int64_t)a.window) + 512);
    LB_CHECK_ARG(p->many ? a.cache->n_kv_head * rows * walked <= (int64_t)1 << 42 : p->rows.fits, "attention4: a request of %d rows and %d keys is more than one launch takes", (int)rows, keys);
    p->scores = 0;
    p->log_sums = a.total != nullptr ? up(units * rows * keys * 4) : 0;
    p->partial = p->log_sums + (a.total != nullptr ? up(units * rows * 4) : 0);
    if (p->many) {
        p->starts = p->bytes = p->partial + up(p->tiles.states);
    } else {
        p->starts = p->partial + up(p->rows.states);
        p->bytes = p->starts + up(p->rows.starts);
    }
    uint8_t* at = static_cast<uint8_t*>(a.scratch);
    c->scores = a.total != nullptr ? reinterpret_cast<float*>(at + p->scores) : nullptr;
    c->log_sums = a.total != nullptr ? reinterpret_cast<float*>(at + p->log_sums) : nullptr;
    c->partial = reinterpret_cast<float*>(at + p->partial);
    c->starts = reinterpret_cast<int*>(at + p->starts);
    return LB_OK;
}

}  // namespace

namespace lb_a4 {

bool rows_apart(const WeightRows& a) {
    if (a.n <= 0) return true;
    if ((a.heads > 1 && a.head < a.width) || (a.n > 1 && a.row < a.width)) return false;
    return a.heads <= 1 || a.n <= 1 || a.row >= (a.heads - 1) * a.head + a.width || a.head >= (a.n - 1) * a.row + a.width;
}

bool rows_disjoint(const WeightRows& a, const WeightRows& b) {
    if (a.n <= 0 || b.n <= 0 || a.width <= 0 || b.width <= 0) return true;
    auto stride = [](int64_t s, int64_t n) { return n > 1 ? s : 0; };                       // (that of a single row is any number)
    auto first = [](const WeightRows& w) { return (int64_t)(reinterpret_cast<uintptr_t>(w.at) / sizeof(float)); };
    auto last = [&](const WeightRows& w) { return first(w) + stride(w.row, w.n) * (w.n - 1) + stride(w.head, w.heads) * (w.heads - 1) + w.width - 1; };
    if (last(a) < first(b) || last(b) < first(a)) return true;
    const int64_t row = std::max(stride(a.row, a.n), stride(b.row, b.n)), head = std::max(stride(a.head, a.heads), stride(b.head, b.heads));
    if ((a.n > 1 && a.row != row) || (b.n > 1 && b.row != row) || (a.heads > 1 && a.head != head) || (b.heads > 1 && b.head != head)) return false;
    // A row of b starts at x, counted from one of a's: dr rows and dh heads on.  They overlap where -b.width < x < a.width.
    for (int64_t dh = 1 - a.heads; dh < b.heads; ++dh) {
        const int64_t x = first(b) - first(a) + dh * head;
        if (row == 0) {
            if (x > -b.width && x < a.width) return false;
        } else {
            // The least dr that takes x past -b.width.
            const int64_t short_of = 1 - b.width - x, dr = std::max(1 - a.n, short_of >= 0 ? (short_of + row - 1) / row : -(-short_of / row));
            if (dr < b.n && x + dr * row < a.width) return false;
        }
    }
    return true;
}

}  // namespace lb_a4

extern "C" int64_t lb_attention4_scratch(const lb_attention4_args* args) {
    Call c;
    Plan p;
    return check(args, &c, &p) == LB_OK ? p.bytes : 0;
}

extern "C" int lb_attention4_plan(const lb_attention4_args* args, int* plan) {
    Call c;
    Plan p;
    LB_CHECK_ARG(plan != nullptr, "attention4: no place for the plan");
    if (int rc = check(args, &c, &p)) return rc;
    plan[0] = p.many ? 1 : 0;
    plan[1] = p.many ? 256 : p.rows.rows;
    plan[2] = p.many ? p.tiles.splits : p.rows.whole ? 1 : p.rows.blocks;
    plan[3] = p.many || p.rows.whole ? 1 : p.rows.per_row;
    return LB_OK;
}

extern "C" int lb_attention4(const lb_attention4_args* args) {
    Call c;
    Plan p;
    if (int rc = check(args, &c, &p)) return rc;
    const lb_attention4_args& a = *args;
    if (a.n_seq == 0 || a.n_tokens == 0) return LB_OK;
    LB_CHECK_ARG(a.q != nullptr && a.last != nullptr && a.block_table != nullptr && a.out != nullptr, "attention4: a pointer is missing");
    LB_CHECK_ARG(reinterpret_cast<uintptr_t>(a.q) % 2 == 0 && reinterpret_cast<uintptr_t>(a.out) % 2 == 0, "attention4: pointers off their type's alignment");
    const int64_t width = (int64_t)a.n_head * a.cache->head_dim;
    LB_CHECK_ARG(a.n_tokens < 2 || (a.q_stride >= width && a.out_stride >= width), "attention4: rows overlap");
    LB_CHECK_ARG(p.bytes == 0 || (a.scratch != nullptr && reinterpret_cast<uintptr_t>(a.scratch) % 16 == 0), "attention4: scratch memory is missing or not 16-byte aligned");
    if (a.total != nullptr) {
        const int64_t n = a.n_mass, heads = a.cache->n_kv_head, keys = c.score_keys;
        const WeightRows mass = {a.mass, a.mass_stride, a.mass_head_stride, n, heads, keys}, total = {a.total, a.total_stride, a.total_head_stride, n, heads, keys};
        LB_CHECK_ARG(rows_apart(total), "attention4: the keys' weights go to rows that overlap (%lld and %lld numbers apart, of %d keys)", (long long)a.total_stride, (long long)a.total_head_stride,
                     c.score_keys);
        const bool same = a.total == a.mass && (n <= 1 || a.total_stride == a.mass_stride) && (heads <= 1 || a.total_head_stride == a.mass_head_stride);
        LB_CHECK_ARG(same || rows_disjoint(mass, total), "attention4: the keys' weights go to memory that overlaps where they come from, and is not the same");
    }
    if (int rc = device_check("attention4", a.cache->device)) return rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
    c.withhold = g_withhold_next;
    g_withhold_next = 0;
    if (p.many) return many_rows(c, a.cache->head_dim, p.tiles, stream);
    if (int rc = few_rows(c, a.cache->head_dim, p.rows, stream)) return rc;
    if (a.total != nullptr) {
        const Mass w = {a.mass, a.total, a.mass_rows, a.mass_stride, a.mass_head_stride, a.total_stride, a.total_head_stride, a.n_mass};
        LB_CHECK_CUDA(lb_launch_overlapped(attention4_mass_kernel, dim3((c.score_keys + 255) / 256, a.cache->n_kv_head, a.n_seq), dim3(256), 0, stream, c, w));
    }
    return LB_OK;
}

// Tests: the waits of this thread's next call run out.
extern "C" int lb_attention4_withhold_next(int on) {
    g_withhold_next = on;
    return LB_OK;
}
