// The paged cache of include/gradhip.h: gh_cache_*.
#include "api_error.h"
#include "cache_attend.h"
#include "cache_session.h"
#include "device_scope.h"
#include "kernels_cache.h"

#include <climits>
#include <cmath>
#include <cstring>
#include <memory>

namespace gh {

namespace {

[[noreturn]] void refuse(const std::string& why) { throw ApiError{GH_ERR_INVALID_ARGUMENT, "cache: " + why}; }

[[noreturn]] void no_workspace(size_t bytes) {
    throw ApiError{GH_ERR_DEVICE, "cache: no memory for a workspace of " + std::to_string(bytes) + " bytes"};
}

struct DeviceBuffer {
    char* at = nullptr;
    size_t bytes = 0;
    ~DeviceBuffer() {
        if (at) (void)hipFree(at);
    }
    enum Outcome { kThere, kMoved, kNone };
    // Room for so many bytes, contents lost if they have to move; what the stream still does with the old ones is waited for.
    // kNone: there is no memory, not even the old.
    Outcome reserve(size_t want, hipStream_t stream) {
        if (want <= bytes) return kThere;
        HIP_CHECK(hipStreamSynchronize(stream));
        if (at) HIP_CHECK(hipFree(at));
        at = nullptr;
        bytes = 0;
        for (const size_t room : {want + want / 2, want}) {
            const size_t whole = (room + 4095) / 4096 * 4096;
            const hipError_t e = hipMalloc(&at, whole);
            if (e == hipSuccess) {
                bytes = whole;
                return kMoved;
            }
            at = nullptr;
            if (e != hipErrorOutOfMemory) HIP_CHECK(e);
            (void)hipGetLastError();
        }
        return kNone;
    }
    void need(size_t want, hipStream_t stream) {
        if (reserve(want, stream) == kNone) no_workspace(want);
    }
};

// Pinned host memory that a kernel reads, two buffers in turn: a buffer is written again when the kernel that read it is done.
struct Staging {
    struct Slot {
        char* at = nullptr;
        size_t bytes = 0;
        hipEvent_t read = nullptr;
        bool pending = false;
    } slots[2];
    int turn = 0;

    ~Staging() {
        for (Slot& s : slots) {
            if (s.at) (void)hipHostFree(s.at);
            if (s.read) (void)hipEventDestroy(s.read);
        }
    }
    char* reserve(size_t want) {
        turn ^= 1;
        Slot& s = slots[turn];
        if (!s.read) HIP_CHECK(hipEventCreateWithFlags(&s.read, hipEventDisableTiming));
        if (s.pending) HIP_CHECK(hipEventSynchronize(s.read));
        s.pending = false;
        if (want > s.bytes) {
            if (s.at) HIP_CHECK(hipHostFree(s.at));
            s.at = nullptr;
            s.bytes = 0;
            const size_t room = (want + want / 2 + 4095) / 4096 * 4096;
            HIP_CHECK(hipHostMalloc(&s.at, room, hipHostMallocDefault));
            s.bytes = room;
        }
        return s.at;
    }
    // The last reserved buffer's first bytes to the device.
    void send(char* to, size_t bytes, hipStream_t stream) {
        Slot& s = slots[turn];
        const size_t words = (bytes + 15) / 16;
        if (words == 0) return;
        if (words <= kWordsListed) {  // with the launch itself: no trip over the bus, no event
            WordList list;
            std::memcpy(list.words, s.at, bytes);
            hipLaunchKernelGGL(cache_hand_kernel, dim3(1), dim3(256), 0, stream, list, reinterpret_cast<u32x4*>(to), static_cast<int>(words));
            HIP_CHECK(hipGetLastError());
            return;
        }
        const int groups = static_cast<int>(std::min<size_t>(256, (words + 255) / 256));
        hipLaunchKernelGGL(cache_load_kernel, dim3(groups), dim3(256), 0, stream, reinterpret_cast<const u32x4*>(s.at),
                           reinterpret_cast<u32x4*>(to), words);
        HIP_CHECK(hipGetLastError());
        HIP_CHECK(hipEventRecord(s.read, stream));
        s.pending = true;
    }
};

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

constexpr int kMaxHeads = 1024;
constexpr int kMaxPageTokens = 1024;
constexpr int kPlans = 4;
// Prefixes are read in common tiles from this many positions on and where their members would read so many bytes of them in all:
// what common tiles leave are parts, to be joined.  us, eight samples, common and apart: fp32, 12 heads of 64: 256 positions (13 MB)
// 11.3 and 9.1, 512 11.6 and 11.9, 1 k (50 MB) 12.1 and 13.1, 2 k 13.4 and 21.4; bf16, 8 kv heads of 128: 1 k (34 MB) 14.9 and 12.6,
// 2 k 15.5 and 20.9, 4 k 19.0 and 30.1.
constexpr int kLeastShared = 128;
constexpr size_t kLeastSharedBytes = 40u << 20;
// ... unless the parts take more than this: each member leaves one of 16 rows at least, whatever it has.  (One kv head of 128 dims: 8 KB.)
constexpr size_t kMostSharedParts = 512u << 20;
// Few rows of sequences that hold so many bytes in all go to the tiles of many rows beside them: there a single token reads its
// sequence 1.2 (16 bit) to 2.4 (fp32) times as slowly, but a launch of its own behind the other is some 15 us.  us, together and
// apart: bf16, beside a chunk of 200 tokens over 64 MB 49 and 69, over 111 MB 68 and 102, over 269 MB 133 and 168, beside 1000 over 68 MB
// 101 and 110, over 154 MB 176 and 181, over 254 MB 317 and 282; fp32, beside 200 over 27 MB 33 and 38, over 96 MB 60 and 68, over
// 167 MB 99 and 99, beside 1000 over 31 MB 51 and 57, over 101 MB 103 and 95, over 230 MB 190 and 158.
constexpr size_t kTogether16 = 320u << 20, kTogether32 = 100u << 20;

}  // namespace

struct Cache {
    gh_cache_opts o{};
    int device = 0;
    int group = 1;
    int bytes = 4;  // of an element
    CacheLayout layout{};
    PageBook book;
    DeviceBuffer pool, speed, pass, parts, arrived;
    Staging staging;
    hipEvent_t done = nullptr;     // the last call's work, if it was on a stream that the caller made
    hipStream_t stream = nullptr;  // of the last call

    // the open pass
    bool open = false;
    int rows = 0;
    std::vector<PassSeq> seqs;
    std::vector<int> numbers;          // theirs in the book
    std::vector<int> news;
    std::vector<int> forgetful;        // which of them have forgotten positions
    std::vector<SharedPrefix> shared;  // among sequences of few rows
    size_t rows_at = 0, table_at = 0;  // in `pass`

    // its attention, as it was last cut up for a mask
    struct Plan {
        bool valid = false;
        bool causal = true;
        int window = 0, sinks = 0;
        // sequences of few rows and of many go to kernels of their own, one behind the other, unless the few fit beside the many
        struct Launch {
            AttendForm form{};
            AttendPlan cut;
        } launches[2];
        DeviceBuffer items;  // empty for the plan that came with the pass
        const char* at = nullptr;
        const AttendItem* items_of(int i) const { return reinterpret_cast<const AttendItem*>(at + place(i)); }
        const AttendJoin* joins_of(int i) const { return reinterpret_cast<const AttendJoin*>(at + place(i) + items_bytes(i)); }
        const int* maps_of(int i) const { return reinterpret_cast<const int*>(at + place(i) + items_bytes(i) + joins_bytes(i)); }
        size_t bytes() const { return place(2); }
        void write(char* host) const {
            for (int i = 0; i < 2; i++) {
                const AttendPlan& c = launches[i].cut;
                char* to = host + place(i);
                if (!c.items.empty()) std::memcpy(to, c.items.data(), sizeof(AttendItem) * c.items.size());
                if (!c.joins.empty()) std::memcpy(to + items_bytes(i), c.joins.data(), sizeof(AttendJoin) * c.joins.size());
                if (!c.maps.empty()) std::memcpy(to + items_bytes(i) + joins_bytes(i), c.maps.data(), sizeof(int) * c.maps.size());
            }
        }

    private:
        size_t items_bytes(int i) const { return sizeof(AttendItem) * launches[i].cut.items.size(); }
        size_t joins_bytes(int i) const { return sizeof(AttendJoin) * launches[i].cut.joins.size(); }
        size_t place(int n) const {
            size_t sum = 0;
            for (int i = 0; i < n; i++) sum += items_bytes(i) + joins_bytes(i) + round16(sizeof(int) * launches[i].cut.maps.size());
            return sum;
        }
    } plans[kPlans];
    int next_plan = 0;
    bool last_causal = true;  // the mask of the last call: the next pass is planned for it
    int last_window = 0, last_sinks = 0;

    Cache(const gh_cache_opts& opts, int pages, int page_tokens) : o(opts), book(pages, page_tokens) {}
    ~Cache() {
        (void)hipDeviceSynchronize();
        if (done) (void)hipEventDestroy(done);
    }

    AttendForm form_for(int rows_of_sequence, bool sinks) const {
        if (sinks)
            return o.type == GH_F32 ? attend_form_sinks_f32(o.head_dim, rows_of_sequence)
                 : o.type == GH_BF16 ? attend_form_sinks_bf16(o.head_dim, rows_of_sequence)
                                     : attend_form_sinks_f16(o.head_dim, rows_of_sequence);
        return o.type == GH_F32 ? attend_form_f32(o.head_dim, rows_of_sequence)
             : o.type == GH_BF16 ? attend_form_bf16(o.head_dim, rows_of_sequence)
                                 : attend_form_f16(o.head_dim, rows_of_sequence);
    }

    // Calls on one cache run in their order whatever streams they name: each waits for the one before, which left an event
    // behind, or was on the default stream and gets one now.  Handles are not compared: a stream may be gone, and its handle another
    // one's (a wait for what the same stream did is free: one-token calls 8.2 to 8.5 us with it, 8.3 to 8.7 without).  The handle that names a stream of each thread's own is refused: waits on events did not hold it back (a second thread's
    // call was done 7 ms before the first's).  So is a stream under capture: a call would be replayed with the pages and lengths of
    // today.
    struct Turn {
        Cache& c;
        Turn(Cache& cache, void* hip_stream) : c(cache) {
            const hipStream_t st = static_cast<hipStream_t>(hip_stream);
            if (st == hipStreamPerThread) refuse("hipStreamPerThread: another stream in every thread");
            hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
            HIP_CHECK(hipStreamIsCapturing(st, &status));
            if (status != hipStreamCaptureStatusNone)
                throw ApiError{GH_ERR_RUNTIME, "cache: the stream is being captured into a graph; a replay would use the pages of the "
                                               "pass that was open at capture"};
            if (st != nullptr || c.stream != nullptr) {
                if (!c.done) HIP_CHECK(hipEventCreateWithFlags(&c.done, hipEventDisableTiming));
                if (c.stream == nullptr) HIP_CHECK(hipEventRecord(c.done, nullptr));
                HIP_CHECK(hipStreamWaitEvent(st, c.done, 0));
                c.stream = st;
            }
        }
        ~Turn() {
            if (c.stream != nullptr) (void)hipEventRecord(c.done, c.stream);
        }
        Turn(const Turn&) = delete;
        Turn& operator=(const Turn&) = delete;
    };

    void close() {
        open = false;
        for (Plan& p : plans) p.valid = false;
    }

    void copy_pages(const char* from, const std::vector<PageCopy>& copies) {
        const int runs = o.layers * 2 * o.kv_heads, token_bytes = o.head_dim * bytes;
        for (size_t at = 0; at < copies.size(); at += kListed) {
            const int n = static_cast<int>(std::min<size_t>(kListed, copies.size() - at));
            CopyList list;
            std::memcpy(list.copies, copies.data() + at, sizeof(PageCopy) * static_cast<size_t>(n));
            const long long pieces = static_cast<long long>(runs) * static_cast<long long>((layout.run_bytes + 4095) / 4096);
            const int x = static_cast<int>(std::max(1ll, std::min<long long>(pieces, 2048 / n)));  // ~2048 workgroups: eight per compute unit
            hipLaunchKernelGGL(cache_copy_kernel, dim3(x, n), dim3(256), 0, stream, from, pool.at, layout.page_bytes, runs,
                               static_cast<int>(layout.run_bytes / 16), token_bytes, list);
            HIP_CHECK(hipGetLastError());
        }
    }

    // How the pass's attention is cut, and room for what its parts leave: with common prefixes, or without them where those would
    // leave more than there is room for.
    void cut(Plan& plan, bool causal, int window, int sinks) {
        plan.causal = causal;
        plan.window = window;
        plan.sinks = sinks;
        if (window == 0 && !shared.empty()) {
            const Room room = cut_with(plan, shared);
            if (room.parts <= kMostSharedParts && reserve(room)) return;
        }
        const Room room = cut_with(plan, {});
        if (room.parts >> 32) refuse("a pass whose parts take more than 4 GB");
        if (!reserve(room)) no_workspace(room.parts);
    }

private:
    struct Room {
        size_t parts = 0, counters = 0;  // bytes
    };

    // false, and no plan is valid any more, if there is no memory.
    bool reserve(const Room& room) {
        const bool there = parts.reserve(room.parts, stream) != DeviceBuffer::kNone;
        const auto counted = there ? arrived.reserve(room.counters, stream) : DeviceBuffer::kNone;
        if (counted == DeviceBuffer::kMoved) HIP_CHECK(hipMemsetAsync(arrived.at, 0, arrived.bytes, stream));
        if (counted == DeviceBuffer::kNone)
            for (Plan& p : plans) p.valid = false;
        return counted != DeviceBuffer::kNone;
    }

    Room cut_with(Plan& plan, const std::vector<SharedPrefix>& prefixes) const {
        const bool causal = plan.causal;
        const int window = plan.window, sinks = plan.sinks;
        Room room;
        int few = few_rows(o.type);
        if (prefixes.empty()) {
            size_t held = 0;  // by the sequences of few rows
            bool many = false;
            for (size_t i = 0; i < news.size(); i++) {
                if (news[i] == 0) continue;
                int k0, k1;
                visible_span(seqs[i], 0, news[i] * group, group, causal, window, k0, k1);
                if (news[i] * group > few) {
                    many = true;
                } else {
                    held += static_cast<size_t>(k1 - k0 + std::min(sinks, k0)) * o.kv_heads * o.head_dim * 2 * static_cast<size_t>(bytes);
                }
            }
            if (many && held <= (bytes == 4 ? kTogether32 : kTogether16)) few = 0;
        }
        for (int many = 0; many < 2; many++) {
            Plan::Launch& l = plan.launches[many];
            std::vector<int> mine(news.size(), 0);
            int most = 0;
            for (size_t i = 0; i < news.size(); i++)
                if ((news[i] * group > few) == (many == 1)) {
                    mine[i] = news[i];
                    most = std::max(most, news[i] * group);
                }
            l.form = form_for(most, sinks > 0);
            // (a launch holds at most 2^32 threads)
            if (static_cast<long long>(most + 15) / 16 * static_cast<long long>(news.size()) * o.kv_heads > (1 << 22)) {
                long long tiles = 0;
                for (int n : mine) tiles += (static_cast<long long>(n) * group + l.form.height - 1) / l.form.height;
                if (tiles * o.kv_heads > (1 << 22)) refuse("a pass of more than 2^22 tiles of rows");
            }
            const bool tiles = l.form.height == kTileRows;
            // Few rows: several workgroups to a compute unit, so that ragged sequences end together (16 sequences of 4 k to
            // 32 k positions, 32/8 heads of 128 in bf16: 256 us, with half as many 262, a quarter 275); parts below 64 KB of
            // keys cost more to join than they save (13 sequences of up to 1 k positions, fp32: 14.5 us, 15.5 in parts of
            // half that), and more than 64 parts of a tile are a long join (one sequence of 128 k positions: 61 us, 71 in 128).
            // Many rows: as many as are resident at once and no more (1024 rows over 16 k positions, bf16: 113 us, 154 with half as
            // many; over 4 k, fp32: 106, 140 with 576), and no more parts than the last one joins in the time that they
            // save (128 rows, bf16: 1 k positions 31 us in 4 parts, 34 in 8; 4 k 44 in 8, 75 in 32; 16 k 75 in 16, 142 in 64;
            // fp32 products take some six times as long: 4 k 48 in 16, 57 in 8, 54 in 32; 16 k 90 in 32, 98 in 16, 121 in 64).
            const int resident = o.head_dim > 128 ? 256 : 512;
            // Windows and sinks: few rows' spans are of one length, nothing has to be evened out, so one workgroup to a compute unit and
            // nothing split that ends no sooner for it (16 sequences with windows of 4 k, 32/8 heads of 128 in bf16: 54 us, with 512
            // workgroups 60, 768 63, 2048 77; 4 sequences 20.2 and 25.8; 64 with windows of 512, 12 heads of 64 in fp32: 40.4 us, in two parts
            // each 47.8; only ragged ones lose a little, 16 of 1 to 4 k, fp32: 95 us, with 512 91).  Windows alone have the rule of all positions, which is
            // not the quickest for them (the same calls on one set of inputs, with sinks and without: 47 and 67 us, 35 and 41).
            const int workgroups = tiles ? resident : sinks > 0 ? 256 : bytes == 4 ? 1024 : 2048;
            const int least = tiles ? 128 : bytes == 4 || sinks > 0 ? 256 : 384;
            l.cut = plan_attend(seqs, mine,
                                AttendCut{group, o.kv_heads, l.form.height, causal, window, workgroups, least, 64,
                                          !tiles ? 0 : bytes == 4 ? 16 : 64, tiles ? resident : 0, sinks, !tiles && sinks > 0 ? 1 : 0},
                                many ? std::vector<SharedPrefix>{} : prefixes);
            room.parts = std::max(room.parts, static_cast<size_t>(l.cut.parts) * o.kv_heads * l.form.part_floats * sizeof(float));
            room.counters = std::max(room.counters, l.cut.joins.size() * o.kv_heads * sizeof(unsigned));
        }
        return room;
    }
};

static void check_rows(const char* what, const gh_rows* r) {
    if (!r || !r->data) refuse(std::string(what) + " is null");
    if (r->row_stride < 0 || r->head_stride < 0) refuse(std::string(what) + " has a negative stride");
}

// Rows that are written must not lie on top of one another.
static void check_apart(const char* what, const gh_rows* r, long long rows, int heads, int dim) {
    const long long row = r->row_stride, head = r->head_stride;
    const bool heads_inside = (heads == 1 || head >= dim) && (rows == 1 || row >= (heads - 1) * head + dim);
    const bool rows_inside = (rows == 1 || row >= dim) && (heads == 1 || head >= (rows - 1) * row + dim);
    if (!heads_inside && !rows_inside) refuse(std::string(what) + "'s rows overlap");
}

static bool aligned(const gh_rows* r, int bytes, bool one_row, bool one_head) {
    return reinterpret_cast<uintptr_t>(r->data) % 16 == 0 && (one_row || r->row_stride * bytes % 16 == 0)
           && (one_head || r->head_stride * bytes % 16 == 0);
}

static CacheRows cache_rows(const gh_rows* r) { return CacheRows{static_cast<char*>(r->data), r->row_stride, r->head_stride}; }

static gh_cache_opts checked(const gh_cache_opts& in) {
    gh_cache_opts o = in;
    if (o.page_tokens == 0) o.page_tokens = 64;
    if (o.layers < 1 || o.layers > 4096) refuse("layers must be 1 to 4096");
    if (o.kv_heads < 1 || o.heads < 1 || o.heads > kMaxHeads) refuse("heads must be 1 to 1024");
    if (o.heads % o.kv_heads != 0) refuse("heads must be a multiple of kv_heads");
    if (o.head_dim < 8 || o.head_dim > 256 || o.head_dim % 8 != 0) refuse("head_dim must be a multiple of 8, 8 to 256");
    if (o.type != GH_F32 && o.type != GH_BF16 && o.type != GH_F16) refuse("unknown element type");
    if (o.page_tokens < 16 || o.page_tokens > kMaxPageTokens || (o.page_tokens & (o.page_tokens - 1)))
        refuse("page_tokens must be a power of two, 16 to 1024");
    if (o.pages < 1 || o.pages > (INT_MAX - kMaxPageTokens) / o.page_tokens) refuse("pages x page_tokens must be 1 to 2^31");
    if (!(o.rope_base >= 0.0f) || std::isinf(o.rope_base)) refuse("rope_base must be a finite number, 0 for no rotation");
    return o;
}

static std::unique_ptr<Cache> create_cache(const gh_cache_opts& in) {
    const gh_cache_opts o = checked(in);
    require_gpu();
    auto c = std::make_unique<Cache>(o, o.pages, o.page_tokens);
    HIP_CHECK(hipGetDevice(&c->device));
    c->group = o.heads / o.kv_heads;
    c->bytes = o.type == GH_F32 ? 4 : 2;
    CacheLayout& l = c->layout;
    l.run_bytes = static_cast<size_t>(o.page_tokens) * o.head_dim * c->bytes;
    l.page_bytes = l.run_bytes * o.kv_heads * 2 * o.layers;
    l.kv_heads = o.kv_heads;
    l.dim = o.head_dim;
    l.layers = o.layers;
    while ((1 << l.page_shift) < o.page_tokens) l.page_shift++;
    const size_t bytes = l.page_bytes * static_cast<size_t>(o.pages);
    const hipError_t e = hipMalloc(&c->pool.at, bytes);
    if (e == hipErrorOutOfMemory) {
        (void)hipGetLastError();
        throw ApiError{GH_ERR_DEVICE, "cache: no memory for a pool of " + std::to_string(bytes) + " bytes"};
    }
    HIP_CHECK(e);
    c->pool.bytes = bytes;
    l.pool = c->pool.at;
    if (o.rope_base > 0.0f) {
        // in turns per position, 64 bits
        std::vector<double> speed(static_cast<size_t>(o.head_dim) / 2);
        for (size_t j = 0; j < speed.size(); j++)
            speed[j] = std::pow(static_cast<double>(o.rope_base), -2.0 * static_cast<double>(j) / o.head_dim) / (2.0 * M_PI);
        HIP_CHECK(hipMalloc(&c->speed.at, speed.size() * sizeof(double)));
        c->speed.bytes = speed.size() * sizeof(double);
        HIP_CHECK(hipMemcpy(c->speed.at, speed.data(), c->speed.bytes, hipMemcpyHostToDevice));
    }
    return c;
}

// A sequence's pages' contents into a new sequence of `to`.
static int copy_sequence(Cache& from, Cache& to, int seq, void* stream) {
    const int length = from.book.at(seq).length;
    const Cache::Turn turn(to, stream);
    std::unique_ptr<Cache::Turn> other;
    if (&from != &to) other = std::make_unique<Cache::Turn>(from, stream);
    std::vector<PageCopy> copies;
    copies.reserve(from.book.at(seq).pages.size());
    const int id = to.book.add_like(from.book.at(seq));
    to.close();  // (a refusal leaves the open pass)
    const std::vector<int>& a = from.book.at(seq).pages;
    const std::vector<int>& b = to.book.at(id).pages;
    for (size_t i = 0; i < a.size(); i++)
        if (a[i] != PageBook::kNone) copies.push_back({a[i], b[i], std::min(from.o.page_tokens, length - static_cast<int>(i) * from.o.page_tokens)});
    to.copy_pages(from.pool.at, copies);
    return id;
}

static void extend_cache(Cache& c, const int32_t* seqs, const int32_t* counts, int n, void* stream) {
    long long rows = 0, pages = 0;
    c.close();
    for (int i = 0; i < n; i++) {
        const int length = c.book.at(seqs[i]).length;
        if (counts[i] < 0) refuse("negative number of positions");
        rows += counts[i];
        pages += (static_cast<long long>(length) + counts[i] + c.o.page_tokens - 1) / c.o.page_tokens - c.book.hole_of(c.book.at(seqs[i])).pages();
        if (rows > (1 << 23) || rows * c.group > (1 << 30) || pages > (1 << 28)) refuse("a pass of more than 2^23 rows");
    }
    const Cache::Turn turn(c, stream);
    // everything that may be refused or find no memory comes before the pages change hands
    c.seqs.assign(static_cast<size_t>(n), PassSeq{});
    c.news.assign(counts, counts + n);
    c.numbers.assign(seqs, seqs + n);
    c.forgetful.clear();
    int row0 = 0, table = 0;
    for (int i = 0; i < n; i++) {
        const int first = c.book.at(seqs[i]).length;
        if (counts[i] > INT_MAX - kMaxPageTokens - first) throw ApiError{GH_ERR_OUT_OF_RANGE, "cache: a sequence of more than 2^31 positions"};
        const int hole = c.book.hole_of(c.book.at(seqs[i])).pages();
        c.seqs[static_cast<size_t>(i)] = {first + counts[i], first, row0, table, hole};
        row0 += counts[i];
        table += c.book.pages_for(first + counts[i]) - hole;
    }
    // prefixes that sequences of few rows share are read once for all of them
    std::vector<const std::vector<int>*> pages_of(static_cast<size_t>(n));
    std::vector<char> few(static_cast<size_t>(n));
    for (int i = 0; i < n; i++) {
        pages_of[static_cast<size_t>(i)] = &c.book.at(seqs[i]).pages;
        const PageBook::Sequence& s = c.book.at(seqs[i]);
        const bool whole = s.gone_from == s.gone_to;
        if (!whole && counts[i] > 0) c.forgetful.push_back(i);
        few[static_cast<size_t>(i)] = whole && counts[i] > 0 && static_cast<long long>(counts[i]) * c.group <= kFewTile;
    }
    c.shared = shared_prefixes(pages_of, c.seqs, few, c.o.page_tokens, kLeastShared);
    const size_t position = static_cast<size_t>(c.o.kv_heads) * c.o.head_dim * 2 * static_cast<size_t>(c.bytes);
    const auto slight = [&](const SharedPrefix& s) { return position * static_cast<size_t>(s.prefix) * s.members.size() < kLeastSharedBytes; };
    c.shared.erase(std::remove_if(c.shared.begin(), c.shared.end(), slight), c.shared.end());
    Cache::Plan& plan = c.plans[0];
    c.cut(plan, c.last_causal, c.last_window, c.last_sinks);
    c.next_plan = 1;
    const size_t rows_at = 0, table_at = round16(sizeof(RowAt) * static_cast<size_t>(rows));
    const size_t items_at = table_at + round16(sizeof(int) * static_cast<size_t>(table));
    const size_t bytes = items_at + plan.bytes();
    c.pass.need(bytes, c.stream);
    char* host = c.staging.reserve(bytes);
    const std::vector<PageCopy> copies = c.book.extend(seqs, counts, n);

    RowAt* row = reinterpret_cast<RowAt*>(host + rows_at);
    int* page = reinterpret_cast<int*>(host + table_at);
    for (int i = 0; i < n; i++) {
        const PageBook::Sequence& s = c.book.at(seqs[i]);
        page = c.book.write_list(s, page);
        for (int t = s.length - counts[i]; t < s.length; t++)
            *row++ = {s.pages[static_cast<size_t>(t >> c.layout.page_shift)] * c.o.page_tokens + (t & (c.o.page_tokens - 1)), t};
    }
    plan.write(host + items_at);
    c.staging.send(c.pass.at, bytes, c.stream);
    c.copy_pages(c.pool.at, copies);
    plan.at = c.pass.at + items_at;
    plan.valid = true;
    c.rows_at = rows_at;
    c.table_at = table_at;
    c.rows = static_cast<int>(rows);
    c.open = true;
}

static void check_pass(const Cache& c, int layer) {
    if (!c.open)
        throw ApiError{GH_ERR_RUNTIME, "cache: no pass is open (extend opens one; fork, truncate, forget, drop, compact and a copy into the cache end it)"};
    if (layer < 0 || layer >= c.o.layers) throw ApiError{GH_ERR_OUT_OF_RANGE, "cache: no layer " + std::to_string(layer)};
}

static void append_rows(Cache& c, int layer, const gh_rows* k, const gh_rows* v, const gh_rows* q, const gh_rows* q_out, bool rotate, void* stream) {
    check_pass(c, layer);
    if ((q == nullptr) != (q_out == nullptr)) refuse("queries and a place for them go together");
    if (c.rows == 0) return;
    const int dim = c.o.head_dim;
    check_rows("k", k);
    check_rows("v", v);
    if (q) {
        check_rows("q", q);
        check_rows("q_out", q_out);
        check_apart("q_out", q_out, c.rows, c.o.heads, dim);
    }
    const DeviceScope on(c.device);
    const Cache::Turn turn(c, stream);
    AppendParams p{};
    p.cache = c.layout;
    p.k = cache_rows(k);
    p.v = cache_rows(v);
    const bool one_row = c.rows == 1, one_kv = c.o.kv_heads == 1, one_head = c.o.heads == 1;
    p.vector_rows = aligned(k, c.bytes, one_row, one_kv) && aligned(v, c.bytes, one_row, one_kv);
    if (q) {
        p.q = cache_rows(q);
        p.q_out = cache_rows(q_out);
        p.vector_rows = p.vector_rows && aligned(q, c.bytes, one_row, one_head) && aligned(q_out, c.bytes, one_row, one_head);
    }
    p.rows = reinterpret_cast<const RowAt*>(c.pass.at + c.rows_at);
    p.speed = rotate ? reinterpret_cast<const double*>(c.speed.at) : nullptr;
    p.layer = layer;
    p.heads = c.o.heads;
    const auto kernel = c.o.type == GH_F32 ? cache_append_kernel<kCacheF32>
                      : c.o.type == GH_BF16 ? cache_append_kernel<kCacheBf16>
                                            : cache_append_kernel<kCacheF16>;
    hipLaunchKernelGGL(kernel, dim3(c.rows), dim3(256), 0, c.stream, p);
    HIP_CHECK(hipGetLastError());
}

// Rows see nothing that is forgotten: it lies between the sinks and the first row's window.
static void check_forgotten(const Cache& c, int window, int sinks) {
    for (int i : c.forgetful) {
        const PassSeq& s = c.seqs[static_cast<size_t>(i)];
        const PageBook::Sequence& held = c.book.at(c.numbers[static_cast<size_t>(i)]);
        const int low = window > 0 ? std::max(0, s.first - window + 1) : 0;
        if (window == 0 || held.gone_from < sinks || held.gone_to > low)
            throw ApiError{GH_ERR_OUT_OF_RANGE, "cache: sequence " + std::to_string(c.numbers[static_cast<size_t>(i)]) + " has forgotten positions "
                                                    + std::to_string(held.gone_from) + " to " + std::to_string(held.gone_to) + ", which a row would see"};
    }
}

static void attend(Cache& c, int layer, const gh_rows* q, const gh_rows* out, float scale, bool causal, int window, int sinks, void* stream) {
    check_pass(c, layer);
    if (window < 0) refuse("negative window");
    if (sinks < 0) refuse("negative number of sinks");
    sinks = window == 0 ? 0 : std::min(sinks, INT_MAX - 15);  // (rounded up to 16, and behind any position)
    if (!(scale >= 0.0f) || std::isinf(scale)) refuse("scale must be a finite number, 0 for 1 / sqrt(head_dim)");
    const float scale2 = (scale > 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(c.o.head_dim))) * 1.44269504088896340736f;  // for powers of two
    if (std::isinf(scale2)) refuse("scale must be below 2.35e38");  // (2^128 / log2(e): infinity times a score of zero is none)
    if (c.rows == 0) return;
    check_rows("q", q);
    check_rows("out", out);
    check_apart("out", out, c.rows, c.o.heads, c.o.head_dim);
    check_forgotten(c, window, sinks);
    const DeviceScope on(c.device);
    const Cache::Turn turn(c, stream);
    c.last_causal = causal;
    c.last_window = window;
    c.last_sinks = sinks;
    Cache::Plan* plan = nullptr;
    for (Cache::Plan& p : c.plans)
        if (p.valid && p.causal == causal && p.window == window && p.sinks == sinks) plan = &p;
    if (!plan) {  // another mask than the pass was planned for
        plan = &c.plans[c.next_plan];
        c.next_plan = c.next_plan % (kPlans - 1) + 1;  // (the first stays: its items are the pass's own)
        plan->valid = false;
        c.cut(*plan, causal, window, sinks);
        const size_t bytes = plan->bytes();
        plan->items.need(bytes, c.stream);
        plan->write(c.staging.reserve(bytes));
        c.staging.send(plan->items.at, bytes, c.stream);
        plan->at = plan->items.at;
        plan->valid = true;
    }
    AttendParams p{};
    p.cache = c.layout;
    p.q = cache_rows(q);
    p.out = cache_rows(out);
    p.table = reinterpret_cast<const int*>(c.pass.at + c.table_at);
    p.layer = layer;
    p.group = c.group;
    p.scale = scale2;
    p.causal = causal;
    p.window = window;
    p.sinks = sinks;
    p.lead = sinks_lead(sinks);
    p.vector_rows = aligned(q, c.bytes, c.rows == 1, c.o.heads == 1) && aligned(out, c.bytes, c.rows == 1, c.o.heads == 1);
    p.parts = reinterpret_cast<float*>(c.parts.at);
    p.arrived = reinterpret_cast<unsigned*>(c.arrived.at);
    for (int i = 0; i < 2; i++) {
        const Cache::Plan::Launch& l = plan->launches[i];
        if (l.cut.items.empty()) continue;
        p.items = plan->items_of(i);
        p.joins = plan->joins_of(i);
        p.maps = plan->maps_of(i);
        hipLaunchKernelGGL(l.form.kernel, dim3(static_cast<unsigned>(l.cut.items.size()) * c.o.kv_heads), dim3(l.form.threads), 0, c.stream, p);
        HIP_CHECK(hipGetLastError());
    }
}

static void read_positions(Cache& c, int seq, int layer, int layers, int start, int count, const gh_rows* k, long long k_layer, const gh_rows* v,
                           long long v_layer, void* stream) {
    const PageBook::Sequence& s = c.book.at(seq);
    if (layer < 0 || layers < 0 || layer > c.o.layers || layers > c.o.layers - layer) throw ApiError{GH_ERR_OUT_OF_RANGE, "cache: layers out of range"};
    if (start < 0 || count < 0 || start > s.length || count > s.length - start)
        throw ApiError{GH_ERR_OUT_OF_RANGE, "cache: positions out of range"};
    if (s.forgot(start, start + count))
        throw ApiError{GH_ERR_OUT_OF_RANGE, "cache: sequence " + std::to_string(seq) + " has forgotten positions " + std::to_string(s.gone_from) + " to "
                                                + std::to_string(s.gone_to)};
    if (count == 0 || layers == 0) return;
    const int dim = c.o.head_dim, heads = c.o.kv_heads;
    check_rows("k", k);
    check_rows("v", v);
    check_apart("k", k, count, heads, dim);
    check_apart("v", v, count, heads, dim);
    if (layers > 1)
        for (const auto& [r, stride, name] : {std::tuple{k, k_layer, "k"}, std::tuple{v, v_layer, "v"}})
            if (stride < (count - 1) * r->row_stride + (heads - 1) * r->head_stride + dim) refuse(std::string(name) + "'s layers overlap");
    const DeviceScope on(c.device);
    const Cache::Turn turn(c, stream);
    ReadParams p{};
    p.cache = c.layout;
    p.k = cache_rows(k);
    p.v = cache_rows(v);
    p.k_layer = k_layer;
    p.v_layer = v_layer;
    p.layer = layer;
    p.vector_rows = aligned(k, c.bytes, count == 1, heads == 1) && aligned(v, c.bytes, count == 1, heads == 1)
                    && (layers == 1 || (k_layer * c.bytes % 16 == 0 && v_layer * c.bytes % 16 == 0));
    const auto kernel = c.o.type == GH_F32 ? cache_read_kernel<kCacheF32>
                      : c.o.type == GH_BF16 ? cache_read_kernel<kCacheBf16>
                                            : cache_read_kernel<kCacheF16>;
    // as many positions to a launch as its list of pages takes
    const int shift = c.layout.page_shift;
    for (int at = start; at < start + count;) {
        const int first = at >> shift, last = std::min((start + count - 1) >> shift, first + 2 * kListed - 1);
        const int end = std::min(start + count, static_cast<int>(std::min<long long>(INT_MAX, (last + 1ll) << shift)));
        PageList list;
        std::memcpy(list.pages, s.pages.data() + first, sizeof(int) * static_cast<size_t>(last - first + 1));
        p.start = at;
        p.count = end - at;
        hipLaunchKernelGGL(kernel, dim3((p.count + kReadPositions - 1) / kReadPositions, layers, 2), dim3(256), 0, c.stream, p, list);
        HIP_CHECK(hipGetLastError());
        p.k.at += static_cast<long long>(p.count) * p.k.row * c.bytes;
        p.v.at += static_cast<long long>(p.count) * p.v.row * c.bytes;
        at = end;
    }
}

}  // namespace gh

struct gh_cache {
    std::unique_ptr<gh::Cache> impl;
};

using namespace gh;

static Cache& cache_of(gh_cache* c) {
    if (!c) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null cache"};
    return *c->impl;
}

static void check_session(const Cache& c, const KvLayout& kv, int layers) {
    if (c.o.type != GH_F32 || c.o.layers != layers || c.o.kv_heads != kv.heads || c.o.head_dim != kv.head_size)
        refuse("a session's context needs a cache of GH_F32 with the model's layers, heads (as kv_heads) and head size");
    hipPointerAttribute_t at{};
    HIP_CHECK(hipPointerGetAttributes(&at, kv.pool));
    if (at.device != c.device) refuse("the session is on another device");
}

static void copy_session(Cache& c, const KvLayout& kv, int layers, int seq, const std::vector<int>& pages, int length, bool to_session) {
    SessionCopyParams p{};
    p.cache = c.layout;
    p.kv = kv;
    p.seq = seq;
    p.to_session = to_session;
    const int shift = c.layout.page_shift;
    for (int at = 0; at < length;) {
        const int first = at >> shift, last = std::min((length - 1) >> shift, first + 2 * kListed - 1);
        const int end = static_cast<int>(std::min<long long>(length, (last + 1ll) << shift));
        PageList list;
        std::memcpy(list.pages, pages.data() + first, sizeof(int) * static_cast<size_t>(last - first + 1));
        p.start = at;
        p.count = end - at;
        hipLaunchKernelGGL(cache_session_kernel, dim3((p.count + kReadPositions - 1) / kReadPositions, layers, 2), dim3(256), 0, c.stream, p, list);
        HIP_CHECK(hipGetLastError());
        at = end;
    }
}

namespace gh {

int cache_from_session(gh_cache* cache, const KvLayout& kv, int layers, int seq, int length, hipStream_t stream) {
    Cache& c = cache_of(cache);
    check_session(c, kv, layers);
    const DeviceScope on(c.device);
    const Cache::Turn turn(c, stream);
    const int id = c.book.add_filled(length);
    c.close();
    copy_session(c, kv, layers, seq, c.book.at(id).pages, length, /*to_session=*/false);
    return id;
}

void cache_to_session(gh_cache* cache, const int32_t* seqs, int batch, const KvLayout& kv, int layers, int length, hipStream_t stream) {
    Cache& c = cache_of(cache);
    check_session(c, kv, layers);
    for (int b = 0; b < batch; b++)
        if (c.book.at(seqs[b]).forgot(0, length))
            throw ApiError{GH_ERR_OUT_OF_RANGE, "cache: sequence " + std::to_string(seqs[b]) + " has forgotten some of its positions"};
    for (int b = 0; b < batch; b++)
        if (c.book.at(seqs[b]).length < length)
            throw ApiError{GH_ERR_OUT_OF_RANGE, "cache: sequence " + std::to_string(seqs[b]) + " holds " + std::to_string(c.book.at(seqs[b]).length)
                                                    + " positions, " + std::to_string(length) + " are wanted"};
    const DeviceScope on(c.device);
    const Cache::Turn turn(c, stream);
    for (int b = 0; b < batch; b++) copy_session(c, kv, layers, b, c.book.at(seqs[b]).pages, length, /*to_session=*/true);
}

}  // namespace gh

extern "C" {

gh_status gh_cache_create(const gh_cache_opts* opts, gh_cache** out) {
    return guard([&] {
        if (!opts || !out) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
        *out = nullptr;
        *out = new gh_cache{create_cache(*opts)};
    });
}

void gh_cache_free(gh_cache* c) {
    if (!c) return;
    (void)guard([&] {
        const DeviceScope on(c->impl->device);
        c->impl.reset();
    });
    delete c;
}

gh_status gh_cache_get_info(const gh_cache* c, gh_cache_info* out) {
    return guard([&] {
        if (!c || !out) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
        const Cache& m = *c->impl;
        *out = gh_cache_info{m.device, m.book.pages(), m.book.pages_free(), m.book.sequences(), m.open ? m.rows : -1, 0, m.pool.bytes};
    });
}

gh_status gh_cache_add(gh_cache* c, int32_t* seq) {
    return guard([&] {
        if (!seq) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
        *seq = cache_of(c).book.add();
    });
}

int32_t gh_cache_length(const gh_cache* c, int32_t seq) {
    int32_t length = -1;
    if (c) (void)guard([&] { length = c->impl->book.at(seq).length; });
    return length;
}

gh_status gh_cache_fork(gh_cache* c, int32_t seq, int32_t length, int32_t* out) {
    return guard([&] {
        if (!out) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
        Cache& m = cache_of(c);
        const int id = m.book.fork(seq, length == -1 ? m.book.at(seq).length : length);
        m.close();
        *out = id;
    });
}

gh_status gh_cache_truncate(gh_cache* c, int32_t seq, int32_t length) {
    return guard([&] {
        Cache& m = cache_of(c);
        m.book.truncate(seq, length);
        m.close();
    });
}

gh_status gh_cache_forget(gh_cache* c, int32_t seq, int32_t start, int32_t end) {
    return guard([&] {
        Cache& m = cache_of(c);
        m.book.forget(seq, start, end);
        m.close();
    });
}

gh_status gh_cache_drop(gh_cache* c, int32_t seq) {
    return guard([&] {
        Cache& m = cache_of(c);
        m.book.drop(seq);
        m.close();
    });
}

gh_status gh_cache_copy(gh_cache* from, int32_t seq, gh_cache* to, void* hip_stream, int32_t* out) {
    return guard([&] {
        if (!out) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
        Cache &a = cache_of(from), &b = cache_of(to);
        if (a.o.layers != b.o.layers || a.o.kv_heads != b.o.kv_heads || a.o.head_dim != b.o.head_dim || a.o.type != b.o.type
            || a.o.page_tokens != b.o.page_tokens)
            refuse("a copy between caches of different layers, kv_heads, head_dim, type or page_tokens");
        if (a.device != b.device) refuse("a copy between devices");
        (void)a.book.at(seq);
        const DeviceScope on(b.device);
        *out = copy_sequence(a, b, seq, hip_stream);
    });
}

gh_status gh_cache_compact(gh_cache* c, void* hip_stream, int32_t* pages_used) {
    return guard([&] {
        Cache& m = cache_of(c);
        const DeviceScope on(m.device);
        const Cache::Turn turn(m, hip_stream);
        const int used = m.book.pages() - m.book.pages_free();
        const std::vector<PageCopy> moves = m.book.compact();
        m.close();
        m.copy_pages(m.pool.at, moves);
        if (pages_used) *pages_used = used;
    });
}

gh_status gh_cache_extend(gh_cache* c, const int32_t* seqs, const int32_t* counts, int32_t n, void* hip_stream) {
    return guard([&] {
        Cache& m = cache_of(c);
        if (n < 0 || (n > 0 && (!seqs || !counts))) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
        const DeviceScope on(m.device);
        extend_cache(m, seqs, counts, n, hip_stream);
    });
}

gh_status gh_cache_append(gh_cache* c, int32_t layer, const gh_rows* k, const gh_rows* v, const gh_rows* q, const gh_rows* q_out,
                          int32_t rotate, void* hip_stream) {
    return guard([&] { append_rows(cache_of(c), layer, k, v, q, q_out, rotate != 0, hip_stream); });
}

gh_status gh_cache_attend(gh_cache* c, int32_t layer, const gh_rows* q, const gh_rows* out, float scale, int32_t causal, int32_t window,
                          void* hip_stream) {
    return guard([&] { attend(cache_of(c), layer, q, out, scale, causal != 0, window, 0, hip_stream); });
}

gh_status gh_cache_attend_sinks(gh_cache* c, int32_t layer, const gh_rows* q, const gh_rows* out, float scale, int32_t causal, int32_t window,
                                int32_t sinks, void* hip_stream) {
    return guard([&] { attend(cache_of(c), layer, q, out, scale, causal != 0, window, sinks, hip_stream); });
}

gh_status gh_cache_read(gh_cache* c, int32_t seq, int32_t layer, int32_t layers, int32_t start, int32_t count, const gh_rows* k,
                        int64_t k_layer_stride, const gh_rows* v, int64_t v_layer_stride, void* hip_stream) {
    return guard([&] { read_positions(cache_of(c), seq, layer, layers, start, count, k, k_layer_stride, v, v_layer_stride, hip_stream); });
}

}  // extern "C"
