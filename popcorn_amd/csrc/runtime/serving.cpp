// Kernels.* descriptors of a batch of requests over a paged cache: page tables,
// the paged cache write, paged attention, with prefixes that requests share, the
// weights that it gives the keys, eviction by them, and the draw of the next token.
// No counterparts in the reference; validation and errors are as for its own
// operations (kernels.cpp).
#include <algorithm>

#include "popcorn.hpp"

namespace popcorn {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool isFloat(DataType t) { return t == DataType::f32 || t == DataType::f16 || t == DataType::bf16; }
bool aligned(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

void requireRank(const Tensor &t, int rank) {
    if (t.shape.rank() != rank) throw Error::tensorInvalidRank(rank, t.shape.rank());
}

// Every size below 2^31 (the kernels count in 32 bits), the bytes below 2^62, and the data's place.
void requireTensor(const Tensor &t, const std::string &what) {
    int64_t bytes = stride(t.dataType);
    for (int64_t d : t.shape.dims) {
        if (d >= (int64_t{1} << 31)) throw Error::tensorShapeMismatch(what + " dimensions must be below 2^31; got " + t.shape.str() + ".");
        if (__builtin_mul_overflow(bytes, d, &bytes) || bytes >= (int64_t{1} << 62))
            throw Error::tensorShapeMismatch(what + " is too large: " + t.shape.str() + ".");
    }
    if (bytes > 0 && !t.data) throw Error::invalidArgument(what + ": null data pointer");
    if (!aligned(t.data, stride(t.dataType))) throw Error::invalidArgument(what + ": data is not aligned to its elements");
}

void requireShape(const Tensor &t, DataType type, std::initializer_list<int64_t> dims, const std::string &what) {
    if (t.dataType != type)
        throw Error::unsupportedDataTypeCombination(what + " must be " + name(type) + "; got " + name(t.dataType) + ".");
    const Shape want(dims);
    requireRank(t, want.rank());
    if (t.shape != want) throw Error::tensorShapeMismatch(what + " must have shape " + want.str() + "; got " + t.shape.str() + ".");
    requireTensor(t, what);
}

// Blocks read the inputs while others write: the outputs lie apart from them, and from each other.
using Named = std::pair<const Tensor *, const char *>;
void requireApart(const std::string &op, const std::vector<Named> &outputs, const std::vector<Named> &inputs) {
    auto apart = [&](const Named &a, const Named &b) {
        const auto at = reinterpret_cast<uintptr_t>(a.first->data), bt = reinterpret_cast<uintptr_t>(b.first->data);
        const size_t an = a.first->byteCount(), bn = b.first->byteCount();
        if (an && bn && at < bt + bn && bt < at + an)
            throw Error::invalidArgument(op + " " + a.second + " must not overlap " + b.second + ".");
    };
    for (size_t i = 0; i < outputs.size(); ++i) {
        for (size_t j = i + 1; j < outputs.size(); ++j) apart(outputs[i], outputs[j]);
        for (const Named &in : inputs) apart(outputs[i], in);
    }
}

// The runtime counts a grid's threads in 32 bits.
void requireGrid(int64_t blocks, int64_t threads, const std::string &op, const Tensor &t) {
    if (blocks > UINT32_MAX / threads) throw Error::tensorShapeMismatch(op + " takes fewer rows in one call; got " + t.shape.str() + ".");
}

// The caches [pages, Nkv, page size, Hd] of one shape and dtype.
void requireCaches(const Tensor &k, const Tensor &v, const std::string &op) {
    requireRank(k, 4);
    if (v.shape != k.shape) throw Error::tensorShapeMismatch(op + " caches must share a shape; got " + k.shape.str() + " and " + v.shape.str() + ".");
    requireTensor(k, op + " k_cache");
    requireTensor(v, op + " v_cache");
    if (k.shape[2] <= 0) throw Error::tensorShapeMismatch(op + " page size must be positive; got " + k.shape.str() + ".");
    if (k.shape[0] * k.shape[2] >= (int64_t{1} << 31))
        throw Error::tensorShapeMismatch(op + " cache must hold fewer than 2^31 slots; got " + k.shape.str() + ".");
}

// The sizes of a paged attention call, checked.
PagedAttentionConstants pagedConstants(const std::string &op, const Tensor &q, const Tensor &kCache, const Tensor &vCache, const Tensor &pageTables,
                                       const Tensor &queryStarts, const Tensor &keyLens, const Tensor &out, float scale, AttentionMask mask,
                                       int64_t sinks, int64_t maxQueryLen) {
    using D = DataType;
    const D t = q.dataType;
    if (!isFloat(t) || kCache.dataType != t || vCache.dataType != t || out.dataType != t)
        throw Error::unsupportedDataTypeCombination(op + std::string(" needs one floating dtype for q, the caches and out; got ") +
                                                    name(t) + ", " + name(kCache.dataType) + ", " + name(vCache.dataType) + ", " +
                                                    name(out.dataType) + ".");
    if (mask.kind > 2) throw Error::invalidArgument("unknown attention mask kind");
    if (sinks < 0 || sinks >= (int64_t{1} << 31)) throw Error::invalidArgument(op + " sinks must be at least 0 and below 2^31.");
    if (sinks > 0 && mask.kind != 1) throw Error::invalidArgument(op + " sinks go with a sliding window.");
    if (maxQueryLen < 0) throw Error::invalidArgument(op + " max_query_len must not be negative.");
    requireCaches(kCache, vCache, op);
    requireRank(q, 3);
    requireRank(pageTables, 2);
    const int64_t T = q.shape[0], Nq = q.shape[1], Hd = q.shape[2], Nkv = kCache.shape[1], page = kCache.shape[2];
    const int64_t R = pageTables.shape[0], M = pageTables.shape[1];
    if (Nkv <= 0 || Nq <= 0 || Nq % Nkv != 0)
        throw Error::tensorShapeMismatch(op + " query heads must be divisible by KV heads; got " + std::to_string(Nq) + " and " +
                                         std::to_string(Nkv) + ".");
    if (Hd <= 0 || Hd > 512)
        throw Error::tensorShapeMismatch(op + " head dim must be 1 to 512 (kernel limit); got " + std::to_string(Hd) + ".");
    if (kCache.shape[3] != Hd)
        throw Error::tensorShapeMismatch(op + " caches must have q's head dim; got " + q.shape.str() + " and " + kCache.shape.str() + ".");
    if (page % 16 != 0)
        throw Error::tensorShapeMismatch(op + " page size must be a multiple of 16; got " + std::to_string(page) + ".");
    requireShape(q, t, {T, Nq, Hd}, op + " q");
    requireShape(out, t, {T, Nq, Hd}, op + " out");
    requireShape(pageTables, D::i32, {R, M}, op + " page_tables");
    requireShape(queryStarts, D::i32, {R + 1}, op + " query_starts");
    requireShape(keyLens, D::i32, {R}, op + " key_lens");
    requireGrid(T * Nq, 256, op, q);
    return PagedAttentionConstants{(uint32_t)T, (uint32_t)R, (uint32_t)Nq, (uint32_t)Nkv, (uint32_t)Hd, (uint32_t)page,
                                   (uint32_t)kCache.shape[0], (uint32_t)M, mask.kind, mask.window, (uint32_t)sinks, scale};
}

// 16-byte rows: the matrix cores
bool fastRows(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &out) {
    return q.shape[2] % (16 / stride(q.dataType)) == 0 && aligned(q.data, 16) && aligned(k.data, 16) && aligned(v.data, 16) && aligned(out.data, 16);
}
std::string plainName(const Tensor &q, const Tensor &k, const Tensor &v) {
    const int run = 4 * stride(q.dataType);
    return name(q.dataType) + std::string(q.shape[2] % 4 || !aligned(k.data, run) || !aligned(v.data, run) ? "_any" : "");
}

// Keys that a table's row has room for, counted in 32 bits by the kernels.
int64_t requireRoom(const std::string &op, int64_t columns, int64_t pageSize) {
    if (columns >= (int64_t{1} << 31) / pageSize)
        throw Error::tensorShapeMismatch(op + " tables must hold fewer than 2^31 keys a request; got " + std::to_string(columns) + " pages of " +
                                         std::to_string(pageSize) + ".");
    return columns * pageSize;
}

std::unique_ptr<Kernel> fixed(const std::string &fn, std::vector<Binding> b, std::vector<uint8_t> c, dim3 grid, unsigned block) {
    return Kernels::Custom(fn, std::move(b), {std::move(c)}, grid, dim3(block, 1, 1));
}

int deviceCUs() {
    static thread_local int cachedDev = -1, cachedCUs = 256;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) {
        (void)hipGetLastError();
        return cachedCUs;
    }
    if (dev != cachedDev) {
        int cus = 0;
        if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && cus > 0) cachedCUs = cus;
        (void)hipGetLastError();
        cachedDev = dev;
    }
    return cachedCUs;
}

// Rows (new tokens x heads of a KV head's group) up to which a request counts as one of few, and of the longest request.
constexpr uint32_t kFewRows = 32;
int64_t longestRows(const PagedAttentionConstants &pc, int64_t maxQueryLen) {
    return std::min<int64_t>(maxQueryLen > 0 ? maxQueryLen : pc.T, pc.T) * (pc.Nq / pc.Nkv);
}
int tilesPerCU(int64_t hdp) { return hdp == 256 ? 1 : 2; }

// What PagedAttention uses its tile kernel for: nothing, all requests, or (apart) those of many rows, beside a launch for the others.
struct TileUse {
    bool tiles, apart;
};
TileUse tileUse(const Tensor &q, const PagedAttentionConstants &pc, int64_t hdp, int64_t longest) {
    // The tile kernel works on the magnitude of the scale (not 0) and 16-bit K and V of up to 256 dims. For requests of up to
    // 32 rows, or so few rows in all, the tiles' 128 rows cost more than reading keys again: us of the few-row kernel and of
    // tiles, 4 heads to a KV head, 8 KV heads, 4000 keys: one request of 64 rows 26 and 33 (Hd 128), 34 and 43 (256), of 128
    // rows 27 and 40, 38 and 46 (but 96 and 67 behind 16000 keys), of 256 rows 33 and 39, 54 and 47.
    const bool tiles = q.dataType != DataType::f32 && hdp <= 256 && pc.scale != 0.0f && pc.scale == pc.scale && longest > kFewRows &&
                       (int64_t)pc.T * (pc.Nq / pc.Nkv) > (hdp == 256 ? 64 : 128);
    // Beside tiles, the requests of few rows have a launch of their own where there are more units than blocks: one request of
    // 500 tokens among 256 of up to 1000 keys on 8 KV heads of 128, 80 us and 107 in tiles alone, 128 on 4 of 256 72 and 88;
    // but as many units as blocks (64 of up to 8000 keys on 8) 81 and 78, 12 requests of few keys 41 and 31.
    return {tiles, tiles && (int64_t)pc.R * pc.Nkv > tilesPerCU(hdp) * deviceCUs()};
}

// PagedAttention on the matrix cores (paged_attention.hip): requests of few
// rows (new tokens x heads of a KV head's group) and of many by a launch each,
// with plans of tiles where the blocks do not lay them out themselves, and the
// merge of what several blocks shared.
class PagedAttentionKernel : public Kernel {
public:
    PagedAttentionKernel(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &tables, const Tensor &starts, const Tensor &lens,
                         const Tensor &out, const PagedAttentionConstants &pc, int64_t maxQueryLen)
        : q_(q), k_(k), v_(v), tables_(tables), starts_(starts), lens_(lens), out_(out), pc_(pc) {
        const int64_t longest = longestRows(pc, maxQueryLen);
        const bool f32 = q.dataType == DataType::f32;
        hdp_ = pc.Hd <= 64 ? 64 : pc.Hd <= 128 ? 128 : pc.Hd <= 256 ? 256 : 512;
        const std::string type = name(q.dataType), hd = "_d" + std::to_string(hdp_);
        merge_ = "paged_attention_merge_" + type + hd;
        const auto [tiles, apart] = tileUse(q, pc, hdp_, longest);
        if (!tiles || apart) {
            // 16 rows per wave or 32: 16 requests of 32 rows, 2000 keys, us: Hd 64 31.1 and 26.5, Hd 256 90 and 60, of 16 rows 22.5
            // and 25.0, 54 and 56. Registers for 32 are wanting at Hd 512 and in f32 at 256 (84 and 198 there).
            const int rt = hdp_ == 512 || (f32 && hdp_ == 256) || longest <= 16 || tiles ? 1 : 2;
            // as many blocks as run at once (the kernels' registers)
            const int perCU = hdp_ == 64 ? 5 - rt : hdp_ == 128 ? 4 - rt : hdp_ == 256 && rt == 1 && !f32 ? 2 : 1;
            add("paged_attention_few_" + type + hd + "_r" + std::to_string(rt), 16 * rt, f32 ? 16 : 32, 0, tiles ? kFewRows : UINT32_MAX, perCU);
        }
        if (tiles) add("paged_attention_tile_" + type + hd, 128, 64, apart ? kFewRows : 0, UINT32_MAX, tilesPerCU(hdp_));
    }
    std::vector<Binding> tensors() const override {
        return {{q_, kRead}, {k_, kRead}, {v_, kRead}, {tables_, kRead}, {starts_, kRead}, {lens_, kRead}, {out_, kWrite}};
    }
    std::string describe() const override {
        std::string s;
        for (const Work &w : work_) s += (w.c.ownPlan ? "" : "paged_plan,") + w.fn + ",";
        return s + merge_;
    }
    void encode(KernelCommandEncoder &enc) const override {
        // one buffer: the states' O, their m and l, what is shared, the plans
        int64_t states = 0, workers = 0, tiles = 0;
        for (const Work &w : work_) {
            states += 2 * (int64_t)w.c.workers * w.c.rows;
            workers += w.c.workers;
            tiles += w.c.ownPlan ? 0 : (int64_t)w.c.maxTiles + 1;
        }
        const int64_t o = states * hdp_ * 4, ml = states * 8, shared = workers * 32;
        enc.withTemporaryTensor(ScratchSpec{{o + ml + shared + tiles * 16}, DataType::u8}, [&](Tensor scratch) {
            auto part = [&](int64_t at, int64_t bytes) { return Tensor((char *)scratch.data + at, Shape({bytes}), DataType::u8); };
            const Tensor pO = part(0, o), pML = part(o, ml);
            int64_t at = o + ml, plan = o + ml + shared;
            for (const Work &w : work_) {
                const Tensor sh = part(at, (int64_t)w.c.workers * 32), pl = part(plan, ((int64_t)w.c.maxTiles + 1) * 16);
                const std::vector<std::vector<uint8_t>> consts = {bytesOf(pc_), bytesOf(w.c)};
                if (!w.c.ownPlan) {
                    launch(enc, "paged_plan", {{starts_, kRead}, {lens_, kRead}, {pl, kWrite}}, consts, dim3(1, 1, 1), 1024);
                    plan += ((int64_t)w.c.maxTiles + 1) * 16;
                }
                launch(enc, w.fn,
                       {{q_, kRead}, {k_, kRead}, {v_, kRead}, {tables_, kRead}, {starts_, kRead}, {lens_, kRead}, {pl, kRead}, {pO, kWrite},
                        {pML, kWrite}, {sh, kWrite}, {out_, kWrite}},
                       consts, dim3(w.c.workers, 1, 1), 256);
                at += (int64_t)w.c.workers * 32;
            }
            launch(enc, merge_, {{pO, kRead}, {pML, kRead}, {part(o + ml, shared), kRead}, {out_, kWrite}}, {bytesOf(pc_)},
                   dim3((unsigned)workers, work_.back().c.rows / 16, 1), 256);
        });
    }

private:
    struct Work {
        std::string fn;
        PagedWorkConstants c;
    };

    void add(const std::string &fn, uint32_t rows, uint32_t stepKeys, uint32_t few, uint32_t many, int perCU) {
        const int64_t G = pc_.Nq / pc_.Nkv;
        PagedWorkConstants w{};
        w.rows = rows;
        w.stepKeys = stepKeys;
        w.fewRows = few;
        w.manyRows = many;
        w.maxTiles = (uint32_t)(cdiv((int64_t)pc_.T * G, rows) + std::min(pc_.R, pc_.T));
        // A worker's least work, and what a unit counts beside its steps (its start: about 10 us). One request of 4096 keys, us:
        // 18.4 with 128 keys at least, 20.1 with 64, 19.9 with 256; 64 requests of 100 to 16000: 136 with 384 keys counted, 146
        // with none, 142 with 768; chunks of prompts among them: 57 with 384, 94 with none, 62 with 768.
        w.minSteps = 128 / stepKeys;
        w.unitSteps = 384 / stepKeys;
        // Caches of more than the 256 MB of the memory-side cache are read once a step: V past the caches reads 766 MB
        // (64 requests) in 137 us instead of 149; 17 MB of one request take 18.7 us that way and 18.0 otherwise.
        w.stream = k_.byteCount() + v_.byteCount() > (size_t{256} << 20);
        // no more workers than the longest requests that the tables can name could give work to
        const double tileSteps = (double)cdiv((int64_t)pc_.columns * pc_.pageSize + stepKeys, stepKeys) + w.unitSteps;
        const double steps = (double)w.maxTiles * tileSteps;
        w.workers = (uint32_t)std::max(1.0, std::min((double)perCU * deviceCUs(), steps * pc_.Nkv / w.minSteps + 1));
        // (a launch less: one request 18.4 us and 21.3, 256 requests 78 and 81)
        w.ownPlan = w.maxTiles <= 1024 && pc_.R <= 1024 && steps < 2147483648.0;
        w.stateBase = work_.empty() ? 0 : 2 * work_.back().c.workers * work_.back().c.rows;
        work_.push_back({fn, w});
    }
    void launch(KernelCommandEncoder &enc, const std::string &fn, std::vector<Binding> b, std::vector<std::vector<uint8_t>> consts, dim3 grid,
                unsigned block) const {
        enc.encode(*Kernels::Custom(fn, std::move(b), std::move(consts), grid, dim3(block, 1, 1)));
    }

    Tensor q_, k_, v_, tables_, starts_, lens_, out_;
    PagedAttentionConstants pc_;
    std::vector<Work> work_;
    std::string merge_;
    int64_t hdp_ = 0;
};

// SharedPrefixAttention (shared_prefix.hip): PagedAttention's two kernels over units of groups' rows against their prefixes and of
// requests' rows against their pages, side by side in one launch behind their plan where there are units of many rows, then a merge
// of each row's pieces.
class SharedPrefixKernel : public Kernel {
public:
    SharedPrefixKernel(std::vector<Tensor> inputs, const Tensor &out, const Tensor *lse, const PagedAttentionConstants &pc,
                       const SharedPrefixConstants &sc, int64_t maxQueryLen)
        : in_(std::move(inputs)), out_(out), lse_(lse ? *lse : out), pc_(pc), sc_(sc) {
        const Tensor &q = in_[0];
        const int64_t G = pc.Nq / pc.Nkv, all = (int64_t)pc.T * G;
        // a group's rows may be all there are
        const int64_t longest = sc.groups ? all : longestRows(pc, maxQueryLen);
        const bool f32 = q.dataType == DataType::f32;
        hdp_ = pc.Hd <= 64 ? 64 : pc.Hd <= 128 ? 128 : pc.Hd <= 256 ? 256 : 512;
        const std::string type = name(q.dataType), hd = "_d" + std::to_string(hdp_);
        merge_ = "shared_prefix_merge_" + type + hd;
        // the kernels and their limits as for PagedAttention
        both_ = !f32 && hdp_ <= 256 && pc.scale != 0.0f && pc.scale == pc.scale && longest > kFewRows && all > (sc.groups || hdp_ == 256 ? 64 : 128);
        if (both_) {
            // one launch of both kinds of rows, or at 256 dims one after the other
            fn_ = (hdp_ == 256 ? "shared_prefix_many_" : "shared_prefix_both_") + type + hd;
            // No row's weights have fewer bits than PagedAttention gives them for the same max_query_len: f16 tiles have two words
            // where its few-row kernel would take some of the rows that share them here. (64 requests, a token each, behind 8192 keys, 2-norm
            // against 64 bits: 2.1e-4, the result's rounding, and 2.8e-4 with one word; 60.5 us and 56.8. But 2048 tokens of one
            // request behind as many, 32 heads of 128 on 8, 560 us and 415; 8 of 256 on 4 273 and 240.)
            const TileUse alone = tileUse(q, pc, hdp_, longestRows(pc, maxQueryLen));
            if (q.dataType == DataType::f16 && sc.groups && (!alone.tiles || alone.apart)) fn_ += "_two";
            if (hdp_ == 256) before_ = "shared_prefix_few_" + type + hd + "_r1";
            blocks_ = (hdp_ == 256 ? 1 : 2) * deviceCUs();
            many_ = work(128, 64, kFewRows, UINT32_MAX, blocks_, 384);
            few_ = work(16, 32, 0, kFewRows, 4 * 2 * deviceCUs(), 96);
            few_.stateBase = 2 * many_.workers * many_.rows;
        } else {
            const int rt = hdp_ == 512 || (f32 && hdp_ == 256) || longest <= 16 ? 1 : 2;
            const int perCU = hdp_ == 64 ? 5 - rt : hdp_ == 128 ? 4 - rt : hdp_ == 256 && rt == 1 && !f32 ? 2 : 1;
            fn_ = "shared_prefix_few_" + type + hd + "_r" + std::to_string(rt);
            // a worker is a wave, or at 512 dims a block
            const int team = hdp_ == 512 ? 1 : 4;
            few_ = work(16 * rt, f32 ? 16 : 32, 0, UINT32_MAX, 0, team == 4 ? 96 : 384);
            const double steps = (double)few_.maxTiles * tileSteps(few_);
            blocks_ = (unsigned)std::max(1.0, std::min((double)perCU * deviceCUs(), (steps * pc.Nkv / few_.minSteps + 1) / team));
            few_.workers = blocks_ * team;
            few_.ownPlan = few_.maxTiles <= 1024 && pc.R + sc.groups <= 1024 && steps < 2147483648.0;
        }
        sc_.rows = pc.T * pc.Nq;
        sc_.rowBase = few_.stateBase + 2 * few_.workers * few_.rows;
        sc_.states = sc_.rowBase + (sc.groups ? 2 * sc_.rows : 0);
        sc_.most = std::max(many_.workers, few_.workers);
        sc_.parts = sc_.rows < 4096 ? 4 : 1;
    }
    std::vector<Binding> tensors() const override {
        std::vector<Binding> b;
        for (const Tensor &t : in_) b.push_back({t, kRead});
        b.push_back({out_, kWrite});
        if (sc_.hasLse) b.push_back({lse_, kWrite});
        return b;
    }
    std::string describe() const override {
        return (both_ ? "shared_prefix_plan," : std::string(sc_.windowed ? "shared_prefix_positions," : "") + (few_.ownPlan ? "" : "shared_prefix_plan,")) +
               (before_.empty() ? "" : before_ + ",") + fn_ + "," + merge_;
    }
    void encode(KernelCommandEncoder &enc) const override {
        // one buffer: the states' O, their m and l, the rows' records, the plans, the positions
        const int64_t tiles = both_ ? (int64_t)many_.maxTiles + few_.maxTiles + 2 : few_.ownPlan ? 0 : (int64_t)few_.maxTiles + 1;
        const int64_t o = (int64_t)sc_.states * hdp_ * 4, ml = cdiv((int64_t)sc_.states * 8, 16) * 16, rec = 2 * (int64_t)sc_.rows * 16;
        const int64_t positions = sc_.windowed ? ((int64_t)pc_.T + sc_.groups) * 4 : 0;
        enc.withTemporaryTensor(ScratchSpec{{o + ml + rec + tiles * kTile + positions}, DataType::u8}, [&](Tensor scratch) {
            auto part = [&](int64_t at, int64_t bytes) { return Tensor((char *)scratch.data + at, Shape({bytes}), DataType::u8); };
            const Tensor pO = part(0, o), pML = part(o, ml), records = part(o + ml, rec), plan = part(o + ml + rec, tiles * kTile);
            const Tensor pos = part(o + ml + rec + tiles * kTile, positions);
            const Tensor &starts = in_[4], &lens = in_[5], &prefixLens = in_[7], &groups = in_[8];
            const std::vector<Binding> lengths = {{starts, kRead}, {lens, kRead}, {prefixLens, kRead}, {groups, kRead}};
            auto with = [](std::vector<Binding> b, std::initializer_list<Binding> more) {
                b.insert(b.end(), more);
                return b;
            };
            std::vector<std::vector<uint8_t>> consts = {bytesOf(pc_)};
            if (both_) consts.push_back(bytesOf(many_));
            consts.push_back(bytesOf(few_));
            consts.push_back(bytesOf(sc_));
            if (both_) {
                launch(enc, "shared_prefix_plan", with(lengths, {{pos, kReadWrite}, {plan, kWrite}}), consts,
                       2 + (sc_.windowed ? cdiv(pc_.T, 1024) : 0), 1024);
            } else {
                if (sc_.windowed)
                    launch(enc, "shared_prefix_positions", with(lengths, {{pos, kWrite}}), {bytesOf(pc_), bytesOf(sc_)},
                           cdiv(pc_.T, 256) + cdiv(sc_.groups, 4), 256);
                if (!few_.ownPlan)  // (writes the groups' least again, the same)
                    launch(enc, "shared_prefix_plan", with(lengths, {{pos, kReadWrite}, {plan, kWrite}}),
                           {bytesOf(pc_), bytesOf(few_), bytesOf(few_), bytesOf(sc_)}, 1, 1024);
            }
            std::vector<Binding> b;
            for (const Tensor &t : in_) b.push_back({t, kRead});
            auto attend = [&](const std::string &fn, const Tensor &pl, const std::vector<std::vector<uint8_t>> &c, int64_t blocks) {
                launch(enc, fn, with(b, {{pos, kRead}, {pl, kRead}, {pO, kWrite}, {pML, kWrite}, {records, kWrite}, {out_, kWrite}, {lse_, kWrite}}), c,
                       blocks, 256);
            };
            if (before_.empty()) {
                attend(fn_, plan, consts, blocks_);
            } else {
                const int64_t first = ((int64_t)many_.maxTiles + 1) * kTile;
                attend(before_, part(o + ml + rec + first, tiles * kTile - first), {bytesOf(pc_), bytesOf(few_), bytesOf(sc_)}, few_.workers / 4);
                attend(fn_, plan, {bytesOf(pc_), bytesOf(many_), bytesOf(sc_)}, blocks_);
            }
            launch(enc, merge_,
                   {{pO, kRead}, {pML, kRead}, {records, kRead}, {starts, kRead}, {out_, kWrite}, {lse_, kWrite}},
                   {bytesOf(pc_), bytesOf(sc_)}, cdiv(sc_.rows, 4 / sc_.parts), 256);
        });
    }

private:
    static constexpr int64_t kTile = 48;  // bytes of a plan's entry

    double tileSteps(const PagedWorkConstants &w) const {
        return (double)cdiv((int64_t)std::max(pc_.columns, sc_.columns) * pc_.pageSize + w.stepKeys, w.stepKeys) + w.unitSteps;
    }
    PagedWorkConstants work(uint32_t rows, uint32_t stepKeys, uint32_t few, uint32_t many, uint32_t workers, uint32_t unitKeys) const {
        PagedWorkConstants w{};
        w.rows = rows;
        w.stepKeys = stepKeys;
        w.fewRows = few;
        w.manyRows = many;
        w.workers = workers;
        const int64_t tiles = cdiv((int64_t)pc_.T * (pc_.Nq / pc_.Nkv), rows);
        w.maxTiles = (uint32_t)(tiles + std::min(pc_.R, pc_.T) + (sc_.groups ? tiles + std::min(sc_.groups, pc_.T) : 0));
        w.minSteps = 64 / stepKeys;
        w.unitSteps = unitKeys / stepKeys;
        w.stream = in_[1].byteCount() + in_[2].byteCount() > (size_t{256} << 20);
        return w;
    }
    void launch(KernelCommandEncoder &enc, const std::string &fn, std::vector<Binding> b, std::vector<std::vector<uint8_t>> consts, int64_t blocks,
                unsigned block) const {
        enc.encode(*Kernels::Custom(fn, std::move(b), std::move(consts), dim3((unsigned)blocks, 1, 1), dim3(block, 1, 1)));
    }

    std::vector<Tensor> in_;  // q, k, v, tables, starts, lens, prefix tables, prefix lens, group starts
    Tensor out_, lse_;
    PagedAttentionConstants pc_;
    SharedPrefixConstants sc_;
    PagedWorkConstants many_{}, few_{};
    std::string before_, fn_, merge_;
    bool both_ = false;
    unsigned blocks_ = 1;
    int64_t hdp_ = 0;
};

// PagedAttentionWeights (attention_weights.hip).
class AttentionWeightsKernel : public Kernel {
public:
    AttentionWeightsKernel(std::vector<Tensor> inputs, const Tensor &weights, const PagedAttentionConstants &pc, int64_t lastRows, int64_t maxQueryLen)
        : in_(std::move(inputs)), weights_(weights), pc_(pc) {
        const Tensor &q = in_[0];
        const int64_t groups = cdiv((int64_t)pc.columns * pc.pageSize, 16);
        const std::string type = name(q.dataType);
        const int hdp = pc.Hd <= 64 ? 64 : pc.Hd <= 128 ? 128 : pc.Hd <= 256 ? 256 : 512;
        fn_ = "attention_weights_few_" + type + "_d" + std::to_string(hdp);
        wc_ = AttentionWeightsConstants{(uint32_t)std::min<int64_t>(lastRows, pc.T), 0, UINT32_MAX,
                                        pc.R <= 1024 && (double)groups * pc.R < 4294967296.0, pc.maskKind == 2};
        const int perCU = q.dataType == DataType::f32 ? (hdp <= 64 ? 3 : hdp <= 256 ? 2 : 1) : (hdp <= 64 ? 4 : hdp <= 128 ? 3 : 2);
        blocks_ = (unsigned)std::clamp<double>((double)groups * pc.R * pc.Nkv / 4, 1, (double)perCU * deviceCUs());
        const int64_t G = pc.Nq / pc.Nkv;
        int64_t longest = std::min<int64_t>(maxQueryLen > 0 ? maxQueryLen : pc.T, pc.T);
        if (lastRows > 0) longest = std::min(longest, lastRows);
        // 16-bit keys of up to 256 dims, rows divided by G as the kernel does, and a step's rows within reach of one offset
        if (q.dataType == DataType::f32 || hdp > 256 || !(pc.scale < 0.0f || pc.scale > 0.0f) || longest * G <= kFewRows || G > 256 || (int64_t)64 * pc.Nq * pc.Hd >= (int64_t{1} << 29)) return;
        tile_ = "attention_weights_tile_" + type + "_d" + std::to_string(hdp);
        // Requests of few rows have a launch of their own where there are many of them, or where their keys may be: a tile's start is
        // as long as 10 of its steps, for 256 keys that a single token's row reads in one. us with the launch and without:
        //   6 requests of 32 rows, 2 KV heads 20.3 and 18.5; 48, 4 heads, 6 prompts 63.8 and 70.7; 48, 8 heads, one prompt 84 and 131
        //   (but 24, 4 heads, 3 prompts among 500 keys 31.3 and 25.0, 40, 4 heads, 800 keys 41.1 and 40.2);
        //   8, 8 heads of 128, a prompt of 500, the others 1000, 2000, 4000, 30000 keys 26.6 and 23.5, 28.6 and 29.0, 34 and 39,
        //   119 and 222; of 64 dims 28.4 and 21.9, 29.3 and 29.4, 32 and 37; of 256, 500 to 4000 keys, 28.7 and 30.5, 32 and 38,
        //   36 and 48, 50 and 81 (4 heads, 1000 keys 32.0 and 29.1); 16 tokens behind 20000 keys, 4 heads, 84 and 148.
        // Where the tables have room for more than there is, the launch takes 2 for nothing (8 prompts of 300 35.5 and 33.5).
        const double room = (double)pc.R * pc.Nkv * pc.columns * pc.pageSize;
        few_ = (int64_t)pc.R * pc.Nkv > 64 || (pc.R > 1 && room > (hdp > 128 ? 1 << 15 : 1 << 17));
        wc_.manyRows = kFewRows;
        work_.fewRows = few_ ? kFewRows : 0;
        work_.manyRows = UINT32_MAX;
        const int64_t blocks = cdiv((int64_t)pc.columns * pc.pageSize, 256);
        work_.maxTiles = (uint32_t)std::min<int64_t>((int64_t)pc.R * blocks, INT32_MAX);
        work_.minSteps = 1;
        // A unit's start (its keys, the first rows) takes as long as about 10 steps. A prompt of 4096, 8192 tokens, 32 heads of 128 on 8,
        // us: 98.9, 319; with 3 steps counted 108.6, 358; with 14 99.9, 311 (8 heads of 256 on 4: 64.9, 177; 67.6, 192; 68.2, 187).
        work_.unitSteps = 10;
        const double steps = (double)work_.maxTiles * ((double)cdiv((int64_t)pc.T * G, 64) + work_.unitSteps);
        work_.workers = (uint32_t)std::max(1.0, std::min((hdp > 128 ? 1.0 : 2.0) * deviceCUs(), steps * pc.Nkv));
        work_.ownPlan = work_.maxTiles <= 1024 && pc.R <= 1024 && steps < 2147483648.0;
    }
    std::vector<Binding> tensors() const override {
        std::vector<Binding> b;
        for (const Tensor &t : in_) b.push_back({t, kRead});
        b.push_back({weights_, kReadWrite});
        return b;
    }
    std::string describe() const override {
        std::string s;
        if (few_) s = (wc_.ownPlan ? "" : "attention_weights_plan,") + fn_;
        if (!tile_.empty()) s += (few_ ? "," : "") + std::string(work_.ownPlan ? "" : "attention_weights_tiles,") + tile_ + ",attention_weights_join";
        return s;
    }
    void encode(KernelCommandEncoder &enc) const override {
        const std::vector<std::vector<uint8_t>> consts = {bytesOf(pc_), bytesOf(wc_)};
        auto run = [&](const Tensor &plan) {
            std::vector<Binding> b;
            for (const Tensor &t : in_) b.push_back({t, kRead});
            b.push_back({plan, kRead});
            b.push_back({weights_, kReadWrite});
            enc.encode(*Kernels::Custom(fn_, std::move(b), consts, dim3(blocks_, 1, 1), dim3(256, 1, 1)));
        };
        if (few_ && wc_.ownPlan) run(weights_);  // (not read)
        else if (few_)
            enc.withTemporaryTensor(ScratchSpec{{((int64_t)pc_.R + 1) * 8}, DataType::u8}, [&](Tensor plan) {
                enc.encode(*Kernels::Custom("attention_weights_plan", {{in_[3], kRead}, {in_[4], kRead}, {plan, kWrite}}, consts, dim3(1, 1, 1),
                                            dim3(1024, 1, 1)));
                run(plan);
            });
        if (tile_.empty()) return;
        // the partial sums, what is shared, the plan
        const int64_t sums = (int64_t)work_.workers * 2 * 256 * 4, shared = (int64_t)work_.workers * 32;
        const int64_t plan = work_.ownPlan ? 0 : ((int64_t)work_.maxTiles + 1) * 16;
        enc.withTemporaryTensor(ScratchSpec{{sums + shared + plan}, DataType::u8}, [&](Tensor scratch) {
            auto part = [&](int64_t at, int64_t bytes) { return Tensor((char *)scratch.data + at, Shape({bytes}), DataType::u8); };
            const Tensor partial = part(0, sums), left = part(sums, shared), tiles = part(sums + shared, plan);
            const std::vector<std::vector<uint8_t>> all = {bytesOf(pc_), bytesOf(work_), bytesOf(wc_)};
            if (plan)
                enc.encode(*Kernels::Custom("attention_weights_tiles", {{in_[3], kRead}, {in_[4], kRead}, {tiles, kWrite}}, all, dim3(1, 1, 1),
                                            dim3(1024, 1, 1)));
            std::vector<Binding> b;
            for (const Tensor &t : in_) b.push_back({t, kRead});
            for (const Binding &x : {Binding{tiles, kRead}, {partial, kWrite}, {left, kWrite}, {weights_, kReadWrite}}) b.push_back(x);
            enc.encode(*Kernels::Custom(tile_, std::move(b), all, dim3(work_.workers, 1, 1), dim3(256, 1, 1)));
            enc.encode(*Kernels::Custom("attention_weights_join",
                                        {{in_[2], kRead}, {partial, kRead}, {left, kRead}, {weights_, kReadWrite}}, {bytesOf(pc_)},
                                        dim3(work_.workers, 1, 1), dim3(256, 1, 1)));
        });
    }

private:
    std::vector<Tensor> in_;  // q, k, tables, starts, lens, lse
    Tensor weights_;
    PagedAttentionConstants pc_;
    AttentionWeightsConstants wc_{};
    PagedWorkConstants work_{};
    std::string fn_, tile_;
    bool few_ = true;
    unsigned blocks_ = 1;
};

// PagedEviction (evict.hip): the choice, then the moves of K and V.
class EvictionKernel : public Kernel {
public:
    EvictionKernel(const Tensor &weights, const Tensor &k, const Tensor &v, const Tensor &tables, const Tensor &lens, const Tensor &budgets,
                   const Tensor &kept, const Tensor &keptWeights, const EvictConstants &ec)
        : weights_(weights), k_(k), v_(v), tables_(tables), lens_(lens), budgets_(budgets), kept_(kept), keptWeights_(keptWeights), ec_(ec) {
        const int64_t row = k.shape[3] * stride(k.dataType);
        int unit = 16;
        while (row % unit || !aligned(k.data, unit) || !aligned(v.data, unit)) unit /= 2;
        fn_ = "evict_move_b" + std::to_string(unit * 8);
        ec_.rowUnits = (uint32_t)(row / unit);
        // A block's slice of the rows is 8 units, 128 bytes (48 requests cut to 1000 keys, 8 heads of 128: 58 us; of 4 units 78, of 16 65);
        // narrower while that gives fewer blocks than CUs (one request of 4 heads of 256, moved row by row: 12 us, and 23 in slices of 8).
        const int64_t rows = (int64_t)ec_.R * ec_.Nkv * 2;
        ec_.units = 8;
        while (ec_.units > 2 && rows * cdiv(ec_.rowUnits, ec_.units) < deviceCUs()) ec_.units /= 2;
    }
    std::vector<Binding> tensors() const override {
        return {{weights_, kRead}, {k_, kReadWrite}, {v_, kReadWrite}, {tables_, kRead}, {lens_, kRead}, {budgets_, kRead}, {kept_, kWrite}, {keptWeights_, kWrite}};
    }
    std::string describe() const override { return "evict_select," + fn_; }
    void encode(KernelCommandEncoder &enc) const override {
        const unsigned rows = ec_.R * ec_.Nkv;
        if (rows == 0) return;
        enc.encode(*Kernels::Custom("evict_select", {{weights_, kRead}, {lens_, kRead}, {budgets_, kRead}, {kept_, kWrite}, {keptWeights_, kWrite}},
                                    {bytesOf(ec_)}, dim3(rows, 1, 1), dim3(1024, 1, 1)));
        if (ec_.rowUnits == 0) return;
        enc.encode(*Kernels::Custom(fn_, {{kept_, kRead}, {tables_, kRead}, {lens_, kRead}, {budgets_, kRead}, {k_, kReadWrite}, {v_, kReadWrite}},
                                    {bytesOf(ec_)}, dim3(rows, (ec_.rowUnits + ec_.units - 1) / ec_.units, 2), dim3(1024, 1, 1)));
    }

private:
    Tensor weights_, k_, v_, tables_, lens_, budgets_, kept_, keptWeights_;
    EvictConstants ec_;
    std::string fn_;
};

// Sample (sample.hip): a row of up to SAMPLE_CANDIDATES logits by one block,
// a longer one in slices.
class SampleKernel : public Kernel {
public:
    SampleKernel(const Tensor &logits, const Tensor &uniforms, const Tensor *temperature, const Tensor *topK, const Tensor *topP,
                 const Tensor *minP, const Tensor &tokens)
        : logits_(logits), tokens_(tokens), type_(name(logits.dataType)) {
        const int64_t rows = logits.shape[0], vocab = logits.shape[1];
        options_ = {uniforms};
        for (const Tensor *t : {temperature, topK, topP, minP}) options_.push_back(t ? *t : uniforms);  // (not read where absent)
        sc_ = SampleConstants{(uint32_t)rows, (uint32_t)vocab, temperature != nullptr, topK != nullptr, topP != nullptr, minP != nullptr, 1, (uint32_t)vocab, 1};
        small_ = vocab <= SAMPLE_CANDIDATES;
        requireGrid(rows, 1024, "Sample", logits);
        if (small_ || rows == 0) return;
        // About 4 blocks per CU, in slices of 8192 logits or more, or of 4096 while they are fewer than the CUs: the last launch
        // reads one slice by one block. (One row of 256000 25.5 us, and 27.8 in slices of 8192; 33 rows of 50257 29.8, and
        // 32.2 in slices of 4096.)
        const int64_t most = std::max(cdiv(vocab, 8192), std::min(cdiv(vocab, 4096), deviceCUs() / rows));
        const int64_t slices = std::clamp<int64_t>(cdiv(4 * deviceCUs(), rows), 1, std::min<int64_t>(SAMPLE_MAX_SLICES, most));
        sc_.sliceLen = (uint32_t)cdiv(cdiv(vocab, slices), 8) * 8;
        sc_.slices = (uint32_t)cdiv(vocab, sc_.sliceLen);
        // a block of sample_gather reads the row's bins first: no more of them than run at once (2 per CU)
        sc_.parts = (uint32_t)std::clamp<int64_t>(2 * deviceCUs() / rows, 1, sc_.slices);
    }
    std::vector<Binding> tensors() const override {
        std::vector<Binding> b = options({{logits_, kRead}});
        b.push_back({tokens_, kWrite});
        return b;
    }
    std::string describe() const override {
        if (small_) return "sample_small_" + type_;
        return "sample_top_" + type_ + (cuts() ? ",sample_hist_" + type_ : "") + ",sample_gather_" + type_ + ",sample_finish_" + type_;
    }
    void encode(KernelCommandEncoder &enc) const override {
        if (sc_.rows == 0) return;
        if (small_) {
            std::vector<Binding> b = options({{logits_, kRead}});
            b.push_back({tokens_, kWrite});
            launch(enc, "sample_small_", std::move(b), sc_.rows);
            return;
        }
        const int64_t n = sc_.rows, blocks = n * sc_.slices;
        const int64_t rowBytes = n * (int64_t)sizeof(SampleRow), binBytes = cuts() ? blocks * SAMPLE_BINS * 8 : 0;
        enc.withTemporaryTensor(ScratchSpec{{rowBytes + binBytes}, DataType::u8}, [&](Tensor scratch) {
            const Tensor rows(scratch.data, Shape({rowBytes}), DataType::u8), bins((char *)scratch.data + rowBytes, Shape({binBytes}), DataType::u8);
            auto with = [&](std::initializer_list<Binding> more) {
                std::vector<Binding> b = options({{logits_, kRead}});
                b.insert(b.end(), more);
                return b;
            };
            launch(enc, "sample_top_", {{logits_, kRead}, {rows, kWrite}}, blocks);
            if (cuts()) launch(enc, "sample_hist_", with({{rows, kReadWrite}, {bins, kWrite}}), blocks);
            launch(enc, "sample_gather_", with({{rows, kReadWrite}, {bins, kRead}}), n * sc_.parts);
            launch(enc, "sample_finish_", with({{rows, kRead}, {tokens_, kWrite}}), n);
        });
    }

private:
    // A row may be cut, by top-k or top-p.
    bool cuts() const { return sc_.hasTopK || sc_.hasTopP; }
    std::vector<Binding> options(std::vector<Binding> b) const {
        for (const Tensor &t : options_) b.push_back({t, kRead});
        return b;
    }
    void launch(KernelCommandEncoder &enc, const char *fn, std::vector<Binding> b, int64_t blocks) const {
        enc.encode(*Kernels::Custom(fn + type_, std::move(b), {bytesOf(sc_)}, dim3((unsigned)blocks, 1, 1), dim3(1024, 1, 1)));
    }

    Tensor logits_, tokens_;
    std::vector<Tensor> options_;
    std::string type_;
    SampleConstants sc_{};
    bool small_ = false;
};

}  // namespace

namespace Kernels {

std::unique_ptr<Kernel> PageTables(const Tensor &pastLens, const Tensor &newLens, const Tensor &freePages,
                                   const Tensor &pageTables, int64_t pageSize, const Tensor &queryStarts,
                                   const Tensor &keyLens, const Tensor &positions, const Tensor &slots, const Tensor &counts) {
    using D = DataType;
    requireRank(pastLens, 1);
    requireRank(freePages, 1);
    requireRank(pageTables, 2);
    requireRank(positions, 1);
    const int64_t R = pastLens.shape[0], F = freePages.shape[0], M = pageTables.shape[1], T = positions.shape[0];
    if (pageSize <= 0 || pageSize >= (int64_t{1} << 31)) throw Error::invalidArgument("PageTables page size must be positive and below 2^31.");
    if (R >= (int64_t{1} << 31) - 1) throw Error::tensorShapeMismatch("PageTables takes fewer than 2^31 - 1 requests.");
    requireShape(pastLens, D::i32, {R}, "PageTables past_lens");
    requireShape(newLens, D::i32, {R}, "PageTables new_lens");
    requireShape(freePages, D::i32, {F}, "PageTables free_pages");
    requireShape(pageTables, D::i32, {R, M}, "PageTables page_tables");
    requireShape(queryStarts, D::i32, {R + 1}, "PageTables query_starts");
    requireShape(keyLens, D::i32, {R}, "PageTables key_lens");
    requireShape(positions, D::i32, {T}, "PageTables positions");
    requireShape(slots, D::i32, {T}, "PageTables slots");
    requireShape(counts, D::i32, {2}, "PageTables counts");
    requireApart("PageTables",
                 {{&pageTables, "page_tables"}, {&queryStarts, "query_starts"}, {&keyLens, "key_lens"}, {&positions, "positions"},
                  {&slots, "slots"}, {&counts, "counts"}},
                 {{&pastLens, "past_lens"}, {&newLens, "new_lens"}, {&freePages, "free_pages"}});
    const PageTablesConstants pc{(uint32_t)R, (uint32_t)M, (uint32_t)F, (uint32_t)T, (uint32_t)pageSize};
    const int64_t blocks = std::clamp<int64_t>(cdiv(T, 256), 1, 256);
    return fixed("page_tables",
                 {{pastLens, kRead}, {newLens, kRead}, {freePages, kRead}, {pageTables, kReadWrite}, {queryStarts, kWrite},
                  {keyLens, kWrite}, {positions, kWrite}, {slots, kWrite}, {counts, kWrite}},
                 bytesOf(pc), dim3((unsigned)blocks, 1, 1), 256);
}

std::unique_ptr<Kernel> PagedKVCacheWrite(const Tensor &k, const Tensor &v, const Tensor &slots, const Tensor &kCache,
                                          const Tensor &vCache) {
    using D = DataType;
    const D s = k.dataType, c = kCache.dataType;
    const char *fn = s == D::f32 && c == D::f32    ? "paged_kv_write_f32"
                     : s == D::f16 && c == D::f16   ? "paged_kv_write_f16"
                     : s == D::bf16 && c == D::bf16 ? "paged_kv_write_bf16"
                     : s == D::f32 && c == D::bf16  ? "paged_kv_write_f32_to_bf16"
                                                    : nullptr;
    if (!fn || v.dataType != s || vCache.dataType != c)
        throw Error::unsupportedDataTypeCombination(std::string("Unsupported paged KV cache data type combination: ") + name(s) + ", " +
                                                    name(v.dataType) + ", " + name(c) + ", " + name(vCache.dataType) + ".");
    requireCaches(kCache, vCache, "PagedKVCacheWrite");
    requireRank(k, 3);
    const int64_t T = k.shape[0], Nkv = kCache.shape[1], page = kCache.shape[2], Hd = kCache.shape[3];
    requireShape(k, s, {T, Nkv, Hd}, "PagedKVCacheWrite k");
    requireShape(v, s, {T, Nkv, Hd}, "PagedKVCacheWrite v");
    requireShape(slots, D::i32, {T}, "PagedKVCacheWrite slots");
    const int64_t run = 16 / stride(s), perToken = Nkv * cdiv(Hd, run);
    if (perToken >= (int64_t{1} << 30)) throw Error::tensorShapeMismatch("PagedKVCacheWrite rows are too long: " + k.shape.str() + ".");
    requireApart("PagedKVCacheWrite", {{&kCache, "k_cache"}, {&vCache, "v_cache"}}, {{&k, "k"}, {&v, "v"}, {&slots, "slots"}});
    const int64_t blocks = cdiv(T * perToken, 1024);
    requireGrid(blocks, 256, "PagedKVCacheWrite", k);
    const PagedKVWriteConstants pc{(uint32_t)T, (uint32_t)Nkv, (uint32_t)Hd, (uint32_t)page, (uint32_t)kCache.shape[0]};
    return fixed(fn, {{k, kRead}, {v, kRead}, {slots, kRead}, {kCache, kWrite}, {vCache, kWrite}}, bytesOf(pc),
                 dim3((unsigned)blocks, blocks ? 2 : 0, 1), 256);
}

std::unique_ptr<Kernel> PagedAttention(const Tensor &q, const Tensor &kCache, const Tensor &vCache, const Tensor &pageTables,
                                       const Tensor &queryStarts, const Tensor &keyLens, const Tensor &out, float scale,
                                       AttentionMask mask, int64_t sinks, int64_t maxQueryLen) {
    const PagedAttentionConstants pc =
        pagedConstants("PagedAttention", q, kCache, vCache, pageTables, queryStarts, keyLens, out, scale, mask, sinks, maxQueryLen);
    requireApart("PagedAttention", {{&out, "out"}},
                 {{&q, "q"}, {&kCache, "k_cache"}, {&vCache, "v_cache"}, {&pageTables, "page_tables"}, {&queryStarts, "query_starts"},
                  {&keyLens, "key_lens"}});
    if (pc.R && pc.T && fastRows(q, kCache, vCache, out))
        return std::make_unique<PagedAttentionKernel>(q, kCache, vCache, pageTables, queryStarts, keyLens, out, pc, maxQueryLen);
    return fixed("paged_attention_plain_" + plainName(q, kCache, vCache), {{q, kRead}, {kCache, kRead}, {vCache, kRead}, {pageTables, kRead}, {queryStarts, kRead}, {keyLens, kRead}, {out, kWrite}},
                 bytesOf(pc), dim3(pc.R ? pc.T * pc.Nq : 0, 1, 1), 256);
}

std::unique_ptr<Kernel> SharedPrefixAttention(const Tensor &q, const Tensor &kCache, const Tensor &vCache, const Tensor *prefixTables,
                                              const Tensor *prefixLens, const Tensor *groupStarts, const Tensor &pageTables,
                                              const Tensor &queryStarts, const Tensor &keyLens, const Tensor &out, const Tensor *lse,
                                              float scale, AttentionMask mask, int64_t sinks, int64_t maxQueryLen) {
    using D = DataType;
    const std::string op = "SharedPrefixAttention";
    if (!prefixTables != !prefixLens || !prefixTables != !groupStarts)
        throw Error::invalidArgument(op + " takes prefix_tables, prefix_lens and group_starts together, or none of them.");
    const PagedAttentionConstants pc = pagedConstants(op, q, kCache, vCache, pageTables, queryStarts, keyLens, out, scale, mask, sinks, maxQueryLen);
    std::vector<Named> inputs = {{&q, "q"}, {&kCache, "k_cache"}, {&vCache, "v_cache"}, {&pageTables, "page_tables"},
                                 {&queryStarts, "query_starts"}, {&keyLens, "key_lens"}};
    SharedPrefixConstants sc{};
    if (prefixTables) {
        requireRank(*prefixTables, 2);
        const int64_t g = prefixTables->shape[0];
        if (g >= (int64_t{1} << 31) - 1 - pc.R) throw Error::tensorShapeMismatch(op + " takes fewer groups and requests than 2^31 - 1.");
        requireShape(*prefixTables, D::i32, {g, prefixTables->shape[1]}, op + " prefix_tables");
        requireShape(*prefixLens, D::i32, {g}, op + " prefix_lens");
        requireShape(*groupStarts, D::i32, {g + 1}, op + " group_starts");
        sc.groups = (uint32_t)g;
        sc.columns = (uint32_t)prefixTables->shape[1];
        for (const Named &n : {Named{prefixTables, "prefix_tables"}, {prefixLens, "prefix_lens"}, {groupStarts, "group_starts"}}) inputs.push_back(n);
    }
    std::vector<Named> outputs = {{&out, "out"}};
    if (lse) {
        requireShape(*lse, D::f32, {q.shape[0], q.shape[1]}, op + " lse");
        outputs.push_back({lse, "lse"});
    }
    requireApart(op, outputs, inputs);
    sc.hasLse = lse != nullptr;
    sc.windowed = mask.kind == 1 && sc.groups > 0;
    const Tensor &none = queryStarts;  // (not read where there is no group)
    std::vector<Tensor> in = {q, kCache, vCache, pageTables, queryStarts, keyLens, prefixTables ? *prefixTables : none,
                              prefixLens ? *prefixLens : none, groupStarts ? *groupStarts : none};
    if (pc.R && pc.T && fastRows(q, kCache, vCache, out)) return std::make_unique<SharedPrefixKernel>(std::move(in), out, lse, pc, sc, maxQueryLen);
    sc.rows = pc.T * pc.Nq;
    std::vector<Binding> b;
    for (const Tensor &t : in) b.push_back({t, kRead});
    b.push_back({out, kWrite});
    b.push_back({lse ? *lse : out, kWrite});
    return Kernels::Custom("shared_prefix_plain_" + plainName(q, kCache, vCache), std::move(b), {bytesOf(pc), bytesOf(sc)},
                           dim3(pc.R ? pc.T * pc.Nq : 0, 1, 1), dim3(256, 1, 1));
}

std::unique_ptr<Kernel> PagedAttentionWeights(const Tensor &q, const Tensor &kCache, const Tensor &pageTables, const Tensor &queryStarts,
                                              const Tensor &keyLens, const Tensor &lse, const Tensor &weights, float scale,
                                              AttentionMask mask, int64_t lastRows, int64_t maxQueryLen) {
    using D = DataType;
    const std::string op = "PagedAttentionWeights";
    if (mask.kind == 1)
        throw Error::invalidArgument(op + " takes causal or bidirectional attention: a sliding window's places are lost with the keys that are evicted.");
    if (lastRows < 0) throw Error::invalidArgument(op + " last_rows must not be negative.");
    const PagedAttentionConstants pc = pagedConstants(op, q, kCache, kCache, pageTables, queryStarts, keyLens, q, scale, mask, 0, maxQueryLen);
    requireShape(lse, D::f32, {q.shape[0], q.shape[1]}, op + " lse");
    requireShape(weights, D::f32, {(int64_t)pc.R, (int64_t)pc.Nkv, (int64_t)pc.columns * pc.pageSize}, op + " weights");
    requireApart(op, {{&weights, "weights"}},
                 {{&q, "q"}, {&kCache, "k_cache"}, {&pageTables, "page_tables"}, {&queryStarts, "query_starts"}, {&keyLens, "key_lens"}, {&lse, "lse"}});
    std::vector<Tensor> in = {q, kCache, pageTables, queryStarts, keyLens, lse};
    if (pc.R && pc.T && fastRows(q, kCache, kCache, q))
        return std::make_unique<AttentionWeightsKernel>(std::move(in), weights, pc, lastRows, maxQueryLen);
    const AttentionWeightsConstants wc{(uint32_t)std::min<int64_t>(lastRows, pc.T), 0, UINT32_MAX, 0, 0};
    std::vector<Binding> b;
    for (const Tensor &t : in) b.push_back({t, kRead});
    b.push_back({weights, kReadWrite});
    requireGrid((int64_t)pc.R * pc.Nkv, 256, op, weights);
    // about 2 blocks per CU, of 16 keys and more
    const int64_t pairs = std::max<int64_t>((int64_t)pc.R * pc.Nkv, 1);
    const int64_t parts = std::clamp<int64_t>(2 * deviceCUs() / pairs, 1, std::max<int64_t>(1, cdiv((int64_t)pc.columns * pc.pageSize, 16)));
    return Kernels::Custom(std::string("attention_weights_plain_") + name(q.dataType), std::move(b), {bytesOf(pc), bytesOf(wc)},
                           dim3(pc.T ? pc.R * pc.Nkv : 0, (unsigned)parts, 1), dim3(256, 1, 1));
}

std::unique_ptr<Kernel> PagedEviction(const Tensor &weights, const Tensor &kCache, const Tensor &vCache, const Tensor &pageTables,
                                      const Tensor &keyLens, const Tensor &budgets, const Tensor &kept, const Tensor &keptWeights,
                                      int64_t first, int64_t last) {
    using D = DataType;
    const std::string op = "PagedEviction";
    if (!isFloat(kCache.dataType) || vCache.dataType != kCache.dataType)
        throw Error::unsupportedDataTypeCombination(op + " needs caches of one floating dtype; got " + name(kCache.dataType) + ", " + name(vCache.dataType) + ".");
    if (first < 0 || last < 0 || first >= (int64_t{1} << 31) || last >= (int64_t{1} << 31))
        throw Error::invalidArgument(op + " first and last must be at least 0 and below 2^31.");
    requireCaches(kCache, vCache, op);
    requireRank(pageTables, 2);
    const int64_t R = pageTables.shape[0], M = pageTables.shape[1], Nkv = kCache.shape[1], page = kCache.shape[2];
    const int64_t room = requireRoom(op, M, page);
    requireShape(pageTables, D::i32, {R, M}, op + " page_tables");
    requireShape(keyLens, D::i32, {R}, op + " key_lens");
    requireShape(budgets, D::i32, {R}, op + " budgets");
    requireShape(weights, D::f32, {R, Nkv, room}, op + " weights");
    requireShape(kept, D::i32, {R, Nkv, room}, op + " kept");
    requireShape(keptWeights, D::f32, {R, Nkv, room}, op + " kept_weights");
    requireGrid(R * Nkv, 1024, op, weights);
    const int64_t slices = cdiv(kCache.shape[3] * stride(kCache.dataType), 4);  // (of 2 units of 2 bytes)
    if (slices > 65535) throw Error::tensorShapeMismatch(op + " rows are too long: " + kCache.shape.str() + ".");
    requireApart(op, {{&kCache, "k_cache"}, {&vCache, "v_cache"}, {&kept, "kept"}, {&keptWeights, "kept_weights"}},
                 {{&weights, "weights"}, {&pageTables, "page_tables"}, {&keyLens, "key_lens"}, {&budgets, "budgets"}});
    const EvictConstants ec{(uint32_t)R, (uint32_t)Nkv, (uint32_t)M, (uint32_t)page, (uint32_t)kCache.shape[0], (uint32_t)first, (uint32_t)last, 0, 8};
    return std::make_unique<EvictionKernel>(weights, kCache, vCache, pageTables, keyLens, budgets, kept, keptWeights, ec);
}

std::unique_ptr<Kernel> ReleasePages(const Tensor &keyLens, const Tensor &budgets, const Tensor &pageTables, int64_t pageSize,
                                     const Tensor &newLens, const Tensor &freed, const Tensor &counts) {
    using D = DataType;
    const std::string op = "ReleasePages";
    requireRank(pageTables, 2);
    const int64_t R = pageTables.shape[0], M = pageTables.shape[1];
    if (pageSize <= 0 || pageSize >= (int64_t{1} << 31)) throw Error::invalidArgument(op + " page size must be positive and below 2^31.");
    requireShape(pageTables, D::i32, {R, M}, op + " page_tables");
    requireRoom(op, M, pageSize);
    requireShape(keyLens, D::i32, {R}, op + " key_lens");
    requireShape(budgets, D::i32, {R}, op + " budgets");
    requireShape(newLens, D::i32, {R}, op + " new_lens");
    requireShape(freed, D::i32, {R * M}, op + " freed");
    requireShape(counts, D::i32, {1}, op + " counts");
    requireApart(op, {{&newLens, "new_lens"}, {&freed, "freed"}, {&counts, "counts"}},
                 {{&keyLens, "key_lens"}, {&budgets, "budgets"}, {&pageTables, "page_tables"}});
    const EvictConstants ec{(uint32_t)R, 1, (uint32_t)M, (uint32_t)pageSize, 0, 0, 0, 0, 0};
    const int64_t blocks = std::clamp<int64_t>(cdiv(R, 16), 1, 256);
    return fixed("release_pages", {{keyLens, kRead}, {budgets, kRead}, {pageTables, kRead}, {newLens, kWrite}, {freed, kWrite}, {counts, kWrite}},
                 bytesOf(ec), dim3((unsigned)blocks, 1, 1), 256);
}

std::unique_ptr<Kernel> Sample(const Tensor &logits, const Tensor &uniforms, const Tensor *temperature, const Tensor *topK,
                               const Tensor *topP, const Tensor *minP, const Tensor &tokens) {
    using D = DataType;
    if (!isFloat(logits.dataType))
        throw Error::unsupportedDataTypeCombination(std::string("Sample logits must be f32, f16 or bf16; got ") + name(logits.dataType) + ".");
    requireRank(logits, 2);
    const int64_t rows = logits.shape[0], vocab = logits.shape[1];
    if (vocab <= 0 || vocab > (int64_t{1} << 22))
        throw Error::tensorShapeMismatch("Sample takes 1 to 2^22 logits a row; got " + std::to_string(vocab) + ".");
    requireTensor(logits, "Sample logits");
    requireShape(uniforms, D::f32, {rows}, "Sample uniforms");
    requireShape(tokens, D::i32, {rows}, "Sample tokens");
    if (temperature) requireShape(*temperature, D::f32, {rows}, "Sample temperature");
    if (topK) requireShape(*topK, D::i32, {rows}, "Sample top_k");
    if (topP) requireShape(*topP, D::f32, {rows}, "Sample top_p");
    if (minP) requireShape(*minP, D::f32, {rows}, "Sample min_p");
    std::vector<Named> inputs = {{&logits, "logits"}, {&uniforms, "uniforms"}};
    for (const Named &n : {Named{temperature, "temperature"}, {topK, "top_k"}, {topP, "top_p"}, {minP, "min_p"}})
        if (n.first) inputs.push_back(n);
    requireApart("Sample", {{&tokens, "tokens"}}, inputs);
    return std::make_unique<SampleKernel>(logits, uniforms, temperature, topK, topP, minP, tokens);
}

}  // namespace Kernels
}  // namespace popcorn
