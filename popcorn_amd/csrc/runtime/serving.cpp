// Kernels.* descriptors of a batch of requests over a paged cache: page tables,
// the paged cache write, paged attention, and the draw of the next token.
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

// PagedAttention on the matrix cores (paged_attention.hip): requests of few
// rows (new tokens x heads of a KV head's group) and of many by a launch each,
// with plans of tiles where the blocks do not lay them out themselves, and the
// merge of what several blocks shared.
class PagedAttentionKernel : public Kernel {
public:
    PagedAttentionKernel(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &tables, const Tensor &starts, const Tensor &lens,
                         const Tensor &out, const PagedAttentionConstants &pc, int64_t maxQueryLen)
        : q_(q), k_(k), v_(v), tables_(tables), starts_(starts), lens_(lens), out_(out), pc_(pc) {
        const int64_t G = pc.Nq / pc.Nkv, longest = std::min<int64_t>(maxQueryLen > 0 ? maxQueryLen : pc.T, pc.T) * G;
        const bool f32 = q.dataType == DataType::f32;
        hdp_ = pc.Hd <= 64 ? 64 : pc.Hd <= 128 ? 128 : pc.Hd <= 256 ? 256 : 512;
        const std::string type = name(q.dataType), hd = "_d" + std::to_string(hdp_);
        merge_ = "paged_attention_merge_" + type + hd;
        // The tile kernel works on the magnitude of the scale (not 0) and 16-bit K and V of up to 256 dims. For requests of up to
        // 32 rows, or so few rows in all, the tiles' 128 rows cost more than reading keys again: us of the few-row kernel and of
        // tiles, 4 heads to a KV head, 8 KV heads, 4000 keys: one request of 64 rows 26 and 33 (Hd 128), 34 and 43 (256), of 128
        // rows 27 and 40, 38 and 46 (but 96 and 67 behind 16000 keys), of 256 rows 33 and 39, 54 and 47.
        const int tilesPerCU = hdp_ == 256 ? 1 : 2;
        const bool tiles = !f32 && hdp_ <= 256 && pc.scale != 0.0f && pc.scale == pc.scale && longest > kFewRows &&
                           (int64_t)pc.T * G > (hdp_ == 256 ? 64 : 128);
        // Beside tiles, the requests of few rows have a launch of their own where there are more units than blocks: one request of
        // 500 tokens among 256 of up to 1000 keys on 8 KV heads of 128, 80 us and 107 in tiles alone, 128 on 4 of 256 72 and 88;
        // but as many units as blocks (64 of up to 8000 keys on 8) 81 and 78, 12 requests of few keys 41 and 31.
        const bool apart = tiles && (int64_t)pc.R * pc.Nkv > tilesPerCU * deviceCUs();
        if (!tiles || apart) {
            // 16 rows per wave or 32: 16 requests of 32 rows, 2000 keys, us: Hd 64 31.1 and 26.5, Hd 256 90 and 60, of 16 rows 22.5
            // and 25.0, 54 and 56. Registers for 32 are wanting at Hd 512 and in f32 at 256 (84 and 198 there).
            const int rt = hdp_ == 512 || (f32 && hdp_ == 256) || longest <= 16 || tiles ? 1 : 2;
            // as many blocks as run at once (the kernels' registers)
            const int perCU = hdp_ == 64 ? 5 - rt : hdp_ == 128 ? 4 - rt : hdp_ == 256 && rt == 1 && !f32 ? 2 : 1;
            add("paged_attention_few_" + type + hd + "_r" + std::to_string(rt), 16 * rt, f32 ? 16 : 32, 0, tiles ? kFewRows : UINT32_MAX, perCU);
        }
        if (tiles) add("paged_attention_tile_" + type + hd, 128, 64, apart ? kFewRows : 0, UINT32_MAX, tilesPerCU);
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
    static constexpr uint32_t kFewRows = 32;
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
    using D = DataType;
    const D t = q.dataType;
    if (!isFloat(t) || kCache.dataType != t || vCache.dataType != t || out.dataType != t)
        throw Error::unsupportedDataTypeCombination(std::string("PagedAttention needs one floating dtype for q, the caches and out; got ") +
                                                    name(t) + ", " + name(kCache.dataType) + ", " + name(vCache.dataType) + ", " +
                                                    name(out.dataType) + ".");
    if (mask.kind > 2) throw Error::invalidArgument("unknown attention mask kind");
    if (sinks < 0 || sinks >= (int64_t{1} << 31)) throw Error::invalidArgument("PagedAttention sinks must be at least 0 and below 2^31.");
    if (sinks > 0 && mask.kind != 1) throw Error::invalidArgument("PagedAttention sinks go with a sliding window.");
    if (maxQueryLen < 0) throw Error::invalidArgument("PagedAttention max_query_len must not be negative.");
    requireCaches(kCache, vCache, "PagedAttention");
    requireRank(q, 3);
    requireRank(pageTables, 2);
    const int64_t T = q.shape[0], Nq = q.shape[1], Hd = q.shape[2], Nkv = kCache.shape[1], page = kCache.shape[2];
    const int64_t R = pageTables.shape[0], M = pageTables.shape[1];
    if (Nkv <= 0 || Nq <= 0 || Nq % Nkv != 0)
        throw Error::tensorShapeMismatch("PagedAttention query heads must be divisible by KV heads; got " + std::to_string(Nq) + " and " +
                                         std::to_string(Nkv) + ".");
    if (Hd <= 0 || Hd > 512)
        throw Error::tensorShapeMismatch("PagedAttention head dim must be 1 to 512 (kernel limit); got " + std::to_string(Hd) + ".");
    if (kCache.shape[3] != Hd)
        throw Error::tensorShapeMismatch("PagedAttention caches must have q's head dim; got " + q.shape.str() + " and " + kCache.shape.str() + ".");
    if (page % 16 != 0)
        throw Error::tensorShapeMismatch("PagedAttention page size must be a multiple of 16; got " + std::to_string(page) + ".");
    requireShape(q, t, {T, Nq, Hd}, "PagedAttention q");
    requireShape(out, t, {T, Nq, Hd}, "PagedAttention out");
    requireShape(pageTables, D::i32, {R, M}, "PagedAttention page_tables");
    requireShape(queryStarts, D::i32, {R + 1}, "PagedAttention query_starts");
    requireShape(keyLens, D::i32, {R}, "PagedAttention key_lens");
    requireGrid(T * Nq, 256, "PagedAttention", q);
    requireApart("PagedAttention", {{&out, "out"}},
                 {{&q, "q"}, {&kCache, "k_cache"}, {&vCache, "v_cache"}, {&pageTables, "page_tables"}, {&queryStarts, "query_starts"},
                  {&keyLens, "key_lens"}});
    const PagedAttentionConstants pc{(uint32_t)T, (uint32_t)R, (uint32_t)Nq, (uint32_t)Nkv, (uint32_t)Hd, (uint32_t)page,
                                     (uint32_t)kCache.shape[0], (uint32_t)M, mask.kind, mask.window, (uint32_t)sinks, scale};
    // 16-byte rows: the matrix cores
    if (R && T && Hd % (16 / stride(t)) == 0 && aligned(q.data, 16) && aligned(kCache.data, 16) && aligned(vCache.data, 16) && aligned(out.data, 16))
        return std::make_unique<PagedAttentionKernel>(q, kCache, vCache, pageTables, queryStarts, keyLens, out, pc, maxQueryLen);
    std::string fn = std::string("paged_attention_plain_") + name(t);
    const int run = 4 * stride(t);
    if (Hd % 4 || !aligned(kCache.data, run) || !aligned(vCache.data, run)) fn += "_any";
    return fixed(fn, {{q, kRead}, {kCache, kRead}, {vCache, kRead}, {pageTables, kRead}, {queryStarts, kRead}, {keyLens, kRead}, {out, kWrite}},
                 bytesOf(pc), dim3((unsigned)(R ? T * Nq : 0), 1, 1), 256);
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
