// session.cpp -- cached generation: the page bookkeeping (PageTable) and the
// sequences of one model over a paged 8-bit key/value cache (Session).  The
// reference's generate loop has neither: it runs the whole prefix again for
// every token (transformer.cu:986-1036).
//
// The bookkeeping is on the host, since it decides what a step launches; the
// pages' contents never leave the GPU (gbx_kv_append, gbx_attn_cached,
// gbx_kv_copy_pages).
#include <algorithm>
#include <cstring>
#include <functional>

#include <cuda_runtime.h>

#include "gbx_model.hpp"

namespace gbx {

// kv_cache.cu: pages src of one pool become pages dst of another
int kv_copy_across(const gbx_kv_cache* from, const gbx_kv_cache* to, const int32_t* src, const int32_t* dst, int n, int* err,
                   gbx_stream_t stream);

// ---------------------------------------------------------------- pages
// (pages of no tokens: none)
PageTable::PageTable(int64_t pages, int pageSize)
    : pageSize_(pageSize < 1 ? 1 : pageSize), refs_((size_t)(pages < 0 || pageSize < 1 ? 0 : pages), 0)
{
    free_.resize(refs_.size());
    for (size_t i = 0; i < free_.size(); ++i) free_[i] = (int32_t)i;   // sorted: a heap already
}

int32_t PageTable::take()
{
    std::pop_heap(free_.begin(), free_.end(), std::greater<int32_t>());
    const int32_t p = free_.back();
    free_.pop_back();
    refs_[p] = 1;
    return p;
}

void PageTable::drop(int32_t page)
{
    if (--refs_[page] == 0) {
        free_.push_back(page);
        std::push_heap(free_.begin(), free_.end(), std::greater<int32_t>());
    }
}

int PageTable::newSequence()
{
    size_t i = 0;
    while (i < seqs_.size() && seqs_[i].live) ++i;
    if (i == seqs_.size()) seqs_.emplace_back();
    seqs_[i] = Seq();
    seqs_[i].live = true;
    return (int)i;
}

int PageTable::fork(int seq)
{
    if (!known(seq)) return -1;
    const int id = newSequence();   // may move seqs_
    seqs_[id].pages = seqs_[seq].pages;
    seqs_[id].length = seqs_[seq].length;
    for (int32_t p : seqs_[id].pages) ++refs_[p];
    return id;
}

bool PageTable::release(int seq)
{
    if (!known(seq)) return false;
    for (int32_t p : seqs_[seq].pages) drop(p);
    seqs_[seq] = Seq();
    return true;
}

bool PageTable::truncate(int seq, int64_t length)
{
    if (!known(seq) || length < 0 || length > seqs_[seq].length) return false;
    Seq& s = seqs_[seq];
    const size_t keep = (size_t)((length + pageSize_ - 1) / pageSize_);
    while (s.pages.size() > keep) {
        drop(s.pages.back());
        s.pages.pop_back();
    }
    s.length = length;
    return true;
}

bool PageTable::append(const std::vector<int>& seqs, const std::vector<int>& n, Copies* copies)
{
    if (seqs.size() != n.size()) return false;
    std::vector<int> sorted = seqs;
    std::sort(sorted.begin(), sorted.end());
    if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end()) return false;
    // what it takes: new pages, and a copy of a last page that others hold too.
    // Of r sequences of this call that share such a page with nobody else, the
    // last one keeps it.
    int64_t need = 0;
    std::map<int32_t, int> left;   // references of shared last pages, counted down
    auto writes = [&](const Seq& s, int count) { return count > 0 && s.length % pageSize_ != 0; };
    for (size_t i = 0; i < seqs.size(); ++i) {
        if (!known(seqs[i]) || n[i] < 0) return false;
        const Seq& s = seqs_[seqs[i]];
        need += (s.length + n[i] + pageSize_ - 1) / pageSize_ - (int64_t)s.pages.size();
        if (writes(s, n[i])) {
            auto it = left.emplace(s.pages.back(), refs_[s.pages.back()]).first;
            if (it->second > 1) {
                --it->second;
                ++need;
            }
        }
    }
    if (need > (int64_t)free_.size()) return false;
    for (size_t i = 0; i < seqs.size(); ++i) {
        Seq& s = seqs_[seqs[i]];
        if (writes(s, n[i]) && refs_[s.pages.back()] > 1) {
            const int32_t old = s.pages.back(), own = take();
            copies->src.push_back(old);
            copies->dst.push_back(own);
            s.pages.back() = own;
            drop(old);
        }
        s.length += n[i];
        while ((int64_t)s.pages.size() * pageSize_ < s.length) s.pages.push_back(take());
    }
    return true;
}

PageTable::Copies PageTable::compact()
{
    Copies c;
    const int64_t used = pages() - freePages();
    std::vector<int32_t> to(refs_.size(), -1);
    int32_t low = 0;
    for (int64_t p = used; p < pages(); ++p) {
        if (!refs_[p]) continue;
        while (refs_[low]) ++low;   // a free page below `used` for every page in use above it
        c.src.push_back((int32_t)p);
        c.dst.push_back(low);
        to[p] = low;
        refs_[low] = refs_[p];
        refs_[p] = 0;
    }
    for (Seq& s : seqs_)
        for (int32_t& p : s.pages)
            if (to[p] >= 0) p = to[p];
    free_.clear();
    for (int64_t p = used; p < pages(); ++p) free_.push_back((int32_t)p);
    return c;
}

// ---------------------------------------------------------------- sessions
namespace {

// A device array that grows to the largest use.
struct Array {
    void* p = nullptr;
    size_t bytes = 0;
    bool ensure(size_t want)
    {
        if (want <= bytes) return true;
        release();
        if (cudaMalloc(&p, want) != cudaSuccess) {
            cudaGetLastError();
            p = nullptr;
            return false;
        }
        bytes = want;
        return true;
    }
    void release()
    {
        if (p) cudaFree(p);
        p = nullptr;
        bytes = 0;
    }
};

struct OnDevice {   // the model's device current, for a scope
    int before = -1;
    explicit OnDevice(int device)
    {
        if (cudaGetDevice(&before) == cudaSuccess && before != device && device >= 0) cudaSetDevice(device);
        else before = -1;
    }
    ~OnDevice()
    {
        if (before >= 0) cudaSetDevice(before);
    }
};

}  // namespace

struct Session::Impl {
    gbx_kv_cache cache = {};
    Array k, v, ks, vs;      // the pool
    Array step;              // a step's integers: table, lengths, counts, positions
    Array ws;                // of gbx_attn_cached
    Array select;            // of token selection and verification
    Array pairs;             // of page copies
    Array rows;              // a verification's QKV rows of every layer, as tf32 pairs
    // What a step's appends can change of the tokens before it: a sequence's last
    // page, where it is not full, has its scales raised and its codes rounded anew
    // (or, by a NaN, lost).  Such pages are copied here first.
    gbx_kv_cache saved = {};
    Array sk, sv, sks, svs;
    std::vector<int32_t> savedPages;           // page of the pool that saved page i is a copy of
    const int32_t* savedIds = nullptr;         // the same on the device, and after them 0, 1, ..
    int32_t* err = nullptr;
    int device = -1;
    cudaStream_t stream = nullptr;   // the model's
    ~Impl()
    {
        OnDevice on(device);
        for (Array* a : {&k, &v, &ks, &vs, &step, &ws, &select, &pairs, &rows, &sk, &sv, &sks, &svs}) a->release();
        if (err) cudaFree(err);
    }
    // Room for n pages beside the pool.
    bool ensureSaved(size_t n)
    {
        const size_t scales = (size_t)cache.layers * n * cache.heads, codes = scales * cache.page * cache.hd;
        if (!sk.ensure(codes) || !sv.ensure(codes) || !sks.ensure(scales * 4) || !svs.ensure(scales * 4)) return false;
        saved = cache;
        saved.k = (int8_t*)sk.p;
        saved.v = (int8_t*)sv.p;
        saved.k_scale = (float*)sks.p;
        saved.v_scale = (float*)svs.p;
        saved.pages = (int64_t)n;
        return true;
    }
    // The saved pages' contents back in the pool.
    bool putBack()
    {
        if (savedPages.empty()) return true;
        OnDevice on(device);
        const int n = (int)savedPages.size();
        savedPages.clear();
        return kv_copy_across(&saved, &cache, savedIds + n, savedIds, n, nullptr, reinterpret_cast<gbx_stream_t>(stream)) == GBX_OK &&
               cudaStreamSynchronize(stream) == cudaSuccess;
    }
};

// Undoes a step that does not come to its end: the pages that it wrote to have
// their contents back, and the page table is as it was, so that pages it copied
// from, or took, are again whose they were.
struct Session::Undo {
    Session& s;
    PageTable before;
    bool done = false;
    explicit Undo(Session& session) : s(session), before(session.table_) { s.impl_->savedPages.clear(); }
    ~Undo()
    {
        if (done) return;
        if (!s.impl_->putBack()) s.ok_ = false;   // the sequences' last pages are lost: none of them can be used
        s.table_ = std::move(before);
    }
};

bool Session::fail(const std::string& msg)
{
    err_ = msg;
    return false;
}

Session::Session(TransformerModel& model, int64_t pages, int pageSize)
    : model_(model), table_(pages, pageSize), impl_(new Impl)
{
    Impl& m = *impl_;
    gbx_stream_t gs = nullptr;
    if (!model.isModelLoaded() || !model.streamAndDevice(&gs, &m.device)) {
        fail("session: model not loaded");
        return;
    }
    m.stream = reinterpret_cast<cudaStream_t>(gs);
    if (pages <= 0 || pages > 0x7fffffffLL || (pageSize != 16 && pageSize != 32 && pageSize != 64 && pageSize != 128)) {
        fail("session: " + std::to_string(pages) + " pages of " + std::to_string(pageSize) + " tokens (16, 32, 64 or 128)");
        return;
    }
    const int heads = model.getNumHeads(), hd = model.getEmbedDim() / heads, layers = model.getNumLayers();
    if (hd % 16 || hd > 128) {
        fail("session: head width " + std::to_string(hd) + " (a multiple of 16 up to 128)");
        return;
    }
    OnDevice on(m.device);
    const size_t scales = (size_t)layers * pages * heads, codes = scales * pageSize * hd;
    if (!m.k.ensure(codes ? codes : 16) || !m.v.ensure(codes ? codes : 16) || !m.ks.ensure(scales * 4 + 4) || !m.vs.ensure(scales * 4 + 4) ||
        cudaMalloc(&m.err, sizeof(int32_t)) != cudaSuccess) {
        cudaGetLastError();
        fail("session: cudaMalloc of the cache failed");
        return;
    }
    m.cache.k = (int8_t*)m.k.p;
    m.cache.v = (int8_t*)m.v.p;
    m.cache.k_scale = (float*)m.ks.p;
    m.cache.v_scale = (float*)m.vs.p;
    m.cache.pages = pages;
    m.cache.layers = layers;
    m.cache.page = pageSize;
    m.cache.heads = heads;
    m.cache.hd = hd;
    ok_ = true;
}

Session::~Session() = default;

// The arguments of a step; *padded: ids in rows of S, zeros behind a sequence's own.
bool Session::check(const std::vector<int>& seqs, const std::vector<int>& ids, const std::vector<int>& counts, int* S,
                    std::vector<int>* padded)
{
    err_.clear();
    if (!ok_) return fail("session: not open");
    if (seqs.empty() || seqs.size() != counts.size()) return fail("session: a count for each of at least one sequence");
    int64_t all = 0;
    *S = 0;
    for (size_t i = 0; i < seqs.size(); ++i) {
        if (!table_.known(seqs[i])) return fail("session: no sequence " + std::to_string(seqs[i]));
        if (counts[i] <= 0) return fail("session: every sequence needs a token");
        if (table_.length(seqs[i]) + counts[i] > model_.getMaxSeqLen())
            return fail("session: " + std::to_string(table_.length(seqs[i]) + counts[i]) + " tokens exceed the " +
                        std::to_string(model_.getMaxSeqLen()) + " position rows");
        all += counts[i];
        *S = std::max(*S, counts[i]);
    }
    if (all != (int64_t)ids.size())
        return fail("session: " + std::to_string(ids.size()) + " ids for " + std::to_string(all) + " tokens");
    padded->assign(seqs.size() * (size_t)*S, 0);
    size_t at = 0;
    for (size_t i = 0; i < seqs.size(); ++i)
        for (int j = 0; j < counts[i]; ++j) (*padded)[i * *S + j] = ids[at++];
    return true;
}

// Appends and runs the model; the logits stay in the model's buffer.  The caller's
// Undo takes it back if this, or what it does with the logits, fails.  keepRows:
// the layers' QKV rows stay, for keepOnly.
bool Session::step(const std::vector<int>& seqs, const std::vector<int>& ids, const std::vector<int>& counts, bool allRows,
                   const std::vector<int>& padded, int S, bool keepRows)
{
    Impl& m = *impl_;
    OnDevice on(m.device);
    const size_t rowFloats = keepRows ? padded.size() * 3 * (size_t)model_.getEmbedDim() * m.cache.layers : 0;
    if (!m.rows.ensure(rowFloats * 8)) return fail("session: cudaMalloc of the step's rows failed");
    std::vector<int64_t> before;
    bool even = true;
    for (size_t i = 0; i < seqs.size(); ++i) {
        before.push_back(table_.length(seqs[i]));
        even = even && counts[i] == S;
    }
    PageTable::Copies copies;
    if (!table_.append(seqs, counts, &copies))
        return fail("session: a sequence is listed twice, or the cache has too few free pages (" +
                    std::to_string(table_.freePages()) + ")");
    const int B = (int)seqs.size();
    size_t most = 1;
    for (int s : seqs) most = std::max(most, table_.pagesOf(s).size());
    // the pages that hold tokens of before and get new ones (each one sequence's own by now)
    std::vector<int32_t> partial;
    for (int b = 0; b < B; ++b)
        if (before[b] % table_.pageSize()) partial.push_back(table_.pagesOf(seqs[b])[(size_t)(before[b] / table_.pageSize())]);
    // one array: table, lengths, counts, counts of the sequences that go on, positions, the pairs of page copies, the partial pages and 0, 1, ..
    const size_t nCopies = copies.src.size(), nPartial = partial.size();
    std::vector<int32_t> host((size_t)B * most + 3 * (size_t)B + (size_t)B * S, 0);
    const size_t atCopies = host.size(), atPartial = atCopies + 2 * nCopies;
    host.insert(host.end(), copies.src.begin(), copies.src.end());
    host.insert(host.end(), copies.dst.begin(), copies.dst.end());
    host.insert(host.end(), partial.begin(), partial.end());
    for (size_t i = 0; i < nPartial; ++i) host.push_back((int32_t)i);
    int32_t *kvLen = host.data() + (size_t)B * most, *nNew = kvLen + B, *nGoing = nNew + B, *pos = nGoing + B;
    for (int b = 0; b < B; ++b) {
        const std::vector<int32_t>& pages = table_.pagesOf(seqs[b]);
        std::copy(pages.begin(), pages.end(), host.begin() + (size_t)b * most);
        kvLen[b] = (int32_t)table_.length(seqs[b]);
        nNew[b] = counts[b];
        nGoing[b] = before[b] ? counts[b] : 0;
        for (int j = 0; j < counts[b]; ++j) pos[(size_t)b * S + j] = (int32_t)(before[b] + j);
    }
    const int64_t wsFloats = gbx_attn_cached_workspace(&m.cache, B, S, m.cache.heads, (int)most);
    const gbx_stream_t gs = reinterpret_cast<gbx_stream_t>(m.stream);
    bool good = wsFloats >= 0 && m.step.ensure(host.size() * 4) && m.ws.ensure((size_t)wsFloats * 4 + 4) &&
                (!nPartial || m.ensureSaved(nPartial)) &&
                cudaMemcpyAsync(m.step.p, host.data(), host.size() * 4, cudaMemcpyHostToDevice, m.stream) == cudaSuccess;
    const int32_t* ints = (const int32_t*)m.step.p;
    // (the page table makes no pair that clashes or leaves the pool: nothing to report)
    if (good && nCopies)
        good = gbx_kv_copy_pages(&m.cache, ints + atCopies, ints + atCopies + nCopies, (int)nCopies, nullptr, gs) == GBX_OK;
    if (good && nPartial)
        good = kv_copy_across(&m.cache, &m.saved, ints + atPartial, ints + atPartial + nPartial, (int)nPartial, nullptr, gs) == GBX_OK;
    if (!good) {
        cudaStreamSynchronize(m.stream);
        return fail(std::string("session: preparing the step failed: ") + gbx_last_error());
    }
    m.savedIds = ints + atPartial;
    m.savedPages = std::move(partial);
    TransformerModel::CachedStep st;
    st.cache = &m.cache;
    st.table = ints;
    st.maxPages = (int)most;
    st.kvLen = st.table + (size_t)B * most;
    st.nNew = st.kvLen + B;
    st.nGoing = st.nNew + B;
    st.posIds = st.nGoing + B;
    st.workspace = (float*)m.ws.p;
    st.workspaceFloats = wsFloats;
    st.counts = counts;
    st.even = even;
    st.allFresh = true;
    for (int b = 0; b < B; ++b) {
        if (before[b]) st.allFresh = false;
        else if (!st.fresh.empty() && st.fresh.back().second == b) ++st.fresh.back().second;
        else st.fresh.emplace_back(b, b + 1);
    }
    st.allRows = allRows;
    st.rows = keepRows ? (float*)m.rows.p : nullptr;
    st.rowsLo = st.rows + rowFloats;
    return model_.runForward(padded, B, nullptr, &st) || fail(model_.lastError());
}

// Leaves in the cache what a step of keep[b] tokens of sequence b would have: the
// last step's rejected tokens have raised scales and rounded kept tokens by them.
// The pages of the sequences with fewer tokens than counts[b] start again from
// what they held before that step, and the kept rows are appended to them.
bool Session::keepOnly(const std::vector<int>& seqs, const std::vector<int64_t>& before, const std::vector<int>& counts,
                       const std::vector<int>& keep, int S)
{
    Impl& m = *impl_;
    const int B = (int)seqs.size(), d = model_.getEmbedDim();
    // page and place among the saved ones of those to start again, then lengths and counts
    std::vector<int32_t> pages, places, lens(B), news(B, 0);
    size_t most = 1;
    int saved = 0;
    bool any = false;
    for (int b = 0; b < B; ++b) {
        const std::vector<int32_t>& p = table_.pagesOf(seqs[b]);
        most = std::max(most, p.size());
        const bool partial = before[b] % table_.pageSize() != 0, fewer = keep[b] < counts[b];
        if (partial && fewer) {
            pages.push_back(m.savedPages[saved]);
            places.push_back(saved);
        }
        saved += partial;
        lens[b] = (int32_t)(before[b] + keep[b]);
        if (fewer) news[b] = keep[b];
        any = any || fewer;
    }
    if (!any) return true;
    const size_t n = pages.size();
    std::vector<int32_t> host(pages);
    host.insert(host.end(), places.begin(), places.end());
    host.insert(host.end(), lens.begin(), lens.end());
    host.insert(host.end(), news.begin(), news.end());
    const gbx_stream_t gs = reinterpret_cast<gbx_stream_t>(m.stream);
    int32_t bits = 0;
    bool good = m.pairs.ensure(host.size() * 4) &&
                cudaMemcpyAsync(m.pairs.p, host.data(), host.size() * 4, cudaMemcpyHostToDevice, m.stream) == cudaSuccess &&
                cudaMemsetAsync(m.err, 0, 4, m.stream) == cudaSuccess;
    const int32_t* ints = (const int32_t*)m.pairs.p;
    if (good && n) good = kv_copy_across(&m.saved, &m.cache, ints + n, ints, (int)n, m.err, gs) == GBX_OK;
    const size_t layer = (size_t)B * S * 3 * d;
    const float *hi = (const float*)m.rows.p, *lo = hi + layer * m.cache.layers;
    for (int l = 0; l < m.cache.layers && good; ++l, hi += layer, lo += layer)
        good = gbx_kv_append(&m.cache, l, (const int32_t*)m.step.p, (int)most, ints + 2 * n, ints + 2 * n + B, B, S, hi + d, lo + d,
                             hi + 2 * d, lo + 2 * d, 3 * d, m.err, gs) == GBX_OK;
    good = good && cudaMemcpyAsync(&bits, m.err, 4, cudaMemcpyDeviceToHost, m.stream) == cudaSuccess &&
           cudaStreamSynchronize(m.stream) == cudaSuccess && !bits;
    return good || fail(std::string("session: the accepted tokens could not be kept: ") + gbx_last_error());
}

std::vector<float> Session::forward(const std::vector<int>& seqs, const std::vector<int>& ids, const std::vector<int>& counts,
                                    bool allRows)
{
    int S = 0;
    std::vector<int> padded;
    std::vector<float> out;
    if (!check(seqs, ids, counts, &S, &padded)) return out;
    Undo undo(*this);
    if (!step(seqs, ids, counts, allRows, padded, S)) return out;
    OnDevice on(impl_->device);
    const size_t V = (size_t)model_.getVocabSize();
    const float* logits = model_.deviceLogits();
    bool good = true;
    if (allRows) {
        out.resize(ids.size() * V);
        size_t at = 0;
        for (size_t b = 0; b < seqs.size() && good; ++b) {
            good = cudaMemcpy(out.data() + at * V, logits + b * S * V, counts[b] * V * sizeof(float), cudaMemcpyDeviceToHost) == cudaSuccess;
            at += counts[b];
        }
    } else {
        out.resize(seqs.size() * V);
        good = cudaMemcpy(out.data(), logits, out.size() * sizeof(float), cudaMemcpyDeviceToHost) == cudaSuccess;
    }
    if (!good) {
        fail("session: device-to-host copy of the logits failed");
        out.clear();
    }
    undo.done = good;
    return out;
}

std::vector<int> Session::nextTokens(const std::vector<int>& seqs, const std::vector<int>& ids, const std::vector<int>& counts,
                                     double temperature, const std::vector<double>& u)
{
    int S = 0;
    std::vector<int> padded, out;
    if (!check(seqs, ids, counts, &S, &padded)) return out;
    const bool draws = !(temperature <= 0.01);
    if (temperature != temperature || (draws && u.size() != seqs.size())) {
        fail("session: a draw for each sequence");
        return out;
    }
    Impl& m = *impl_;
    OnDevice on(m.device);
    const size_t B = seqs.size();
    if (!m.select.ensure(B * 12)) {
        fail("session: cudaMalloc failed");
        return out;
    }
    Undo undo(*this);
    if (!step(seqs, ids, counts, false, padded, S)) return out;
    double* du = (double*)m.select.p;
    int32_t* dids = (int32_t*)(du + B);
    std::vector<int32_t> got(B);
    if ((draws && cudaMemcpyAsync(du, u.data(), B * 8, cudaMemcpyHostToDevice, m.stream) != cudaSuccess) ||
        gbx_select_tokens(model_.deviceLogits(), (int64_t)B, model_.getVocabSize(), temperature, draws ? du : nullptr, dids, nullptr,
                          nullptr, reinterpret_cast<gbx_stream_t>(m.stream)) != GBX_OK ||
        cudaMemcpyAsync(got.data(), dids, B * 4, cudaMemcpyDeviceToHost, m.stream) != cudaSuccess ||
        cudaStreamSynchronize(m.stream) != cudaSuccess) {
        fail(std::string("session: token selection failed: ") + gbx_last_error());
        return out;
    }
    out.assign(got.begin(), got.end());
    undo.done = true;
    return out;
}

bool Session::verify(const std::vector<int>& seqs, const std::vector<int>& ids, int nDraft, const std::vector<int>& draftLen,
                     const float* draftLogits, double temperature, const std::vector<double>& u, std::vector<int>* outIds,
                     std::vector<int>* accepted)
{
    err_.clear();
    const size_t B = seqs.size(), n1 = (size_t)nDraft + 1;
    if (nDraft < 0 || nDraft > 256) return fail("session: " + std::to_string(nDraft) + " drafts");
    if (ids.size() != B * n1) return fail("session: a pending token and the drafts for each sequence");
    if (!draftLen.empty() && draftLen.size() != B) return fail("session: a draft count for each sequence");
    const bool draws = !(temperature <= 0.01);
    if (temperature != temperature || (draws && u.size() != B * n1)) return fail("session: a draw for each row");
    if (!outIds || !accepted) return fail("session: null output");
    std::vector<int> counts(B), given;
    std::vector<int32_t> drafts(B * (size_t)nDraft, 0), lens(B);
    for (size_t b = 0; b < B; ++b) {
        lens[b] = draftLen.empty() ? nDraft : draftLen[b];
        if (lens[b] < 0 || lens[b] > nDraft) return fail("session: a draft count out of range");
        counts[b] = lens[b] + 1;
        for (int j = 0; j < counts[b]; ++j) given.push_back(ids[b * n1 + j]);
        for (int j = 0; j < lens[b]; ++j) drafts[b * nDraft + j] = ids[b * n1 + 1 + j];
    }
    int S = 0;
    std::vector<int> padded;
    if (!check(seqs, given, counts, &S, &padded)) return false;
    // the rows of the verification are the rows of the step
    const int V = model_.getVocabSize(), steps = S - 1;
    std::vector<int32_t> cut(B * (size_t)steps);
    std::vector<double> du(B * (size_t)S, 0.0);
    for (size_t b = 0; b < B; ++b) {
        for (int j = 0; j < steps; ++j) cut[b * steps + j] = drafts[b * nDraft + j];
        if (draws) {
            for (int j = 0; j < steps; ++j) du[b * S + j] = u[b * n1 + j];
            du[b * S + steps] = u[b * n1 + nDraft];
        }
    }
    Impl& m = *impl_;
    OnDevice on(m.device);
    // device: draws, drafts' logits, drafts, counts, results
    const bool withLogits = draws && draftLogits && steps > 0;
    const size_t logitBytes = withLogits ? B * (size_t)steps * V * 4 : 0;
    const size_t offLogits = du.size() * 8, offIds = offLogits + logitBytes, offLens = offIds + cut.size() * 4,
                 offOut = offLens + B * 4, offAcc = offOut + B * (size_t)S * 4;
    if (!m.select.ensure(offAcc + B * 4)) return fail("session: cudaMalloc failed");
    Undo undo(*this);
    std::vector<int64_t> before;
    for (int s : seqs) before.push_back(table_.length(s));
    if (!step(seqs, given, counts, true, padded, S, steps > 0)) return false;
    uint8_t* p = (uint8_t*)m.select.p;
    std::vector<int32_t> out(B * (size_t)S), acc(B);
    bool good = cudaMemcpyAsync(p, du.data(), du.size() * 8, cudaMemcpyHostToDevice, m.stream) == cudaSuccess &&
                (cut.empty() || cudaMemcpyAsync(p + offIds, cut.data(), cut.size() * 4, cudaMemcpyHostToDevice, m.stream) == cudaSuccess) &&
                cudaMemcpyAsync(p + offLens, lens.data(), B * 4, cudaMemcpyHostToDevice, m.stream) == cudaSuccess &&
                cudaMemsetAsync(m.err, 0, 4, m.stream) == cudaSuccess;
    for (size_t b = 0; b < B && good && withLogits; ++b)
        good = cudaMemcpyAsync(p + offLogits + b * (size_t)steps * V * 4, draftLogits + b * (size_t)nDraft * V, (size_t)steps * V * 4,
                               cudaMemcpyHostToDevice, m.stream) == cudaSuccess;
    int32_t bits = 0;
    good = good &&
           gbx_verify_tokens(model_.deviceLogits(), withLogits ? (const float*)(p + offLogits) : nullptr, (const int32_t*)(p + offIds),
                             (const int32_t*)(p + offLens), (int64_t)B, steps, V, temperature, draws ? (const double*)p : nullptr,
                             (int32_t*)(p + offOut), (int32_t*)(p + offAcc), m.err, reinterpret_cast<gbx_stream_t>(m.stream)) == GBX_OK &&
           cudaMemcpyAsync(out.data(), p + offOut, out.size() * 4, cudaMemcpyDeviceToHost, m.stream) == cudaSuccess &&
           cudaMemcpyAsync(acc.data(), p + offAcc, B * 4, cudaMemcpyDeviceToHost, m.stream) == cudaSuccess &&
           cudaMemcpyAsync(&bits, m.err, 4, cudaMemcpyDeviceToHost, m.stream) == cudaSuccess &&
           cudaStreamSynchronize(m.stream) == cudaSuccess;
    if (!good || bits)
        return fail(good ? std::string("session: a logits row gives no distribution") : std::string("session: verification failed: ") + gbx_last_error());
    std::vector<int> keep(B);
    for (size_t b = 0; b < B; ++b) keep[b] = 1 + acc[b];
    if (!keepOnly(seqs, before, counts, keep, S)) return false;
    outIds->assign(B * n1, -1);
    accepted->assign(acc.begin(), acc.end());
    for (size_t b = 0; b < B; ++b) {
        for (int j = 0; j < S; ++j) (*outIds)[b * n1 + j] = out[b * S + j];
        table_.truncate(seqs[b], before[b] + keep[b]);
    }
    undo.done = true;
    return true;
}

int64_t Session::compact()
{
    err_.clear();
    if (!ok_) {
        fail("session: not open");
        return -1;
    }
    Impl& m = *impl_;
    OnDevice on(m.device);
    if (!m.pairs.ensure((size_t)(table_.pages() / 2 + 1) * 8)) {   // at most half the pages move
        fail("session: cudaMalloc failed");
        return -1;
    }
    const PageTable::Copies c = table_.compact();
    const size_t n = c.src.size();
    if (!n) return 0;
    int32_t bits = 0;
    if (cudaMemsetAsync(m.err, 0, 4, m.stream) != cudaSuccess ||
        cudaMemcpyAsync(m.pairs.p, c.src.data(), n * 4, cudaMemcpyHostToDevice, m.stream) != cudaSuccess ||
        cudaMemcpyAsync((int32_t*)m.pairs.p + n, c.dst.data(), n * 4, cudaMemcpyHostToDevice, m.stream) != cudaSuccess ||
        gbx_kv_copy_pages(&m.cache, (int32_t*)m.pairs.p, (int32_t*)m.pairs.p + n, (int)n, m.err, reinterpret_cast<gbx_stream_t>(m.stream)) !=
            GBX_OK ||
        cudaMemcpyAsync(&bits, m.err, 4, cudaMemcpyDeviceToHost, m.stream) != cudaSuccess ||
        cudaStreamSynchronize(m.stream) != cudaSuccess || bits) {
        // the sequences' pages are where their data is not: none of them can be used
        ok_ = false;
        fail("session: the page copies failed; the session is closed");
        return -1;
    }
    return (int64_t)n;
}

}  // namespace gbx
