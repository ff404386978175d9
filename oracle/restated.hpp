// TEST INFRASTRUCTURE ONLY -- nothing under shasta_amd/ may include, link or call this.
//
// CPU restatement of the Shasta overlap-detection hot path, one function per
// reference function, each citing the /root/reference/ file:line it follows.
// It is pinned (tests/test_oracle_*.py) against
//   - the golden digests SURVEY.md section 8c records for tests/TinyTest.fasta.gz,
//   - fixtures under tests/golden/ generated by running the reference itself
//     (oracle/_ref, built from /root/reference/src in place),
//   - the reference's testAlignmentCompression table (src/compressAlignment.cpp:160-220),
//   - oracle/_ref live, whenever that library is present.
// The banded DP (banded_dp.hpp) is the only part whose parity is UNPINNED.
#ifndef ORACLE_RESTATED_HPP
#define ORACLE_RESTATED_HPP

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <limits>
#include <map>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "banded_dp.hpp"
#include "sparse_chain.hpp"
#include "anchored_chain.hpp"
#include <atomic>

namespace oracle {

// Bookkeeping of the sparse path's prototype (oracle/sparse_chain.hpp) over the DP tasks of real candidates: see oracle_sparse_census_read.
struct SparseCensus {
    static constexpr int N = 22;
    bool anchored = false;              // also run the anchored form (oracle/anchored_chain.hpp) on every task: [13] tasks where it differs from the dense DP (must stay 0), [14] dense cells it solved, [15] windows, [16] tasks it ran whole, [17] anchors, [18] cells of the largest rectangle, [19] tasks with a rectangle of more than 16384 cells, [20] ambiguous tasks with an optimal link of a live hit more than 29 hits back, [21] tasks with more than 128 windows
    bool on = false;
    uint32_t scanBudget = 64; bool oneHitPerMarker = false, runningMaxBound = false;
    std::atomic<uint64_t> counters[N];
    SparseCensus() { for(auto& c : counters) c.store(0); }
    template<class T> void note(const T* k0, uint32_t nx, const T* k1, uint32_t ny, int32_t bandMin, int32_t bandMax, const BandedDpResult& dp,
        const std::vector< std::pair<uint32_t, uint32_t> >& denseOrdinals)
    {
        SparseChainResult r;
        sparseChainAlignment(k0, nx, k1, ny, bandMin, bandMax, r, scanBudget, oneHitPerMarker, runningMaxBound);
        const uint64_t cells = uint64_t(nx) * uint64_t(bandMax - bandMin + 1);
        counters[0] += 1; counters[3] += cells; counters[4] += r.hits; counters[5] += r.scanSteps; counters[r.reason < 4 ? 6 + r.reason : 12] += 1;
        counters[11] += denseOrdinals.size();
        if(r.certified) {
            counters[1] += 1; counters[10] += cells;
            if(!dp.ok || r.score != dp.score || r.ordinals != denseOrdinals) counters[2] += 1;
        }
        if(anchored) {
            AnchoredResult a;
            anchoredAlignment(k0, nx, k1, ny, bandMin, bandMax, a);
            if(!dp.ok || a.score != dp.score || a.ordinals != denseOrdinals) counters[13] += 1;
            counters[14] += a.denseCells; counters[15] += a.windows; counters[16] += a.wholeTaskDense ? 1 : 0; counters[17] += a.anchors;
            if(a.largestWindow > counters[18]) counters[18] = a.largestWindow;
            if(a.largestWindow > 16384) counters[19] += 1;
            if(!r.certified && a.longestLink > 29) counters[20] += 1;
            if(a.windows > 128) counters[21] += 1;
        }
    }
};
inline SparseCensus& sparseCensus() { static SparseCensus census; return census; }


// ---------------------------------------------------------------------------
// MurmurHash64A -- src/MurmurHash2.cpp:96-140 (public-domain MurmurHash2, 64-bit
// variant A, Austin Appleby).  Little-endian, unaligned 8-byte reads.
// ---------------------------------------------------------------------------
inline uint64_t murmurHash64A(const void* key, int len, uint64_t seed)
{
    const uint64_t m = 0xc6a4a7935bd1e995ULL;
    const int r = 47;
    uint64_t h = seed ^ (uint64_t(len) * m);
    const unsigned char* p = static_cast<const unsigned char*>(key);
    const int blockCount = len / 8;
    for(int i = 0; i < blockCount; i++, p += 8) {
        uint64_t k;
        std::memcpy(&k, p, 8);
        k *= m; k ^= k >> r; k *= m;
        h ^= k; h *= m;
    }
    const int tail = len & 7;
    if(tail) {
        for(int i = tail - 1; i >= 0; i--) h ^= uint64_t(p[i]) << (8 * i);
        h *= m;
    }
    h ^= h >> r; h *= m; h ^= h >> r;
    return h;
}

// ---------------------------------------------------------------------------
// Markers: packed 7-byte CompressedMarker {u32 kmerId, u24 position}
// (src/Marker.hpp:56-70).  LowHash0::createKmerIds (src/LowHash0.cpp:261-308).
// ---------------------------------------------------------------------------
inline void extractKmerIds(const uint8_t* data7, uint64_t markerCount, std::vector<uint32_t>& kmerIds)
{
    kmerIds.resize(markerCount);
    for(uint64_t i = 0; i < markerCount; i++) {
        std::memcpy(&kmerIds[i], data7 + 7 * i, 4);
    }
}

// ---------------------------------------------------------------------------
// LowHash0 -- src/LowHash0.cpp:23-257 and the pass functions :314-484.
// ---------------------------------------------------------------------------
struct LowHash0Params {
    uint64_t m;
    double hashFraction;
    uint64_t minHashIterationCount;
    double alignmentCandidatesPerRead;
    uint64_t log2MinHashBucketCount;
    uint64_t minBucketSize, maxBucketSize, minFrequency;
};

struct Candidate {                 // src/LowHash0.hpp:112-136
    uint32_t readId1;
    uint8_t strand;                // 0 = same strand
    uint16_t frequency;
    bool operator==(const Candidate& t) const { return readId1 == t.readId1 && strand == t.strand; }
    bool operator<(const Candidate& t) const
    { return std::tie(readId1, strand) < std::tie(t.readId1, t.strand); }
};

struct LowHash0Output {
    std::vector< std::array<uint32_t, 3> > candidates;    // readId0, readId1, isSameStrand
    std::vector< std::array<uint64_t, 3> > statistics;    // per read: sparse, good, crowded
    std::vector<uint64_t> highFrequency, total;           // per iteration
    std::vector< std::array<uint64_t, 3> > histogram;     // iteration, bucketSize, bucketCount
    uint32_t log2BucketCount = 0;
};

// src/LowHash0.cpp:493-562, restated as "append in merged order, folding equal keys".
inline void mergeCandidates(const std::vector<Candidate>& x0, const std::vector<Candidate>& x1,
    std::vector<Candidate>& y)
{
    y.clear();
    size_t i0 = 0, i1 = 0;
    auto add = [&y](const Candidate& c) {
        if(!y.empty() && y.back() == c) y.back().frequency = uint16_t(y.back().frequency + c.frequency);
        else y.push_back(c);
    };
    while(i0 < x0.size() || i1 < x1.size()) {
        if(i0 == x0.size()) add(x1[i1++]);
        else if(i1 == x1.size()) add(x0[i0++]);
        else if(x0[i0] < x1[i1]) add(x0[i0++]);
        else add(x1[i1++]);
    }
}

inline void lowHash0(
    uint64_t readCount, const uint64_t* toc, const uint32_t* kmerIds, const uint8_t* readFlags,
    const LowHash0Params& p, LowHash0Output& out)
{
    const uint64_t orientedReadCount = 2 * readCount;
    const uint64_t totalMarkerCount = toc[orientedReadCount];

    // Bucket count: src/LowHash0.cpp:73-98.
    const uint64_t estimate = uint64_t(p.hashFraction * double(totalMarkerCount));
    // __builtin_clzl(0) is undefined in the reference; an empty marker set never gets there.
    const uint32_t log2Estimate = estimate ? 64 - uint32_t(__builtin_clzl(estimate)) : 0;
    uint64_t log2BucketCount = p.log2MinHashBucketCount;
    if(log2BucketCount == 0) log2BucketCount = 5 + log2Estimate;
    else if(log2BucketCount < log2Estimate) throw std::runtime_error("log2MinHashBucketCount is unreasonably small.");
    if(log2BucketCount > 31) log2BucketCount = 31;
    const uint64_t bucketCount = 1ULL << log2BucketCount;
    const uint64_t mask = bucketCount - 1;
    out.log2BucketCount = uint32_t(log2BucketCount);

    // :109
    const uint64_t hashThreshold =
        uint64_t(double(p.hashFraction) * double(std::numeric_limits<uint64_t>::max()));

    out.statistics.assign(readCount, {0, 0, 0});
    std::vector< std::vector<Candidate> > candidates(readCount);

    struct LowHash { uint64_t hash; uint32_t orientedReadId; };
    std::vector<LowHash> lowHashes;            // in (orientedReadId, feature) order
    std::vector<uint64_t> lowHashBegin(orientedReadCount + 1);
    struct Entry { uint32_t bucketId, orientedReadId, hashHigh; };
    std::vector<Entry> entries;
    std::vector<Candidate> newCandidates, merged;

    uint64_t highFrequency = 0;
    for(uint64_t iteration = 0; ; iteration++) {
        // Iteration control: :136-157.
        if(p.minHashIterationCount == 0) {
            const double current = 2. * double(highFrequency) / double(readCount);
            if(current >= p.alignmentCandidatesPerRead) break;
        } else if(iteration == p.minHashIterationCount) {
            break;
        }

        // Pass 1 (:314-360): low hashes of every oriented read.
        const uint64_t seed = iteration * 37;
        const int featureByteCount = int(p.m * 4);
        lowHashes.clear();
        for(uint64_t readId = 0; readId < readCount; readId++) {
            for(uint32_t strand = 0; strand < 2; strand++) {
                const uint64_t o = 2 * readId + strand;
                lowHashBegin[o] = lowHashes.size();
                if(readFlags && (readFlags[readId] & 1)) continue;      // :325 palindromic
                const uint64_t n = toc[o + 1] - toc[o];
                if(n < p.m) continue;                                    // :337
                const uint32_t* k = kmerIds + toc[o];
                for(uint64_t j = 0; j + p.m <= n; j++) {
                    const uint64_t h = murmurHash64A(k + j, featureByteCount, seed);
                    if(h < hashThreshold) lowHashes.push_back({h, uint32_t(o)});
                }
            }
        }
        lowHashBegin[orientedReadCount] = lowHashes.size();

        // Pass 2 (:365-398): buckets = groups of equal (hash & mask).
        entries.resize(lowHashes.size());
        for(size_t i = 0; i < lowHashes.size(); i++) {
            entries[i] = {uint32_t(lowHashes[i].hash & mask), lowHashes[i].orientedReadId,
                uint32_t(lowHashes[i].hash >> 32)};
        }
        std::stable_sort(entries.begin(), entries.end(),
            [](const Entry& a, const Entry& b) { return a.bucketId < b.bucketId; });
        // bucketBegin/bucketEnd per entry, histogram (:566-613), statistics (:386-393).
        std::map<uint64_t, uint64_t> histogram;
        uint64_t nonEmpty = 0;
        for(size_t b = 0; b < entries.size(); ) {
            size_t e = b;
            while(e < entries.size() && entries[e].bucketId == entries[b].bucketId) ++e;
            const uint64_t size = e - b;
            ++histogram[size];
            ++nonEmpty;
            for(size_t i = b; i < e; i++) {
                const uint32_t readId = entries[i].orientedReadId >> 1;
                if(size < p.minBucketSize) ++out.statistics[readId][0];
                else if(size > p.maxBucketSize) ++out.statistics[readId][2];
                else ++out.statistics[readId][1];
            }
            b = e;
        }
        if(bucketCount > nonEmpty) histogram[0] += bucketCount - nonEmpty;
        for(const auto& h : histogram) out.histogram.push_back({iteration, h.first, h.second});

        // Pass 3 (:403-484).  For each oriented read, for each of its low hashes,
        // scan its bucket.  Equivalent statement: every ordered pair (a,b) of
        // entries of one valid bucket with equal hashHigh and readId(a) < readId(b).
        std::vector< std::vector<Candidate> > perRead(readCount);
        const uint64_t minSize = std::max<uint64_t>(2, p.minBucketSize);
        for(size_t b = 0; b < entries.size(); ) {
            size_t e = b;
            while(e < entries.size() && entries[e].bucketId == entries[b].bucketId) ++e;
            const uint64_t size = e - b;
            if(size >= minSize && size <= p.maxBucketSize) {
                for(size_t i = b; i < e; i++) {
                    const uint32_t readId0 = entries[i].orientedReadId >> 1;
                    const uint32_t strand0 = entries[i].orientedReadId & 1;
                    for(size_t j = b; j < e; j++) {
                        if(entries[j].hashHigh != entries[i].hashHigh) continue;     // :443
                        const uint32_t readId1 = entries[j].orientedReadId >> 1;
                        if(readId1 <= readId0) continue;                               // :450
                        const bool same = (entries[j].orientedReadId & 1) == strand0;
                        perRead[readId0].push_back({readId1, uint8_t(same ? 0 : 1), 1});
                    }
                }
            }
            b = e;
        }
        uint64_t total = 0;
        highFrequency = 0;
        for(uint64_t readId0 = 0; readId0 < readCount; readId0++) {
            newCandidates.swap(perRead[readId0]);
            std::sort(newCandidates.begin(), newCandidates.end());                     // :462
            mergeCandidates(candidates[readId0], newCandidates, merged);               // :468
            candidates[readId0] = merged;
            total += merged.size();
            for(const Candidate& c : merged) if(c.frequency >= p.minFrequency) ++highFrequency;
            newCandidates.clear();
        }
        out.highFrequency.push_back(highFrequency);
        out.total.push_back(total);
    }

    // :204-214
    out.candidates.clear();
    for(uint64_t readId0 = 0; readId0 < readCount; readId0++) {
        for(const Candidate& c : candidates[readId0]) {
            if(c.frequency >= p.minFrequency) {
                out.candidates.push_back({uint32_t(readId0), c.readId1, uint32_t(c.strand == 0 ? 1 : 0)});
            }
        }
    }
}


// ---------------------------------------------------------------------------
// AlignmentInfo::create -- src/Alignment.cpp:67-113; accessors src/Alignment.hpp:100-330.
// ---------------------------------------------------------------------------
struct Info {
    uint32_t markerCounts[2] = {0, 0}, firstOrdinal[2] = {0, 0}, lastOrdinal[2] = {0, 0};
    uint32_t markerCount = 0;
    int32_t minOrdinalOffset = 0, maxOrdinalOffset = 0, averageOrdinalOffset = 0;
    uint32_t maxSkip = 0, maxDrift = 0;

    uint32_t leftTrim(int i) const { return firstOrdinal[i]; }
    uint32_t rightTrim(int i) const { return markerCounts[i] - 1 - lastOrdinal[i]; }
    uint32_t range(int i) const { return lastOrdinal[i] + 1 - firstOrdinal[i]; }
    double alignedFraction(int i) const { return double(markerCount) / double(range(i)); }
    double minAlignedFraction() const { return std::min(alignedFraction(0), alignedFraction(1)); }
    std::pair<uint32_t, uint32_t> computeTrim() const
    {
        return std::make_pair(std::min(leftTrim(0), leftTrim(1)), std::min(rightTrim(0), rightTrim(1)));
    }
    bool isContaining(uint32_t maxTrim) const
    {
        for(int i = 0; i < 2; i++) if(leftTrim(i) <= maxTrim && rightTrim(i) <= maxTrim) return true;
        return false;
    }
};

using Ordinals = std::vector< std::pair<uint32_t, uint32_t> >;

inline void createInfo(const Ordinals& ord, uint32_t nx, uint32_t ny, Info& info)
{
    info = Info();
    info.markerCount = uint32_t(ord.size());
    info.markerCounts[0] = nx; info.markerCounts[1] = ny;
    if(!ord.empty()) {
        info.firstOrdinal[0] = ord.front().first;  info.firstOrdinal[1] = ord.front().second;
        info.lastOrdinal[0] = ord.back().first;    info.lastOrdinal[1] = ord.back().second;
    }
    info.minOrdinalOffset = std::numeric_limits<int32_t>::max();
    info.maxOrdinalOffset = std::numeric_limits<int32_t>::min();
    double sum = 0.;
    for(size_t i = 0; i < ord.size(); i++) {
        const int32_t offset = int32_t(ord[i].first) - int32_t(ord[i].second);
        info.minOrdinalOffset = std::min(info.minOrdinalOffset, offset);
        info.maxOrdinalOffset = std::max(info.maxOrdinalOffset, offset);
        sum += double(offset);
        if(i) {
            info.maxSkip = std::max(info.maxSkip, uint32_t(std::abs(int32_t(ord[i].first) - int32_t(ord[i-1].first))));
            info.maxSkip = std::max(info.maxSkip, uint32_t(std::abs(int32_t(ord[i].second) - int32_t(ord[i-1].second))));
            const int32_t previousOffset = int32_t(ord[i-1].first) - int32_t(ord[i-1].second);
            info.maxDrift = std::max(info.maxDrift, uint32_t(std::abs(offset - previousOffset)));
        }
    }
    // An empty alignment makes the reference evaluate int32_t(round(0./0.)) (undefined);
    // it is never stored, so the value is pinned to 0 here.
    info.averageOrdinalOffset = ord.empty() ? 0 : int32_t(std::round(sum / double(info.markerCount)));
}


// ---------------------------------------------------------------------------
// shasta::compress / decompress -- src/compressAlignment.cpp:11-140, formats
// src/compressAlignment.hpp:101-321 (GCC little-endian bitfield layout).
// ---------------------------------------------------------------------------
inline void appendStreak(int32_t skip0, int32_t skip1, uint32_t n, std::vector<uint8_t>& s)
{
    auto put = [&s](uint64_t v, int bytes) { for(int i = 0; i < bytes; i++) s.push_back(uint8_t(v >> (8 * i))); };
    const uint64_t u0 = uint32_t(skip0), u1 = uint32_t(skip1), nm1 = uint64_t(n) - 1;
    if(skip0 >= 0 && skip0 <= 3 && skip1 >= 0 && skip1 <= 3 && n >= 1 && n <= 8) {
        put(0 | (u0 & 3) << 1 | (u1 & 3) << 3 | (nm1 & 7) << 5, 1);                          // Format0
    } else if(skip0 >= -8 && skip0 <= 7 && skip1 >= -8 && skip1 <= 7 && n >= 1 && n <= 32) {
        put(1 | (u0 & 0xf) << 3 | (u1 & 0xf) << 7 | (nm1 & 0x1f) << 11, 2);                   // Format1
    } else if(skip0 >= -512 && skip0 <= 511 && skip1 >= -512 && skip1 <= 511 && n >= 1 && n <= 512) {
        put(3 | (u0 & 0x3ff) << 3 | (u1 & 0x3ff) << 13 | (nm1 & 0x1ff) << 23, 4);             // Format2
    } else if(skip0 >= -524288 && skip0 <= 524287 && skip1 >= -524288 && skip1 <= 524287 && n >= 1 && n <= 2097152) {
        put(5 | (u0 & 0xfffff) << 3 | (u1 & 0xfffff) << 23 | (nm1 & 0x1fffff) << 43, 8);      // Format3
    } else {
        put(7, 4); put(u0, 4); put(u1, 4); put(nm1 & 0xffffffffULL, 4);                      // Format4
    }
}

inline void compress(const Ordinals& ord, std::vector<uint8_t>& s)
{
    s.clear();
    uint32_t ordinal0 = 0, ordinal1 = 0;
    for(size_t i = 0; i < ord.size(); ) {
        const int32_t skip0 = int32_t(ord[i].first) - int32_t(ordinal0);
        const int32_t skip1 = int32_t(ord[i].second) - int32_t(ordinal1);
        ordinal0 = ord[i].first; ordinal1 = ord[i].second;
        uint32_t n = 1;
        for(size_t j = i + 1; j < ord.size(); j++, n++) {
            if(ord[j].first != ordinal0 + 1 || ord[j].second != ordinal1 + 1) break;
            ++ordinal0; ++ordinal1;
        }
        i += n;
        appendStreak(skip0, skip1, n, s);
    }
}

inline void decompress(const uint8_t* s, size_t size, Ordinals& ord)
{
    ord.clear();
    uint32_t ordinal0 = 0, ordinal1 = 0;
    auto get = [&s](size_t pos, int bytes) { uint64_t v = 0; for(int i = 0; i < bytes; i++) v |= uint64_t(s[pos+i]) << (8*i); return v; };
    auto sext = [](uint64_t v, int bits) { const uint64_t m = 1ULL << (bits - 1); return int32_t(int64_t((v ^ m) - m)); };
    size_t pos = 0;
    while(pos < size) {
        int32_t skip0, skip1; uint32_t n;
        const uint8_t c = s[pos];
        if((c & 1) == 0) { const uint64_t v = get(pos, 1); pos += 1;
            skip0 = int32_t((v >> 1) & 3); skip1 = int32_t((v >> 3) & 3); n = uint32_t((v >> 5) & 7) + 1;
        } else if((c & 7) == 1) { const uint64_t v = get(pos, 2); pos += 2;
            skip0 = sext((v >> 3) & 0xf, 4); skip1 = sext((v >> 7) & 0xf, 4); n = uint32_t((v >> 11) & 0x1f) + 1;
        } else if((c & 7) == 3) { const uint64_t v = get(pos, 4); pos += 4;
            skip0 = sext((v >> 3) & 0x3ff, 10); skip1 = sext((v >> 13) & 0x3ff, 10); n = uint32_t((v >> 23) & 0x1ff) + 1;
        } else if((c & 7) == 5) { const uint64_t v = get(pos, 8); pos += 8;
            skip0 = sext((v >> 3) & 0xfffff, 20); skip1 = sext((v >> 23) & 0xfffff, 20); n = uint32_t((v >> 43) & 0x1fffff) + 1;
        } else {
            skip0 = int32_t(get(pos + 4, 4)); skip1 = int32_t(get(pos + 8, 4)); n = uint32_t(get(pos + 12, 4)) + 1; pos += 16;
        }
        ordinal0 += uint32_t(skip0); ordinal1 += uint32_t(skip1);
        for(uint32_t i = 0; i < n; i++) ord.push_back(std::make_pair(ordinal0 + i, ordinal1 + i));
        ordinal0 += n - 1; ordinal1 += n - 1;
    }
}


// ---------------------------------------------------------------------------
// Align4 -- src/Align4.cpp.  Options: src/Align4.hpp:106-121.
// ---------------------------------------------------------------------------
struct Align4Options {
    uint64_t deltaX, deltaY, minEntryCountPerCell, maxDistanceFromBoundary, minAlignedMarkerCount;
    double minAlignedFraction;
    uint64_t maxSkip, maxDrift, maxTrim, maxBand;
};

struct Cell { uint32_t iX, iY; bool nearLeftOrTop, nearRightOrBottom, forward = false, backward = false; };

struct Align4Trace {            // intermediate products, exposed for stage-level parity tests
    std::vector<Cell> cells;                                   // sorted by (iY, iX)
    std::vector< std::pair<int32_t, int32_t> > bands;          // (bandMin, bandMax) per component, ordered by (iYMin, first cell)
    uint64_t dpCells = 0;
    bool tie = false;
};

// getxy, src/Align4.cpp:184-191.
inline void getxy(uint32_t X, uint32_t Y, uint32_t nx, int32_t& x, int32_t& y)
{
    const int32_t Xs = int32_t(X), Ys = int32_t(Y);
    x = (Xs - Ys + int32_t(nx) - 1) / 2;
    y = (Xs + Ys - int32_t(nx) + 1) / 2;
}

// An oriented read's markers as (kmerId, ordinal), sorted by kmerId: src/AssemblerAlign4.cpp:243-258.
using SortedMarkers = std::vector< std::pair<uint32_t, uint32_t> >;
inline void sortMarkers(const uint32_t* k, uint32_t n, std::pair<uint32_t, uint32_t>* sorted)
{
    for(uint32_t i = 0; i < n; i++) sorted[i] = std::make_pair(k[i], i);
    std::sort(sorted, sorted + n, [](const std::pair<uint32_t, uint32_t>& a, const std::pair<uint32_t, uint32_t>& b) { return a.first < b.first; });
}

// sorted0 / sorted1: sortMarkers of the two reads where the caller has it (once for all candidates, as the reference does).
inline void align4(
    const uint32_t* k0, uint32_t nx, const uint32_t* k1, uint32_t ny,
    const Align4Options& o, Ordinals& bestOrdinals, Info& bestInfo, Align4Trace* traceOut = nullptr,
    const std::pair<uint32_t, uint32_t>* sorted0 = nullptr, const std::pair<uint32_t, uint32_t>* sorted1 = nullptr)
{
    const uint32_t deltaX = uint32_t(int32_t(o.deltaX)), deltaY = uint32_t(int32_t(o.deltaY));

    // createAlignmentMatrix (:195-267): only the number of entries per cell matters downstream.
    SortedMarkers own0, own1;
    if(!sorted0) { own0.resize(nx); sortMarkers(k0, nx, own0.data()); sorted0 = own0.data(); }
    if(!sorted1) { own1.resize(ny); sortMarkers(k1, ny, own1.data()); sorted1 = own1.data(); }
    std::map< std::pair<uint32_t, uint32_t>, uint64_t > cellCount;     // key (iY, iX)
    {
        size_t i0 = 0, i1 = 0;
        while(i0 < nx && i1 < ny) {
            if(sorted0[i0].first < sorted1[i1].first) ++i0;
            else if(sorted1[i1].first < sorted0[i0].first) ++i1;
            else {
                const uint32_t kmerId = sorted0[i0].first;
                size_t e0 = i0, e1 = i1;
                while(e0 < nx && sorted0[e0].first == kmerId) ++e0;
                while(e1 < ny && sorted1[e1].first == kmerId) ++e1;
                for(size_t a = i0; a < e0; a++) for(size_t b = i1; b < e1; b++) {
                    const uint32_t x = sorted0[a].second, y = sorted1[b].second;
                    const uint32_t X = x + y, Y = nx + y - x - 1;                 // getXY :171-177
                    ++cellCount[std::make_pair(Y / deltaY, X / deltaX)];
                }
                i0 = e0; i1 = e1;
            }
        }
    }

    // createCells (:380-436) with the four boundary distances (:530-626).
    std::vector<Cell> cells;
    for(const auto& p : cellCount) {
        if(p.second < o.minEntryCountPerCell) continue;
        Cell c;
        c.iY = p.first.first; c.iX = p.first.second;
        int32_t x, y;
        getxy(c.iX * deltaX, (c.iY + 1) * deltaY, nx, x, y);
        const uint32_t left = x < 0 ? 0 : uint32_t(x);
        getxy((c.iX + 1) * deltaX, c.iY * deltaY, nx, x, y);
        const uint32_t right = (x >= int32_t(nx) - 1) ? 0 : uint32_t(nx - 1 - uint32_t(x));
        getxy(c.iX * deltaX, c.iY * deltaY, nx, x, y);
        const uint32_t top = y < 0 ? 0 : uint32_t(y);
        getxy((c.iX + 1) * deltaX, (c.iY + 1) * deltaY, nx, x, y);
        const uint32_t bottom = (y >= int32_t(ny) - 1) ? 0 : uint32_t(ny - 1 - uint32_t(y));
        c.nearLeftOrTop = (left < o.maxDistanceFromBoundary) || (top < o.maxDistanceFromBoundary);
        c.nearRightOrBottom = (right < o.maxDistanceFromBoundary) || (bottom < o.maxDistanceFromBoundary);
        cells.push_back(c);
    }
    std::map< std::pair<uint32_t, uint32_t>, size_t > index;           // (iY,iX) -> position in cells
    for(size_t i = 0; i < cells.size(); i++) index[std::make_pair(cells[i].iY, cells[i].iX)] = i;
    auto find = [&index](int64_t iX, int64_t iY) -> int64_t {
        if(iX < 0 || iY < 0) return -1;
        const auto it = index.find(std::make_pair(uint32_t(iY), uint32_t(iX)));
        return it == index.end() ? -1 : int64_t(it->second);
    };

    // forwardSearch (:682-729): children dY in {-1,0,1}, dX in {0,1}.
    std::vector<size_t> stack;
    for(size_t i = 0; i < cells.size(); i++) if(cells[i].nearLeftOrTop) { cells[i].forward = true; stack.push_back(i); }
    while(!stack.empty()) {
        const size_t i = stack.back(); stack.pop_back();
        for(int dY = -1; dY <= 1; dY++) for(int dX = 0; dX <= 1; dX++) {
            const int64_t j = find(int64_t(cells[i].iX) + dX, int64_t(cells[i].iY) + dY);
            if(j >= 0 && !cells[size_t(j)].forward) { cells[size_t(j)].forward = true; stack.push_back(size_t(j)); }
        }
    }
    // backwardSearch (:736-787): parents dY in {-1,0,1}, dX in {-1,0}; seeds must be forward accessible.
    for(size_t i = 0; i < cells.size(); i++) if(cells[i].nearRightOrBottom && cells[i].forward) { cells[i].backward = true; stack.push_back(i); }
    while(!stack.empty()) {
        const size_t i = stack.back(); stack.pop_back();
        for(int dY = -1; dY <= 1; dY++) for(int dX = -1; dX <= 0; dX++) {
            const int64_t j = find(int64_t(cells[i].iX) + dX, int64_t(cells[i].iY) + dY);
            if(j >= 0 && !cells[size_t(j)].backward) { cells[size_t(j)].backward = true; stack.push_back(size_t(j)); }
        }
    }

    // findActiveCellsConnectedComponents (:792-868): 8-neighbourhood over active cells.
    // The reference orders components by union-find representative, which depends on
    // libstdc++ unordered_map iteration order; only ties on markerCount can observe
    // that order.  Here: components in order of their first cell in (iY,iX) order.
    std::vector<int32_t> component(cells.size(), -1);
    std::vector< std::pair<uint32_t, uint32_t> > iYRange;       // per component
    for(size_t i = 0; i < cells.size(); i++) {
        if(!(cells[i].forward && cells[i].backward) || component[i] >= 0) continue;
        const int32_t id = int32_t(iYRange.size());
        iYRange.push_back(std::make_pair(cells[i].iY, cells[i].iY));
        component[i] = id; stack.push_back(i);
        while(!stack.empty()) {
            const size_t a = stack.back(); stack.pop_back();
            iYRange[size_t(id)].first = std::min(iYRange[size_t(id)].first, cells[a].iY);
            iYRange[size_t(id)].second = std::max(iYRange[size_t(id)].second, cells[a].iY);
            for(int dY = -1; dY <= 1; dY++) for(int dX = -1; dX <= 1; dX++) {
                const int64_t j = find(int64_t(cells[a].iX) + dX, int64_t(cells[a].iY) + dY);
                if(j >= 0 && cells[size_t(j)].forward && cells[size_t(j)].backward && component[size_t(j)] < 0) {
                    component[size_t(j)] = id; stack.push_back(size_t(j));
                }
            }
        }
    }

    // computeBandedAlignments (:875-988).
    bestOrdinals.clear();
    bool haveBest = false, tie = false;
    Ordinals ordinals;
    Info info;
    BandedDpResult dp;
    if(traceOut) { traceOut->cells = cells; traceOut->bands.clear(); traceOut->dpCells = 0; }
    for(size_t c = 0; c < iYRange.size(); c++) {
        const uint32_t YMin = iYRange[c].first * deltaY;
        const uint32_t YMax = (iYRange[c].second + 1) * deltaY - 1;
        const int32_t bandMin = int32_t(nx) - 1 - int32_t(YMax);
        const int32_t bandMax = int32_t(nx) - 1 - int32_t(YMin);
        const int32_t bandWidth = bandMax - bandMin + 1;
        if(traceOut) traceOut->bands.push_back(std::make_pair(bandMin, bandMax));
        if(bandWidth > int64_t(o.maxBand)) continue;
        // computeBandedAlignment (:993-1088); scores are the class defaults 6/-1/-1
        // (src/Align4.hpp:159-161 -- never assigned from Options).
        bandedOverlapAlignment(k0, nx, k1, ny, 6, -1, -1, bandMin, bandMax, dp);
        if(traceOut) traceOut->dpCells += uint64_t(nx) * uint64_t(bandWidth);
        diagonalMatches(k0, k1, dp, ordinals);
        if(sparseCensus().on) sparseCensus().note(k0, nx, k1, ny, bandMin, bandMax, dp, ordinals);
        createInfo(ordinals, nx, ny, info);
        if(info.markerCount < o.minAlignedMarkerCount) continue;
        if(info.minAlignedFraction() < o.minAlignedFraction) continue;
        if(info.maxSkip > o.maxSkip) continue;
        if(info.maxDrift > o.maxDrift) continue;
        const auto trim = info.computeTrim();
        if(trim.first > o.maxTrim || trim.second > o.maxTrim) continue;
        if(!haveBest || info.markerCount > bestInfo.markerCount) {
            haveBest = true; tie = false; bestOrdinals = ordinals; bestInfo = info;
        } else if(info.markerCount == bestInfo.markerCount) {
            tie = true;
        }
    }
    if(!haveBest) { bestOrdinals.clear(); createInfo(bestOrdinals, nx, ny, bestInfo); }
    if(traceOut) traceOut->tie = tie;
}

// Outer filters of computeAlignmentsThreadFunction, src/AssemblerAlign.cpp:439-472.
inline bool passesOuterFilters(const Ordinals& ord, const Info& info, const Align4Options& o, bool suppressContainments)
{
    if(ord.size() < o.minAlignedMarkerCount) return false;
    if(std::min(info.alignedFraction(0), info.alignedFraction(1)) < o.minAlignedFraction) return false;
    const auto trim = info.computeTrim();
    if(trim.first > o.maxTrim || trim.second > o.maxTrim) return false;
    if(info.maxSkip > o.maxSkip) return false;       // Alignment::maxSkip/maxDrift (src/Alignment.cpp:4-31)
    if(info.maxDrift > o.maxDrift) return false;     // compute the same maxima as AlignmentInfo::create
    if(suppressContainments && info.isContaining(uint32_t(o.maxTrim))) return false;
    return true;
}


// ---------------------------------------------------------------------------
// Align method 3 -- Assembler::alignOrientedReads3, src/AssemblerAlign3.cpp:22-314.
// ---------------------------------------------------------------------------

// MurmurHash2, 32-bit (public-domain MurmurHash2 by Austin Appleby) -- src/MurmurHash2.cpp:37-85.
inline uint32_t murmurHash2(const void* key, int len, uint32_t seed)
{
    const uint32_t m = 0x5bd1e995u;
    uint32_t h = seed ^ uint32_t(len);
    const unsigned char* p = static_cast<const unsigned char*>(key);
    for(; len >= 4; p += 4, len -= 4) {
        uint32_t k;
        std::memcpy(&k, p, 4);
        k *= m; k ^= k >> 24; k *= m;
        h *= m; h ^= k;
    }
    if(len) {
        for(int i = len - 1; i >= 0; i--) h ^= uint32_t(p[i]) << (8 * i);
        h *= m;
    }
    h ^= h >> 13; h *= m; h ^= h >> 15;
    return h;
}

// Id of the reverse complement of the k-mer with this id.  A k-mer id is two k-bit planes,
// (high bits of the k bases) << k | (low bits of the k bases), first base at the most significant
// bit of its plane, A=0 C=1 G=2 T=3 (ShortBaseSequence::id and its inverse constructor,
// src/ShortBaseSequence.hpp:89-105).  Complementing flips both bits of every base, reversing
// reverses each plane (reverseComplement, :109-117).
inline uint64_t reverseComplementKmerId(uint64_t kmerId, uint64_t k)
{
    const uint64_t mask = (1ULL << k) - 1;
    const uint64_t plane[2] = {~kmerId & mask, ~(kmerId >> k) & mask};
    uint64_t reversed[2] = {0, 0};
    for(int p = 0; p < 2; p++) {
        for(uint64_t i = 0; i < k; i++) reversed[p] |= ((plane[p] >> i) & 1ULL) << (k - 1 - i);
    }
    return (reversed[1] << k) | reversed[0];
}

// KmerInfo::hash, the value method 3 down-samples on -- src/AssemblerKmers.cpp:182-186.
inline uint32_t kmerDownsamplingHash(uint64_t kmerId, uint64_t k)
{
    const uint64_t n = kmerId + reverseComplementKmerId(kmerId, k);
    return murmurHash2(&n, 8, 13477);
}

struct Align3Options {
    int32_t matchScore = 6, mismatchScore = -1, gapScore = -1;
    double downsamplingFactor = 0.1;
    int32_t bandExtend = 10, maxBand = 1000;
    uint64_t k = 10;
};

struct Align3Trace {            // intermediate products, exposed for stage-level parity tests
    uint32_t downsampledCount[2] = {0, 0};
    bool downsampledAligned = false;      // step 1 produced at least one aligned column
    int32_t offsetMin = 0, offsetMax = 0; // over the step-1 columns with equal kmer ids (:200-223)
    int32_t bandMin = 0, bandMax = 0;
    bool bandTooWide = false;
    uint64_t dpCells = 0;                 // nx * band width, both steps
};

// Returns false where the reference throws (SeqAn failure, :128-130, :265-267): the caller
// skips the candidate (src/AssemblerAlign.cpp:419-435).
inline bool align3(
    const uint32_t* k0, uint32_t nx, const uint32_t* k1, uint32_t ny,
    const Align3Options& o, Ordinals& ord, Info& info, Align3Trace* traceOut = nullptr)
{
    Align3Trace trace;
    ord.clear();
    auto finish = [&](bool ok) {
        createInfo(ord, nx, ny, info);
        if(traceOut) *traceOut = trace;
        return ok;
    };

    // Step 1 inputs: the markers whose k-mer hash is under the threshold (:66-82).
    const uint32_t hashThreshold = uint32_t(o.downsamplingFactor * double(std::numeric_limits<uint32_t>::max()));
    std::vector<uint32_t> dsKmer[2], dsOrdinal[2];
    const uint32_t* seq[2] = {k0, k1};
    const uint32_t n[2] = {nx, ny};
    for(int i = 0; i < 2; i++) {
        for(uint32_t ordinal = 0; ordinal < n[i]; ordinal++) {
            if(kmerDownsamplingHash(seq[i][ordinal], o.k) < hashThreshold) {
                dsKmer[i].push_back(seq[i][ordinal]);
                dsOrdinal[i].push_back(ordinal);
            }
        }
        trace.downsampledCount[i] = uint32_t(dsKmer[i].size());
    }
    if(dsKmer[0].empty() || dsKmer[1].empty()) return finish(true);          // :101-107

    // Step 1: unbanded overlap alignment of the down-sampled sequences (:118-130).
    const uint32_t n0 = uint32_t(dsKmer[0].size()), n1 = uint32_t(dsKmer[1].size());
    BandedDpResult dp;
    bandedOverlapAlignment(dsKmer[0].data(), n0, dsKmer[1].data(), n1,
        o.matchScore, o.mismatchScore, o.gapScore, -int32_t(n1), int32_t(n0), dp);
    trace.dpCells += uint64_t(n0) * (uint64_t(n0) + n1 + 1);
    if(!dp.ok) return finish(false);

    // No column pairs two markers: empty alignment (:185-192).
    bool anyDiagonal = false;
    for(const uint8_t op : dp.ops) if(op == TRACE_DIAG) { anyDiagonal = true; break; }
    if(!anyDiagonal) return finish(true);
    trace.downsampledAligned = true;

    // Offset range of the aligned columns with equal k-mer ids, in ordinals of the full reads (:198-223).
    int32_t offsetMin = std::numeric_limits<int32_t>::max(), offsetMax = std::numeric_limits<int32_t>::min();
    {
        uint32_t x = dp.iBegin, y = dp.jBegin;
        for(const uint8_t op : dp.ops) {
            if(op == TRACE_DIAG) {
                if(dsKmer[0][x] == dsKmer[1][y]) {
                    const int32_t offset = int32_t(dsOrdinal[0][x]) - int32_t(dsOrdinal[1][y]);
                    offsetMin = std::min(offsetMin, offset);
                    offsetMax = std::max(offsetMax, offset);
                }
                ++x; ++y;
            } else if(op == TRACE_VERT) ++y;
            else ++x;
        }
    }
    // A positive optimal score needs at least one match, and a non-positive one has no columns.
    if(offsetMin > offsetMax) throw std::logic_error("align3: aligned columns without a match");
    trace.offsetMin = offsetMin; trace.offsetMax = offsetMax;
    const int32_t bandMin = offsetMin - o.bandExtend, bandMax = offsetMax + o.bandExtend;      // :224-225
    trace.bandMin = bandMin; trace.bandMax = bandMax;
    if(bandMax - bandMin > o.maxBand) { trace.bandTooWide = true; return finish(true); }      // :236-241

    // Step 2: banded overlap alignment of all markers (:246-267); aligned markers = diagonal
    // steps over equal k-mer ids (:281-297).
    bandedOverlapAlignment(k0, nx, k1, ny, o.matchScore, o.mismatchScore, o.gapScore, bandMin, bandMax, dp);
    {
        const int32_t lo = std::max(bandMin, -int32_t(ny)), hi = std::min(bandMax, int32_t(nx));
        trace.dpCells += uint64_t(nx) * uint64_t(hi - lo + 1);
    }
    if(!dp.ok) return finish(false);
    diagonalMatches(k0, k1, dp, ord);
    return finish(true);
}


// ---------------------------------------------------------------------------
// Marker finding -- MarkerFinder::threadFunction, src/MarkerFinder.cpp:58-127 (both passes).
// Reads are stored as LongBaseSequences (src/LongBaseSequence.hpp:33-41): per block of 64 bases
// two 64-bit words, the low bits of the bases then their high bits, base 0 of the block in the most
// significant bit.  A k-mer id is (high bits of its k bases) << k | (low bits), first base most
// significant (src/ShortBaseSequence.hpp:89-105).
// ---------------------------------------------------------------------------
inline uint32_t baseAt(const uint64_t* words, uint64_t i)
{
    const uint64_t block = i >> 6, bit = 63 - (i & 63);
    return uint32_t(((words[2 * block + 1] >> bit) & 1ULL) << 1 | ((words[2 * block] >> bit) & 1ULL));
}

// Markers of one read: strand 0 in position order, strand 1 = reverse complement, also in its own
// position order (the reference fills it backwards, :96-100).  7-byte records appended to out0 / out1.
inline void findMarkersOfRead(const uint64_t* words, uint64_t baseCount, uint64_t k, const uint8_t* isMarker,
    std::vector<uint8_t>& out0, std::vector<uint8_t>& out1)
{
    out0.clear(); out1.clear();
    if(baseCount < k) return;                                          // :78
    auto append = [](std::vector<uint8_t>& v, uint32_t kmerId, uint32_t position) {
        for(int b = 0; b < 4; b++) v.push_back(uint8_t(kmerId >> (8 * b)));
        for(int b = 0; b < 3; b++) v.push_back(uint8_t(position >> (8 * b)));
    };
    std::vector< std::pair<uint32_t, uint32_t> > reversed;
    for(uint64_t position = 0; position + k <= baseCount; position++) {
        uint64_t low = 0, high = 0;
        for(uint64_t j = 0; j < k; j++) {
            const uint32_t base = baseAt(words, position + j);
            low = (low << 1) | (base & 1u);
            high = (high << 1) | (base >> 1);
        }
        const uint64_t kmerId = (high << k) | low;
        if(!isMarker[kmerId]) continue;
        append(out0, uint32_t(kmerId), uint32_t(position));
        reversed.push_back(std::make_pair(uint32_t(reverseComplementKmerId(kmerId, k)), uint32_t(baseCount - k - position)));
    }
    for(size_t i = reversed.size(); i-- > 0; ) append(out1, reversed[i].first, reversed[i].second);
}

}  // namespace oracle
#endif
