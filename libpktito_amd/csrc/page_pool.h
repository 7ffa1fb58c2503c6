/* Which pages of a cache's pool are in use: a count of holders a page, and a
 * bit for each free one. Host only; nothing is allocated after the pool is
 * made. */
#ifndef PK_PAGE_POOL_H
#define PK_PAGE_POOL_H

#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <vector>

namespace pkq8 {

class PagePool {
public:
    explicit PagePool(uint32_t pages) : holders_(pages, 0), free_((pages + 63) / 64, 0), nfree_(pages) {
        for (uint32_t i = 0; i < pages; i++)
            free_[i / 64] |= 1ull << i % 64;
    }

    uint32_t free_pages() const {
        std::lock_guard<std::mutex> lk(mu_);
        return nfree_;
    }

    uint32_t holders(int32_t id) const {
        std::lock_guard<std::mutex> lk(mu_);
        return (uint32_t)id < holders_.size() ? holders_[(uint32_t)id] : 0;
    }

    bool alloc(int32_t *ids, uint32_t n) {
        std::lock_guard<std::mutex> lk(mu_);
        if (nfree_ < n)
            return false;
        for (uint32_t i = 0; i < n; i++) {
            const uint32_t id = lowest();
            take(id);
            holders_[id] = 1;
            ids[i] = (int32_t)id;
        }
        return true;
    }

    bool share(const int32_t *ids, uint32_t n) {
        std::lock_guard<std::mutex> lk(mu_);
        for (uint32_t i = 0; i < n; i++)
            if ((uint32_t)ids[i] >= holders_.size() || holders_[(uint32_t)ids[i]] == 0 ||
                holders_[(uint32_t)ids[i]] > UINT32_MAX - n)
                return false;
        for (uint32_t i = 0; i < n; i++)
            holders_[(uint32_t)ids[i]]++;
        return true;
    }

    bool release(const int32_t *ids, uint32_t n) {
        std::lock_guard<std::mutex> lk(mu_);
        uint32_t i = 0;
        for (; i < n; i++) {
            if ((uint32_t)ids[i] >= holders_.size() || holders_[(uint32_t)ids[i]] == 0)
                break;
            holders_[(uint32_t)ids[i]]--;
        }
        if (i < n) {                        /* as it was */
            while (i--)
                holders_[(uint32_t)ids[i]]++;
            return false;
        }
        for (i = 0; i < n; i++)
            if (holders_[(uint32_t)ids[i]] == 0)
                give((uint32_t)ids[i]);
        return true;
    }

    /* moves the highest pages in use into the lowest free ones below them */
    uint32_t compact(int32_t *pairs, uint32_t cap) {
        std::lock_guard<std::mutex> lk(mu_);
        uint32_t n = 0, top = (uint32_t)holders_.size();
        while (n < cap && nfree_) {
            while (top > 0 && holders_[top - 1] == 0)
                top--;
            const uint32_t to = lowest();
            if (to >= top)
                break;
            const uint32_t from = top - 1;
            relocate(from, to);
            pairs[2 * n] = (int32_t)from;
            pairs[2 * n + 1] = (int32_t)to;
            n++;
        }
        return n;
    }

    /* undoes compact's pairs, the last first, if each page that one was moved
     * from is still free and the page it went to held */
    bool restore(const int32_t *pairs, uint32_t n) {
        std::lock_guard<std::mutex> lk(mu_);
        uint32_t i = n;
        for (; i > 0; i--) {
            const uint32_t from = (uint32_t)pairs[2 * i - 2], to = (uint32_t)pairs[2 * i - 1];
            if (from >= holders_.size() || to >= from || holders_[from] != 0 || holders_[to] == 0)
                break;
            relocate(to, from);
        }
        if (i > 0) {                        /* as it was */
            for (; i < n; i++)
                relocate((uint32_t)pairs[2 * i], (uint32_t)pairs[2 * i + 1]);
            return false;
        }
        return true;
    }

private:
    /* page `from` in use becomes page `to`, which is free */
    void relocate(uint32_t from, uint32_t to) {
        take(to);
        give(from);
        std::swap(holders_[to], holders_[from]);
    }
    /* the lowest free page; there is one */
    uint32_t lowest() {
        while (free_[low_] == 0)
            low_++;
        return 64 * low_ + (uint32_t)__builtin_ctzll(free_[low_]);
    }
    void take(uint32_t id) {
        free_[id / 64] &= ~(1ull << id % 64);
        nfree_--;
    }
    /* a page named twice in a release is given once */
    void give(uint32_t id) {
        const uint64_t bit = 1ull << id % 64;
        nfree_ += (free_[id / 64] & bit) == 0;
        free_[id / 64] |= bit;
        low_ = std::min(low_, id / 64);
    }

    mutable std::mutex mu_;
    std::vector<uint32_t> holders_;
    std::vector<uint64_t> free_;
    uint32_t nfree_, low_ = 0;              /* no free page in the words before low_ */
};

}  // namespace pkq8

#endif
