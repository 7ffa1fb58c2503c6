"""The plan of a step of a cache's streams on the host, a stream and a page at a
time, from its definition (include/pk_hip.h)."""
import numpy as np

PAGE = 64


class Plan:
    def __init__(self, pages, B, max_pages, rows, max_T):
        self.pages, self.B, self.max_pages, self.rows, self.max_T = pages, B, max_pages, rows, max_T
        self.queue = list(range(pages))
        self.head = 0
        self.table = np.full((B, max_pages), -1, np.int32)
        self.state = np.zeros((B, 2), np.int32)

    def step(self, add, fresh=None, left=None, sinks=0):
        B, cap = self.B, PAGE * self.max_pages
        keep = -(-sinks // PAGE)
        self.len, self.row0 = np.zeros(B, np.int32), np.zeros(B + 1, np.int32)
        asked = at = 0
        for b in range(B):
            had, gone = (int(x) for x in self.state[b])
            new = fresh is not None and fresh[b]
            start = 0 if new else had
            if new:
                back = range(0, -(-had // PAGE))
                gone = 0
            else:
                behind = 0 if left is None else max(0, start - left) // PAGE
                back = range(max(gone, keep), behind)
                gone = max(gone, behind)
            for c in back:
                if 0 <= self.table[b, c] < self.pages:
                    self.queue.append(int(self.table[b, c]))
                self.table[b, c] = -1
            want = min(max(int(add[b]), 0), self.max_T, cap - start)
            asked += max(int(add[b]), 0)
            T = min(want, self.rows - at)
            at += T
            self.len[b], self.row0[b + 1] = start, at
            self.state[b] = start + T, gone
        missing = 0
        for b in range(B):
            start, end = int(self.len[b]), int(self.state[b, 0])
            for c in range(-(-start // PAGE), -(-end // PAGE)):
                if self.queue:
                    self.table[b, c] = self.queue.pop(0)
                    self.head = (self.head + 1) % self.pages
                else:
                    self.table[b, c] = -1
                    missing += 1
        self.slot = np.full(self.rows, -1, np.int32)
        for b in range(B):
            for r in range(self.row0[b], self.row0[b + 1]):
                f = self.len[b] + r - self.row0[b]
                if self.table[b, f // PAGE] >= 0:
                    self.slot[r] = PAGE * self.table[b, f // PAGE] + f % PAGE
        self.told = [at, min(asked - at, 0x7fffffff), missing, len(self.queue)]
