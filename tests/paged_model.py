"""The paged cache restated with Python lists and 64-bit numpy: one sequence, head, chunk and query after the other."""
import numpy as np

GLOBAL, LOCAL, SLIDING = 0, 1, 2
NO_LIMIT, OPEN = 2 ** 31 - 1, 2 ** 31 - 2


class PagedModel:
    def __init__(self, S, H, P, D, num_pages, SW):
        self.S, self.H, self.P, self.D, self.SW = S, H, P, D, SW
        self.refs = [0] * num_pages
        self.k = np.full((num_pages, P, D), np.nan)
        self.v = np.full((num_pages, P, D), np.nan)
        self.rows = [[[] for _ in range(H)] for _ in range(S)]           # [page, start, limit]
        self.length = [0] * S

    def take(self):
        page = self.refs.index(0)
        self.refs[page] = 1
        return page

    def append(self, k, v, roles, n_new, skip_hidden=False):
        P = self.P
        for s in range(self.S):
            n, old = n_new[s], self.length[s]
            total = old + n
            for h in range(self.H):
                row = self.rows[s][h]
                chunks = range(old // P, -(-total // P)) if n else range(0)

                def role(c):
                    i = c - old // P
                    return roles[s, h, i] if roles is not None and i < roles.shape[2] else GLOBAL
                done_globals = [c for c in chunks if (c + 1) * P <= total and role(c) == GLOBAL]
                for e in row:
                    if e[2] == OPEN and done_globals:
                        e[2] = (done_globals[0] + 1) * P - 1
                for c in chunks:
                    limit = NO_LIMIT
                    if (c + 1) * P <= total and role(c) != GLOBAL:
                        later = [g for g in done_globals if g > c]
                        limit = c * P + self.SW + P - 1 if role(c) == SLIDING else (later[0] + 1) * P - 1 if later else OPEN
                    if c * P < old:
                        row[-1][2] = limit
                        page = row[-1][0]
                    elif skip_hidden and limit < total:
                        continue
                    else:
                        page = self.take()
                        row.append([page, c * P, limit])
                    for pos in range(max(old, c * P), min(total, (c + 1) * P)):
                        self.k[page, pos - c * P] = k[s, h, pos - old]
                        self.v[page, pos - c * P] = v[s, h, pos - old]
        self.length = [a + b for a, b in zip(self.length, n_new)]

    def attention(self, q, n_new, scale):
        """(o, softmax . |v|), both [S,Hq,N,D]"""
        S, Hq, N, D = q.shape
        G = Hq // self.H
        out, mag = np.zeros((2, S, Hq, N, D))
        for s in range(S):
            for h in range(self.H):
                row = self.rows[s][h]
                if not row:
                    continue
                pos = np.concatenate([np.arange(e[1], e[1] + self.P) for e in row])
                lim = np.repeat([e[2] for e in row], self.P)
                K, V = (np.concatenate([x[e[0]] for e in row]) for x in (self.k, self.v))
                for i in range(n_new[s]):
                    p = self.length[s] - n_new[s] + i
                    seen = (pos <= p) & (p <= lim)
                    if not seen.any():
                        continue
                    for g in range(G):
                        x = K[seen] @ q[s, h * G + g, i] * scale
                        w = np.exp(x - x.max())
                        w /= w.sum()
                        out[s, h * G + g, i] = w @ V[seen]
                        mag[s, h * G + g, i] = w @ np.abs(V[seen])
        return out, mag

    def give_back(self, page):
        self.refs[page] -= 1

    def evict(self):
        for s in range(self.S):
            for h in range(self.H):
                for e in self.rows[s][h]:
                    if e[2] < self.length[s]:
                        self.give_back(e[0])
                self.rows[s][h] = [e for e in self.rows[s][h] if e[2] >= self.length[s]]

    def reorder(self, src):
        old_rows, old_len, P = self.rows, self.length, self.P
        keeper = {}
        for s, o in enumerate(src):
            if o >= 0 and (src[o] == o or o not in keeper):
                keeper[o] = o if src[o] == o else s
        for s in range(self.S):
            for h in range(self.H):
                for e in old_rows[s][h]:
                    self.give_back(e[0])
        self.rows = [[[] for _ in range(self.H)] for _ in src]
        copies = []
        for s, o in enumerate(src):
            for h in range(self.H if o >= 0 else 0):
                row = [list(e) for e in old_rows[o][h]]
                own = old_len[o] % P > 0 and keeper[o] != s
                for i, e in enumerate(row):
                    if own and i == len(row) - 1:
                        copies.append((e, old_len[o] % P))
                    else:
                        self.refs[e[0]] += 1
                self.rows[s][h] = row
        for e, n in copies:
            page = self.take()
            self.k[page, :n], self.v[page, :n] = self.k[e[0], :n], self.v[e[0], :n]
            e[0] = page
        self.length = [old_len[o] if o >= 0 else 0 for o in src]
