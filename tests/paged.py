"""Plain 64-bit forms of the paged-cache operators and the buffers their tests use."""

import numpy as np

import inferi_amd as I

NP = {I.F16: np.float16, I.F32: np.float32}
NO = 0xFFFFFFFF


def plan_ref(ctx_len, new_len, free, count, table, page, n_pages, n_rows):
    """ifr_paged_plan request by request, in whole numbers."""
    free, table = [int(x) for x in free], table.copy()
    stack = free[:min(int(count), n_pages)]
    most = table.shape[1]
    for r, (c, n) in enumerate(zip(ctx_len, new_len)):
        if n == NO:
            held = min(-(-int(c) // page), most)
            stack += [int(p) for p in table[r, :held] if p < n_pages]
    stack = stack[:n_pages]
    free[:len(stack)] = stack
    top, seen, taken, row = len(stack), 0, 0, 0
    start, kv, ctx_out = [], [], []
    pos, slots = np.full(n_rows, NO, np.uint32), np.full(n_rows, NO << 32 | NO, np.uint64)
    grants = []
    for r, (c, n) in enumerate(zip(ctx_len, new_len)):
        c, n = int(c), int(n)
        gone = n == NO
        n = 0 if gone else n
        start.append(min(row, n_rows))
        fits = not gone and c + n <= most * page and row + n <= n_rows
        held = -(-c // page)
        need = -(-(c + n) // page) - held if fits else 0
        ok = fits and (need == 0 or seen + need <= top)
        seen += need
        if ok:
            for i in range(need):
                table[r, held + i] = free[top - 1 - taken - i]
            taken += need
            grants.append((r, c, n, row))
        kv.append(c + n if ok else 0)
        ctx_out.append(c + n if ok else 0 if gone else c)
        row += n
    for r, c, n, row0 in grants:
        for i in range(n):
            p = int(table[r, (c + i) // page])
            pos[row0 + i] = c + i
            if p < n_pages:
                slots[row0 + i] = p * page + (c + i) % page
    return {"row_start": np.array(start + [min(row, n_rows)], np.uint32), "kv_len": np.array(kv, np.uint32),
            "ctx_len_out": np.array(ctx_out, np.uint32), "block_table": table, "positions": pos, "slots": slots,
            "free_count_out": np.array([top - taken], np.uint32), "free_pages": np.array(free, np.uint32)}


def run_plan(ctx, ctx_len, new_len, free, count, table, page, n_pages, n_rows, in_place=False):
    u = lambda a, t=np.uint32: ctx.upload(np.ascontiguousarray(np.asarray(a, t)))  # noqa: E731
    n = len(ctx_len)
    b = {"ctx_len": u(list(ctx_len) or [0]), "new_len": u(list(new_len) or [0]), "free_pages": u(free), "free_count": u([count]),
         "block_table": u(table if table.size else [0]), "row_start": u([7] * (n + 1)), "kv_len": u([7] * max(n, 1)),
         "positions": u([7] * max(n_rows, 1)), "slots": u([7] * max(n_rows, 1), np.uint64)}
    b["free_count_out"] = b["free_count"] if in_place else u([7])
    b["ctx_len_out"] = b["ctx_len"] if in_place else u([7] * max(n, 1))
    args = I.PagedPlan(n_requests=n, n_rows=n_rows, n_pages=n_pages, page_size=page, max_pages=table.shape[1],
                       **{k: v.ptr for k, v in b.items()})
    ctx.paged_plan(args)
    out = {k: b[k].download(np.uint64 if k == "slots" else np.uint32) for k in
           ("row_start", "kv_len", "ctx_len_out", "block_table", "positions", "slots", "free_count_out", "free_pages")}
    for k, m in (("kv_len", n), ("ctx_len_out", n), ("positions", n_rows), ("slots", n_rows)):
        out[k] = out[k][:m]
    out["block_table"] = out["block_table"][:table.size].reshape(table.shape)
    for v in {id(v): v for v in b.values()}.values():
        v.free()
    return out


def rope_ref(x, pos, base, neox):
    """x [rows][heads][hs] in f64, each row turned at its position."""
    hs = x.shape[-1]
    if not base:
        return x
    ang = np.asarray(pos, np.float64)[:, None] * float(base) ** (-2.0 * np.arange(hs // 2) / hs)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y = x.copy()
    a, b = (slice(0, hs // 2), slice(hs // 2, hs)) if neox else (slice(0, hs, 2), slice(1, hs, 2))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


class Paged:
    """A paged cache in host memory (values of its own type), and its device copy."""

    def __init__(self, ctx, rng, dtype, n_pages, page, kvh, hs, layout="dense", fill=np.nan):
        self.ctx, self.dtype, self.n_pages, self.page, self.kvh, self.hs = ctx, dtype, n_pages, page, kvh, hs
        pad = {"dense": 0, "gap": 8, "heads": 0}[layout]
        if layout == "heads":  # [page][head][row][dim]
            self.row, self.head, self.pg = hs, page * hs, kvh * page * hs
        else:
            self.head, self.row = hs + pad, kvh * (hs + pad) + pad
            self.pg = page * self.row + 2 * pad
        self.strides = {} if layout == "dense" else {"page_stride": self.pg, "row_stride": self.row, "head_stride": self.head}
        self.k = np.full(n_pages * self.pg, fill, NP[dtype])
        self.v = self.k.copy()

    def index(self, page, row):
        """Flat indices [kvh][hs] of one row."""
        return page * self.pg + row * self.row + np.arange(self.kvh)[:, None] * self.head + np.arange(self.hs)[None, :]

    def put(self, page, row, k, v):
        at = self.index(page, row)
        self.k[at], self.v[at] = k, v

    def upload(self):
        self.dk, self.dv = self.ctx.upload(self.k), self.ctx.upload(self.v)
        return self

    def args(self, table, max_pages):
        return I.PagedCache(key=self.dk.ptr, value=self.dv.ptr, block_table=table.ptr if table is not None else None,
                            dtype=self.dtype, n_pages=self.n_pages, page_size=self.page, max_pages=max_pages,
                            n_kv_heads=self.kvh, head_size=self.hs, **self.strides)

    def free(self):
        self.dk.free()
        self.dv.free()


def attn_ref(q, k, v, qpos, window=0, sinks=0, scale=0.0, there=None):
    """One request: q [n][heads][hs], k, v [kv][kvh][hs], positions qpos; in 64 bits.  there: rows whose page is one."""
    n, heads, hs = q.shape
    kv, kvh = k.shape[0], k.shape[1]
    out = np.zeros((n, heads, hs))
    j = np.arange(kv)
    scale = scale or 1.0 / np.sqrt(hs)
    with np.errstate(invalid="ignore", over="ignore"):
        for i in range(n):
            see = j <= qpos[i]
            if window:
                see &= (j > qpos[i] - window) | (j < sinks)
            if there is not None:
                see &= there
            if not see.any():
                continue
            for h in range(heads):
                s = (k[see, h * kvh // heads].astype(np.float64) @ q[i, h].astype(np.float64)) * scale
                p = np.exp(s - s.max())
                out[i, h] = (p / p.sum()) @ v[see, h * kvh // heads].astype(np.float64)
    return out
