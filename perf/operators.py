"""Serving many sequences from one paged cache: the operators around the matmuls, and what each is measured on.

  append   rows of several sequences turned (rope) and written to their pages (Context.paged_rope_append)
  decode   attention of one new token per sequence over its pages (Context.paged_decode_attention)
  prompt   causal attention of whole prompts packed one after the other (Context.prompt_attention) or, with a page
           size, of the new rows of sequences whose earlier positions are cached (Context.paged_prompt_attention)
  branch   sequences dropped, forked anew and given room for their next tokens (Context.pages_free, pages_fork,
           pages_extend)
  compact  a fragmented pool moved together (Context.pages_compact)

A pool is [pages][page][n_kv][head_dim], one for K and one for V; a sequence's row of the table names its pages in order.
Lengths are spread geometrically from `lo` to `hi`, so a case alone says what has to be done.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
THETA = 10000.0


def listed():
    return [
        # one user's chat a few lines in: the latency of a decode step's attention
        case("decode_1seq_len300", "decode", "bf16", 1, 300, 300, 32, 8, 128, 16),
        # a batch of conversations of very different age, the newest of one token
        case("decode_16seq_ragged", "decode", "bf16", 16, 1, 8000, 32, 8, 128, 16),
        # a 70B-class model's layer, a full batch of long conversations: the largest cache
        case("decode_64seq_len4100", "decode", "bf16", 64, 4000, 4200, 64, 8, 128, 64),
        # a 7B-class model without grouped heads, its cache in f32 as the chain of one sequence holds it
        case("decode_4seq_f32", "decode", "f32", 4, 700, 2100, 32, 32, 128, 32),
        # prompts of different lengths packed together, the shortest a single token
        case("prompt_ragged_12seq", "prompt", "bf16", 12, 1, 2500, 28, 4, 128, 0),
        # one long document: the most operations
        case("prompt_8192", "prompt", "bf16", 1, 8192, 8192, 32, 8, 128, 0),
        # short prompts in f32, between f32 matmuls
        case("prompt_f32_2seq", "prompt", "f32", 2, 300, 1000, 16, 16, 64, 0),
        # questions about documents that are cached already: 200 new rows each, keys and values from their pages
        case("prompt_paged_6seq", "prompt", "bf16", 6, 700, 5000, 32, 8, 128, 32, new=200),
        # a decode step's rows on their way into the cache
        case("append_16rows", "append", "bf16", 16, 1, 900, 32, 8, 128, 16, new=1),
        # the same for packed prompts
        case("append_4prompts", "append", "bf16", 4, 500, 2000, 32, 8, 128, 32),
        # eight answers to each of eight prompts: the partial pages of 16 layers copied, room made for the next tokens
        paged("branch_8x8", "branch", "bf16", 72, 8, 8, 30, 900, 16, 8, 128, 32),
        # two of three sequences are gone: what is left of eight layers moves together
        paged("compact_8layers", "compact", "bf16", 48, 0, 0, 100, 1400, 8, 8, 128, 32),
    ]


def case(name, kind, dtype, seqs, lo, hi, n_q, n_kv, head_dim, page, new=0):
    """`new` rows at the end of each sequence are this call's (0: all of them)."""
    return {"name": name, "kind": kind, "dtype": dtype, "seqs": seqs, "lo": lo, "hi": hi, "n_q": n_q, "n_kv": n_kv,
            "head_dim": head_dim, "page": page, "new": new}


def paged(name, kind, dtype, seqs, parents, per, lo, hi, layers, n_kv, head_dim, page):
    return {"name": name, "kind": kind, "dtype": dtype, "seqs": seqs, "parents": parents, "per": per, "lo": lo, "hi": hi,
            "layers": layers, "n_kv": n_kv, "head_dim": head_dim, "page": page}


def logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "prompt", "paged prompt", "append", "branch", "compact"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    head_dim = rng.choice([64, 128, 128, 128, 96])
    n_kv, group = rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([1, 2, 4, 4, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    if kind in ("branch", "compact"):
        per, parents = rng.randint(1, 8), rng.randint(1, 8)
        hi = logint(rng, 100, 1400)
        return {k: v for k, v in paged("", kind, dtype, rng.randint(3, 48) if kind == "compact" else parents * (1 + per),
                                       parents, per, logint(rng, 1, hi), hi, rng.randint(1, 8), rng.choice([1, 2, 4, 8]),
                                       head_dim, rng.choice([16, 32])).items() if k != "name"}
    if kind == "decode":
        seqs = logint(rng, 1, 64)
        hi = logint(rng, 16, min(16000, 64 * 4100 * 8 * 128 // (seqs * n_kv * head_dim * (SIZE[dtype] // 2))))
        c = case("", kind, dtype, seqs, logint(rng, 1, hi), hi, n_kv * group, n_kv, head_dim, page)
    elif kind == "append":
        new, seqs = rng.choice([0, 1, 1, rng.randint(2, 40)]), logint(rng, 1, 32)
        hi = logint(rng, max(new, 16), 8000 // seqs + 40)
        c = case("", kind, dtype, seqs, logint(rng, max(new, 1), hi), hi, n_kv * group, n_kv, head_dim, page, new)
    else:
        seqs = logint(rng, 1, 16)
        n_kv = n_kv if n_kv * group <= 32 else 4
        if kind == "prompt":
            hi = logint(rng, 16, (6000 if dtype == "bf16" else 2000) // seqs + 40)
            c = case("", "prompt", dtype, seqs, logint(rng, 1, hi), hi, n_kv * group, n_kv, head_dim, 0)
        else:
            new = logint(rng, 2, 300)
            hi = logint(rng, new + 16, (16000 if dtype == "bf16" else 4000) // seqs + new + 40)
            c = case("", "prompt", dtype, seqs, logint(rng, new, hi), hi, n_kv * group, n_kv, head_dim, page, new)
    return {k: v for k, v in c.items() if k != "name"}


def spread(c, n):
    """n lengths from lo to hi, evenly over their logarithm."""
    lo, hi = math.log(c["lo"]), math.log(c["hi"])
    return [int(round(math.exp(hi if n == 1 else lo + (hi - lo) * i / (n - 1)))) for i in range(n)]


def lengths(c):
    """(lengths, new rows) of the sequences; every third place is swapped so that they come in no order."""
    a = spread(c, c["seqs"])
    a = a[::3] + a[1::3] + a[2::3]
    return a, [min(c["new"], n) if c["new"] else n for n in a]


# ---- what a program has in hand ----
class State:
    pass


def gen_of(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def prefix(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def prepare(c, seed):
    s, g = State(), gen_of(seed)
    s.c, s.handles = c, None
    if c["kind"] in ("branch", "compact"):
        prepare_pages(s, c, g)
    else:
        prepare_attention(s, c, g)
    return s


def prepare_attention(s, c, g):
    t, page, nq, nkv, hd = TYPES[c["dtype"]], c["page"], c["n_q"], c["n_kv"], c["head_dim"]
    lens, new = lengths(c)
    s.lens, s.rows = ints(lens), sum(new)
    s.cu = ints(prefix(new))
    if page:
        # the pages of a pool that has been in use: in no order, some of them nobody's
        need = [-(-n // page) for n in lens]
        s.width = max(need)
        s.n_pages = sum(need) + sum(need) // 8 + 1
        order = torch.randperm(s.n_pages, generator=g, device="cuda").to(torch.int32)
        s.table = torch.full((len(lens), s.width), -1, dtype=torch.int32, device="cuda")
        for i, at in enumerate(prefix(need)[:-1]):
            s.table[i, :need[i]] = order[at:at + need[i]]
        s.kpool = normal(g, s.n_pages, page, nkv, hd).to(t)
        s.vpool = normal(g, s.n_pages, page, nkv, hd).to(t)
    if c["kind"] == "append":
        s.q, s.k, s.v = normal(g, s.rows, nq, hd), normal(g, s.rows, nkv, hd), normal(g, s.rows, nkv, hd)
        s.out = torch.empty(s.rows, nq, hd, dtype=t, device="cuda")
        return
    s.rows = len(lens) if c["kind"] == "decode" else s.rows
    # heads that look far and wide, and heads that look at little
    sharp = torch.linspace(0.5, 3.0, nq, device="cuda")[:, None]
    s.q = (normal(g, s.rows, nq, hd) * sharp).to(t)
    s.out = torch.empty(s.rows, nq, hd, dtype=t, device="cuda")
    if not page:
        s.k, s.v = normal(g, s.rows, nkv, hd).to(t), normal(g, s.rows, nkv, hd).to(t)


def prepare_pages(s, c, g):
    t, page = TYPES[c["dtype"]], c["page"]
    n_seq = c["parents"] if c["kind"] == "branch" else c["seqs"]
    lens = spread(c, n_seq)
    need = [-(-n // page) for n in lens]
    s.width = max(need) + 2
    full = sum(need)
    s.n_pages = full + (2 * c["parents"] * c["per"] + 8 if c["kind"] == "branch" else full // 8 + 2)
    order = torch.randperm(s.n_pages, generator=g, device="cuda").to(torch.int32)
    s.table = torch.full((c["seqs"], s.width), -1, dtype=torch.int32, device="cuda")
    s.lens = torch.zeros(c["seqs"], dtype=torch.int32, device="cuda")
    s.refs = torch.zeros(s.n_pages, dtype=torch.int32, device="cuda")
    for i, at in enumerate(prefix(need)[:-1]):
        if c["kind"] == "compact" and i % 3:
            continue        # a sequence that has ended
        s.table[i, :need[i]] = order[at:at + need[i]]
        s.refs[order[at:at + need[i]].long()] = 1
        s.lens[i] = lens[i]
    s.kpool = normal(g, c["layers"], s.n_pages, page, c["n_kv"], c["head_dim"]).to(t)
    s.vpool = normal(g, c["layers"], s.n_pages, page, c["n_kv"], c["head_dim"]).to(t)
    if c["kind"] == "branch":
        s.src = ints([i for i in range(c["parents"]) for _ in range(c["per"])])
        s.dst = ints(list(range(c["parents"], c["seqs"])))
        s.counts = ints([1 + i % 3 for i in range(c["parents"] * c["per"])])
    else:
        s.table_out, s.refs_out = torch.empty_like(s.table), torch.empty_like(s.refs)
    s.info = torch.zeros(4, dtype=torch.int32, device="cuda")


# ---- one pass ----
def run(s):
    if own:
        return run_own(s)
    return {"decode": plain_decode, "prompt": plain_prompt, "append": plain_append, "branch": plain_branch,
            "compact": plain_compact}[s.c["kind"]](s)


def run_own(s):
    if s.handles is None:
        s.handles = Handles(s)
    s.handles.call()
    return outputs(s)


def outputs(s):
    kind = s.c["kind"]
    if kind in ("decode", "prompt"):
        return s.out
    if kind == "append":
        return [s.out, s.kpool, s.vpool]
    if kind == "branch":
        return [s.kpool, s.vpool, s.table, s.lens, s.refs, s.info]
    return [s.kpool, s.vpool, s.table_out, s.refs_out, s.info]


class Handles:
    """The library's handles on a state's tensors, made once, and the calls of a pass."""

    def __init__(self, s):
        from raster_b200 import _lib as L
        from raster_b200.runtime import default_context
        self.ctx, c, w = default_context(), s.c, self.wrap
        self.bufs = []
        dt = {"f32": L.F32, "bf16": L.BF16}[c["dtype"]]
        ctx, page, nkv, hd, B = self.ctx, c["page"], c["n_kv"], c["head_dim"], c["seqs"]
        if c["kind"] in ("branch", "compact"):
            row = nkv * hd * SIZE[c["dtype"]]
            k, v, table, lens, refs, info = w(s.kpool), w(s.vpool), w(s.table), w(s.lens), w(s.refs), w(s.info)
            if c["kind"] == "branch":
                src, dst, counts, n = w(s.src), w(s.dst), w(s.counts), c["parents"] * c["per"]
                self.calls = [
                    (ctx.pages_free, (table, lens, refs, dst, info, n, B, s.n_pages, s.width, page)),
                    (ctx.pages_fork, (k, v, table, lens, refs, src, dst, info, n, B, s.n_pages, s.width, page, c["layers"], row)),
                    (ctx.pages_extend, (table, lens, refs, dst, counts, info, n, B, s.n_pages, s.width, page))]
            else:
                self.calls = [(ctx.pages_compact, (k, v, table, lens, refs, w(s.table_out), w(s.refs_out), info, B, s.n_pages,
                                                   s.width, page, c["layers"], row))]
            return
        nq, scale = c["n_q"], hd ** -0.5
        if c["kind"] == "append":
            self.calls = [(ctx.paged_rope_append, (w(s.q), w(s.k), w(s.v), w(s.out), w(s.kpool), w(s.vpool), w(s.table), w(s.lens),
                                                   w(s.cu), s.rows, B, nq, nkv, hd, page, s.n_pages, s.width, THETA, L.F32, dt))]
        elif c["kind"] == "decode":
            self.calls = [(ctx.paged_decode_attention, (w(s.q), w(s.kpool), w(s.vpool), w(s.out), w(s.table), w(s.lens), B, nq,
                                                        nq // nkv, nkv, hd, page, s.n_pages, s.width, scale, dt))]
        elif page:
            self.calls = [(ctx.paged_prompt_attention, (w(s.q), w(s.kpool), w(s.vpool), w(s.out), w(s.table), w(s.cu), w(s.lens),
                                                        s.rows, B, nq, nq // nkv, nkv, hd, page, s.n_pages, s.width, scale, True, dt))]
        else:
            cu = w(s.cu)
            self.calls = [(ctx.prompt_attention, (w(s.q), w(s.k), w(s.v), w(s.out), cu, cu, s.rows, s.rows, B, nq, nq // nkv, nkv,
                                                  hd, scale, True, dt))]

    def wrap(self, t):
        import numpy as np
        kind = {torch.float32: np.float32, torch.bfloat16: np.uint16, torch.int32: np.int32}[t.dtype]
        self.bufs.append(self.ctx.wrap_buffer(t.data_ptr(), t.numel(), kind))
        return self.bufs[-1]

    def call(self):
        for fn, args in self.calls:
            fn(*args)

    def __del__(self):
        for b in self.bufs:
            b.free()


# ---- the plain forms ----
def softmax_values(scores, keep, v):
    """softmax over the kept scores times v; rows that keep nothing are zero."""
    scores.masked_fill_(~keep, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores -= torch.where(torch.isinf(top), torch.zeros_like(top), top)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    return (scores @ v) / torch.where(total > 0, total, torch.ones_like(total))


def plain_decode(s):
    c = s.c
    B, nkv, hd, g = c["seqs"], c["n_kv"], c["head_dim"], c["n_q"] // c["n_kv"]
    pages = s.table.clamp(min=0).long()
    k = s.kpool[pages].reshape(B, -1, nkv, hd).float()
    v = s.vpool[pages].reshape(B, -1, nkv, hd).float()
    q = s.q.float().reshape(B, nkv, g, hd) * hd ** -0.5
    keep = torch.arange(k.shape[1], device="cuda") < s.lens[:, None]
    o = softmax_values(q @ k.permute(0, 2, 3, 1), keep[:, None, None, :], v.permute(0, 2, 1, 3))
    return o.reshape(B, c["n_q"], hd).to(s.q.dtype)


def sequence_of(cu, rows):
    """Which sequence each packed row belongs to."""
    return (torch.arange(rows, device="cuda")[:, None] >= cu[1:]).sum(1)


def plain_prompt(s):
    c = s.c
    nkv, hd, g = c["n_kv"], c["head_dim"], c["n_q"] // c["n_kv"]
    seq = sequence_of(s.cu, s.rows)
    at = torch.arange(s.rows, device="cuda") - s.cu[1:][seq] + s.lens[seq]     # the rows' positions
    if c["page"]:
        pages = s.table.clamp(min=0).long()
        k = s.kpool[pages].reshape(-1, nkv, hd).float()
        v = s.vpool[pages].reshape(-1, nkv, hd).float()
        n = s.width * c["page"]
        j = torch.arange(c["seqs"] * n, device="cuda")
        kseq, kat = j // n, j % n
    else:
        k, v, kseq, kat = s.k.float(), s.v.float(), seq, at
    keep = (seq[:, None] == kseq) & (at[:, None] >= kat)
    q = s.q.float().reshape(s.rows, nkv, g, hd) * hd ** -0.5
    o = softmax_values(q.permute(1, 2, 0, 3) @ k.permute(1, 2, 0)[:, None], keep, v.permute(1, 0, 2)[:, None])
    return o.permute(2, 0, 1, 3).reshape(s.rows, c["n_q"], hd).to(s.q.dtype)


def turned(x, at):
    """Rotate-half rope of x [rows, heads, head_dim] at positions `at`; the angles in 64 bits."""
    h = x.shape[-1] // 2
    angle = at.double()[:, None] * torch.exp(torch.arange(h, device="cuda").double() * (-2.0 / x.shape[-1] * math.log(THETA)))
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def plain_append(s):
    seq = sequence_of(s.cu, s.rows)
    at = torch.arange(s.rows, device="cuda") - s.cu[1:][seq] + s.lens[seq]
    page = s.table[seq, at // s.c["page"]].long()
    slot = at % s.c["page"]
    s.kpool[page, slot] = turned(s.k, at).to(s.kpool.dtype)
    s.vpool[page, slot] = s.v.to(s.vpool.dtype)
    s.out.copy_(turned(s.q, at))
    return outputs(s)


def drop(s, seqs):
    """The pages of the sequences given back: their counts go down, their rows of the table are empty."""
    held = torch.arange(s.width, device="cuda") < ((s.lens[seqs] + s.c["page"] - 1) // s.c["page"])[:, None]
    pages = s.table[seqs].clamp(min=0).long()
    s.refs.scatter_add_(0, pages.reshape(-1), -held.reshape(-1).int())
    s.table[seqs] = -1
    s.lens[seqs] = 0


def free_pages(s):
    return torch.argsort((s.refs > 0).int(), stable=True)     # free pages first, in order


def plain_branch(s):
    src, dst, page = s.src.long(), s.dst.long(), s.c["page"]
    drop(s, dst)
    # fork: full pages are shared, a partial one is copied to a free page
    n = s.lens[src]
    full, part = n // page, n % page > 0
    slot = torch.arange(s.width, device="cuda")
    shared = slot < full[:, None]
    old = s.table[src]
    s.refs.scatter_add_(0, old.clamp(min=0).long().reshape(-1), shared.reshape(-1).int())
    fresh = free_pages(s)[(part.cumsum(0) - 1).clamp(min=0)].int()
    last = old.gather(1, full.clamp(max=s.width - 1)[:, None].long())[:, 0]
    rows = torch.where(shared, old, torch.full_like(old, -1))
    s.table[dst] = torch.where((slot == full[:, None]) & part[:, None], fresh[:, None], rows)
    s.refs.scatter_add_(0, fresh.long(), part.int())
    s.lens[dst] = n
    a, b = last[part].long(), fresh[part].long()
    s.kpool[:, b] = s.kpool[:, a]
    s.vpool[:, b] = s.vpool[:, a]
    # extend: free pages, in order, where the next tokens need them
    n, more = s.lens[dst], s.lens[dst] + s.counts
    have, want = (n + page - 1) // page, (more + page - 1) // page
    add = (slot >= have[:, None]) & (slot < want[:, None])
    rank = add.reshape(-1).int().cumsum(0).reshape(add.shape) - 1
    fresh = free_pages(s)[rank.clamp(min=0)].int()
    s.table[dst] = torch.where(add, fresh, s.table[dst])
    s.refs.scatter_add_(0, fresh.long().reshape(-1), add.reshape(-1).int())
    s.lens[dst] = more
    s.info[0] = 0
    s.info[1] = (s.refs > 0).sum()
    s.info[2:] = 0
    return outputs(s)


def plain_compact(s):
    live = s.refs > 0
    n_live = live.sum()
    index = torch.arange(s.n_pages, device="cuda")
    moves, holes = live & (index >= n_live), ~live & (index < n_live)
    a, b = index[moves], index[holes]
    to = index.clone()
    to[a] = b
    held = torch.arange(s.width, device="cuda") < ((s.lens + s.c["page"] - 1) // s.c["page"])[:, None]
    s.table_out.copy_(torch.where(held, to[s.table.clamp(min=0).long()].int(), s.table))
    s.refs_out.copy_(s.refs)
    s.refs_out[b] = s.refs[a]
    s.refs_out[a] = 0
    s.kpool[:, b] = s.kpool[:, a]
    s.vpool[:, b] = s.vpool[:, a]
    s.info[0] = 0
    s.info[1] = n_live
    s.info[2] = a.numel()
    s.info[3] = 0
    return outputs(s)


# ---- from the definitions, in 64 bits ----
def exact(c, seed):
    if c["kind"] in ("branch", "compact"):
        return None         # copies: nothing is computed
    s = prepare(c, seed)
    lens, cu, hd, g, page = s.lens.tolist(), s.cu.tolist(), c["head_dim"], c["n_q"] // c["n_kv"], c["page"]
    out = torch.zeros(s.rows, c["n_q"], hd, dtype=torch.float64, device="cuda")
    if c["kind"] == "append":
        freq = torch.tensor([THETA ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64, device="cuda")
        k, v = s.kpool.double(), s.vpool.double()

        def rope(x, pos):
            z = torch.complex(x[..., :hd // 2].double(), x[..., hd // 2:].double())
            a = pos[:, None, None] * freq
            z = z * torch.complex(a.cos(), a.sin())
            return torch.cat([z.real, z.imag], -1)

        for b, n in enumerate(lens):
            r = slice(cu[b], cu[b + 1])
            pos = torch.arange(n - (cu[b + 1] - cu[b]), n, device="cuda")
            where = s.table[b].long()[pos // page]
            out[r] = rope(s.q[r], pos.double())
            k[where, pos % page] = rope(s.k[r], pos.double())
            v[where, pos % page] = s.v[r].double()
        return [out, k, v]
    for b, n in enumerate(lens):
        if page:
            at = [p for p in s.table[b].tolist() if p >= 0]
            k, v = s.kpool[at].flatten(0, 1)[:n].double(), s.vpool[at].flatten(0, 1)[:n].double()
        else:
            k, v = s.k[cu[b]:cu[b + 1]].double(), s.v[cu[b]:cu[b + 1]].double()
        first, last = (b, b + 1) if c["kind"] == "decode" else (cu[b], cu[b + 1])
        for h in range(c["n_q"]):
            for r in range(first, last, 2048):      # some rows at a time
                q = s.q[r:min(r + 2048, last), h].double()
                t = q @ k[:, h // g].T / math.sqrt(hd)
                pos = torch.arange(r, r + q.shape[0], device="cuda") + (n - last)
                t = torch.where(torch.arange(n, device="cuda")[None] > pos[:, None], -math.inf, t)
                out[r:r + q.shape[0], h] = torch.softmax(t, 1) @ v[:, h // g]
    return out


# ---- what a pass cannot do without ----
def work(c):
    size, hd, page = SIZE[c["dtype"]], c["head_dim"], c["page"]
    if c["kind"] == "branch":
        lens = spread(c, c["parents"])
        copied = sum(c["per"] for n in lens if n % page)
        return {"bytes": 4 * copied * c["layers"] * page * c["n_kv"] * hd * size, "flops": 0}
    if c["kind"] == "compact":
        lens = spread(c, c["seqs"])
        need = [-(-n // page) for n in lens]
        live = sum(need[::3])
        n_pages = sum(need) + sum(need) // 8 + 2
        moved = live * (n_pages - live) / n_pages       # pages behind the first `live`, of pages in no order
        return {"bytes": 4 * moved * c["layers"] * page * c["n_kv"] * hd * size + 8 * n_pages, "flops": 0}
    lens, new = lengths(c)
    rows = c["seqs"] if c["kind"] == "decode" else sum(new)
    if c["kind"] == "append":
        return {"bytes": rows * hd * (c["n_q"] + 2 * c["n_kv"]) * (4 + size), "flops": rows * hd * (c["n_q"] + c["n_kv"]) * 3}
    pairs = sum(lens) if c["kind"] == "decode" else sum(r * (n - r) + r * (r + 1) // 2 for n, r in zip(lens, new))
    return {"bytes": 2 * sum(lens) * c["n_kv"] * hd * size + 2 * rows * c["n_q"] * hd * size, "flops": 4 * pairs * c["n_q"] * hd}
