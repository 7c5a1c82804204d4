"""The paged cache's operators beyond a sequence's own tokens, whose time this
repository answers for: attention of any rows over cached states of another length,
attention of a batch whose sequences share their first tokens, attention that keeps
count of each key's weights, and the eviction that goes by those. Each with its
inputs, its least work, a plain statement in elementary torch operations and one in
64 bits.

Sizes: 24 heads of 128, contexts of 512 rows, 768 and 27280 video tokens; between and
beyond them sizes without a name. Codes are returned as the whole numbers they are:
eviction moves them, and has to give the same ones."""
import math
import os
import random
import sys

import torch

own = False

_PKG = "self-evolve-diffusion-cpp_amd"
HD = 128


def listed():
    return [
        # One token of each of eight sequences over the states of a text, ragged: latency.
        {"name": "cross_tokens", "kind": "cross", "nseq": 8, "rows": 1, "len": 512, "heads": 24,
         "kv_heads": 24, "page": 64, "pad": 0},
        # Every token of a 720p clip over its text context, a layer of a denoising step.
        {"name": "cross_clip", "kind": "cross", "nseq": 1, "rows": 27280, "len": 512, "heads": 24,
         "kv_heads": 24, "page": 128, "pad": 0},
        # Chunks of a ragged batch over states three times as long, heads shared by four, one
        # sequence without states.
        {"name": "cross_ragged", "kind": "cross", "nseq": 7, "rows": 1031, "len": 3001, "heads": 32,
         "kv_heads": 8, "page": 16, "pad": 5},
        # Sixteen continuations of one prompt, a token each.
        {"name": "shared_tokens", "kind": "shared", "groups": 1, "nseq": 16, "new": 1,
         "prefix": 4099, "len": 67, "heads": 24, "kv_heads": 24, "page": 64, "causal": True,
         "pad": 0},
        # Thirty-two continuations of a very long one, heads shared by four.
        {"name": "shared_long", "kind": "shared", "groups": 1, "nseq": 32, "new": 1,
         "prefix": 131073, "len": 1031, "heads": 32, "kv_heads": 8, "page": 128, "causal": True,
         "pad": 3},
        # Short chunks of six sequences on two clips (with and without guidance).
        {"name": "shared_chunks", "kind": "shared", "groups": 2, "nseq": 6, "new": 96,
         "prefix": 8209, "len": 300, "heads": 24, "kv_heads": 24, "page": 256, "causal": True,
         "pad": 0},
        # One token of each of eight sequences, its weights counted.
        {"name": "weights_tokens", "kind": "weights", "nseq": 8, "new": 1, "len": 4099,
         "heads": 24, "kv_heads": 24, "page": 64, "causal": True, "pad": 3},
        # One token against a very long cache whose heads are shared by four.
        {"name": "weights_long", "kind": "weights", "nseq": 1, "new": 1, "len": 131073,
         "heads": 32, "kv_heads": 8, "page": 128, "causal": True, "pad": 0},
        # A whole prompt over itself, before its cache is thinned out.
        {"name": "weights_prompt", "kind": "weights", "nseq": 1, "new": 4099, "len": 4099,
         "heads": 24, "kv_heads": 8, "page": 16, "causal": True, "pad": 0},
        # A step's cache back to its budget after a few dozen new tokens.
        {"name": "evict_step", "kind": "evict", "nseq": 1, "len": 2111, "keep": 2048, "first": 4,
         "last": 512, "kv_heads": 24, "page": 64},
        # Ragged prompts of a batch to their budget; the shortest are under it.
        {"name": "evict_batch", "kind": "evict", "nseq": 8, "len": 8203, "keep": 2048, "first": 16,
         "last": 256, "kv_heads": 8, "page": 16},
        # Two very long prompts to an eighth.
        {"name": "evict_long", "kind": "evict", "nseq": 2, "len": 131073, "keep": 16384,
         "first": 64, "last": 4096, "kv_heads": 8, "page": 256},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["cross", "shared", "weights", "evict"])
    page = rng.choice([16, 32, 64, 128, 256])
    while True:
        kv = rng.choice([1, 2, 3, 8, 24])
        heads = kv * rng.choice([1, 1, 2, 4, 5, 8])
        if heads > 32:
            continue
        few = rng.choice([1, rng.randint(2, 16)])
        c = {"kind": kind, "nseq": rng.randint(1, 9), "heads": heads, "kv_heads": kv, "page": page}
        if kind == "cross":
            c.update(rows=rng.choice([few, _log(rng, 17, 27280)]), len=_log(rng, 1, 8192),
                     pad=rng.choice([0, 0, 7]))
            if (c["nseq"] * c["rows"] * c["len"] * heads <= 3.3e8
                    and c["nseq"] * c["rows"] * heads <= 27280 * 24):
                return c
        elif kind == "shared":
            groups = rng.choice([1, 1, 2, 3])
            new = rng.choice([few, few, _log(rng, 17, 256)])
            c.update(groups=groups, nseq=groups * rng.randint(2, 32 // groups), new=new,
                     prefix=_log(rng, 1, 131073), len=new + _log(rng, 1, 2048),
                     causal=rng.random() < 0.7, pad=rng.choice([0, 0, 7]))
            if (c["nseq"] * new * (c["prefix"] + c["len"]) * heads <= 1.35e8
                    and (groups * c["prefix"] + c["nseq"] * c["len"]) * kv <= 164065 * 8):
                return c
        elif kind == "weights":
            new = rng.choice([few, few, _log(rng, 17, 4099)])
            c.update(new=new, len=new + _log(rng, 1, 65536), causal=rng.random() < 0.7,
                     pad=rng.choice([0, 0, 7]))
            if (c["nseq"] * new * c["len"] * heads <= 4.0e8
                    and c["nseq"] * c["len"] * kv <= 262145 * 4):
                return c
        else:
            keep = _log(rng, 16, 16384)
            c.update(len=_log(rng, 16, 131073), keep=keep, first=rng.randint(0, keep // 4),
                     last=rng.randint(0, keep // 2))
            del c["heads"]
            if c["nseq"] * c["len"] * kv <= 262146 * 8 and c["len"] > keep // 2:
                return c


def _part(r, most, least=1):
    return r.randint(least, max(least, most))


def _shape(case):
    """Rows and cached tokens of each sequence, and tokens of each shared part: the first
    has the case's own sizes, the others ragged parts of them; of more than five the third
    has no tokens."""
    r = random.Random(case["nseq"] * 1000003 + case["len"] * 31 + case["kv_heads"])
    most = case.get("rows", case.get("new", 0))
    rows, lens = [most], [case["len"]]
    for s in range(1, case["nseq"]):
        n = most if most < 2 else _part(r, most)
        rows.append(n)
        lens.append(_part(r, case["len"], 1 if case["kind"] in ("cross", "evict") else n))
    if case["nseq"] > 5 and case["kind"] in ("cross", "weights"):
        lens[2] = 0
    shared = [case["prefix"]] if case["kind"] == "shared" else []
    shared += [_part(r, case["prefix"]) for _ in range(1, case.get("groups", 0))]
    return rows, lens, shared


# ---- inputs -------------------------------------------------------------

def _sdq():
    for root in (os.getcwd(), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))):
        at = os.path.join(root, _PKG)
        if os.path.isdir(at):
            if at not in sys.path:
                sys.path.insert(0, at)
            break
    import sdq
    return sdq


class _Draws:
    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.dev)
        self.g.manual_seed(int(seed))

    def n(self, *shape, std=1.0):
        t = torch.randn(shape, generator=self.g, device=self.dev, dtype=torch.float32)
        return t if std == 1.0 else t.mul_(std)

    def u(self, *shape):
        return torch.rand(shape, generator=self.g, device=self.dev, dtype=torch.float32)

    def codes(self, shape):
        return torch.randint(-127, 128, shape, generator=self.g, device=self.dev,
                             dtype=torch.int8)


def _int32(dev, v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _pages(r, lists, page):
    """For each list of lengths a page table, all of shuffled pages of their own, and the
    pool's size (a few pages stay free)."""
    need = [[max(1, -(-n // page)) for n in lens] for lens in lists]
    pool = sum(map(sum, need)) + 3
    free = torch.randperm(pool, generator=r.g, device=r.dev).to(torch.int32)
    tables, at = [], 0
    for counts in need:
        table = torch.zeros((len(counts), max(counts, default=1)), dtype=torch.int32, device=r.dev)
        for s, n in enumerate(counts):
            table[s, :n] = free[at:at + n]
            at += n
        tables.append(table)
    return tables, pool


def prepare(case, seed):
    r = _Draws(seed)
    kind, page, h = case["kind"], case["page"], case["kv_heads"]
    rows, lens, shared = _shape(case)
    lists = [lens, [case["keep"]] * len(lens) if kind == "evict" else shared]
    (table, other), pool = _pages(r, lists, page)
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    shape = (pool, h, page)
    st = dict(case)
    st.update(rows=rows, lens=lens, shared=shared, starts=starts, total=starts[-1] + case.get("pad", 0),
              table=table, t_starts=_int32(r.dev, starts), t_lens=_int32(r.dev, lens),
              kc=r.codes(shape + (HD,)), vc=r.codes(shape + (HD,)),
              ks=0.012 * (0.5 + r.u(*shape)), vs=0.02 * torch.exp(r.n(*shape, std=0.5)))
    if kind != "evict":
        c = case["heads"] * HD
        st.update(q=r.n(st["total"], c, std=1.5), out=torch.zeros((st["total"], c), device=r.dev))
    if kind in ("weights", "evict"):
        # sums of many rows' weights: a few keys far above the others, a tenth never looked at
        st["w"] = 8 / max(lens) * torch.exp(r.n(*shape, std=2.0)) * (r.u(*shape) > 0.1)
    if kind == "shared":
        per = case["nseq"] // case["groups"]
        st.update(s_table=other, s_lens=_int32(r.dev, shared),
                  s_start=_int32(r.dev, [g * per for g in range(case["groups"] + 1)]))
    if kind == "evict":
        st.update(to_table=other, to_lens=torch.zeros(case["nseq"], dtype=torch.int32, device=r.dev),
                  kept=torch.zeros((case["nseq"], h, case["keep"]), dtype=torch.int32,
                                   device=r.dev))
    if own:
        sdq = _sdq()
        st["cache"] = sdq.KvCache(st["kc"], st["ks"], st["vc"], st["vs"])
        st["batch"] = sdq.KvBatch(st["t_starts"], st["t_lens"], st["table"])
        if kind == "shared":
            st["prefixes"] = sdq.KvShared(st["s_start"], st["s_lens"], st["s_table"])
    return st


# ---- one pass -----------------------------------------------------------

def run(st):
    return (_run_own if own else _run_plain)[st["kind"]](st)


def _own_cross(st):
    return _sdq().kv_cross_attention(st["cache"], st["batch"], st["q"], st["out"], st["heads"])


def _own_shared(st):
    return _sdq().kv_attention_shared(st["cache"], st["prefixes"], st["batch"], st["q"], st["out"],
                                      st["heads"], causal=st["causal"])


def _own_weights(st):
    _sdq().kv_attention_weights(st["cache"], st["batch"], st["w"], st["q"], st["out"], st["heads"],
                                causal=st["causal"])
    return {"out": st["out"], "weights": st["w"]}


def _own_evict(st):
    _sdq().kv_evict(st["cache"], st["batch"], st["w"], st["to_table"], st["to_lens"], st["kept"],
                    first=st["first"], last=st["last"])
    return _evicted(st)


_run_own = {"cross": _own_cross, "shared": _own_shared, "weights": _own_weights,
            "evict": _own_evict}


def _evicted(st):
    return {"k": st["kc"], "ks": st["ks"], "v": st["vc"], "vs": st["vs"], "weights": st["w"],
            "lens": st["to_lens"], "kept": st["kept"]}


def _cached(st, table, most):
    """Keys and values [n, kv, most, HD] in fp32 of the first `most` tokens that a table
    names, and their (page, slot)."""
    pos = torch.arange(most, device=table.device)
    page = table[:, pos // st["page"]].long()
    slot = (pos % st["page"]).expand_as(page)
    k = st["kc"][page, :, slot].float() * st["ks"][page, :, slot][..., None]
    v = st["vc"][page, :, slot].float() * st["vs"][page, :, slot][..., None]
    return k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous(), page, slot


def _queries(st):
    """Rows of q as [nseq, kv, G * n, HD], n the most rows of a sequence; their row of q and
    whether it is one."""
    n, kv = max(st["rows"]), st["kv_heads"]
    i = torch.arange(n, device=st["q"].device)
    there = i[None] < (st["t_starts"][1:] - st["t_starts"][:-1])[:, None]
    row = (st["t_starts"][:-1, None] + i[None]).long().clamp(max=st["total"] - 1)
    q = st["q"][row].view(len(row), n, kv, -1, HD).permute(0, 2, 3, 1, 4)
    return q.reshape(len(row), kv, -1, HD), row, there


def _scores(q, k):
    return q.contiguous() @ k.transpose(-1, -2).contiguous() * (1 / math.sqrt(HD))


def _own_places(st, n, most):
    """[nseq, n, most]: the keys of its own that row i of a sequence sees."""
    pos = torch.arange(most, device=st["q"].device)
    seen = (pos[None, None] < st["t_lens"][:, None, None]).expand(-1, n, -1)
    if st.get("causal"):
        new = st["t_starts"][1:] - st["t_starts"][:-1]
        at = (st["t_lens"] - new)[:, None] + torch.arange(n, device=pos.device)[None]
        seen = seen & (pos[None, None] <= at[:, :, None])
    return seen


def _masked(s, seen, n):
    """Scores [.., G * n, most] with -inf where a row does not see a key."""
    return s.view(s.shape[0], s.shape[1], -1, n, s.shape[-1]).masked_fill(
        ~seen[:, None, None], -math.inf).view_as(s)


def _finite(top):
    return torch.where(torch.isinf(top), torch.zeros_like(top), top)


def _nonzero(z):
    return torch.where(z == 0, torch.ones_like(z), z)


def _to_rows(st, o, row, there):
    S, n = row.shape
    o = o.view(S, st["kv_heads"], -1, n, HD).permute(0, 3, 1, 2, 4).reshape(S, n, -1)
    out = torch.zeros_like(st["q"])
    out[row[there]] = o[there]
    return out


def _plain_own(st):
    """Attention over a sequence's own tokens: output, weights and the tokens' places."""
    q, row, there = _queries(st)
    k, v, page, slot = _cached(st, st["table"], max(1, max(st["lens"])))
    s = _masked(_scores(q, k), _own_places(st, row.shape[1], k.shape[2]), row.shape[1])
    p = torch.exp(s - _finite(s.amax(-1, keepdim=True)))
    p = p / _nonzero(p.sum(-1, keepdim=True))
    return _to_rows(st, p @ v, row, there), p, there, page, slot


def _plain_cross(st):
    return _plain_own(st)[0]


def _plain_weights(st):
    out, p, there, page, slot = _plain_own(st)
    S, n = there.shape
    p = p.view(S, st["kv_heads"], -1, n, p.shape[-1]).masked_fill(~there[:, None, None, :, None], 0)
    got = p.sum((2, 3)).transpose(1, 2)  # [S, tokens, kv]
    pos = torch.arange(got.shape[1], device=got.device)[None]
    new = (st["t_starts"][1:] - st["t_starts"][:-1])[:, None]
    live, old = pos < st["t_lens"][:, None], pos < st["t_lens"][:, None] - new
    got = got + torch.where(old[..., None], st["w"][page, :, slot], torch.zeros_like(got))
    st["w"][page[live], :, slot[live]] = got[live]
    return {"out": out, "weights": st["w"]}


def _plain_shared(st):
    q, row, there = _queries(st)
    S, n, groups = row.shape[0], row.shape[1], st["groups"]
    k, v, _, _ = _cached(st, st["table"], max(st["lens"]))
    s = _masked(_scores(q, k), _own_places(st, n, k.shape[2]), n)
    # the shared part: the rows of all sequences of a group over one copy of its keys
    pk, pv, _, _ = _cached(st, st["s_table"], max(st["shared"]))
    gq = q.view(groups, S // groups, st["kv_heads"], -1, HD).transpose(1, 2)
    t = _scores(gq.reshape(groups, st["kv_heads"], -1, HD), pk)
    pos = torch.arange(pk.shape[2], device=q.device)
    t = t.masked_fill((pos[None] >= st["s_lens"][:, None])[:, None, None], -math.inf)

    def by_group(x):
        return x.reshape(groups, S // groups, st["kv_heads"], -1, x.shape[-1]).transpose(1, 2).reshape(
            groups, st["kv_heads"], -1, x.shape[-1])

    def by_seq(x):
        return x.view(groups, st["kv_heads"], S // groups, -1, x.shape[-1]).transpose(1, 2).reshape(
            S, st["kv_heads"], -1, x.shape[-1])

    top = _finite(torch.maximum(s.amax(-1, keepdim=True), by_seq(t.amax(-1, keepdim=True))))
    p, g = torch.exp(s - top), torch.exp(t - by_group(top))
    z = p.sum(-1, keepdim=True) + by_seq(g.sum(-1, keepdim=True))
    return _to_rows(st, (p @ v + by_seq(g @ pv)) / _nonzero(z), row, there)


def _plain_evict(st):
    S, keep, most = st["nseq"], st["keep"], max(st["lens"])
    pos = torch.arange(most, device=st["w"].device)
    page = st["table"][:, pos // st["page"]].long()
    slot = (pos % st["page"]).expand(S, -1)
    n = st["t_lens"][:, None]
    always = (pos < st["first"]) | (pos >= n - st["last"])  # [S, tokens]
    w = st["w"][page, :, slot].transpose(1, 2)  # [S, kv, tokens]
    w = w.masked_fill(always[:, None], math.inf).masked_fill((pos >= n)[:, None], -math.inf)
    # the largest first, the lower position of equals, then in order of position
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    order = torch.where(order < n[..., None], order, torch.full_like(order, most))
    order = torch.sort(order, -1).values
    order = torch.cat([order, order.new_full((S, order.shape[1], keep - order.shape[2]), most)], 2)
    live = order < most
    st["kept"].copy_(torch.where(live, order, torch.full_like(order, -1)))
    st["to_lens"].copy_(st["t_lens"].clamp(max=keep))
    at = torch.nonzero(live, as_tuple=True)
    seq, head, to = at
    src = order[at]
    src_page, src_slot = page[seq, src], src % st["page"]
    to_page, to_slot = st["to_table"][seq, to // st["page"]].long(), to % st["page"]
    for name in ("kc", "ks", "vc", "vs", "w"):
        st[name][to_page, head, to_slot] = st[name][src_page, head, src_slot]
    return _evicted(st)


_run_plain = {"cross": _plain_cross, "shared": _plain_shared, "weights": _plain_weights,
              "evict": _plain_evict}


# ---- least work ---------------------------------------------------------

def _pairs(case, rows, lens):
    """Row and own key pairs."""
    if not case.get("causal"):
        return sum(n * length for n, length in zip(rows, lens))
    return sum(sum(range(max(1, length - n + 1), length + 1)) for n, length in zip(rows, lens))


def work(case):
    rows, lens, shared = _shape(case)
    kv = case["kv_heads"]
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        # every weight in; of a kept token codes, scales and weight in and out, its position out
        return {"bytes": kv * (4 * sum(lens) + kept * (2 * (2 * (HD + 4) + 4) + 4)),
                "flops": kv * sum(lens)}
    heads = case["heads"]
    pairs = _pairs(case, rows, lens)
    if shared:
        per = case["nseq"] // case["groups"]
        pairs += sum(n * shared[s // per] for s, n in enumerate(rows))
    counted = case["kind"] == "weights"
    keys = sum(lens) + sum(shared)
    return {"bytes": kv * keys * (2 * (HD + 4) + 8 * counted) + 8 * sum(rows) * heads * HD,
            "flops": heads * pairs * (4 * HD + counted)}


# ---- in 64 bits, from the definitions -----------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return _exact_evict(st) if case["kind"] == "evict" else _exact_attention(st)


def _of(st, name, table, s, h, n):
    """A pool's entries of tokens 0 .. n - 1 of table row s, head h, in 64 bits."""
    used = table[s, :-(-n // st["page"])].long()
    return st[name][used, h].double().flatten(0, 1)[:n]


def _exact_attention(st):
    G = st["heads"] // st["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    sums = st["w"].double() if st["kind"] == "weights" else None
    for s in range(st["nseq"]):
        n, length, first = st["rows"][s], st["lens"][s], st["starts"][s]
        g = s // (st["nseq"] // st["groups"]) if st["shared"] else 0
        ahead = st["shared"][g] if st["shared"] else 0
        if not ahead + length:
            continue
        for h in range(st["kv_heads"]):
            k, v = [], []
            for table, row, count in ((st.get("s_table"), g, ahead), (st["table"], s, length)):
                if count:
                    k.append(_of(st, "kc", table, row, h, count)
                             * _of(st, "ks", table, row, h, count)[:, None])
                    v.append(_of(st, "vc", table, row, h, count)
                             * _of(st, "vs", table, row, h, count)[:, None])
            k, v = torch.cat(k), torch.cat(v)
            total = torch.zeros(length, dtype=torch.float64, device=k.device)
            for j in range(h * G, (h + 1) * G):
                logits = st["q"][first:first + n, j * HD:(j + 1) * HD].double() @ k.t().contiguous()
                logits /= math.sqrt(HD)
                if st.get("causal"):
                    last = ahead + length - n + torch.arange(n, device=k.device)
                    logits[torch.arange(len(k), device=k.device)[None] > last[:, None]] = -math.inf
                weight = torch.softmax(logits, 1)
                out[first:first + n, j * HD:(j + 1) * HD] = weight @ v
                total += weight[:, ahead:].sum(0)
            if sums is not None:
                p = torch.arange(length, device=k.device)
                page, slot = st["table"][s, p // st["page"]].long(), p % st["page"]
                before = sums[page, h, slot]
                before[length - n:] = 0  # the call's own tokens start anew
                sums[page, h, slot] = before + total
    return out if sums is None else {"out": out, "weights": sums}


def _exact_evict(st):
    pools = {"k": st["kc"].clone(), "v": st["vc"].clone()}
    pools.update((name, st[key].double()) for name, key in (("ks", "ks"), ("vs", "vs"),
                                                            ("weights", "w")))
    kept = torch.full_like(st["kept"], -1)
    lens = torch.zeros_like(st["to_lens"])
    for s, n in enumerate(st["lens"]):
        lens[s] = min(n, st["keep"])
        place = torch.arange(n, device=kept.device)
        for h in range(st["kv_heads"]):
            w = _of(st, "w", st["table"], s, h, n)
            must = (place < st["first"]) | (place >= n - st["last"])
            rest = place[~must]
            by_weight = rest[torch.argsort(w[rest], descending=True, stable=True)]
            chosen = torch.cat([place[must], by_weight])[:st["keep"]].sort().values
            to = torch.arange(len(chosen), device=kept.device)
            kept[s, h, :len(chosen)] = chosen.int()
            a = st["table"][s, chosen // st["page"]].long(), h, chosen % st["page"]
            b = st["to_table"][s, to // st["page"]].long(), h, to % st["page"]
            for pool in pools.values():
                pool[b] = pool[a]
    return {**pools, "lens": lens, "kept": kept}
