"""The paged KV cache's operators on cases of real use: their plain forms in elementary torch
operations, and the calls a program makes of this package for the same work.

Kinds of cases (``op``):

* ``attend``: drafted tokens (a tree, a chain, or one decoded token) of ``n`` sequences attend
  their paged cache.
* ``compact``: the kept tokens of a sequence's cache become another sequence (an evicted
  branch, an accepted path of a draft tree).
* ``fork``: sequences that share their prefix's pages with another and own a copy of its last
  page.
* ``append``: room for new tokens is taken, their keys and values are written, and the room is
  given back (a rejected draft, or a finished prompt).
"""

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent /
               "bridge-aware-kv-cache-eviction-for-efficient-long-context-transformers_b200")
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one decoded token of one short sequence: latency
        dict(name="attend_token_short", op="attend", n=1, heads=8, kv=8, dim=64, ctx=299, ragged=0.0, nodes=1,
             tree="chain", page=16, dtype="bf16"),
        # a decode step of a serving batch with grouped heads, lengths spread from about a tenth to the whole
        dict(name="attend_token_batch", op="attend", n=32, heads=32, kv=8, dim=128, ctx=8192, ragged=0.9, nodes=1,
             tree="chain", page=16, dtype="bf16"),
        # a wide draft tree over long contexts (the long-context GQA layer's length): the largest
        dict(name="attend_tree_long", op="attend", n=4, heads=32, kv=8, dim=128, ctx=65536, ragged=0.0, nodes=64,
             tree="parents", page=64, dtype="bf16"),
        # trees of different sizes given as masks, odd lengths, head_dim 64
        dict(name="attend_tree_mask", op="attend", n=7, heads=8, kv=4, dim=64, ctx=5001, ragged=0.7, nodes=25,
             tree="mask", page=32, dtype="f16"),
        # float32, the type of parity runs
        dict(name="attend_chain_f32", op="attend", n=3, heads=8, kv=8, dim=64, ctx=1531, ragged=0.5, nodes=5,
             tree="chain", page=16, dtype="f32"),
        # a prompt's next chunk over what is cached
        dict(name="attend_chunk", op="attend", n=2, heads=8, kv=8, dim=128, ctx=4099, ragged=0.3, nodes=301,
             tree="chain", page=64, dtype="bf16"),
        # eviction of two 128,000-token caches to a twentieth, the full ones kept beside
        dict(name="compact_evicted", op="compact", n=2, layers=1, kv=8, dim=128, ctx=128000, ragged=0.0, kept=6400,
             tail=0, page=64, dtype="bf16"),
        # accepted paths of a batch's draft trees
        dict(name="compact_accepted", op="compact", n=32, layers=4, kv=8, dim=128, ctx=4096, ragged=0.8, kept=4,
             tail=16, page=16, dtype="bf16"),
        # eight samples from one prompt
        dict(name="fork_samples", op="fork", n=8, parents=1, layers=8, kv=8, dim=128, ctx=10007, ragged=0.0, page=64,
             dtype="bf16"),
        # the next beams of 32 sequences
        dict(name="fork_beams", op="fork", n=32, parents=32, layers=4, kv=8, dim=64, ctx=8192, ragged=0.9, page=16,
             dtype="f16"),
        # a batch's drafted tokens, then rolled back
        dict(name="append_draft", op="append", n=32, kv=8, dim=128, ctx=4001, ragged=0.8, new=8, page=16,
             dtype="bf16"),
        # two prompts written and freed
        dict(name="append_prompt", op="append", n=2, kv=8, dim=128, ctx=0, ragged=0.0, new=32768, page=64,
             dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "compact", "fork", "append"])
    page = rng.choice([16, 16, 32, 64, 128])
    kv = rng.choice([1, 2, 4, 8, 8])
    dim = rng.choice([64, 128, 128])
    ragged = round(rng.uniform(0.0, 0.95), 3)
    if op == "attend":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        heads = kv * rng.choice([1, 2, 4, 5, 8])
        nodes = _log_int(rng, 1, 512)
        tree = "chain" if nodes > 128 else rng.choice(["chain", "parents", "mask"])
        n = _log_int(rng, 1, 48)
        # tokens of all sequences such that neither the cache read nor the products pass the largest case's
        most = min(260000 * 8 // kv, int(4e8 // (heads * nodes)))
        if dtype == "f32":
            most = min(most // 8, int(8e6 // (heads * nodes)))
        most = max(1, most // n)
        return dict(op=op, n=n, heads=heads, kv=kv, dim=dim, ctx=_log_int(rng, 1, max(2, min(most, 131072))),
                    ragged=ragged, nodes=nodes, tree=tree, page=page, dtype=dtype)
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "compact":
        n, layers = _log_int(rng, 1, 16), _log_int(rng, 1, 4)
        ctx = _log_int(rng, 64, 180000 // (n * layers))
        if rng.random() < 0.5:
            nodes = rng.randint(2, 64)
            return dict(op=op, n=n, layers=layers, kv=kv, dim=dim, ctx=ctx, ragged=ragged,
                        kept=rng.randint(1, min(nodes, 8)), tail=nodes, page=page, dtype=dtype)
        least = max(1, int(ctx * (1 - ragged)) - 1)
        return dict(op=op, n=n, layers=layers, kv=kv, dim=dim, ctx=ctx, ragged=ragged,
                    kept=_log_int(rng, 1, least), tail=0, page=page, dtype=dtype)
    if op == "fork":
        n, layers = _log_int(rng, 1, 48), _log_int(rng, 1, 8)
        parents = rng.choice([1, max(1, n // 2), n])
        return dict(op=op, n=n, parents=parents, layers=layers, kv=kv, dim=dim,
                    ctx=_log_int(rng, 1, max(64, 256000 // (parents * layers))), ragged=ragged, page=page, dtype=dtype)
    n = _log_int(rng, 1, 48)
    new = _log_int(rng, 1, max(1, 65536 // n))
    return dict(op=op, n=n, kv=kv, dim=dim, ctx=rng.choice([0, _log_int(rng, 1, 100000 // n)]), ragged=ragged, new=new,
                page=page, dtype=dtype)


def _lengths(case, count):
    """Cached tokens of each sequence: spread evenly below the longest, ``ragged`` of it at most."""
    return [int(case["ctx"] * (1.0 - case["ragged"] * ((0.6180339887 * i) % 1.0))) for i in range(count)]


def _node_counts(case):
    """Drafted tokens of each sequence: trees of a batch given as masks differ in size."""
    less = 3 if case["tree"] == "mask" else 1
    return [max(1, case["nodes"] - i % less) for i in range(case["n"])]


def _cdiv(a, b):
    return -(-a // b)


def _cache(case, lens, layers, rows, spare, gen, slack=0):
    """A cache in use: ``rows`` sequence slots, of which the first hold ``lens`` tokens in pages
    scattered over the pool, with room for ``spare`` pages more."""
    S, H, D = case["page"], case["kv"], case["dim"]
    dt = _TYPES[case["dtype"]]
    counts = [_cdiv(x, S) for x in lens]
    width = max(counts + [1]) + slack
    pages = sum(counts) + spare
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(rows, dtype=torch.int64)
    held[:len(lens)] = torch.tensor(counts, dtype=torch.int64)
    held = held.cuda()
    used = torch.arange(width, device="cuda") < held[:, None]
    table[used] = order[:sum(counts)]
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order[:sum(counts)].long()] = 1
    seq = torch.zeros(rows, dtype=torch.int32)
    seq[:len(lens)] = torch.tensor(lens, dtype=torch.int32)
    k = torch.randn(layers, pages, H, S, D, device="cuda", dtype=dt, generator=gen)
    k += torch.randn(H, 1, D, device="cuda", dtype=dt, generator=gen)  # keys have a mean of their own in each channel
    v = torch.randn(layers, pages, H, S, D, device="cuda", dtype=dt, generator=gen)
    return dict(k_pages=k, v_pages=v, block_table=table, seq_lens=seq.cuda(), ref_counts=refs,
                status=torch.zeros(1, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    n, S, H, D = case["n"], case["page"], case["kv"], case["dim"]
    dt = _TYPES[case["dtype"]]
    st = dict(op=case["op"])
    if case["op"] == "attend":
        T, counts = case["nodes"], _node_counts(case)
        lens = [c + m for c, m in zip(_lengths(case, n), counts)]
        st.update(_cache(case, lens, 1, n, 3, gen))
        st["q"] = torch.randn(n, case["heads"], T, D, device="cuda", dtype=dt, generator=gen)
        st["num_nodes"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
        st["parents"] = st["tree_mask"] = None
        at = torch.arange(T, device="cuda")
        par = (torch.rand(n, T, device="cuda", generator=gen) * at).long().clamp(max=T - 1) - (at == 0).long()
        if case["tree"] == "parents":
            st["parents"] = par.to(torch.int32)
        elif case["tree"] == "mask":
            st["tree_mask"] = _ancestors(par)
    elif case["op"] == "compact":
        base = _lengths(case, n)
        K, tail = case["kept"], case["tail"]
        lens = [max(x, K) for x in base] if tail == 0 else [x + tail for x in base]
        fresh = n * (_cdiv(K, S) + 2)
        st.update(_cache(case, lens, case["layers"], 2 * n, 2 * fresh + 3, gen))
        st["src"] = torch.arange(n, dtype=torch.int32, device="cuda")
        st["dst"] = torch.arange(n, 2 * n, dtype=torch.int32, device="cuda")
        room = torch.tensor(lens if tail == 0 else [tail] * n, device="cuda")
        # K different places out of each row's room, ascending
        pick = torch.rand(n, int(room.max()), device="cuda", generator=gen)
        pick[torch.arange(pick.shape[1], device="cuda") >= room[:, None]] = 2.0
        st["keep"] = pick.topk(K, dim=1, largest=False).indices.sort(dim=1).values
        st["keep_num"] = torch.full((n,), K, dtype=torch.int32, device="cuda")
        if tail:
            st["keep_num"] -= torch.arange(n, device="cuda", dtype=torch.int32) % K
        st["start"] = torch.tensor(base, dtype=torch.int32, device="cuda") if tail else None
    elif case["op"] == "fork":
        m = case["parents"]
        lens = [max(1, x) for x in _lengths(case, m)]
        st.update(_cache(case, lens, case["layers"], m + n, 2 * n + 3, gen))
        st["src"] = torch.randint(0, m, (n,), device="cuda", generator=gen, dtype=torch.int32)
        st["dst"] = torch.arange(m, m + n, dtype=torch.int32, device="cuda")
    else:
        lens, new = _lengths(case, n), case["new"]
        more = _cdiv(new, S) + 1
        st.update(_cache(case, lens, 1, n, n * more + 3, gen, slack=more))
        st["new"] = new
        st["before"] = st["seq_lens"].clone()
        st["empty"] = case["ctx"] == 0
        # as a projection's output is viewed by heads: [n, tokens, heads, dim] in memory
        st["k"] = torch.randn(n, new, H, D, device="cuda", dtype=dt, generator=gen).transpose(1, 2)
        st["v"] = torch.randn(n, new, H, D, device="cuda", dtype=dt, generator=gen).transpose(1, 2)
    return st


# ---------------------------------------------------------------- plain forms
def _ancestors(parents):
    """[n, T, T] truth: node u is t or one of t's ancestors (parents come before their children)."""
    n, T = parents.shape
    at = torch.arange(T, device=parents.device)
    step = (parents[:, :, None] == at).float()
    seen = torch.eye(T, device=parents.device) + step
    for _ in range(max(1, (T - 1).bit_length())):  # each product doubles the path length covered
        seen = ((seen @ seen) > 0).float()
    return seen > 0


def _plain_attend(st):
    q, kp, vp = st["q"], st["k_pages"][0], st["v_pages"][0]
    n, Hq, T, D = q.shape
    H, S = kp.shape[1], kp.shape[2]
    table, lens, nodes = st["block_table"].long(), st["seq_lens"].long(), st["num_nodes"].long()
    width = table.shape[1] * S
    at = table.clamp(min=0)
    key = kp[at].transpose(1, 2).reshape(n, H, width, D).float()
    score = q.float().reshape(n, H, Hq // H * T, D) @ key.transpose(2, 3)
    del key
    score = score.reshape(n, Hq, T, width) * (1.0 / math.sqrt(D))
    node = torch.arange(T, device=q.device)
    if st["parents"] is not None:
        tree = _ancestors(st["parents"].long())
    elif st["tree_mask"] is not None:
        tree = st["tree_mask"]
    else:
        tree = (node[None, :] <= node[:, None]).expand(n, T, T)
    pos = torch.arange(width, device=q.device)
    ctx = (lens - nodes)[:, None]
    in_tree = (pos - ctx).clamp(0, T - 1)[:, None, :].expand(n, T, width)
    seen = (pos < ctx)[:, None, :] | ((pos >= ctx) & (pos < lens[:, None]))[:, None, :] & tree.gather(2, in_tree)
    seen = (seen & (node < nodes[:, None])[:, :, None])[:, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(dim=3, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    del score
    total = p.sum(dim=3, keepdim=True)
    val = vp[at].transpose(1, 2).reshape(n, H, width, D).float()
    val = val * (pos < lens[:, None])[:, None, :, None]
    out = (p.reshape(n, H, Hq // H * T, width) @ val).reshape(n, Hq, T, D)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    lse = (torch.log(total) + top).squeeze(3)
    return out.to(q.dtype), lse


def _plain_update(st, src, dst, start, keep, keep_num, grow):
    """Sequence dst becomes the first ``start`` tokens of src and those at start + keep, with room
    for ``grow`` more: pages whose tokens stay in place are shared, the others are the free pages
    of lowest number, taken in order."""
    kp, vp, table, lens, refs = (st[x] for x in ("k_pages", "v_pages", "block_table", "seq_lens", "ref_counts"))
    S, W = kp.shape[3], table.shape[1]
    dev = kp.device
    src, dst = src.long(), dst.long()
    n, K = src.shape[0], keep.shape[1]
    x = torch.arange(K, device=dev)
    kn = keep_num.long()
    moved = (x < kn[:, None]) & (keep != x)
    same = torch.cat([torch.where(moved, x, K), kn[:, None]], dim=1).amin(dim=1)
    intact, held = start + same, start + kn
    size = held + grow
    old, gone = table[src].long(), table[dst].long()
    j = torch.arange(W, device=dev)
    tail = old.gather(1, (held // S).clamp(max=W - 1)[:, None]).squeeze(1).clamp(min=0)
    alone = (src == dst) & (refs[tail] == 1) & ((src[:, None] == src).sum(dim=1) == 1)
    stay = intact // S + ((intact == held) & (held % S > 0) & alone).long()
    pages = (size + S - 1) // S
    need = pages - stay
    first = need.cumsum(0) - need
    free = (refs == 0).nonzero().squeeze(1)
    fresh = (j >= stay[:, None]) & (j < pages[:, None])
    taken = free[(first[:, None] + j - stay[:, None]).clamp(0, free.shape[0] - 1)]
    new = torch.where(j < stay[:, None], old, torch.where(fresh, taken, torch.full_like(taken, -1)))
    was = j < ((lens[dst].long() + S - 1) // S)[:, None]
    refs.index_add_(0, gone[was], torch.full_like(gone[was], -1, dtype=torch.int32))
    refs.index_add_(0, new[j < pages[:, None]], torch.ones_like(new[j < pages[:, None]], dtype=torch.int32))
    # tokens that change their page: [stay * S, held)
    to = (stay * S)[:, None] + torch.arange(K + S, device=dev)
    i, c = (to < held[:, None]).nonzero(as_tuple=True)
    to = to[i, c]
    off = to - start[i]
    if K:
        off = torch.where(off < 0, off, keep[i, off.clamp(0, K - 1)])
    at = start[i] + off
    page_from, page_to = old[i, at // S], new[i, to // S]
    kp[:, page_to, :, to % S] = kp[:, page_from, :, at % S]
    vp[:, page_to, :, to % S] = vp[:, page_from, :, at % S]
    table[dst] = new.to(torch.int32)
    lens[dst] = size.to(torch.int32)


def _plain_write(st):
    kp, vp, k, v = st["k_pages"][0], st["v_pages"][0], st["k"], st["v"]
    n, H, T, D = k.shape
    S = kp.shape[2]
    pos = (st["seq_lens"].long() - T)[:, None] + torch.arange(T, device=k.device)
    page = st["block_table"].long().gather(1, pos // S)
    kp[page, :, pos % S] = k.transpose(1, 2)
    vp[page, :, pos % S] = v.transpose(1, 2)


def _plain(st):
    if st["op"] == "attend":
        return _plain_attend(st)
    dev = st["k_pages"].device
    if st["op"] == "compact":
        start = torch.zeros_like(st["keep_num"]) if st["start"] is None else st["start"]
        _plain_update(st, st["src"], st["dst"], start.long(), st["keep"], st["keep_num"], 0)
    elif st["op"] == "fork":
        none = torch.empty(st["src"].shape[0], 0, dtype=torch.int64, device=dev)
        start = st["seq_lens"].long()[st["src"].long()]
        _plain_update(st, st["src"], st["dst"], start, none, torch.zeros_like(start), 0)
    else:
        rows = torch.arange(st["seq_lens"].shape[0], device=dev)
        none = torch.empty(rows.shape[0], 0, dtype=torch.int64, device=dev)
        nothing = torch.zeros_like(rows)
        _plain_update(st, rows, rows, st["seq_lens"].long(), none, nothing, st["new"])
        _plain_write(st)
        _plain_update(st, rows, rows, st["before"].long(), none, nothing, 0)
    return _state(st)


def _state(st):
    return [st[x] for x in ("k_pages", "v_pages", "block_table", "seq_lens", "ref_counts", "status")]


# ---------------------------------------------------------------- the package's calls
def _handle(st):
    """The cache object a program holds: made from its tensors on the first call, then kept with them."""
    if "cache" not in st:
        if _PACKAGE not in sys.path:
            sys.path.insert(0, _PACKAGE)
        from cab_attention import PagedKVCache
        st["cache"] = PagedKVCache(st["k_pages"], st["v_pages"], st["block_table"], st["seq_lens"],
                                   st["ref_counts"], st["status"])
    return st["cache"]


def _calls(st):
    cache = _handle(st)
    if st["op"] == "attend":
        return cache.attend(0, st["q"], parents=st["parents"], tree_mask=st["tree_mask"],
                            num_nodes=st["num_nodes"], return_lse=True)
    if st["op"] == "compact":
        cache.compact(st["keep"], st["keep_num"], start=st["start"], src=st["src"], dst=st["dst"])
    elif st["op"] == "fork":
        cache.fork(st["src"], st["dst"])
    else:
        cache.extend(st["new"])
        cache.write(0, st["k"], st["v"])
        if st["empty"]:
            cache.free()
        else:
            cache.truncate(st["before"])
    return _state(st)


def run(state):
    if own:
        return _calls(state)
    return _plain(state)


def work(case):
    n, S, H, D, e = case["n"], case["page"], case["kv"], case["dim"], _BYTES[case["dtype"]]
    if case["op"] == "attend":
        counts = _node_counts(case)
        ctx = _lengths(case, n)
        tokens = sum(c + m for c, m in zip(ctx, counts))
        rows = case["heads"] * case["nodes"] * n
        seen = sum(m * c + m * (m + 1) // 2 for c, m in zip(ctx, counts))
        return {"bytes": 2 * tokens * H * D * e + 2 * rows * D * e + 4 * rows + 4 * _cdiv(tokens, S),
                "flops": 4.0 * case["heads"] * D * seen}
    if case["op"] == "compact":
        counts = [case["kept"] - (i % case["kept"] if case["tail"] else 0) for i in range(n)]
        token = 2 * 2 * case["layers"] * H * D * e
        # a path's first page keeps its context: those tokens go along
        before = sum(x % S for x in _lengths(case, n)) if case["tail"] else 0
        return {"bytes": (sum(counts) + before) * token + 8 * sum(counts), "flops": 0}
    if case["op"] == "fork":
        lens = [max(1, x) for x in _lengths(case, case["parents"])]
        token = 2 * 2 * case["layers"] * H * D * e
        mean = sum(x % S for x in lens) / len(lens)
        return {"bytes": n * (mean * token + 8 * _cdiv(sum(lens) // len(lens), S)), "flops": 0}
    return {"bytes": n * case["new"] * 2 * 2 * H * D * e, "flops": 0}


def exact(case, seed):
    """Attention from its definition in 64 bits, one sequence after the other. The other
    operators only move values."""
    if case["op"] != "attend":
        return None
    st = prepare(case, seed)
    q, n, T, D = st["q"], case["n"], case["nodes"], case["dim"]
    group = case["heads"] // case["kv"]
    out = torch.zeros(n, case["heads"], T, D, dtype=torch.float64, device="cuda")
    lse = torch.full((n, case["heads"], T), -math.inf, dtype=torch.float64, device="cuda")
    for b, (m, size) in enumerate(zip(st["num_nodes"].tolist(), st["seq_lens"].tolist())):
        pages = st["block_table"][b, :_cdiv(size, case["page"])].long()
        bias = torch.zeros(m, size, dtype=torch.float64, device="cuda")
        if st["tree_mask"] is not None:
            open_ = st["tree_mask"][b, :m, :m].cpu()
        else:
            up = st["parents"][b].tolist() if st["parents"] is not None else list(range(-1, T - 1))
            open_ = torch.zeros(m, m, dtype=torch.bool)
            for t in range(m):
                u = t
                while u >= 0:
                    open_[t, u] = True
                    u = up[u]
        bias[:, size - m:] = torch.where(open_, 0.0, -math.inf).double().cuda()
        for h in range(case["kv"]):
            key = st["k_pages"][0, pages, h].reshape(-1, D)[:size].double()
            val = st["v_pages"][0, pages, h].reshape(-1, D)[:size].double()
            for g in range(h * group, (h + 1) * group):
                s = torch.einsum("td,sd->ts", q[b, g, :m].double(), key) / math.sqrt(D) + bias
                lse[b, g, :m] = torch.logsumexp(s, dim=1)
                out[b, g, :m] = torch.softmax(s, dim=1) @ val
    return out, lse
