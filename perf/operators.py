"""Soft reads of a store of vectors, and what keeps the store small: cases by which their speed is judged.

A store here is what an index holds: states that a model wrote down once and reads again.  ``search``
reads it the hard way (inner products, then the k largest); these operators read it the soft way, with
a softmax over all inner products in the place of the selection.

``attend``    cross attention of a batch of queries to states of another length (an encoder's, or, ``index``,
              the rows of a flat index by inner product)
``backward``  its gradient with respect to queries, keys and values
``shared``    one step of a batch of sequences that share a long prefix and have rows of their own behind it
``mass``      the attention weight that every row received, added to what it received before
``evict``     the rows of largest weight and the most recent ones move to a smaller cache

Layouts: queries [batch, queries, heads, width], keys and values [batch, keys, key heads, width], log-sums
[batch, queries, heads], weights [batch, key heads, keys].  A group of heads / key heads query heads reads the
same keys.  Synthetic inputs, from the seed alone: normal states that also share a direction which some keys
follow more than others, so that a few rows collect much of the weight, as in a real store.
"""
import math

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


def _attend(name, dtype, batch, lq, lk, heads, kv_heads, d, ragged, op="attend"):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "lq": lq, "lk": lk, "heads": heads,
            "kv_heads": kv_heads, "d": d, "ragged": ragged}


def _index(name, dtype, nb, nq, d):
    return {"name": name, "op": "index", "dtype": dtype, "nb": nb, "nq": nq, "d": d}


def _shared(name, dtype, batch, new, prefix, own_rows, heads, kv_heads, d, ragged):
    return {"name": name, "op": "shared", "dtype": dtype, "batch": batch, "new": new, "prefix": prefix,
            "own_rows": own_rows, "heads": heads, "kv_heads": kv_heads, "d": d, "ragged": ragged}


def _mass(name, dtype, batch, lq, lk, heads, kv_heads, d, ragged, causal):
    return {"name": name, "op": "mass", "dtype": dtype, "batch": batch, "lq": lq, "lk": lk, "heads": heads,
            "kv_heads": kv_heads, "d": d, "ragged": ragged, "causal": causal}


def _evict(name, dtype, batch, lk, kv_heads, d, keep, recent, ragged):
    return {"name": name, "op": "evict", "dtype": dtype, "batch": batch, "lk": lk, "kv_heads": kv_heads, "d": d,
            "keep": keep, "recent": recent, "ragged": ragged}


def listed():
    return [
        # a training step's reader: long targets against twice as many states
        _attend("reader_train", "bf16", 8, 2048, 4096, 16, 4, 128, False),
        # a padded batch of odd lengths, one of them empty, one key head per head
        _attend("reader_ragged", "f16", 3, 771, 1531, 12, 12, 64, True),
        # a server that decodes one token a sequence against stored states
        _attend("reader_token", "bf16", 32, 1, 4096, 32, 8, 128, True),
        # all rows of a flat index read softly by a batch of queries, where search reads the k largest
        _index("index_read", "f16", 100_000, 1_000, 128),
        # the gradient of the training step, the largest case
        _attend("reader_train_backward", "bf16", 8, 2048, 4096, 16, 4, 128, False, op="backward"),
        # the gradient of the padded batch
        _attend("reader_ragged_backward", "f16", 3, 771, 1531, 12, 12, 64, True, op="backward"),
        # a decoding step of 64 conversations behind one long document
        _shared("prefix_decode", "bf16", 64, 1, 32_768, 1_024, 32, 8, 128, True),
        # a few short sequences that check three guessed tokens at once; odd sizes
        _shared("prefix_short", "f16", 5, 3, 1_003, 77, 6, 2, 80, True),
        # weights of one decoding step, over a long cache
        _mass("mass_decode", "bf16", 32, 1, 8_192, 32, 8, 128, True, True),
        # weights that a prompt's own queries leave behind
        _mass("mass_prompt", "f16", 2, 1_111, 2_049, 16, 4, 64, False, True),
        # a server cuts its caches to a quarter
        _evict("evict_quarter", "bf16", 16, 8_192, 8, 128, 2_048, 256, True),
        # one short conversation
        _evict("evict_small", "f16", 1, 700, 2, 64, 129, 16, False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _limits():
    ws = [(c["op"], work(c)) for c in listed()]
    return max(w["flops"] for _, w in ws), max(w["bytes"] for _, w in ws)


def draw(rng):
    flops, nbytes = _limits()
    while True:
        op = rng.choice(["attend", "attend", "index", "backward", "shared", "mass", "evict"])
        dtype = rng.choice(["bf16", "f16"])
        d = rng.choice([64, 64, 128, 128, 80, 96, 8 * rng.randint(1, 16)])
        kv = rng.choice([1, 2, 3, 4, 8, 12, 16])
        heads = kv * rng.choice([1, 1, 2, 3, 4, 6, 8])
        batch = _log_int(rng, 1, 64)
        ragged = rng.random() < 0.6
        if op == "index":
            c = _index(None, dtype, _log_int(rng, 1_000, 400_000), _log_int(rng, 1, 2_000), rng.choice([64, 96, 128]))
        elif op == "shared":
            new = rng.choice([1, 1, 1, rng.randint(2, 9)])
            c = _shared(None, dtype, batch, new, _log_int(rng, 1, 65_536), new + _log_int(rng, 1, 4_096), heads, kv, d, ragged)
        elif op == "evict":
            lk = _log_int(rng, 2, 40_000)
            keep = rng.randint(1, lk)
            c = _evict(None, dtype, batch, lk, kv, d, keep, rng.randint(0, keep), ragged)
        else:
            lq, lk = _log_int(rng, 1, 4_096), _log_int(rng, 1, 16_384)
            if op == "mass":
                c = _mass(None, dtype, batch, lq, max(lq, lk), heads, kv, d, ragged, rng.random() < 0.5)
            else:
                c = _attend(None, dtype, batch, lq, lk, heads, kv, d, ragged, op=op)
        if op in ("attend", "backward", "mass"):
            if c["batch"] * c["heads"] * c["lq"] * c["lk"] > 1 << 30:   # the plain form writes the scores down
                continue
        if op == "shared" and c["batch"] * c["heads"] * c["new"] * (c["prefix"] + c["own_rows"]) > 1 << 29:
            continue
        w = work(c)
        if w["flops"] > flops or w["bytes"] > nbytes:
            continue
        del c["name"]
        return c


# ---- inputs ---------------------------------------------------------------------------------------


def _lengths(case, n, top, low):
    """Visible keys of every sequence; the seed only decides which sequence gets which."""
    if not case["ragged"]:
        return [top] * n
    out = [max(low, top - (i * top * 7) // (8 * n)) for i in range(n)]
    if n >= 3 and low == 0:
        out[-1] = 0
    return out


def _permuted(lengths, gen):
    order = torch.randperm(len(lengths), generator=gen, device="cuda")
    return torch.tensor(lengths, dtype=torch.int32, device="cuda")[order]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _queries(gen, dtype, *shape):
    return (_randn(gen, *shape) + 3.0 / math.sqrt(shape[-1])).to(dtype)


def _keys(gen, dtype, *shape):
    pull = _randn(gen, *shape[:-1], 1).abs() * (2.0 / math.sqrt(shape[-1]))
    return (_randn(gen, *shape) + pull).to(dtype)


def _scale(case):
    return 1.0 / math.sqrt(case["d"])


def prepare(case, seed):
    gen = _gen(seed)
    dt = DTYPE[case["dtype"]]
    op = case["op"]
    st = {"case": case, "scale": _scale(case)}
    if op == "index":
        nb, nq, d = case["nb"], case["nq"], case["d"]
        rows = _keys(gen, dt, nb, d)
        st.update(x=_queries(gen, dt, nq, d), rows=rows, values=_randn(gen, nb, d).to(dt))
        if own:
            import faiss_metal_b200 as fm
            st["resources"] = fm.StandardB200Resources(torch.cuda.current_device())
            st["index"] = fm.B200IndexFlat(st["resources"], d, fm.METRIC_INNER_PRODUCT,
                                           fm.STORAGE_BF16 if case["dtype"] == "bf16" else fm.STORAGE_F16)
            st["index"].add(rows.float())
        return st
    b, hk, d = case["batch"], case["kv_heads"], case["d"]
    if op == "evict":
        lk = case["lk"]
        st.update(k=_keys(gen, dt, b, lk, hk, d), v=_randn(gen, b, lk, hk, d).to(dt),
                  mass=torch.exp(2.0 * _randn(gen, b, hk, lk)),
                  lengths=_permuted(_lengths(case, b, lk, 0), gen))
        return st
    h = case["heads"]
    if op == "shared":
        p, s = case["prefix"], case["own_rows"]
        st.update(q=_queries(gen, dt, b, case["new"], h, d), pk=_keys(gen, dt, p, hk, d), pv=_randn(gen, p, hk, d).to(dt),
                  k=_keys(gen, dt, b, s, hk, d), v=_randn(gen, b, s, hk, d).to(dt),
                  lengths=_permuted(_lengths(case, b, s, case["new"]), gen))
        return st
    lq, lk = case["lq"], case["lk"]
    causal = op == "mass" and case["causal"]
    low = lq if causal else 0
    st.update(q=_queries(gen, dt, b, lq, h, d), k=_keys(gen, dt, b, lk, hk, d),
              lengths=_permuted(_lengths(case, b, lk, low), gen) if case["ragged"] else None)
    if op == "mass":
        st["mass"] = torch.exp(_randn(gen, b, hk, lk))
        st["lse"] = _plain_lse(st, causal)
        return st
    st["v"] = _randn(gen, b, lk, hk, d).to(dt)
    if op == "backward":
        st["out"], st["lse"] = _plain_attend(st)
        st["grad"] = _randn(gen, b, lq, h, d).to(dt)
    return st


# ---- the plain forms -------------------------------------------------------------------------------


def _grouped(x, hk):
    """[batch, n, heads, d] -> [batch, key heads, group * n, d] in 32 bits."""
    b, n, h, d = x.shape
    return x.float().reshape(b, n, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, h // hk * n, d)


def _ungrouped(x, n):
    """[batch, key heads, group * n, d] -> [batch, n, heads, d]."""
    b, hk, gn, d = x.shape
    return x.reshape(b, hk, gn // n, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, hk * (gn // n), d)


def _plain_scores(st, causal):
    q, k = st["q"], st["k"]
    b, lq, h, _ = q.shape
    lk, hk = k.shape[1], k.shape[2]
    s = (_grouped(q, hk) @ k.float().permute(0, 2, 3, 1)) * st["scale"]
    if st["lengths"] is not None or causal:
        n = st["lengths"].long() if st["lengths"] is not None else torch.full((b,), lk, device=q.device)
        end = n.view(b, 1).expand(b, lq)
        if causal:
            end = end - lq + 1 + torch.arange(lq, device=q.device)
        hidden = torch.arange(lk, device=q.device) >= end.unsqueeze(-1)     # [b, lq, lk]
        s.view(b, hk, h // hk, lq, lk).masked_fill_(hidden.view(b, 1, 1, lq, lk), -math.inf)
    return s


def _plain_softmax(s):
    """Weights (0 where a row sees nothing) and log-sums of the rows of s."""
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:-1], 1), -math.inf)
    e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    return e / torch.where(total == 0, torch.ones_like(total), total), lse


def _rows_lse(lse, lq):
    """[batch, key heads, group * lq] -> [batch, lq, heads]."""
    return _ungrouped(lse.unsqueeze(-1), lq).squeeze(-1).contiguous()


def _plain_lse(st, causal):
    s = _plain_scores(st, causal)
    return _rows_lse(_plain_softmax(s)[1], st["q"].shape[1])


def _plain_attend(st):
    lq = st["q"].shape[1]
    p, lse = _plain_softmax(_plain_scores(st, False))
    v = st["v"].float().permute(0, 2, 1, 3)
    return _ungrouped(p @ v, lq).to(st["q"].dtype).contiguous(), _rows_lse(lse, lq)


def _plain_backward(st):
    q, k, v = st["q"], st["k"], st["v"]
    hk, lq = k.shape[2], q.shape[1]
    p, _ = _plain_softmax(_plain_scores(st, False))
    do = _grouped(st["grad"], hk)
    dv = p.transpose(-1, -2) @ do
    dp = do @ v.float().permute(0, 2, 3, 1)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * st["scale"]
    dq = ds @ k.float().permute(0, 2, 1, 3)
    dk = ds.transpose(-1, -2) @ _grouped(q, hk)
    return (_ungrouped(dq, lq).to(q.dtype), dk.permute(0, 2, 1, 3).to(q.dtype), dv.permute(0, 2, 1, 3).to(q.dtype))


def _plain_shared(st):
    q, hk = st["q"], st["k"].shape[2]
    b, t, h, d = q.shape
    first = (_grouped(q, hk).permute(1, 0, 2, 3).reshape(hk, -1, d) @ st["pk"].float().permute(1, 2, 0)) * st["scale"]
    first = first.view(hk, b, h // hk * t, -1).permute(1, 0, 2, 3)
    n_first = first.shape[-1]
    p, lse = _plain_softmax(torch.cat([first, _plain_scores(st, True)], -1))
    o = p[..., :n_first].permute(1, 0, 2, 3).reshape(hk, -1, n_first) @ st["pv"].float().permute(1, 0, 2)
    o = o.view(hk, b, -1, d).permute(1, 0, 2, 3) + p[..., n_first:] @ st["v"].float().permute(0, 2, 1, 3)
    return _ungrouped(o, t).to(q.dtype), _rows_lse(lse, t)


def _plain_index(st):
    p, lse = _plain_softmax((st["x"].float() @ st["rows"].float().T) * st["scale"])
    return (p @ st["values"].float()).to(st["x"].dtype), lse


def _plain_mass(st):
    q, k = st["q"], st["k"]
    b, lq, h, _ = q.shape
    hk = k.shape[2]
    lse = _grouped(st["lse"].unsqueeze(-1), hk)
    s = _plain_scores(st, st["case"]["causal"])
    p = torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse))
    return st["mass"] + p.sum(2)


def _plain_evict(st):
    k, v, mass, lengths = st["k"], st["v"], st["mass"], st["lengths"].long()
    keep, recent = st["case"]["keep"], st["case"]["recent"]
    b, lk, hk, d = k.shape
    pos = torch.arange(lk, device=k.device)
    n = lengths.view(b, 1, 1)
    weight = torch.where(pos >= n - recent, torch.full_like(mass, math.inf), mass)
    weight = torch.where(pos >= n, torch.full_like(mass, -math.inf), weight)
    order = torch.sort(weight, dim=-1, descending=True, stable=True).indices[..., :keep]
    count = torch.clamp(n, max=keep)
    kept = torch.where(torch.arange(keep, device=k.device) < count, order, lk)
    kept = torch.sort(kept, dim=-1).values
    live = kept < lk
    rows = torch.where(live, kept, torch.zeros_like(kept))                    # [b, hk, keep]
    at = rows.permute(0, 2, 1).unsqueeze(-1).expand(b, keep, hk, d)
    on = live.permute(0, 2, 1).unsqueeze(-1)
    new_k = torch.where(on, torch.gather(k, 1, at), torch.zeros((), dtype=k.dtype, device=k.device))
    new_v = torch.where(on, torch.gather(v, 1, at), torch.zeros((), dtype=k.dtype, device=k.device))
    new_mass = torch.where(live, torch.gather(mass, 2, rows), torch.zeros_like(mass[..., :keep]))
    return (new_k, new_v, new_mass, torch.where(live, kept, torch.full_like(kept, -1)).int(),
            count.view(b).int())


_PLAIN = {"attend": _plain_attend, "backward": _plain_backward, "shared": _plain_shared, "index": _plain_index,
          "mass": _plain_mass, "evict": _plain_evict}


def _own(st):
    import faiss_metal_b200 as fm
    op, scale = st["case"]["op"], st["scale"]
    if op == "attend":
        return fm.attend(st["q"], st["k"], st["v"], key_lengths=st["lengths"], scale=scale, return_lse=True)
    if op == "backward":
        return fm.attend_backward(st["grad"], st["q"], st["k"], st["v"], st["out"], st["lse"], key_lengths=st["lengths"],
                                  scale=scale)
    if op == "shared":
        return fm.attend_shared(st["q"], st["pk"], st["pv"], st["k"], st["v"], st["lengths"], scale=scale,
                                return_lse=True)
    if op == "index":
        return st["index"].attend(st["x"], st["values"], scale=scale, return_lse=True)
    if op == "mass":
        return fm.attention_mass(st["q"], st["k"], st["lse"], key_lengths=st["lengths"], scale=scale,
                                 causal=st["case"]["causal"], mass=st["mass"])
    return fm.evict(st["k"], st["v"], st["mass"], st["lengths"], st["case"]["keep"], recent=st["case"]["recent"])


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    op, d = case["op"], case["d"]
    if op == "index":
        nb, nq = case["nb"], case["nq"]
        return {"bytes": 2 * d * (2 * nb + 2 * nq) + 4 * nq, "flops": 4 * nb * nq * d}
    b, hk = case["batch"], case["kv_heads"]
    if op == "evict":
        kept = sum(min(n, case["keep"]) for n in _lengths(case, b, case["lk"], 0)) * hk
        seen = sum(_lengths(case, b, case["lk"], 0)) * hk
        slots = b * hk * case["keep"]
        return {"bytes": 4 * seen + 2 * 2 * d * (kept + slots) + 2 * 4 * slots, "flops": seen}
    h = case["heads"]
    if op == "shared":
        t, p = case["new"], case["prefix"]
        ns = _lengths(case, b, case["own_rows"], t)
        pairs = h * (b * t * p + sum(t * n - t * (t - 1) // 2 for n in ns))
        rows = b * t * h
        return {"bytes": 2 * d * (2 * rows + 2 * hk * (p + sum(ns))) + 4 * rows, "flops": 4 * pairs * d}
    lq, lk = case["lq"], case["lk"]
    causal = op == "mass" and case["causal"]
    ns = _lengths(case, b, lk, lq if causal else 0)
    pairs = h * sum(lq * n - (lq * (lq - 1) // 2 if causal else 0) for n in ns)
    rows, keys = b * lq * h, hk * sum(ns)
    if op == "mass":
        return {"bytes": 2 * d * (rows + keys) + 4 * rows + 8 * b * hk * lk, "flops": 2 * pairs * d}
    if op == "attend":
        return {"bytes": 2 * d * (2 * rows + 2 * keys) + 4 * rows, "flops": 4 * pairs * d}
    return {"bytes": 2 * d * (4 * rows + 2 * keys + 2 * b * lk * hk) + 4 * rows, "flops": 10 * pairs * d}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------


def _visible(st, i, lq, lk, causal):
    """[lq, lk] of sequence i: which keys each query sees."""
    n = int(st["lengths"][i]) if st["lengths"] is not None else lk
    end = torch.full((lq,), n, device="cuda")
    if causal:
        end = n - lq + 1 + torch.arange(lq, device="cuda")
    return torch.arange(lk, device="cuda")[None, :] < end[:, None]


def _exact_rows(s):
    """Row weights and log-sums of 64-bit scores; hidden ones are -inf."""
    lse = torch.logsumexp(s, -1) if s.shape[-1] else s.new_full(s.shape[:-1], -math.inf)
    p = torch.exp(s - lse.unsqueeze(-1))
    return torch.where(lse.unsqueeze(-1) == -math.inf, torch.zeros((), dtype=s.dtype, device=s.device), p), lse


def exact(case, seed):
    st = prepare(case, seed)
    op, scale = case["op"], st["scale"]
    if op == "index":
        outs, lses = [], []
        rows, values = st["rows"].double().T, st["values"].double()
        for x in st["x"].double().split(256):
            p, lse = _exact_rows(x @ rows * scale)
            outs.append(p @ values)
            lses.append(lse)
        return torch.cat(outs), torch.cat(lses)
    if op == "evict":
        return _exact_evict(st)
    q, k = st["q"].double(), st["k"].double()
    b, lq, h, d = q.shape
    lk, group = k.shape[1], h // k.shape[2]
    causal = op == "shared" or (op == "mass" and case["causal"])
    out, lse = torch.zeros_like(q), torch.zeros(b, lq, h, dtype=torch.float64, device="cuda")
    v = st["v"].double() if op != "mass" else None
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)
    mass = st["mass"].double() if op == "mass" else None
    for i in range(b):
        seen = _visible(st, i, lq, lk, causal)
        for head in range(h):
            kh = head // group
            s = (q[i, :, head] @ k[i, :, kh].T * scale).masked_fill(~seen, -math.inf)
            if op == "shared":
                s = torch.cat([q[i, :, head] @ st["pk"][:, kh].double().T * scale, s], 1)
            if op == "mass":
                row = st["lse"][i, :, head].double().unsqueeze(1)
                mass[i, kh] += torch.exp(s - torch.where(row == -math.inf, torch.zeros_like(row), row)).sum(0)
                continue
            p, lse[i, :, head] = _exact_rows(s)
            if op == "shared":
                out[i, :, head] = p @ torch.cat([st["pv"][:, kh].double(), v[i, :, kh]])
                continue
            if op == "attend":
                out[i, :, head] = p @ v[i, :, kh]
                continue
            g = st["grad"][i, :, head].double()
            dv[i, :, kh] += p.T @ g
            dp = g @ v[i, :, kh].T
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
            dq[i, :, head] = ds @ k[i, :, kh]
            dk[i, :, kh] += ds.T @ q[i, :, head]
    if op == "mass":
        return mass
    if op == "backward":
        return dq, dk, dv
    return out, lse


def _exact_evict(st):
    case = st["case"]
    keep, recent = case["keep"], case["recent"]
    k, v, mass = st["k"], st["v"], st["mass"]
    b, lk, hk, d = k.shape
    new_k, new_v = k.new_zeros(b, keep, hk, d).double(), k.new_zeros(b, keep, hk, d).double()
    new_mass = mass.new_zeros(b, hk, keep).double()
    rows = torch.full((b, hk, keep), -1, dtype=torch.int32, device="cuda")
    lengths = []
    for i in range(b):
        n = int(st["lengths"][i])
        lengths.append(min(n, keep))
        for head in range(hk):
            if n <= keep:
                chosen = list(range(n))
            else:
                weights = mass[i, head, :n - recent].tolist()
                best = sorted(range(n - recent), key=lambda j: (-weights[j], j))[:keep - recent]
                chosen = sorted(best) + list(range(n - recent, n))
            at = torch.tensor(chosen, dtype=torch.long, device="cuda")
            rows[i, head, :len(chosen)] = at.int()
            new_k[i, :len(chosen), head] = k[i, at, head].double()
            new_v[i, :len(chosen), head] = v[i, at, head].double()
            new_mass[i, head, :len(chosen)] = mass[i, head, at].double()
    return new_k, new_v, new_mass, rows, torch.tensor(lengths, dtype=torch.int32, device="cuda")
