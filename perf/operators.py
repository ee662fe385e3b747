"""Cases of the serving operators: attention of ragged chunks of new tokens
over paged caches, log probabilities of given tokens with entropy, rank and
top alternatives, and copies between pages of a cache.

Each operator has a plain form in elementary torch operations and the
library's call (`own`).  Sizes follow the model shapes of
llama3.go_b200/synthetic.py and the batched decode benchmark."""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

PAGE = 256  # positions of one page


def _l3g():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama3.go_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import l3g
    return l3g


def _attn(name, heads, heads_kv, hd, f16, seqs, q, kv, lens_seed):
    return {"name": name, "op": "attention", "heads": heads, "heads_kv": heads_kv, "hd": hd, "f16": f16,
            "seqs": seqs, "q_min": q[0], "q_max": q[1], "kv_min": kv[0], "kv_max": kv[1],
            "lens_seed": lens_seed}


def _logp(name, rows, vocab, top_k, masked):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top_k": top_k, "masked": masked}


def _pages(name, hd, f16, n, pool, rows_min, rows_max, lens_seed):
    return {"name": name, "op": "pages", "hd": hd, "f16": f16, "n": n, "pool": pool, "rows_min": rows_min,
            "rows_max": rows_max, "lens_seed": lens_seed}


def listed():
    return [
        # one session's next token early in a chat (the 1B shape, the cache's default type): latency
        _attn("attn-1x1-f32-hd64", 32, 8, 64, False, 1, (1, 1), (300, 300), 1),
        # a batched decode step: 64 sessions of 512 to 8192 positions, the 8B shape
        _attn("attn-64x1-f16-hd128", 32, 8, 128, True, 64, (1, 1), (512, 8192), 2),
        # a long prompt's next pass of 512 tokens after 4096
        _attn("attn-1x512-f16-hd128", 32, 8, 128, True, 1, (512, 512), (4608, 4608), 3),
        # sessions with a few to a couple of hundred new tokens each, a group of three query heads, f32 cache
        _attn("attn-24xragged-f32-hd128", 24, 8, 128, False, 24, (1, 200), (1, 2048), 4),
        # several short prompts at once from position zero, the 1B shape in f16
        _attn("attn-7x300-f16-hd64", 32, 8, 64, True, 7, (100, 300), (100, 300), 5),
        # long documents scored in large chunks: 8 sessions of 8000 positions
        _attn("attn-8x1000-f16-hd128", 32, 8, 128, True, 8, (1000, 1000), (8000, 8192), 6),
        # the log probability of one sampled token and its five best alternatives
        _logp("logp-1x128256-top5", 1, 128256, 5, 0.0),
        # a pass of prompt scoring: 512 positions, 20 alternatives each
        _logp("logp-512x128256-top20", 512, 128256, 20, 0.0),
        # answers restricted by a grammar: a third of the vocabulary masked, no alternatives asked
        _logp("logp-131x8000-masked", 131, 8000, 0, 0.33),
        # one session of a small model forked: the last, part-filled page of each (layer, kv head)
        _pages("pages-fork-16x37", 64, False, 16, 64, 37, 37, 1),
        # eight forks of an 8B session: 32 layers x 8 kv heads part-filled pages each
        _pages("pages-fork-2048", 128, True, 2048, 4608, 1, 255, 2),
        # compacting a pool: whole pages moved
        _pages("pages-compact-1500", 128, False, 1500, 4000, 256, 256, 3),
    ]


SHAPES = [(32, 8, 128), (32, 8, 64), (24, 8, 128), (8, 2, 128), (4, 1, 128), (4, 2, 64), (4, 2, 32), (6, 2, 32),
          (2, 1, 32)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "logprobs", "pages"])
    if kind == "attention":
        heads, heads_kv, hd = rng.choice(SHAPES)
        while True:
            seqs = _log_int(rng, 1, 64)
            q_max = _log_int(rng, 1, 1024)
            kv_max = max(q_max, _log_int(rng, 1, 8192))
            # padded score values of the plain form, at most those of the largest listed case
            if seqs * heads * q_max * kv_max <= 8 * 32 * 1000 * 8000 and seqs * kv_max <= 64 * 8192:
                break
        q_min = rng.choice([1, q_max, max(1, q_max // 2)])
        kv_min = rng.choice([q_min, max(q_min, kv_max // 4), kv_max])
        c = _attn("", heads, heads_kv, hd, rng.random() < 0.5, seqs, (q_min, q_max), (kv_min, kv_max),
                  rng.randrange(1 << 30))
    elif kind == "logprobs":
        vocab = rng.choice([97, 500, 2048, 8000, 128256, _log_int(rng, 50, 130000)])
        rows = _log_int(rng, 1, max(1, min(2048, 60_000_000 // vocab)))
        c = _logp("", rows, vocab, rng.choice([0, 1, 5, 20, 40]), rng.choice([0.0, 0.0, 0.25, 0.9]))
    else:
        n = _log_int(rng, 1, 2048)
        r = rng.choice([(1, 255), (PAGE, PAGE), (n % 255 + 1, n % 255 + 1)])
        hd = rng.choice([32, 64, 128])
        f16 = rng.random() < 0.5
        if not f16 and hd == 128:
            n = min(n, 1024)
        c = _pages("", hd, f16, n, 2 * n + rng.randrange(1, 500), r[0], r[1], rng.randrange(1 << 30))
    del c["name"]
    return c


def _lens(case):
    """(new tokens, cache length) of each session, from the case alone."""
    rng = random.Random(case["lens_seed"])
    out = []
    for _ in range(case["seqs"]):
        nq = rng.randint(case["q_min"], case["q_max"])
        out.append((nq, max(nq, rng.randint(case["kv_min"], case["kv_max"]))))
    return out


def _copies(case):
    """(source page, destination page, rows) of each copy, from the case alone."""
    rng = random.Random(case["lens_seed"])
    ids = list(range(case["pool"]))
    rng.shuffle(ids)
    n = case["n"]
    rows = [rng.randint(case["rows_min"], case["rows_max"]) for _ in range(n)]
    return ids[:n], ids[n:2 * n], rows


def work(case):
    if case["op"] == "attention":
        es = 2 if case["f16"] else 4
        lens = _lens(case)
        width = case["heads"] * case["hd"]
        tokens = sum(q for q, _ in lens)
        keys = sum(k for _, k in lens)
        pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in lens)
        return {"bytes": 2 * tokens * width * 4 + keys * case["heads_kv"] * 2 * case["hd"] * es,
                "flops": 4 * width * pairs}
    if case["op"] == "logprobs":
        r = case["rows"]
        return {"bytes": r * case["vocab"] * 4 + r * (16 + 8 * case["top_k"]), "flops": 5 * r * case["vocab"]}
    es = 2 if case["f16"] else 4
    return {"bytes": 2 * sum(_copies(case)[2]) * 2 * case["hd"] * es, "flops": 0}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_attention(case, seed):
    g = _gen(seed)
    heads, hk, hd = case["heads"], case["heads_kv"], case["hd"]
    lens = _lens(case)
    total = sum(q for q, _ in lens)
    pps = max(1, max(-(-k // PAGE) for _, k in lens))
    need = sum(-(-k // PAGE) for _, k in lens) * hk
    n_pages = need + 3
    dt = torch.float16 if case["f16"] else torch.float32
    pool = torch.empty(n_pages, PAGE, 2, hd, dtype=dt, device="cuda")
    for a in range(0, n_pages, 512):  # K and V rows
        b = min(n_pages, a + 512)
        pool[a:b] = torch.randn(b - a, PAGE, 2, hd, generator=g, device="cuda")
    q = torch.randn(total, heads, hd, generator=g, device="cuda") * 1.3
    # pages handed out in the order a shared pool would: scattered
    perm = np.random.RandomState(seed % (1 << 31)).permutation(n_pages)[:need]
    table = np.zeros((case["seqs"], hk, pps), np.int32)
    at = 0
    for s, (_, k) in enumerate(lens):
        n = -(-k // PAGE)
        table[s, :, :n] = perm[at:at + hk * n].reshape(hk, n)
        at += hk * n
    nq = [a for a, _ in lens]
    q0 = np.concatenate([[0], np.cumsum(nq)[:-1]])
    st = {"case": case, "pool": pool, "q": q, "table": torch.from_numpy(table).cuda(), "nq": _ints(nq),
          "kv": _ints([k for _, k in lens]), "q0": _ints(q0), "max_q": max(nq),
          "max_kv": max(k for _, k in lens),
          # session and place in its chunk of each row
          "row_seq": torch.from_numpy(np.repeat(np.arange(case["seqs"]), nq)).cuda(),
          "row_tok": torch.from_numpy(np.concatenate([np.arange(a) for a in nq])).cuda(), "out": torch.empty(total, heads, hd, device="cuda")}
    if own:
        l3g = _l3g()
        st["op"] = l3g.ChunkAttention(heads, hk, hd, l3g.L3G_KV_F16 if case["f16"] else l3g.L3G_KV_F32)
        seqs = l3g.chunk_seqs(case["seqs"])
        seqs["pool"] = pool.data_ptr()
        seqs["n_pages"] = n_pages
        seqs["pages"] = st["table"].data_ptr() + np.arange(case["seqs"], dtype=np.uint64) * (hk * pps * 4)
        seqs["pps"] = pps
        seqs["q0"], seqs["n_q"], seqs["kv_len"] = q0, nq, [k for _, k in lens]
        st["seqs"] = torch.from_numpy(seqs.view(np.uint8)).cuda()
    return st


def _prepare_logprobs(case, seed):
    g = _gen(seed)
    n, v = case["rows"], case["vocab"]
    x = torch.randn(n, v, generator=g, device="cuda") * 2.5
    top = torch.randint(0, v, (n, 8), generator=g, device="cuda")  # a few likely tokens per row
    x.scatter_add_(1, top, torch.rand(n, 8, generator=g, device="cuda") * 10)
    target = top[:, 0].clone()
    if case["masked"]:
        x = x.masked_fill(torch.rand(n, v, generator=g, device="cuda") < case["masked"], -math.inf)
        x.scatter_(1, target[:, None], torch.rand(n, 1, generator=g, device="cuda") * 4)
    st = {"case": case, "logits": x, "target": target.to(torch.int32)}
    k = min(case["top_k"], v)
    f = dict(dtype=torch.float32, device="cuda")
    i = dict(dtype=torch.int32, device="cuda")
    st["out"] = {"logprob": torch.empty(n, **f), "entropy": torch.empty(n, **f), "rank": torch.empty(n, **i),
                 "top_ids": torch.empty(n, k, **i), "top_logprobs": torch.empty(n, k, **f)}
    if own:
        st["op"] = _l3g().LogProbs(n, v)
    return st


def _prepare_pages(case, seed):
    g = _gen(seed)
    dt = torch.float16 if case["f16"] else torch.float32
    pool = torch.empty(case["pool"], PAGE, 2 * case["hd"], dtype=dt, device="cuda")
    for a in range(0, case["pool"], 512):
        b = min(case["pool"], a + 512)
        pool[a:b] = torch.randn(b - a, PAGE, 2 * case["hd"], generator=g, device="cuda")
    src, dst, rows = _copies(case)
    if own:
        _l3g().lib()
    return {"case": case, "pool": pool, "src": _ints(src), "dst": _ints(dst), "rows": _ints(rows)}


def prepare(case, seed):
    return {"attention": _prepare_attention, "logprobs": _prepare_logprobs, "pages": _prepare_pages}[case["op"]](
        case, seed)


def _plain_attention(st):
    c = st["case"]
    hk, hd, G = c["heads_kv"], c["hd"], c["heads"] // c["heads_kv"]
    n, mq, mk = c["seqs"], st["max_q"], st["max_kv"]
    pos = torch.arange(mk, device="cuda")
    # every session's keys and values, padded to the longest: [n][hk][mk][hd]
    page = st["table"].long()[:, :, pos // PAGE]
    rows = st["pool"][page, pos % PAGE].float()
    k, v = rows[..., 0, :], rows[..., 1, :]
    v = torch.where((pos < st["kv"][:, None])[:, None, :, None], v, 0.0)
    tok = torch.arange(mq, device="cuda")
    at = (st["q0"][:, None] + tok).clamp(max=st["q"].shape[0] - 1).long()
    q = st["q"][at].reshape(n, mq, hk, G, hd).permute(0, 2, 3, 1, 4).reshape(n, hk, G * mq, hd)
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    last = (st["kv"] - st["nq"])[:, None] + tok  # the last key each token sees
    see = pos <= last[..., None]
    s = torch.where(see[:, None, None], s.reshape(n, hk, G, mq, mk), -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(n, hk, G * mq, mk), v).reshape(n, hk, G, mq, hd)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, mq, c["heads"], hd)
    return o[st["row_seq"], st["row_tok"]]


def _plain_logprobs(st):
    x, t = st["logits"], st["target"].long()[:, None]
    k = min(st["case"]["top_k"], st["case"]["vocab"])
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    S = e.sum(-1, keepdim=True)
    xt = x.gather(1, t)
    ids = torch.arange(x.shape[1], device="cuda")
    before = (x > xt) | ((x == xt) & (ids < t))
    ent = torch.log(S) - torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / S
    if k:
        val, at = torch.sort(x, dim=-1, descending=True, stable=True)
        val, at = val[:, :k], at[:, :k]
    else:
        val, at = x[:, :0], ids[:0].expand(x.shape[0], 0)
    return {"logprob": (xt - m - torch.log(S))[:, 0], "entropy": ent[:, 0],
            "rank": before.sum(-1).to(torch.int32), "top_ids": at.to(torch.int32),
            "top_logprobs": val - m - torch.log(S)}


def _plain_pages(st):
    pool, src, dst = st["pool"], st["src"].long(), st["dst"].long()
    keep = torch.arange(PAGE, device="cuda") < st["rows"][:, None]
    pool[dst] = torch.where(keep[..., None], pool[src], pool[dst])
    return pool


def _own_attention(st):
    stream = torch.cuda.current_stream().cuda_stream
    c, q, out = st["case"], st["q"], st["out"]
    st["op"].run(st["seqs"].data_ptr(), c["seqs"], q.shape[0], q.data_ptr(), q.stride(0), out.data_ptr(),
                 out.stride(0), stream=stream)
    return out


def _own_logprobs(st):
    stream = torch.cuda.current_stream().cuda_stream
    x, o = st["logits"], st["out"]
    st["op"].run(x.data_ptr(), x.stride(0), x.shape[0], st["target"].data_ptr(), o["logprob"].data_ptr(),
                 o["entropy"].data_ptr(), o["rank"].data_ptr(), o["top_ids"].shape[1], o["top_ids"].data_ptr(),
                 o["top_logprobs"].data_ptr(), stream=stream)
    return o


def _own_pages(st):
    stream = torch.cuda.current_stream().cuda_stream
    pool = st["pool"]
    row_bytes = pool.stride(1) * pool.element_size()
    _l3g().kv_copy_pages(pool.data_ptr(), pool.shape[0], pool.data_ptr(), pool.shape[0], row_bytes,
                         st["src"].data_ptr(), st["dst"].data_ptr(), st["rows"].data_ptr(), st["src"].shape[0],
                         stream=stream)
    return pool


def run(st):
    if own:
        return {"attention": _own_attention, "logprobs": _own_logprobs, "pages": _own_pages}[st["case"]["op"]](st)
    return {"attention": _plain_attention, "logprobs": _plain_logprobs, "pages": _plain_pages}[st["case"]["op"]](st)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        # session by session, kv head by kv head, from the definition
        hk, hd, G = case["heads_kv"], case["hd"], case["heads"] // case["heads_kv"]
        out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
        row = 0
        for s, (nq, kv) in enumerate(_lens(case)):
            j = torch.arange(kv, device="cuda")
            hidden = j[None, :] > (kv - nq + torch.arange(nq, device="cuda"))[:, None]
            for h in range(hk):
                cells = st["pool"][st["table"][s, h].long()].reshape(-1, 2, hd)[:kv].double()
                for g in range(G):
                    qs = st["q"][row:row + nq, h * G + g].double()
                    w = torch.softmax((qs @ cells[:, 0].T / math.sqrt(hd)).masked_fill(hidden, -math.inf), 1)
                    out[row:row + nq, h * G + g] = w @ cells[:, 1]
            row += nq
        return out
    if case["op"] == "logprobs":
        o = {k: torch.empty(v.shape, dtype=torch.float64 if v.is_floating_point() else v.dtype, device="cuda")
             for k, v in st["out"].items()}
        k = o["top_ids"].shape[1]
        for r in range(case["rows"]):
            x = st["logits"][r].double()
            t = int(st["target"][r])
            lp = torch.log_softmax(x, 0)
            order = torch.argsort(x, descending=True, stable=True)
            o["logprob"][r] = lp[t]
            o["entropy"][r] = torch.special.entr(lp.exp()).sum()
            o["rank"][r] = (order == t).nonzero()[0, 0]
            o["top_ids"][r] = order[:k]
            o["top_logprobs"][r] = lp[order[:k]]
        return o
    want = st["pool"].clone()
    for a, b, n in zip(*_copies(case)):
        want[b, :n] = st["pool"][a, :n]
    return want.double()
