"""The operators of speculative decoding over the paged K/V cache, as cases to time:
attention of a drafted token tree (three row formats), log probabilities of given
tokens with entropy and top alternatives, and keeping the accepted nodes' rows.

Head shapes, windows and vocabularies are those of spkv.SHAPES; the cache is the
library's: pages of 64 positions, [K, V][kv head][position][row].  `run` computes
the operators in elementary torch operations, or, where `own` is true, calls the
library on the same memory.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 64
# q heads, kv heads, head dim, sliding window of the window layers, layers
SHAPES = {
    "qwen3-0.6b": (16, 8, 128, 0, 28),
    "qwen3-8b": (32, 8, 128, 0, 36),
    "gemma3-12b": (16, 8, 256, 1024, 48),
}
VOCABS = {"qwen3": 151936, "gemma3": 262144}
REWIND = 128                     # positions a window layer's ring keeps behind its window
DEV = "cuda"


def listed():
    return [
        # a draft of one token behind a short question: nothing but latency
        dict(name="tree 0.6b 1 node at 100", op="tree", shape="qwen3-0.6b", rows="f32", window=0, seqs=1, lo=100, hi=100, nlo=1, nhi=1),
        # a chat with a usual draft tree, four q heads per kv head
        dict(name="tree 8b 24 nodes at 4k", op="tree", shape="qwen3-8b", rows="f32", window=0, seqs=1, lo=4095, hi=4095, nlo=24, nhi=24),
        # a server's step: ragged sessions, each with its own tree
        dict(name="tree 8b 16 sessions", op="tree", shape="qwen3-8b", rows="f32", window=0, seqs=16, lo=256, hi=4096, nlo=3, nhi=17),
        # the headline context with a wide tree
        dict(name="tree 12b 64 nodes at 32k", op="tree", shape="gemma3-12b", rows="f32", window=0, seqs=1, lo=32703, hi=32703, nlo=64, nhi=64),
        # the same model's window layers, K/V in a ring of pages
        dict(name="tree 12b window 33 nodes", op="tree", shape="gemma3-12b", rows="f32", window=1024, seqs=1, lo=6001, hi=6001, nlo=33, nhi=33),
        # a session with the compressed K/V codec
        dict(name="tree 12b spinor 16 at 6k", op="tree", shape="gemma3-12b", rows="spinor", window=0, seqs=1, lo=6001, hi=6001, nlo=16, nhi=16),
        # exact arithmetic: a chain of seven guesses
        dict(name="tree 0.6b exact 7 at 4k", op="tree", shape="qwen3-0.6b", rows="exact", window=0, seqs=1, lo=4095, hi=4095, nlo=7, nhi=7),
        # ... and the headline context
        dict(name="tree 12b exact 48 at 32k", op="tree", shape="gemma3-12b", rows="exact", window=0, seqs=1, lo=32703, hi=32703, nlo=48, nhi=48),
        # one sampled token's log probability and its alternatives
        dict(name="logprob 1 row of 151936", op="logprob", vocab="qwen3", rows=1, given=1, top=5),
        # every node of a wide tree, its children's tokens given
        dict(name="logprob 64 rows of 262144", op="logprob", vocab="gemma3", rows=64, given=4, top=20),
        # one session accepts a path of five in all 48 layers
        dict(name="keep 12b 5 of 64", op="keep", shape="gemma3-12b", seqs=1, lo=32703, hi=32703, nodes=64, keep=5),
        # a server's step accepts in every session
        dict(name="keep 8b 16 sessions", op="keep", shape="qwen3-8b", seqs=16, lo=256, hi=4096, nodes=17, keep=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "logprob", "keep"])
    if op == "logprob":
        return dict(op=op, vocab=rng.choice(sorted(VOCABS)), rows=_log_int(rng, 1, 128), given=rng.randint(0, 6), top=rng.randint(0, 20))
    shape = rng.choice(sorted(SHAPES))
    if op == "keep":
        seqs, nodes = _log_int(rng, 1, 16), _log_int(rng, 2, 64)
        lo = _log_int(rng, 1, 4096)
        return dict(op=op, shape=shape, seqs=seqs, lo=lo, hi=lo + _log_int(rng, 1, 300), nodes=nodes, keep=rng.randint(1, min(nodes, 12)))
    rows, nhi = rng.choice(["f32", "f32", "spinor", "exact"]), _log_int(rng, 1, 64)
    seqs = rng.choice([1, 1, _log_int(rng, 2, 16)])
    lo = _log_int(rng, 1, 32000 if seqs == 1 else 2048)
    window = SHAPES[shape][3] if rng.random() < 0.4 else 0
    # no dearer than the longest listed tree, and spans of a few hundred in a batch
    if rows != "f32" or SHAPES[shape][0] > 16:
        nhi = min(nhi, 32)
    if seqs > 1:
        nhi = min(nhi, 24)
    return dict(op=op, shape=shape, rows=rows, window=window, seqs=seqs, lo=lo, hi=lo + (0 if seqs == 1 else _log_int(rng, 1, 2048)),
                nlo=rng.randint(1, nhi), nhi=nhi)


# ---------------------------------------------------------------- inputs
def _sizes(what, lo, hi, n):
    """n sizes of [lo, hi], the case's own: outputs have one shape whatever the seed."""
    return np.random.default_rng([what, lo, hi, n]).integers(lo, hi + 1, n)


def _row_format(rows, hd):
    """Spinor rows: hd int8 codes, one f32 multiplier per chunk of at most 55, padded to 16 bytes."""
    nb = -(-hd // 55)
    return nb, (hd + 4 * nb + 15) // 16 * 16


def _chunk_of(hd):
    """The chunk of each coordinate: the first hd % nb chunks are one longer."""
    nb = -(-hd // 55)
    base, extra = hd // nb, hd % nb
    return np.repeat(np.arange(nb), [base + (b < extra) for b in range(nb)])


def _pages(g, cached, nodes, ring, extra=0):
    """Page numbers [sequence][slot] of every sequence's positions, in shuffled order."""
    need = [-(-int(c + n) // PAGE) for c, n in zip(cached, nodes)]
    need = [min(n, ring) if ring else n for n in need]
    table = np.zeros((len(need), max(need) if not ring else ring), np.int64)
    order = g.permutation(sum(need) + extra)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, len(order)


def prepare(case, seed):
    g = np.random.default_rng([seed & 0x7FFFFFFF, 5])
    gen = torch.Generator(DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    def put(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)

    st = dict(case=case, plan=None)
    if case["op"] == "logprob":
        V, R = VOCABS[case["vocab"]], case["rows"]
        x = randn(R, V) * 2.5
        hot = torch.randint(0, V, (R, 24), generator=gen, device=DEV)
        x.scatter_add_(1, hot, 6 + 2 * randn(R, 24))             # a model's few likely tokens
        x[:, V - 267:] = -math.inf                               # entries of a padded vocabulary
        st["logits"] = x
        st["given"] = torch.randint(0, V - 267, (R, case["given"]), generator=gen, device=DEV, dtype=torch.int32)
        st["scale"] = float(np.float32(1 / 0.8))
        return st
    NH, NKV, HD, _, layers = SHAPES[case["shape"]]
    S = case["seqs"]
    cached = _sizes(1, case["lo"], case["hi"], S)
    if case["op"] == "keep":
        nodes = np.full(S, case["nodes"])
        tables = [_pages(g, [c % PAGE for c in cached], nodes, 0) for _ in range(layers)]
        base = np.cumsum([0] + [n for _, n in tables])
        page = np.stack([t + b for (t, _), b in zip(tables, base)])              # [layer][seq][page of the tree's positions]
        keep = np.stack([np.concatenate([[0], 1 + np.sort(g.permutation(case["nodes"] - 1)[:case["keep"] - 1])]) for _ in range(S)])
        st.update(pool=randn(int(base[-1]), 2, NKV, PAGE, HD), page=put(page), keep=put(keep.astype(np.int32)),
                  base=put((cached % PAGE).astype(np.int32)), start=put((np.arange(S + 1) * case["keep"]).astype(np.int32)),
                  seq=put(np.tile(np.arange(S), layers).astype(np.int32)))
        st["tables"] = st["pool"].data_ptr() + st["page"] * (2 * NKV * PAGE * HD * 4)     # page addresses
        st["lists"] = st["tables"].data_ptr() + 8 * page.shape[2] * torch.arange(layers * S, device=DEV)
        return st
    nodes = _sizes(2, case["nlo"], case["nhi"], S)
    ring = -(-(case["window"] + REWIND) // PAGE) + 1 if case["window"] else 0
    table, n_pages = _pages(g, cached, nodes, ring)
    n = int(nodes.sum())
    start = np.concatenate([[0], np.cumsum(nodes)])
    # node 0 is the last accepted token; each other node hangs below one of the few before it
    words = (int(nodes.max()) + 63) // 64
    mask, depth = np.zeros((n, words), np.uint64), np.zeros(n, np.int32)
    for s in range(S):
        for j in range(int(nodes[s])):
            i = start[s] + j
            if j:
                up = start[s] + int(g.integers(max(0, (j - 1) // 3 - 1), max(1, (j + 2) // 2)))
                mask[i], depth[i] = mask[up], depth[up] + 1
            mask[i, j // 64] |= np.uint64(1 << (j % 64))
    if case["rows"] == "spinor":
        nb, rb = _row_format("spinor", HD)
        pool = torch.zeros(n_pages, 2, NKV, PAGE, rb, dtype=torch.uint8, device=DEV)
        codes = (randn(n_pages, 2, NKV, PAGE, HD) * 40).round_().clamp_(-127, 127).to(torch.int8)
        pool[..., :HD] = codes.view(torch.uint8)
        scale = 0.02 + 0.01 * torch.rand(n_pages, 2, NKV, PAGE, nb, generator=gen, device=DEV)
        pool[..., HD:HD + 4 * nb] = scale.view(torch.uint8)
    else:
        pool = randn(n_pages, 2, NKV, PAGE, HD)
        if case["rows"] == "exact":
            pool = (pool * 65536).round_().to(torch.int32)
    st.update(pool=pool, page=put(table), cached=put(cached.astype(np.int32)), start=put(start.astype(np.int32)), depth=put(depth),
              mask=put(mask.view(np.int64)), q=randn(n, NH, HD), max_nodes=int(nodes.max()), max_positions=int((cached + nodes).max()),
              ring=ring, seq=put(np.repeat(np.arange(S), nodes)), node=put(np.concatenate([np.arange(k) for k in nodes])),
              out=torch.empty(n, NH, HD, device=DEV))
    st["tables"] = pool.data_ptr() + st["page"] * (pool[0].numel() * pool.element_size())
    st["lists"] = st["tables"].data_ptr() + 8 * table.shape[1] * torch.arange(S, device=DEV)
    return st


# ---------------------------------------------------------------- plain forms
def _span(st):
    """First position and length of the positions gathered (window layers: the ring's reach)."""
    W = st["case"]["window"]
    if not W:
        return torch.zeros_like(st["cached"]), st["max_positions"]
    return (st["cached"] - (W - 1)).clamp(min=0), min(st["max_positions"], W - 1 + st["max_nodes"])


def _tree_plain(st):
    c, q = st["case"], st["q"]
    NH, NKV, HD, _, _ = SHAPES[c["shape"]]
    S, N, G = c["seqs"], st["max_nodes"], NH // NKV
    first, n = _span(st)
    pos = first.long()[:, None] + torch.arange(n, device=DEV)                     # [S, n]
    slot = pos // PAGE % st["ring"] if st["ring"] else pos // PAGE
    page = st["page"].gather(1, slot.clamp(max=st["page"].shape[1] - 1))
    rows = st["pool"][page, :, :, pos % PAGE]                                     # [S, n, 2, NKV, row]
    if c["rows"] == "spinor":
        nb, rb = _row_format("spinor", HD)
        mul = rows[..., HD:HD + 4 * nb].contiguous().view(torch.float32)
        chunk = torch.from_numpy(_chunk_of(HD)).to(DEV)
        rows = rows[..., :HD].contiguous().view(torch.int8).float() * mul[..., chunk]
    k, v = rows[:, :, 0].transpose(1, 2).contiguous(), rows[:, :, 1].transpose(1, 2).contiguous()   # [S, NKV, n, HD]
    qp = q.new_zeros(S, N, NH, HD)
    qp[st["seq"], st["node"]] = q
    qp = qp.view(S, N, NKV, G, HD).transpose(1, 2).reshape(S, NKV, N * G, HD)
    # what node i of sequence s sees
    low = (st["cached"].long()[st["seq"]] + st["depth"] - c["window"] + 1) if c["window"] else torch.zeros_like(st["seq"])
    p, cached = pos[st["seq"]], st["cached"].long()[st["seq"], None]
    tail = (p - cached).clamp(min=0)
    inside = tail < (st["start"][1:] - st["start"][:-1]).long()[st["seq"], None]
    bit = st["mask"].gather(1, (tail // 64).clamp(max=st["mask"].shape[1] - 1)) >> (tail % 64) & 1
    see = torch.where(p < cached, p >= low[:, None], inside & (bit == 1))
    seen = torch.zeros(S, N, n, dtype=torch.bool, device=DEV)
    seen[st["seq"], st["node"]] = see
    seen = seen[:, None, :, None].expand(S, NKV, N, G, n).reshape(S, NKV, N * G, n)
    scale = float(np.float32(1) / np.sqrt(np.float32(HD)))
    if c["rows"] == "exact":
        o = _exact_weights(torch.round(qp * 65536).double(), k, v, seen, scale)
    else:
        s = (qp @ k.transpose(2, 3)) * scale
        s = s.masked_fill(~seen, -math.inf)
        m = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
        o = (w @ v) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(S, NKV, N, G, HD).transpose(1, 2).reshape(S, N, NH, HD)
    return o[st["seq"], st["node"]]


# round((ln 2)^k / k! 2^30): 2^f on a 30-bit grid
_EXP = [1073741824, 744261118, 257941248, 59597083, 10327387, 1431680, 165394]
_LOG2E = 1549082005


def _exact_weights(qi, ki, vi, seen, scale):
    """The integer attention: scores on a grid of 2^-14, weights of 22 bits, in 64 bits throughout."""
    ip = qi @ ki.double().transpose(2, 3)                         # integers below 2^53
    z = (ip / 4294967296.0).float() * scale
    z = z.double() * 16384
    z = torch.trunc(z + torch.where(z < 0, -0.5, 0.5)).long()
    top = z.masked_fill(~seen, -(1 << 40)).amax(-1, keepdim=True)
    d = (top - z).clamp(0, 1 << 19)
    e = (d * _LOG2E + 16383) >> 14
    n, r = e >> 30, e & 1073741823
    f = 1073741824 - r
    acc = torch.full_like(f, _EXP[6])
    acc = (acc * f >> 30) + _EXP[5]
    acc = (acc * f >> 30) + _EXP[4]
    acc = (acc * f >> 30) + _EXP[3]
    acc = (acc * f >> 30) + _EXP[2]
    acc = (acc * f >> 30) + _EXP[1]
    acc = (acc * f >> 30) + _EXP[0]
    w = torch.where(r > 0, acc >> (n + 1).clamp(max=63), 1073741824 >> n.clamp(max=63)) >> 8
    w = w.masked_fill(~seen | (n >= 32), 0)
    wd = w.double()
    hi = vi.double().div(4096).floor()
    lo = vi.double() - hi * 4096
    num = (wd @ hi) * 4096 + wd @ lo
    return (num / (wd.sum(-1, keepdim=True).clamp(min=1) * 65536)).float()


def _logprob_plain(st):
    x, c = st["logits"], st["case"]
    y = x * st["scale"]
    m = y.amax(1, keepdim=True)
    # 1 + others: the sum beside its largest term, which 32 bits would swallow where a row is sure of a token
    d = (y - m).clamp(min=-200.0)
    e = torch.where(d < 0, torch.exp(d), torch.zeros_like(d))
    others = e.sum(1, keepdim=True) + ((d == 0).sum(1, keepdim=True) - 1)
    lse = m + torch.log1p(others)
    ent = torch.log1p(others) - (e * d).sum(1, keepdim=True) / (1 + others)
    given = y.gather(1, st["given"].long()) - lse
    # the value's order in the high bits, the lower index first among equals
    bits = (x + 0.0).view(torch.int32)                            # one zero
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = (order << 32) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=DEV))
    ids = (x.shape[1] - 1) - (torch.topk(key, c["top"], dim=1).values & 0xFFFFFFFF)
    return dict(given=given, entropy=ent[:, 0], lse=lse[:, 0], top_ids=ids.int(), top=y.gather(1, ids) - lse)


def _keep_plain(st):
    pool, page = st["pool"], st["page"]                           # page: [layer][seq][page]
    n = st["keep"].shape[1]
    src = st["base"].long()[:, None] + st["keep"]
    dst = st["base"].long()[:, None] + torch.arange(n, device=DEV)
    seq = torch.arange(page.shape[1], device=DEV)[:, None]
    rows = pool[page[:, seq, src // PAGE], :, :, src % PAGE]      # [layer][seq][kept][2][kv head][row]
    pool[page[:, seq, dst // PAGE], :, :, dst % PAGE] = rows
    return pool


# ---------------------------------------------------------------- the library's
def _spkv():
    if "spkv" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "shannon-prime-system_amd"))
    import spkv
    return spkv


def _plan(st):
    """The argument block and the buffers that a program keeps for its calls."""
    spkv, c = _spkv(), st["case"]
    if c["op"] == "logprob":
        R, V = st["logits"].shape
        f = dict(device=DEV, dtype=torch.float32)
        st["outs"] = dict(given=torch.empty(R, c["given"], **f), entropy=torch.empty(R, **f), lse=torch.empty(R, **f),
                          top_ids=torch.empty(R, c["top"], device=DEV, dtype=torch.int32), top=torch.empty(R, c["top"], **f))
        o = st["outs"]
        a = spkv.LogprobArgs(n_rows=R, vocab=V, n_given=c["given"], n_top=c["top"], scale=st["scale"], logits=st["logits"].data_ptr(), stride=V,
                             given=st["given"].data_ptr(), given_logprob=o["given"].data_ptr(), entropy=o["entropy"].data_ptr(),
                             lse=o["lse"].data_ptr(), top_ids=o["top_ids"].data_ptr(), top_logprob=o["top"].data_ptr())
        need = spkv.token_logprobs_work(a)
    elif c["op"] == "keep":
        _, NKV, HD, _, layers = SHAPES[c["shape"]]
        a = spkv.KeepArgs(n_kv_heads=NKV, row_bytes=4 * HD, n_tables=layers * c["seqs"], n_seqs=c["seqs"], max_keep=c["keep"],
                          max_positions=PAGE + c["nodes"], tables=st["lists"].data_ptr(), seq=st["seq"].data_ptr(), ring_pages=None,
                          cached=st["base"].data_ptr(), keep_start=st["start"].data_ptr(), keep=st["keep"].data_ptr())
        need = 0
    else:
        NH, NKV, HD, _, _ = SHAPES[c["shape"]]
        rows = dict(f32=spkv.ROWS_F32, exact=spkv.ROWS_EXACT, spinor=spkv.ROWS_SPINOR)[c["rows"]]
        a = spkv.TreeArgs(n_heads=NH, n_kv_heads=NKV, head_dim=HD, rows=rows, n_seqs=c["seqs"], n_nodes=st["q"].shape[0],
                          max_nodes=st["max_nodes"], max_positions=st["max_positions"], window=c["window"], ring_pages=st["ring"],
                          mask_words=st["mask"].shape[1], scale=float(np.float32(1) / np.sqrt(np.float32(HD))),
                          node_start=st["start"].data_ptr(), cached=st["cached"].data_ptr(), depth=st["depth"].data_ptr(),
                          visible=st["mask"].data_ptr(), tables=st["lists"].data_ptr(), q=st["q"].data_ptr(), q_stride=NH * HD,
                          out=st["out"].data_ptr(), out_stride=NH * HD)
        need = spkv.tree_attention_work(a)
    if need:
        st["work"] = torch.empty(need, dtype=torch.uint8, device=DEV)
        a.work, a.work_bytes = st["work"].data_ptr(), need
    st["plan"] = (spkv, a)


def run(st):
    op = st["case"]["op"]
    if not own:
        return _tree_plain(st) if op == "tree" else _logprob_plain(st) if op == "logprob" else _keep_plain(st)
    if st["plan"] is None:
        _plan(st)
    spkv, a = st["plan"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "tree":
        spkv.tree_attention(a, stream)
        return st["out"]
    if op == "logprob":
        spkv.token_logprobs(a, stream)
        return st["outs"]
    spkv.keep_rows(a, stream)
    return st["pool"]


def work(case):
    """Each input read once, each output written once; sequences and trees of middling size."""
    if case["op"] == "logprob":
        V, R = VOCABS[case["vocab"]], case["rows"]
        return dict(bytes=4.0 * R * (V + 2 * case["given"] + 2 * case["top"] + 2), flops=4.0 * R * V)
    NH, NKV, HD, _, layers = SHAPES[case["shape"]]
    if case["op"] == "keep":
        return dict(bytes=2.0 * case["seqs"] * layers * case["keep"] * 2 * NKV * HD * 4, flops=0.0)
    nodes, n = (case["nlo"] + case["nhi"]) / 2, (case["lo"] + case["hi"]) / 2
    if case["window"]:
        n = min(n, case["window"])
    row = 4 * HD if case["rows"] != "spinor" else HD + 4 * _row_format("spinor", HD)[0]
    return dict(bytes=case["seqs"] * (2.0 * NKV * (n + nodes) * row + 8.0 * nodes * NH * HD), flops=4.0 * case["seqs"] * nodes * NH * HD * (n + nodes / 2))


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprob":
        y = st["logits"].double() * st["scale"]
        p = torch.softmax(y, 1)
        lse = torch.logsumexp(y, 1)
        ent = -(torch.special.xlogy(p, p)).sum(1)
        ids = torch.sort(st["logits"], dim=1, descending=True, stable=True).indices[:, :case["top"]]
        return dict(given=y.gather(1, st["given"].long()) - lse[:, None], entropy=ent, lse=lse, top_ids=ids.int(), top=y.gather(1, ids) - lse[:, None])
    if case["op"] == "keep":
        pool, page = st["pool"], st["page"].cpu().numpy()
        keep, base = st["keep"].cpu().numpy(), st["base"].cpu().numpy()
        for layer in page:
            for s in range(case["seqs"]):
                for i, j in enumerate(keep[s]):                    # ascending: a row is read before it is written over
                    a, b = int(base[s] + j), int(base[s] + i)
                    pool[layer[s, b // PAGE], :, :, b % PAGE] = pool[layer[s, a // PAGE], :, :, a % PAGE].clone()
        return pool.double()
    NH, NKV, HD, _, _ = SHAPES[case["shape"]]
    G, W = NH // NKV, case["window"]
    start, cached = st["start"].tolist(), st["cached"].tolist()
    depth, mask = st["depth"].tolist(), st["mask"].cpu().numpy().view(np.uint64)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    scale = float(np.float32(1) / np.sqrt(np.float32(HD)))
    for s in range(case["seqs"]):
        nodes = start[s + 1] - start[s]
        n = cached[s] + nodes
        lo = max(0, cached[s] - W + 1) if W else 0
        pos = torch.arange(lo, n, device=DEV)
        slot = pos // PAGE % st["ring"] if st["ring"] else pos // PAGE
        rows = st["pool"][st["page"][s][slot], :, :, pos % PAGE]                # [n, 2, NKV, row]
        if case["rows"] == "spinor":
            nb, _ = _row_format("spinor", HD)
            mul = rows[..., HD:HD + 4 * nb].contiguous().view(torch.float32)
            code = rows[..., :HD].contiguous().view(torch.int8)
            rows = torch.cat([code[..., torch.from_numpy(_chunk_of(HD) == b).to(DEV)].double() * mul[..., b:b + 1].double() for b in range(nb)], -1)
        for j in range(nodes):
            i = start[s] + j
            sees = [b for b in range(nodes) if int(mask[i, b // 64]) >> (b % 64) & 1]
            first = max(0, cached[s] + depth[i] - W + 1) if W else 0
            at = torch.cat([torch.arange(first - lo, cached[s] - lo, device=DEV), torch.tensor(sees, device=DEV, dtype=torch.long) + cached[s] - lo])
            r = rows[at]
            for h in range(NH):
                k, v = r[:, 0, h // G], r[:, 1, h // G]
                if case["rows"] == "exact":
                    out[i, h] = _exact_row(torch.round(st["q"][i, h] * 65536).long(), k.long(), v.long(), scale)
                else:
                    p = torch.softmax(k.double() @ st["q"][i, h].double() * scale, 0)
                    out[i, h] = p @ v.double()
    return out


def _exact_row(q, k, v, scale):
    z = ((k * q).sum(1).double() / 2.0 ** 32).float() * torch.tensor(scale, dtype=torch.float32, device=DEV)
    z = torch.sign(z) * torch.floor(z.abs().double() * 16384 + 0.5)
    steps = z.long().max() - z.long()                              # of 2^-14 below the largest score
    near = steps < 1 << 19                                         # beyond: e^-32 and less, no bit left
    g = -((-steps.clamp(max=1 << 19) * _LOG2E) >> 14)              # powers of two, rounded up, 30 bits of fraction
    n, f = g >> 30, g % (1 << 30)
    t = torch.zeros_like(f) + _EXP[-1]
    for c in _EXP[-2::-1]:
        t = (t * ((1 << 30) - f) >> 30) + c
    w = torch.where(f == 0, torch.full_like(t, 1 << 30) >> n.clamp(0, 60), t >> (n + 1).clamp(0, 60)) >> 8
    w = torch.where(near & (n < 32), w, torch.zeros_like(w))
    return (w[:, None] * v).sum(0).double() / (w.sum() * 65536).double()
