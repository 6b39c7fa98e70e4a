"""Operators of serving within a fixed memory, as cases that can be timed.

  paged   attention of new tokens (one of each sequence, or a piece of a prompt)
          over 4-bit K and V in pages of one pool, which each sequence's table names
          (eakv_attention_paged_device)
  append  K and V of new tokens into those pages (eakv_append_paged_device)
  weights the attention weight that each cached token gets from a window's queries,
          added to what it had before (eakv_attention_weights_batch_device)
  select  which tokens of a full cache stay: the first, the most recent and those of
          most weight (eakv_evict_select_device)
  logprob log probabilities of given tokens, the entropies of their distributions and
          the most likely alternatives (eakv_token_logprobs_device)

Where `own` is false a pass computes the same in elementary torch operations.  A
pool or cache is then three tensors (packed codes, scales, biases: 64 values in 32 bytes
and two floats, byte k holding value k in its low and value k + 32 in its high four
bits); else it is an eakv_amd.Cache of the same values.
"""
import math
import random

import torch

own = False

# q heads, kv heads, head_dim
HEADS = [(8, 8, 128), (32, 4, 64), (32, 32, 128), (32, 8, 128), (64, 8, 128), (40, 8, 128),
         (16, 8, 128), (12, 12, 64)]

# The largest listed case of each kind, which no drawn case exceeds
MOST_FLOPS = 1.36e11
MOST_BYTES = 4.51e8


def listed():
    def paged(name, heads, dtype, seqs, ctx, page, spread=1, new=1, prompts=0):
        return dict(name=name, op="paged", n_q=heads[0], n_kv=heads[1], d=heads[2], dtype=dtype,
                    seqs=seqs, ctx=ctx, spread=spread, page=page, new=new, prompts=prompts)

    def append(name, heads, dtype, seqs, ctx, page, spread=1, new=1, prompts=0):
        return dict(paged(name, heads, dtype, seqs, ctx, page, spread, new, prompts), op="append")

    def weights(name, heads, dtype, seqs, tokens, ctx, spread=1):
        return dict(name=name, op="weights", n_q=heads[0], n_kv=heads[1], d=heads[2], dtype=dtype,
                    seqs=seqs, tokens=tokens, ctx=ctx, spread=spread)

    def select(name, heads, seqs, ctx, keep, spread=1):
        return dict(name=name, op="select", heads=heads, seqs=seqs, ctx=ctx, keep=keep, first=4,
                    recent=min(keep // 4, 256), spread=spread)

    def logprob(name, dtype, rows, vocab, top, allowed=0):
        return dict(name=name, op="logprob", dtype=dtype, rows=rows, vocab=vocab, top=top,
                    allowed=allowed)

    return [
        # one chat's next token at a short context: latency
        paged("paged token x1 2K bf16", (32, 8, 128), "bf16", 1, 2048, 16),
        # a server's decode step, sequences of all lengths
        paged("paged token x64 ragged bf16", (32, 8, 128), "bf16", 64, 16384, 64, 16),
        # a step that decodes 15 sequences beside a piece of a new one's prompt
        paged("paged 512 + 15 tokens f32", (64, 8, 128), "f32", 16, 8200, 32, 4, 512, 1),
        # pieces of four prompts on a small model
        paged("paged 1500 x4 d64 bf16", (32, 4, 64), "bf16", 4, 6001, 16, 4, 1500, 4),
        # the decode step's K and V
        append("append token x64 bf16", (32, 8, 128), "bf16", 64, 4096, 64, 16),
        # a piece of a long prompt
        append("append 4000 x2 f32", (32, 32, 128), "f32", 2, 9001, 16, 1, 4000, 2),
        # one decode step's weights, long contexts
        weights("weights 1 x8 32K f32", (32, 8, 128), "f32", 8, 1, 32768),
        # the last 32 tokens of each prompt vote for the others
        weights("weights 32 x4 ragged bf16", (64, 8, 128), "bf16", 4, 32, 20011, 4),
        # sequences held at a small budget, a token at a time or a few
        select("select 2048 of 2100 x8", 8, 8, 2100, 2048),
        # long prompts reduced once
        select("select 20000 of 131072 x2", 8, 2, 131072, 20000),
        # one chat's token, a small vocabulary
        logprob("logprob x1 32000 f32", "f32", 1, 32000, 5),
        # a prompt's tokens or a batch's, a large vocabulary of odd size
        logprob("logprob x500 151665 bf16", "bf16", 500, 151665, 20),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["paged"] * 4 + ["append"] + ["weights"] * 2 + ["select"] + ["logprob"] * 2)
    n_q, n_kv, d = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "f32"])
    spread = rng.choice([1, 4, 16])
    if op in ("paged", "append"):
        seqs = _log(rng, 1, 128)
        case = dict(op=op, n_q=n_q, n_kv=n_kv, d=d, dtype=dtype, seqs=seqs, ctx=_log(rng, 16, 65536),
                    spread=spread, page=rng.choice([16, 32, 64, 128, 256]), new=_log(rng, 1, 2048))
        case["prompts"] = rng.randint(0, min(seqs, 4))
    elif op == "weights":
        case = dict(op=op, n_q=n_q, n_kv=n_kv, d=d, dtype=dtype, seqs=_log(rng, 1, 32),
                    tokens=rng.choice([1, _log(rng, 1, 256)]), ctx=_log(rng, 16, 131072), spread=spread)
    elif op == "select":
        ctx = _log(rng, 64, 262144)
        keep = rng.randint(16, ctx - 1)
        case = dict(op=op, heads=n_kv * rng.randint(1, 2), seqs=_log(rng, 1, 32), ctx=ctx, keep=keep,
                    first=rng.randint(0, 8), recent=rng.randint(0, keep // 2), spread=spread)
    else:
        vocab = _log(rng, 1000, 200000)
        case = dict(op=op, dtype=dtype, rows=_log(rng, 1, 1024), vocab=vocab, top=rng.randint(0, 32),
                    allowed=rng.choice([0, 0, _log(rng, 2, vocab)]))
    big = "rows" if op == "logprob" else "seqs"
    while work(case)["flops"] > MOST_FLOPS or _held(case) > MOST_BYTES:
        if case[big] > 1:
            case[big] = case[big] * 2 // 3
        elif op == "logprob":
            case["vocab"] = case["vocab"] * 2 // 3
        else:
            case["ctx"] = case["ctx"] * 2 // 3
        if "prompts" in case:
            case["prompts"] = min(case["prompts"], case["seqs"])
        if op == "select":
            case["keep"] = max(16, min(case["keep"], case["ctx"] - 1))
            case["recent"] = min(case["recent"], case["keep"] // 2)
    return case


def _held(case):
    """Bytes that a case's largest buffers have."""
    if case["op"] == "append":
        return 2.0 * sum(a + m for a, m in _lengths(case)) * case["n_kv"] * case["d"] // 64 * 40
    return work(case)["bytes"]


# ---------------------------------------------------------------- the inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _spread(n, ctx, spread, r):
    """Lengths log-uniform from ctx/spread to ctx, one of them ctx."""
    total = [max(1, int(round(ctx * spread ** -r.random()))) for _ in range(n)]
    total[n // 3] = ctx
    return total


def _lengths(case):
    """(tokens before the new ones, new ones) of each sequence.  Where lengths differ a piece
    of a prompt, and a window, is of any length up to the longest."""
    n, ctx, spread = case["seqs"], case["ctx"], case["spread"]
    r = random.Random(n * 1000003 + ctx * 131 + spread)
    total = _spread(n, ctx, spread, r)
    if "tokens" in case:
        most, many = case["tokens"], set(range(n))
    else:
        most, many = case["new"], set((n // 3 + i) % n for i in range(case["prompts"]))
    new = [min(t, most if spread == 1 or i == n // 3 else r.randint(1, most)) if i in many else 1
           for i, t in enumerate(total)]
    return [(t - m, m) for t, m in zip(total, new)]


def _channels(g, n_kv, d):
    """Key channel scales f32[n_kv][1][d]: log-uniform in [0.5, 4], two
    channels of each head ten times larger."""
    c = torch.exp(torch.rand(n_kv, 1, d, generator=g, device="cuda") * math.log(8.0) + math.log(0.5))
    for h in range(n_kv):
        c[h, 0, torch.randperm(d, generator=g, device="cuda")[:2]] *= 10
    return c


def _kv(g, n_kv, tokens, d, chan):
    """K and V f32[2][n_kv][tokens][d], as model states are: K with scales and
    outliers by channel, V normal."""
    x = torch.randn(2, n_kv, tokens, d, generator=g, device="cuda")
    x[0] *= chan
    return x


def _quantize(x):
    """The cache's codes, scales and biases of x [..., d]: groups of 64, bias the
    minimum, scale range/15 (quotients by way of 64 bits, where they are rounded
    once), each step rounded to f32."""
    v = x.unflatten(-1, (x.shape[-1] // 64, 64))
    mn, mx = v.aminmax(dim=-1)
    r = mx - mn
    some = r > 0
    scale = torch.where(some, (r.double() / 15.0).float(), torch.ones_like(r))
    inv = torch.where(some, (15.0 / r.double()).float(), torch.zeros_like(r))
    n = (v - mn[..., None]).mul_(inv[..., None]).add_(0.5).floor_().clamp_(0, 15).to(torch.uint8)
    return ((n[..., 32:] << 4) | n[..., :32]).flatten(-2), scale, mn


def _tables(case, seed):
    """(pages of the pool, i32 tables [seqs][most pages], each sequence's pages): every
    page of the pool named once, in any order, a tenth of them free; places behind a
    sequence's last page are -1."""
    page, lens = case["page"], _lengths(case)
    need = [-(-(a + m) // page) for a, m in lens]
    n_pages = sum(need) + max(1, sum(need) // 10)
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).split(
        need + [n_pages - sum(need)])[:-1]
    return n_pages, torch.nn.utils.rnn.pad_sequence(order, batch_first=True, padding_value=-1).to(
        torch.int32).cuda(), [o.cuda() for o in order]


def _pool(case, seed):
    """The pool's planes [2][n_kv][tokens][...] with every sequence's tokens before (paged:
    and with) its new ones in its pages, the tables, and the generator and channels
    that filled it."""
    g = _gen(seed)
    n_kv, d, page = case["n_kv"], case["d"], case["page"]
    n_pages, tables, pages = _tables(case, seed)
    chan = _channels(g, n_kv, d)
    room = n_pages * page
    planes = (torch.zeros(2, n_kv, room, d // 2, dtype=torch.uint8, device="cuda"),
              torch.zeros(2, n_kv, room, d // 64, device="cuda"),
              torch.zeros(2, n_kv, room, d // 64, device="cuda"))
    for (a, m), p in zip(_lengths(case), pages):
        n = a + (m if case["op"] == "paged" else 0)
        if n:
            at = (p[:, None] * page + torch.arange(page, device="cuda")).flatten()[:n]
            for to, x in zip(planes, _quantize(_kv(g, n_kv, n, d, chan))):
                to[:, :, at] = x
    return planes, tables, g, chan


def _typed(x, case):
    return x.bfloat16() if case["dtype"] == "bf16" else x


def _weights_inputs(case, seed):
    """Each sequence's K and V, then the queries of all windows and the weights so far
    [seqs][n_kv][room]."""
    g = _gen(seed)
    n_kv, d, lens = case["n_kv"], case["d"], _lengths(case)
    chan = _channels(g, n_kv, d)
    for a, m in lens:
        yield _kv(g, n_kv, a + m, d, chan)
    q = torch.randn(sum(m for _, m in lens), case["n_q"], d, generator=g, device="cuda")
    w = torch.rand(case["seqs"], n_kv, case["ctx"], generator=g, device="cuda").pow_(4)
    for i, (a, m) in enumerate(lens):
        w[i, :, a:] = 0.0       # the window's own tokens have none yet
    yield _typed(q, case), w


def _select_inputs(case, seed):
    """Weights f32 [seqs][heads][ctx] of many sizes, tokens that none looked at among them;
    behind a sequence's last token anything."""
    g = _gen(seed)
    shape = case["seqs"], case["heads"], case["ctx"]
    w = torch.exp(2.0 * torch.randn(shape, generator=g, device="cuda"))
    w *= torch.rand(shape[0], 1, shape[2], generator=g, device="cuda") > 0.05
    total = _spread(shape[0], shape[2], case["spread"], random.Random(seed))
    least = case["first"] + case["recent"]
    keep = [min(t, max(1, least, case["keep"] * t // case["ctx"])) for t in total]
    return w, total, keep


def _logprob_inputs(case, seed):
    """Logits of usual size; where `allowed` is set all but some of that many tokens are
    masked.  The given tokens are drawn from the distributions."""
    g = _gen(seed)
    n, v = case["rows"], case["vocab"]
    x = torch.randn(n, v, generator=g, device="cuda").mul_(3.0)
    if case["allowed"]:
        few = torch.rand(n, v, generator=g, device="cuda") * v >= case["allowed"]
        few[:, 0] = False
        x.masked_fill_(few, -math.inf)
    gumbel = torch.empty_like(x).exponential_(generator=g).log_().neg_()
    token = (x + gumbel).argmax(-1).to(torch.int32)
    return _typed(x, case), token


def prepare(case, seed):
    op = case["op"]
    st = dict(case=case)
    if op in ("paged", "append"):
        st["lens"] = lens = _lengths(case)
        planes, st["tables"], g, chan = _pool(case, seed)
        n = sum(m for _, m in lens)
        shape = n, case["n_kv"], case["d"]
        if op == "paged":
            st["q"] = _typed(torch.randn(n, case["n_q"], case["d"], generator=g, device="cuda"), case)
        else:
            x = _kv(g, shape[1], n, shape[2], chan).transpose(1, 2)
            st["new"] = [_typed(x[i].contiguous(), case) for i in (0, 1)]
        first = [0]
        for _, m in lens:
            first.append(first[-1] + m)
        st["first"] = first
        st["d_first"] = torch.tensor(first, dtype=torch.int32, device="cuda")
        st["d_lens"] = torch.tensor([a + m for a, m in lens], dtype=torch.int32, device="cuda")
        st["planes"] = _own_cache(planes) if own else planes
        st["alike"] = [(torch.tensor(some, device="cuda"),
                        torch.tensor([first[i] for i in some], device="cuda"), lens[some[0]][1],
                        sum(lens[some[0]])) for some in _alike(lens)]
    elif op == "weights":
        xs = list(_weights_inputs(case, seed))
        st["q"], st["w"] = xs.pop()
        st["lens"] = _lengths(case)
        st["caches"] = [_own_cache(_quantize(x), case["ctx"]) if own else _quantize(x) for x in xs]
    elif op == "select":
        st["w"], st["total"], st["keep"] = _select_inputs(case, seed)
        st["d_total"] = torch.tensor(st["total"], device="cuda")
        st["d_keep"] = torch.tensor(st["keep"], device="cuda")
    else:
        st["x"], st["token"] = _logprob_inputs(case, seed)
    if own:
        _own_prepare(st)
    return st


# ------------------------------------------------------- one pass, plain form

def _values(w, s, b):
    """f32 [..., d] of codes [..., d/2], scales and biases [..., d/64]."""
    w = w.unflatten(-1, (-1, 32))
    n = torch.cat([w & 15, w >> 4], -1).float()
    return n.mul_(s[..., None]).add_(b[..., None]).flatten(-2)


def _alike(lens):
    """Sequences with equally many new tokens and contexts of about one length, which a
    pass takes as one padded batch."""
    got = []
    for i in sorted(range(len(lens)), key=lambda i: (-lens[i][1], -sum(lens[i]))):
        a, m = lens[i]
        top = lens[got[-1][0]] if got else None
        held = (len(got[-1]) + 1) * sum(top) if got else 0
        if got and top[1] == m and a + m >= 0.75 * sum(top) and held < 1 << 19 and held * m < 1 << 24:
            got[-1].append(i)
        else:
            got.append([i])
    return got


def _paged(st):
    q, out = st["q"], torch.empty_like(st["q"])
    page = st["case"]["page"]
    n_q, d = q.shape[1:]
    for some, first, m, most in st["alike"]:
        at = torch.arange(most, device="cuda")
        table = st["tables"][some].long()
        index = (table[:, at // page] * page + at % page).clamp_(min=0)
        k, v = (_values(*(p[i][:, index] for p in st["planes"])).transpose(0, 1) for i in (0, 1))
        n_kv = k.shape[1]
        rows = first[:, None] + torch.arange(m, device="cuda")
        x = q[rows].float().unflatten(2, (n_kv, -1)).transpose(1, 2).flatten(2, 3)
        s = torch.matmul(x, k.transpose(2, 3).contiguous()).div_(math.sqrt(d))
        seen = st["d_lens"][some][:, None] - m + 1 + torch.arange(m, device="cuda")
        s = s.unflatten(2, (m, -1)).masked_fill_(
            (at >= seen[..., None])[:, None, :, None], -math.inf)
        p = s.sub_(s.amax(-1, keepdim=True)).exp_()
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.flatten(2, 3), v.contiguous()).unflatten(2, (m, -1)).div_(total)
        out[rows] = o.transpose(1, 2).flatten(2, 3).to(q.dtype)
    return out


def _append(st):
    page = st["case"]["page"]
    new = st["d_first"].diff()
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), new,
                                  output_size=st["first"][-1])
    at = torch.arange(st["first"][-1], device="cuda") - st["d_first"][seq] + (st["d_lens"] - new)[seq]
    index = st["tables"][seq, at // page].long() * page + at % page
    for i, x in enumerate(st["new"]):
        for to, y in zip(st["planes"], _quantize(x.float().transpose(0, 1))):
            to[i][:, index] = y
    return st["planes"]


KEEP = 0.96875      # of the weights so far


def _weights(st):
    ms = [m for _, m in st["lens"]]

    def one(cache, q, w, a):
        m, n_q, d = q.shape
        k = _values(*(p[0] for p in cache))
        n_kv, t = k.shape[:2]
        x = q.float().unflatten(1, (n_kv, -1)).transpose(0, 1).flatten(1, 2)
        s = torch.matmul(x, k.transpose(1, 2).contiguous()).div_(math.sqrt(d)).unflatten(1, (m, -1))
        at = torch.arange(m, device="cuda")
        s[..., a:].masked_fill_((at[:, None] < at)[:, None], -math.inf)
        p = s.sub_(s.amax(-1, keepdim=True)).exp_()
        p = p.div_(p.sum(-1, keepdim=True)).sum((1, 2))
        w[:, :t].mul_(KEEP).add_(p)

    [one(c, q, w, a) for c, q, w, (a, _) in zip(st["caches"], st["q"].split(ms), st["w"], st["lens"])]
    return st["w"]


def _select(st):
    """Scores: the heads' sums in 64 bits, rounded to 32.  (Sorting a number made of the score's
    bits and the position keeps ties in order.)"""
    case, w = st["case"], st["w"]
    at = torch.arange(case["ctx"], device="cuda")
    n = st["d_total"][:, None]
    score = w.double().sum(1).float()
    score = score.masked_fill((at < case["first"]) | (at >= n - case["recent"]), math.inf)
    score = score.masked_fill(at >= n, -math.inf)
    bits = score.view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits) * 2 ** 32 + (2 ** 31 - at)
    most = max(st["keep"])
    index = key.topk(most, 1).indices
    index = index.masked_fill(torch.arange(most, device="cuda") >= st["d_keep"][:, None], case["ctx"])
    index = index.sort(1).values
    kept = w.gather(2, index.clamp(max=case["ctx"] - 1)[:, None].expand(-1, w.shape[1], -1))
    kept = kept * (index < case["ctx"])[:, None]
    return index[index < case["ctx"]].to(torch.int32), kept


def _logprob(st):
    x, k = st["x"].float(), st["case"]["top"]
    top = x.amax(-1, keepdim=True)
    z = x - top
    p = z.exp()
    total = p.sum(-1, keepdim=True)
    log_total = total.log()
    entropy = log_total[:, 0] - torch.where(p > 0, p * z, 0.0).sum(-1) / total[:, 0]
    given = z.gather(1, st["token"].long()[:, None]) - log_total
    bits = (x + 0.0).view(torch.int32).long()
    at = torch.arange(x.shape[1], device="cuda")
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits) * 2 ** 32 + (2 ** 31 - at)
    best = key.topk(k, 1).indices
    lp = z.gather(1, best) - log_total
    return given[:, 0], entropy, torch.where(lp > -math.inf, best, -1).to(torch.int32), lp


# --------------------------------------------------- one pass, the library's

class _Memory:
    """A cache's plane as an array in device memory."""

    def __init__(self, ptr, shape, strides, typestr):
        self.__cuda_array_interface__ = dict(data=(ptr, False), shape=shape, strides=strides,
                                             typestr=typestr, version=3)


def _own_views(c):
    """Views of a cache's first layer's planes, [2][n_kv][tokens][...], that keep the cache."""
    at_0, at_1 = c.planes_device(0, 0), c.planes_device(0, 1)
    step, gpd = at_1[0] - at_0[0], c.head_dim // 64
    got = []
    for ptr, per, kind, size in zip(at_0, (32 * gpd, gpd, gpd), ("|u1", "<f4", "<f4"), (1, 4, 4)):
        row = per * size
        got.append(torch.as_tensor(_Memory(ptr, (2, c.n_heads, c.max_seq_len, per),
                                           (step, c.max_seq_len * row, row, size), kind),
                                   device="cuda"))
        got[-1].cache = c       # the memory lives as long as the view
    return got


def _own_cache(planes, room=None):
    # the same codes as the plain form's
    import eakv_amd
    _, n_kv, t, half = planes[0].shape
    c = eakv_amd.Cache(1, n_kv, 2 * half, room or t)
    for to, plane in zip(_own_views(c), planes):
        to[:, :, :t].copy_(plane)
    if room:
        c.advance(t)
    torch.cuda.synchronize()
    return c


def _own_prepare(st):
    import eakv_amd
    case, L, op = st["case"], eakv_amd.lib(), st["case"]["op"]

    def scratch(n):
        st["work"] = torch.empty(n, dtype=torch.uint8, device="cuda")
        return st["work"].data_ptr(), n

    if op in ("paged", "append"):
        pool = st["planes"]
        st["batch"] = eakv_amd.PagedBatch(
            pool, case["page"], st["tables"].data_ptr(), st["tables"].shape[1], st["d_lens"].data_ptr(),
            case["seqs"], max_len=max(a + m for a, m in st["lens"]), max_new=max(m for _, m in st["lens"]),
            d_first=st["d_first"].data_ptr(), n_new=st["first"][-1])
        if op == "paged":
            st["out"] = torch.empty_like(st["q"])
            scratch(st["batch"].work_bytes(case["n_q"], case["n_kv"], case["dtype"]))
        else:
            st["views"] = _own_views(pool)
    elif op == "weights":
        st["plan"] = eakv_amd.WeightsPlan(st["caches"], [m for _, m in st["lens"]], case["n_q"],
                                          case["n_kv"], starts=[a for a, _ in st["lens"]],
                                          dtype=case["dtype"])
        scratch(st["plan"].work_bytes)
    elif op == "select":
        n, keep = case["seqs"], st["keep"]
        st["index"] = torch.empty(sum(keep), dtype=torch.int32, device="cuda")
        st["kept"] = torch.zeros(n, case["heads"], max(keep), device="cuda")
        st["lists"] = eakv_amd.ints(st["total"]), eakv_amd.ints(keep)
        scratch(L.eakv_evict_select_work_bytes(n, st["lists"][0]))
    else:
        n, k = case["rows"], case["top"]
        st["given"], st["entropy"] = (torch.empty(n, device="cuda") for _ in range(2))
        st["best"] = torch.empty(n, k, dtype=torch.int32, device="cuda")
        st["best_lp"] = torch.empty(n, k, device="cuda")
        scratch(L.eakv_token_logprobs_work_bytes(n, case["vocab"], k))


def _must(rc):
    import eakv_amd
    if rc != eakv_amd.EAKV_OK:
        raise RuntimeError("%d: %s" % (rc, eakv_amd.last_error()[1]))


def _own_paged(st):
    case = st["case"]
    st["batch"].attend(0, st["q"].data_ptr(), st["out"].data_ptr(), case["n_q"], case["n_kv"], case["dtype"],
                       st["work"].data_ptr(), st["work"].numel())
    return st["out"]


def _own_append(st):
    k, v = st["new"]
    st["batch"].append(0, k.data_ptr(), v.data_ptr(), st["case"]["dtype"])
    return st["views"]


def _own_weights(st):
    st["plan"].run(0, st["q"].data_ptr(), st["w"].data_ptr(), st["w"].shape[2], KEEP,
                   st["work"].data_ptr(), st["work"].numel())
    return st["w"]


def _own_select(st):
    import eakv_amd
    case, w, (total, keep) = st["case"], st["w"], st["lists"]
    _must(eakv_amd.lib().eakv_evict_select_device(
        case["seqs"], case["heads"], w.data_ptr(), case["ctx"], total, case["first"], case["recent"], keep,
        st["index"].data_ptr(), st["kept"].data_ptr(), st["kept"].shape[2], st["work"].data_ptr(),
        st["work"].numel(), None))
    return st["index"], st["kept"]


def _own_logprob(st):
    import eakv_amd
    case = st["case"]
    _must(eakv_amd.lib().eakv_token_logprobs_device(
        case["rows"], case["vocab"], st["x"].data_ptr(),
        eakv_amd.EAKV_BF16 if case["dtype"] == "bf16" else eakv_amd.EAKV_F32, case["vocab"],
        st["token"].data_ptr(), case["top"], st["given"].data_ptr(), st["entropy"].data_ptr(),
        st["best"].data_ptr(), st["best_lp"].data_ptr(), st["work"].data_ptr(), st["work"].numel(), None))
    return st["given"], st["entropy"], st["best"], st["best_lp"]


_PLAIN = dict(paged=_paged, append=_append, weights=_weights, select=_select, logprob=_logprob)
_OWN = dict(paged=_own_paged, append=_own_append, weights=_own_weights, select=_own_select,
            logprob=_own_logprob)


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------- what a pass stands for

def work(case):
    """Each input read once and each output written once; a cached token of one kv head
    is 40 bytes for each 64 dims of K and the same of V."""
    op = case["op"]
    size = 2 if case.get("dtype") == "bf16" else 4
    if op == "logprob":
        n, v, k = case["rows"], case["vocab"], case["top"]
        return dict(bytes=float(n * v * size + n * (12 + 8 * k)), flops=4.0 * n * v)
    if op == "select":
        n, h = case["seqs"], case["heads"]
        return dict(bytes=4.0 * n * (h * case["ctx"] + case["keep"] * (h + 1)), flops=float(n * h * case["ctx"]))
    lens, n_kv, d = _lengths(case), case["n_kv"], case["d"]
    per, new = n_kv * d // 64 * 40, sum(m for _, m in lens)
    if op == "append":
        return dict(bytes=2.0 * new * (n_kv * d * size + per), flops=6.0 * new * n_kv * d)
    held, pairs = sum(a + m for a, m in lens), sum(m * a + m * (m + 1) / 2 for a, m in lens)
    rows = float(new * case["n_q"] * d * size)
    if op == "weights":
        return dict(bytes=held * (per + 8.0 * n_kv) + rows, flops=2.0 * case["n_q"] * d * pairs)
    return dict(bytes=2.0 * held * per + 2.0 * rows, flops=4.0 * case["n_q"] * d * pairs)


# ------------------------------------------------------------- in 64 bits

def _wide(w, s, b):
    """f64 [t][d] of one head's codes [t][d/2], scales and biases."""
    t, groups = s.shape
    codes = w.reshape(t, groups, 32)
    n = torch.stack([codes % 16, codes // 16], 2).reshape(t, groups, 64).double()
    return (n * s.double()[..., None] + b.double()[..., None]).reshape(t, -1)


def _softmax(q, k, a):
    """f64 weights [m][q heads][t] of queries [m][q heads][d] at a, a + 1, .."""
    m, t = q.shape[0], k.shape[0]
    s = torch.tensordot(q.double() / math.sqrt(q.shape[2]), k.t().contiguous(), 1)
    see = torch.ones(m, t, dtype=torch.bool, device="cuda").tril(a)
    return torch.softmax(s.masked_fill(~see[:, None], -math.inf), -1)


def exact(case, seed):
    op = case["op"]
    if op == "select":
        return None, _kept(case, seed)
    if op == "logprob":
        x, token = _logprob_inputs(case, seed)
        some = []
        for r in range(case["rows"]):
            lp = torch.log_softmax(x[r].double(), 0)
            value, index = torch.sort(lp, descending=True, stable=True)
            full = torch.where(lp > -math.inf, lp.exp() * lp, 0.0)
            some.append((lp[int(token[r])], -full.sum(), value[:case["top"]]))
        given, entropy, best = (torch.stack(y) for y in zip(*some))
        return given, entropy, None, best
    lens, n_kv = _lengths(case), case["n_kv"]
    if op == "weights":
        xs = list(_weights_inputs(case, seed))
        q, w = xs.pop()
        w, row, per = w.double(), 0, case["n_q"] // n_kv
        for i, (x, (a, m)) in enumerate(zip(xs, lens)):
            planes = _quantize(x[0])
            for h in range(n_kv):
                p = _softmax(q[row:row + m, h * per:(h + 1) * per], _wide(*(y[h] for y in planes)), a)
                w[i, h, :a + m] = w[i, h, :a + m] * KEEP + p.sum((0, 1))
            row += m
        return w
    planes, tables, g, chan = _pool(case, seed)
    n, d, page = sum(m for _, m in lens), case["d"], case["page"]
    if op == "append":
        x = _kv(g, n_kv, n, d, chan).transpose(1, 2)
        scales, biases = (p.double() for p in planes[1:])
        row = 0
        for i, (a, m) in enumerate(lens):
            at = torch.arange(a, a + m, device="cuda")
            at = tables[i, at // page].long() * page + at % page
            for j in (0, 1):
                y = _typed(x[j, row:row + m], case).double().reshape(m, n_kv, -1, 64)
                lo, hi = y.amin(-1), y.amax(-1)
                scales[j][:, at] = torch.where(hi > lo, (hi - lo) / 15, 1.0).transpose(0, 1)
                biases[j][:, at] = lo.transpose(0, 1)
            row += m
        return None, scales, biases
    q = _typed(torch.randn(n, case["n_q"], d, generator=g, device="cuda"), case)
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    row, per = 0, case["n_q"] // n_kv
    for i, (a, m) in enumerate(lens):
        at = torch.arange(a + m, device="cuda")
        at = tables[i, at // page].long() * page + at % page
        for h in range(n_kv):
            k, v = (_wide(*(p[j, h, at] for p in planes)) for j in (0, 1))
            for b in range(0, m, 512):      # rows that fit the memory
                c = min(m, b + 512)
                p = _softmax(q[row + b:row + c, h * per:(h + 1) * per], k[:a + c], a + b)
                out[row + b:row + c, h * per:(h + 1) * per] = torch.tensordot(p, v[:a + c], 1)
        row += m
    return out


def _kept(case, seed):
    """The kept tokens' weights: scores sorted one sequence at a time."""
    w, total, keep = _select_inputs(case, seed)
    kept = torch.zeros(case["seqs"], case["heads"], max(keep), dtype=torch.float64, device="cuda")
    for i, (t, k) in enumerate(zip(total, keep)):
        x = w[i, :, :t].double()
        score = x.sum(0).float()
        lo, hi = min(case["first"], t), max(0, t - case["recent"])
        score[:lo] = math.inf
        score[hi:] = math.inf
        stay = torch.sort(score, descending=True, stable=True).indices[:k].sort().values
        kept[i, :, :k] = x[:, stay]
    return kept
