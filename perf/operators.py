"""Operators of serving with the 4-bit cache, as cases that can be timed.

  window  attention of several new tokens of each sequence over its cache: the
          tokens of a draft (a chain, or a tree with a mask of ancestors) or a
          piece of a prompt (eakv_attention_window_batch_device)
  verify  which drafted tokens the target model keeps, and the token after
          them, from given random numbers (eakv_verify_drafts_device)
  copy    a cache's tokens into other caches: forking a sequence
          (eakv_cache_copy_batch_device)
  gather  a cache reduced to chosen tokens: the accepted path of a tree, the
          first and the most recent tokens, the tokens of most weight
          (eakv_cache_gather_batch_device)

Where `own` is false a pass computes the same in elementary torch operations.
A cache is then three tensors (packed codes, scales, biases: 64 values in 32
bytes and two floats, byte k holding value k in its low and value k + 32 in
its high four bits); else it is an eakv_amd.Cache of the same values.

The copied and gathered outputs are the caches' planes as they stand in
memory: these operators move them and compute nothing.
"""
import math
import random

import torch

own = False

# q heads, kv heads, head_dim
HEADS = [(8, 8, 128), (32, 4, 64), (32, 32, 128), (32, 8, 128), (64, 8, 128), (40, 8, 128),
         (16, 8, 128), (12, 12, 64)]

# The largest listed case of each kind, which no drawn case exceeds
MOST_FLOPS = 1.1e12
MOST_BYTES = 1.0e9


def listed():
    def window(name, heads, dtype, seqs, tokens, ctx, spread=1, tree=False):
        return dict(name=name, op="window", n_q=heads[0], n_kv=heads[1], d=heads[2], dtype=dtype,
                    seqs=seqs, tokens=tokens, ctx=ctx, spread=spread, tree=tree)

    return [
        # one chat, a short draft at a short context: latency
        window("draft 4 x1 2K bf16", (32, 8, 128), "bf16", 1, 4, 2048),
        # serving with drafts at long contexts
        window("draft 8 x8 32K bf16", (32, 8, 128), "bf16", 8, 8, 32768),
        # trees of drafts on a 70B-shaped model, sequences of several lengths
        window("tree 24 x6 ragged f32", (64, 8, 128), "f32", 6, 24, 30011, 16, True),
        # the first piece of a prompt on a model with one q head per kv head
        window("prompt 2000 f32", (32, 32, 128), "f32", 1, 2000, 2000),
        # ragged pieces of prompts on a small model
        window("prompt 1100 x4 d64 bf16", (32, 4, 64), "bf16", 4, 1100, 5003, 4),
        # a further piece of a long prompt
        window("prompt 2048 at 30K bf16", (32, 8, 128), "bf16", 1, 2048, 32768),
        # one chat's draft, a small vocabulary
        dict(name="verify 4 x1 32000", op="verify", seqs=1, drafts=4, vocab=32000, onehot=False),
        # a batch's drafts, a large vocabulary of odd size
        dict(name="verify 7 x64 151665", op="verify", seqs=64, drafts=7, vocab=151665,
             onehot=False),
        # a short chat forked once
        dict(name="fork 2K", op="copy", n_kv=8, d=128, layers=2, ctx=2047, copies=1),
        # a long prompt's cache forked for parallel samples
        dict(name="fork 32K x4", op="copy", n_kv=8, d=128, layers=4, ctx=32768, copies=4),
        # the accepted path of each sequence's tree, in place
        dict(name="keep 5 of 24 x8", op="gather", how="tree", n_kv=8, d=128, layers=8, seqs=8,
             ctx=4120, keep=5),
        # a long context reduced to the tokens of most weight, into a cache of its own
        dict(name="keep 13001 of 30011", op="gather", how="weight", n_kv=8, d=128, layers=8,
             seqs=1, ctx=30011, keep=13001),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["window"] * 5 + ["verify"] * 2 + ["copy", "gather", "gather"])
    n_q, n_kv, d = rng.choice(HEADS)
    if op == "window":
        ctx = _log(rng, 16, 131072)
        tree = rng.random() < 0.3
        case = dict(op=op, n_q=n_q, n_kv=n_kv, d=d, dtype=rng.choice(["bf16", "bf16", "f32"]),
                    seqs=_log(rng, 1, 32), tokens=_log(rng, 1, 64 if tree else min(4096, ctx)),
                    ctx=ctx, spread=rng.choice([1, 1, 4, 16]), tree=tree)
        case["tokens"] = min(case["tokens"], ctx)
        while work(case)["flops"] > MOST_FLOPS or work(case)["bytes"] > MOST_BYTES / 2:
            if case["seqs"] > 1:
                case["seqs"] = case["seqs"] * 2 // 3
            else:
                case["ctx"] = case["ctx"] * 2 // 3
                case["tokens"] = min(case["tokens"], case["ctx"])
        return case
    if op == "verify":
        case = dict(op=op, seqs=_log(rng, 1, 128), drafts=rng.randint(1, 15),
                    vocab=_log(rng, 1000, 160000), onehot=rng.random() < 0.3)
        while case["seqs"] * case["drafts"] * case["vocab"] > 64 * 7 * 151665:
            case["seqs"] = case["seqs"] * 2 // 3
        return case
    case = dict(op=op, n_kv=n_kv, d=d, layers=rng.randint(1, 8), ctx=_log(rng, 64, 65536))
    if op == "copy":
        case.update(copies=_log(rng, 1, 16))
        size = "copies"
    else:
        how = rng.choice(["tree", "recent", "weight"])
        case.update(how=how, seqs=_log(rng, 1, 16))
        if how == "tree":
            case["keep"] = rng.randint(1, 8)
        else:
            case["keep"] = rng.randint(8, case["ctx"] // 2 if how == "recent" else case["ctx"])
        size = "seqs"
    while work(case)["bytes"] > MOST_BYTES:
        if case[size] > 1:
            case[size] = case[size] * 2 // 3
        else:
            case["ctx"] = case["ctx"] * 2 // 3
            case["keep"] = case.get("keep", 0) * 2 // 3
    return case


# ---------------------------------------------------------------- the inputs

TREE = 24       # a drafted tree's nodes, where a gather keeps one path of it


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case):
    """(tokens before the window, tokens of the window) of each sequence:
    contexts log-uniform from ctx/spread to ctx, one of them ctx; windows of
    one length, or, where the contexts differ, of any up to it."""
    n, ctx, m, spread = case["seqs"], case["ctx"], case["tokens"], case["spread"]
    r = random.Random(n * 1000003 + ctx * 131 + m)
    total = [max(1, int(round(ctx * spread ** -r.random()))) for _ in range(n)]
    total[n // 3] = ctx
    win = [min(t, m if spread == 1 else r.randint(1, m)) for t in total]
    win[n // 3] = min(m, ctx)
    return [(t - w, w) for t, w in zip(total, win)]


def _channels(g, n_kv, d):
    """Key channel scales f32[n_kv][1][d]: log-uniform in [0.5, 4], two
    channels of each head ten times larger."""
    c = torch.exp(torch.rand(n_kv, 1, d, generator=g, device="cuda") * math.log(8.0) + math.log(0.5))
    for h in range(n_kv):
        c[h, 0, torch.randperm(d, generator=g, device="cuda")[:2]] *= 10
    return c


def _kv(g, layers, n_kv, tokens, d, chan):
    """K and V f32[layers][2][n_kv][tokens][d], as model states are: K with
    scales and outliers by channel, V normal."""
    x = torch.randn(layers, 2, n_kv, tokens, d, generator=g, device="cuda")
    x[:, 0] *= chan
    return x


def _quantize(x):
    """The cache's codes, scales and biases of x [..., t, d]: groups of 64,
    bias the minimum, scale range/15, each step rounded to f32."""
    v = x.unflatten(-1, (x.shape[-1] // 64, 64))
    mn, mx = v.aminmax(dim=-1)
    r = mx - mn
    some = r > 0
    scale = torch.where(some, r / 15.0, torch.ones_like(r))
    inv = torch.where(some, 15.0 / r, torch.zeros_like(r))
    n = (v - mn[..., None]).mul_(inv[..., None]).add_(0.5).floor_().clamp_(0, 15).to(torch.uint8)
    w = (n[..., 32:] << 4) | n[..., :32]
    return w.flatten(-2), scale, mn


def _tree(r, m):
    """Ancestor masks of a random tree of m drafted tokens: bit j of word i
    says that token i sees token j."""
    words = []
    for i in range(m):
        up = r.randint(-1, i - 1) if i else -1
        words.append((words[up] if up >= 0 else 0) | 1 << i)
    return [w - (1 << 64) if w >> 63 else w for w in words]


def _window_inputs(case, seed):
    """The sequences' K and V in turn (the window's tokens at the end), then
    the queries [tokens of all windows][n_q][d] and the tree's words."""
    g = _gen(seed)
    n_kv, d = case["n_kv"], case["d"]
    chan = _channels(g, n_kv, d)
    lens = _lengths(case)
    for start, m in lens:
        yield _kv(g, 1, n_kv, start + m, d, chan)[0]
    total = sum(m for _, m in lens)
    q = torch.randn(total, case["n_q"], d, generator=g, device="cuda")
    if case["dtype"] == "bf16":
        q = q.bfloat16()
    r = random.Random(seed)
    tree = [w for _, m in lens for w in _tree(r, m)] if case["tree"] else None
    yield q, None if tree is None else torch.tensor(tree, dtype=torch.int64, device="cuda")


def _verify_inputs(case, seed):
    """Target and draft distributions a few tenths of a nat apart, the drafted
    tokens from the latter, drafts of any length up to the longest."""
    g = _gen(seed)
    n, k, v = case["seqs"], case["drafts"], case["vocab"]
    logits = torch.randn(n, k + 1, v, generator=g, device="cuda").mul_(3.0)
    target = torch.softmax(logits, -1)
    near = logits[:, :k].add_(torch.randn(n, k, v, generator=g, device="cuda"), alpha=0.5)
    draft = torch.softmax(near, -1)
    del logits, near
    pick = torch.rand(n, k, 1, generator=g, device="cuda") * 0.999
    token = (draft.cumsum(-1) <= pick).sum(-1).clamp_(max=v - 1).to(torch.int32)
    if case["onehot"]:      # drafts without a distribution: the likeliest token, or one copied
        likely = target[:, :k].argmax(-1).to(torch.int32)
        token = torch.where(torch.rand(n, k, generator=g, device="cuda") < 0.7, likely, token)
        draft = None
    uniform = torch.rand(n, k + 1, generator=g, device="cuda")
    count = torch.randint(0, k + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    count[0] = k
    return count, token, draft, target, uniform


def _kept(case, seed, s):
    """Sequence s's first changed position and the positions that it keeps
    from there on."""
    r = random.Random(seed * 131 + s)
    ctx, keep = case["ctx"], case["keep"]
    if case["how"] == "tree":
        # the tree's tokens are its levels one after the other: a path through
        # its root and nodes behind the first levels
        at = max(0, ctx - TREE)
        n = ctx - at
        k = min(keep, max(1, n // 2))
        return at, [at] + sorted(at + i for i in r.sample(range(k, n), k - 1))
    if case["how"] == "recent":
        first = min(4, keep // 2)
        return first, list(range(ctx - (keep - first), ctx))
    return 0, sorted(r.sample(range(ctx), keep))


def prepare(case, seed):
    op = case["op"]
    st = dict(case=case)
    if op == "window":
        caches, lens = [], _lengths(case)
        for x in _window_inputs(case, seed):
            if isinstance(x, tuple):
                st.update(q=x[0], tree=x[1])
            else:
                caches.append(_cache(x[None], case["ctx"]))
            del x
        st.update(caches=caches, lens=lens)
    elif op == "verify":
        st["in"] = _verify_inputs(case, seed)
    else:
        g = _gen(seed)
        n_kv, d, layers, ctx = case["n_kv"], case["d"], case["layers"], case["ctx"]
        chan = _channels(g, n_kv, d)
        src = [_cache(_kv(g, layers, n_kv, ctx, d, chan), ctx) for _ in range(case.get("seqs", 1))]
        empty = torch.zeros(layers, 2, n_kv, 1, d, device="cuda")
        if op == "copy":
            st.update(src=src, dst=[_cache(empty, ctx) for _ in range(case["copies"])], at=0, n=ctx)
        else:
            kept = [_kept(case, seed, s) for s in range(case["seqs"])]
            st.update(src=src, dst=src, at=[a for a, _ in kept], n=[len(i) for _, i in kept],
                      index=torch.tensor([p for _, i in kept for p in i], dtype=torch.int32,
                                         device="cuda"))
            if case["how"] == "weight":
                st["dst"] = [_cache(empty, case["keep"]) for _ in src]
    if own:
        _own_prepare(st)
    return st


# ------------------------------------------------------- one pass, plain form

def _cache(x, room):
    """A cache with room for `room` tokens that holds x [layers][2][n_kv][t][d]."""
    if own:
        return _own_cache(x, room)
    w, s, b = _quantize(x)
    more = room - x.shape[3]
    if more > 0:
        w, s, b = (torch.cat([p, p.new_zeros(p.shape[:3] + (more,) + p.shape[4:])], 3)
                   for p in (w, s, b))
    return w, s, b


def _values(planes):
    """f32 [n_kv][t][d] of one block's codes, scales and biases."""
    w, s, b = planes
    w = w.unflatten(-1, (-1, 32))
    n = torch.cat([w & 15, w >> 4], -1).float()
    return n.mul_(s[..., None]).add_(b[..., None]).flatten(-2)


def _attend(cache, q, start, tree):
    """softmax(q.k/sqrt(d)).v of the tokens of one window, [m][n_q][d]."""
    m, n_q, d = q.shape
    seen = start + m
    k, v = (_values([p[0, i, :, :seen] for p in cache]) for i in (0, 1))
    n_kv = k.shape[0]
    rows = q.float().reshape(m, n_kv, n_q // n_kv, d).transpose(0, 1).reshape(n_kv, -1, d)
    s = torch.matmul(rows, k.transpose(1, 2).contiguous()).div_(math.sqrt(d))
    s = s.view(n_kv, m, n_q // n_kv, seen)
    at = torch.arange(m, device=q.device)
    if tree is None:
        hidden = at[:, None] < at
    else:
        hidden = (tree[:, None] >> at & 1) == 0
    s[..., start:].masked_fill_(hidden[:, None, :], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n_kv, -1, seen), v).view(n_kv, m, n_q // n_kv, d)
    o = (o / total).masked_fill(total == 0, 0.0)
    return o.transpose(0, 1).reshape(m, n_q, d).to(q.dtype)


def _window(st):
    ms = [m for _, m in st["lens"]]
    qs = st["q"].split(ms)
    trees = st["tree"].split(ms) if st["tree"] is not None else [None] * len(ms)
    return torch.cat([_attend(c, q, start, t)
                      for c, q, t, (start, _) in zip(st["caches"], qs, trees, st["lens"])])


def _verify(st):
    """(tokens kept, the token after them) of each sequence.  Sums in 64 bits:
    a step of the cumulative sum near the drawn number decides."""
    count, token, draft, target, uniform = st["in"]
    n, k = token.shape
    seq = torch.arange(n, device=token.device)
    pos = torch.arange(k, device=token.device)
    x = token.long()[..., None]
    p = target[:, :k].gather(-1, x)[..., 0].double()
    q = torch.ones_like(p) if draft is None else draft.gather(-1, x)[..., 0].double()
    ok = (uniform[:, :k].double() * q < p) & (pos < count[:, None])
    kept = ok.long().cumprod(1).sum(1)
    rest = target[seq, kept].double()
    last = kept.clamp(max=k - 1)
    if draft is None:
        less = rest.scatter(1, token.long()[seq, last][:, None], 0.0)
    else:
        less = (rest - draft[seq, last].double()).clamp_(min=0.0)
    r = torch.where((kept < count)[:, None], less, rest)
    r = torch.where(r.sum(1, keepdim=True) > 0, r, rest)
    upto = r.cumsum(1)
    want = uniform[:, k:].double() * upto[:, -1:]
    at = (upto <= want).sum(1)
    end = torch.where(r > 0, torch.arange(r.shape[1], device=r.device), -1).amax(1)
    return kept.to(torch.int32), torch.minimum(at, end).to(torch.int32)


def _copy(st):
    n = st["n"]
    return [[d[:, :, :, :n].copy_(s[:, :, :, :n]) for s, d in zip(st["src"][0], dst)]
            for dst in st["dst"]]


def _gather(st):
    index = st["index"].long().split(st["n"])

    def one(src, dst, i, at):
        return [d[:, :, :, at:at + i.numel()].copy_(s.index_select(3, i)) for s, d in zip(src, dst)]

    return [one(*a) for a in zip(st["src"], st["dst"], index, st["at"])]


# --------------------------------------------------- one pass, the library's

class _Memory:
    """A cache's plane as an array in device memory."""

    def __init__(self, ptr, shape, strides, typestr):
        self.__cuda_array_interface__ = dict(data=(ptr, False), shape=shape, strides=strides,
                                             typestr=typestr, version=3)


def _own_cache(x, room):
    # the same codes as the plain form's, bit for bit, not requantized
    import eakv_amd
    layers, _, n_kv, t, d = x.shape
    c = eakv_amd.Cache(layers, n_kv, d, room)
    for to, plane in zip(_own_planes(c, 0, t), _quantize(x)):
        to.copy_(plane)
    c.advance(t)
    torch.cuda.synchronize()
    return c


def _must(rc):
    import eakv_amd
    if rc != eakv_amd.EAKV_OK:
        raise RuntimeError("%d: %s" % (rc, eakv_amd.last_error()[1]))


def _own_planes(c, at, n):
    """Views of tokens [at, at + n) of every block's planes,
    [layers][2][n_kv][n][...], that keep the cache."""
    at_0, at_1 = c.planes_device(0, 0), c.planes_device(0, 1)
    step, gpd = at_1[0] - at_0[0], c.head_dim // 64
    got = []
    for ptr, per, kind, size in zip(at_0, (32 * gpd, gpd, gpd), ("|u1", "<f4", "<f4"), (1, 4, 4)):
        row = per * size
        got.append(torch.as_tensor(_Memory(ptr + at * row, (2 * c.n_layers, c.n_heads, n, per),
                                           (step, c.max_seq_len * row, row, size), kind),
                                   device="cuda").unflatten(0, (c.n_layers, 2)))
        got[-1].cache = c       # the memory lives as long as the view
    return got


def _own_prepare(st):
    import eakv_amd
    case, L = st["case"], eakv_amd.lib()
    if case["op"] == "window":
        st["plan"] = eakv_amd.WindowPlan(st["caches"], [m for _, m in st["lens"]], case["n_q"],
                                         case["n_kv"], starts=[a for a, _ in st["lens"]],
                                         dtype=case["dtype"])
        st["out"] = torch.empty_like(st["q"])
        st["work"] = torch.empty(st["plan"].work_bytes, dtype=torch.uint8, device="cuda")
    elif case["op"] == "verify":
        n, k, v = case["seqs"], case["drafts"], case["vocab"]
        st["kept"] = torch.empty(n, dtype=torch.int32, device="cuda")
        st["next"] = torch.empty(n, dtype=torch.int32, device="cuda")
        st["work"] = torch.empty(L.eakv_verify_drafts_work_bytes(n, k, v), dtype=torch.uint8,
                                 device="cuda")
    elif case["op"] == "copy":
        st["src_h"], st["dst_h"] = st["src"][0].h, eakv_amd.handles(st["dst"])
        st["planes"] = [_own_planes(c, 0, st["n"]) for c in st["dst"]]
    else:
        st["src_h"], st["dst_h"] = eakv_amd.handles(st["src"]), eakv_amd.handles(st["dst"])
        st["at_h"], st["n_h"] = eakv_amd.ints(st["at"]), eakv_amd.ints(st["n"])
        st["planes"] = [_own_planes(c, a, n) for c, a, n in zip(st["dst"], st["at"], st["n"])]


def _own_window(st):
    tree = st["tree"]
    st["plan"].run(0, st["q"].data_ptr(), st["out"].data_ptr(),
                   None if tree is None else tree.data_ptr(), st["work"].data_ptr(),
                   st["work"].numel())
    return st["out"]


def _own_verify(st):
    import eakv_amd
    n, k, v = (st["case"][x] for x in ("seqs", "drafts", "vocab"))
    count, token, draft, target, uniform = st["in"]
    _must(eakv_amd.lib().eakv_verify_drafts_device(
        n, k, v, count.data_ptr(), token.data_ptr(), None if draft is None else draft.data_ptr(), v,
        target.data_ptr(), v, uniform.data_ptr(), st["kept"].data_ptr(), st["next"].data_ptr(),
        st["work"].data_ptr(), st["work"].numel(), None))
    return st["kept"], st["next"]


def _own_copy(st):
    import eakv_amd
    _must(eakv_amd.lib().eakv_cache_copy_batch_device(st["src_h"], 0, st["dst_h"], len(st["dst"]),
                                                     st["at"], st["n"], None))
    return st["planes"]


def _own_gather(st):
    import eakv_amd
    _must(eakv_amd.lib().eakv_cache_gather_batch_device(st["src_h"], st["dst_h"], len(st["dst"]),
                                                       st["at_h"], st["index"].data_ptr(),
                                                       st["n_h"], None))
    return st["planes"]


_PLAIN = dict(window=_window, verify=_verify, copy=_copy, gather=_gather)
_OWN = dict(window=_own_window, verify=_own_verify, copy=_own_copy, gather=_own_gather)


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------- what a pass stands for

def work(case):
    """Each input read once and each output written once; a cached token of
    one kv head is 40 bytes for each 64 dims of K and the same of V."""
    op = case["op"]
    if op == "verify":
        # one row of the target, one of the draft where there is one
        n, v = case["seqs"], case["vocab"]
        return dict(bytes=float(n * v * 4 * (1 if case["onehot"] else 2) + n * case["drafts"] * 16),
                    flops=4.0 * n * v)
    n_kv, d = case["n_kv"], case["d"]
    per = n_kv * d // 64 * 40
    if op == "copy":
        return dict(bytes=2.0 * case["layers"] * case["ctx"] * per * (1 + case["copies"]), flops=0.0)
    if op == "gather":
        return dict(bytes=4.0 * case["layers"] * case["seqs"] * case["keep"] * per, flops=0.0)
    lens = _lengths(case)
    # the tokens before the window, and half of the window (a tree: less)
    pairs = sum(m * start + m * (m + 1) / 2 for start, m in lens)
    size = 2 if case["dtype"] == "bf16" else 4
    return dict(bytes=2.0 * sum(a + m for a, m in lens) * per
                + 2.0 * sum(m for _, m in lens) * case["n_q"] * d * size,
                flops=4.0 * case["n_q"] * d * pairs)


# ------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """The window's attention in f64, one kv head at a time; the other
    operators give whole numbers and copies."""
    if case["op"] != "window":
        return None
    xs = list(_window_inputs(case, seed))
    q, tree = xs.pop()
    n_kv, d = case["n_kv"], case["d"]
    per = case["n_q"] // n_kv
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    row = 0
    for x, (start, m) in zip(xs, _lengths(case)):
        w, s, b = _quantize(x)
        see = torch.ones(m, start + m, dtype=torch.bool, device="cuda").tril(start)
        if tree is not None:
            for j in range(m):
                see[:, start + j] = torch.bitwise_and(tree[row:row + m] >> j, 1).bool()
        for h in range(n_kv):
            kv = []
            for i in (0, 1):
                codes = w[i, h].reshape(-1, d // 64, 32)
                n = torch.stack([codes % 16, codes // 16], 2).double().reshape(-1, d // 64, 64)
                kv.append((n * s[i, h].double()[..., None] + b[i, h].double()[..., None]).reshape(-1, d))
            for a in range(0, m, 512):      # rows that fit the memory
                z = q[row + a:row + min(m, a + 512), h * per:(h + 1) * per].double()
                p = torch.matmul(z.reshape(-1, d) / math.sqrt(d), kv[0].t().contiguous())
                p = p.reshape(z.shape[0], per, -1)
                p = p.masked_fill(~see[a:a + 512, None, :], -math.inf)
                p = torch.softmax(p, -1)
                o = torch.matmul(p.reshape(-1, start + m), kv[1]).reshape(z.shape)
                out[row + a:row + min(m, a + 512), h * per:(h + 1) * per] = o
        row += m
    return out
