"""Performance cases of the paged cache (append with rotation, attention of new tokens, accepted paths) and of the gated recurrence.

A case is a dict of plain values; `kind` names what is timed:

  append             paged_append: new keys, rotated, and values go to their pages; queries are rotated on the way
  attention          paged_attention: new tokens of each sequence -- one, a chunk of a prompt, or a tree of drafted ones -- against the pages
  keep               paged_keep: the accepted path of each tree moves to the places behind the tokens before it
  recurrence_prompt  gated_recurrence: outputs and the state behind the last token
  recurrence_train   the same and its gradients, the states' among them
  recurrence_step    gated_recurrence_step: one new token of each sequence, state updated in place

`lengths` is a text of the sequences' new tokens, `cached` one of the tokens before them.  `tree` is 0 for new tokens in a row; otherwise trees
are drawn with it: a token's parent is one of the four before it, as often as not the last.  Queries, keys, values are standard normal, as behind a norm;
log decays are -rate sigmoid(gate), rates of the channels spread between 0.001 and 1.
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BASE = 10000.0


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _text(lengths):
    return ",".join(str(n) for n in lengths)


def _paged(name, kind, dtype, heads, kv_heads, width, page, lengths, cached, tree=0, window=0, sinks=0, rotated=0, interleaved=False):
    """window 0: every token before; rotated: columns that are rotated"""
    c = dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, width=width, page=page, lengths=_text(lengths), cached=_text(cached),
             tree=tree, window=window, sinks=sinks, rotated=rotated, interleaved=interleaved)
    return dict(c, name=name) if name else c


def _recurrence(name, kind, dtype, channels, lengths, carried):
    c = dict(kind=kind, dtype=dtype, channels=channels, lengths=_text(lengths), carried=carried)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token for each sequence of a serving batch; latency counts
        _paged("append_batch", "append", "bf16", 32, 8, 128, 16, [1] * 64, [2048 - 61 * (i % 29) - i for i in range(64)], rotated=128),
        # prompts of a batch of requests as they come, some behind a prefix that the cache holds already
        _paged("append_prompts", "append", "fp16", 32, 8, 128, 64, [4096, 1021, 1, 2500, 57, 333, 1600, 513], [0, 3000, 177, 0, 1024, 0, 0, 511], rotated=64,
               interleaved=True),
        # one conversation, a small tree of drafted tokens, few heads
        _paged("attention_one", "attention", "bf16", 8, 2, 64, 16, [9], [1500], tree=1),
        # one new token for each sequence of a serving batch, conversations of many lengths
        _paged("attention_token", "attention", "bf16", 32, 8, 128, 64, [1] * 32, [16384 - 509 * (i % 31) - 37 * i for i in range(31)] + [2]),
        # drafted trees behind the same
        _paged("attention_trees", "attention", "bf16", 32, 8, 128, 64, [32 - i % 7 for i in range(32)], [16384 - 509 * (i % 31) - 37 * i for i in range(31)] + [2], tree=2),
        # the next chunks of two long prompts, window with sinks
        _paged("attention_chunk", "attention", "fp16", 32, 8, 128, 128, [2048, 1021], [8192, 5000], window=4096, sinks=4),
        # the accepted paths of the trees, of one conversation and of a batch
        _paged("keep_one", "keep", "bf16", 8, 2, 64, 16, [24], [1500], tree=3),
        _paged("keep_batch", "keep", "fp16", 32, 8, 128, 64, [64 - i % 7 for i in range(64)], [1024 - 13 * i for i in range(64)], tree=2),
        # a short prompt, odd length
        _recurrence("recurrence_prompt_short", "recurrence_prompt", "fp16", 512, [129], False),
        # one long document
        _recurrence("recurrence_prompt_long", "recurrence_prompt", "bf16", 2048, [65536], False),
        # a training step on packed documents
        _recurrence("recurrence_train_packed", "recurrence_train", "bf16", 4096, [4096, 1500, 777, 5000, 1011], True),
        # a serving batch
        _recurrence("recurrence_step_batch", "recurrence_step", "bf16", 4096, [1] * 256, True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "attention", "attention", "attention", "keep", "recurrence_prompt", "recurrence_train", "recurrence_step"))
    if kind.startswith("recurrence"):
        dtype, channels = rng.choice(("bf16", "bf16", "fp16", "fp32")), 8 * _log_uniform(rng, 8, 512)
        if kind == "recurrence_step":
            return _recurrence("", kind, dtype, channels, [1] * _log_uniform(rng, 1, 256), True)
        longest = _log_uniform(rng, 16, 32768 if kind == "recurrence_prompt" else 8192)
        n = rng.randint(1, max(1, min(8, (1 << 25) // (channels * longest))))
        return _recurrence("", kind, dtype, channels, [longest] + [_log_uniform(rng, 1, longest) for _ in range(n - 1)], rng.random() < 0.5)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    kv = rng.choice((1, 2, 4, 8))
    heads, width, page = kv * rng.choice((1, 2, 3, 4, 5, 8)), rng.choice((32, 64, 80, 96, 128)), rng.choice((16, 32, 64, 128, 256))
    rotated, interleaved = rng.choice((width, width, 32)), rng.random() < 0.5
    if kind == "append":
        longest = _log_uniform(rng, 1, 4096)
        n = rng.randint(1, 8) if longest > 256 else _log_uniform(rng, 1, 64)
        tree = rng.randint(1, 99) if 1 < longest <= 128 and rng.random() < 0.5 else 0
        lengths = [longest] + [_log_uniform(rng, 1, longest) for _ in range(n - 1)]
        return _paged("", kind, dtype, heads, kv, width, page, lengths, [rng.randint(0, 2048) for _ in lengths], tree, rotated=rotated, interleaved=interleaved)
    if kind == "keep":
        n = _log_uniform(rng, 1, 64)
        return _paged("", kind, dtype, heads, kv, width, page, [rng.randint(1, 64) for _ in range(n)], [rng.randint(0, 1024) for _ in range(n)], rng.randint(1, 99))
    form = rng.choice(("token", "tree", "tree", "chunk"))
    cache = _log_uniform(rng, 64, 16384)
    longest = 1 if form == "token" else rng.randint(2, 128) if form == "tree" else _log_uniform(rng, 16, 2048)
    # the plain form holds heads * sequences * longest * cache numbers: no more than the largest listed case's
    n = min(_log_uniform(rng, 1, 64), max(1, (1 << 19) // cache), max(1, int(5e8 // (heads * longest * (cache + longest)))))
    lengths = [longest] + [1 if form == "token" else rng.randint(max(1, longest // 2), longest) for _ in range(n - 1)]
    cached = [_log_uniform(rng, 1, cache) if rng.random() < 0.3 else rng.randint(cache // 2, cache) for _ in range(n)]
    window, sinks = (0, 0) if rng.random() < 0.5 else (_log_uniform(rng, 16, cache), rng.choice((0, 1, 4, 16, rng.randint(2, 200))))
    return _paged("", kind, dtype, heads, kv, width, page, lengths, cached, rng.randint(1, 99) if form == "tree" else 0, window, sinks)


def _numbers(text):
    return [int(n) for n in text.split(",")]


def _trees(case):
    """Parents of the new tokens, sequence by sequence, -1 at the roots"""
    rng = random.Random(case["tree"])
    return [[-1 if i == 0 else i - 1 if rng.random() < 0.5 else rng.randrange(max(0, i - 4), i) for i in range(n)] for n in _numbers(case["lengths"])]


def _paths(case):
    """Of each tree the path to one of its tokens"""
    rng, paths = random.Random(case["tree"] + 1000), []
    for parents in _trees(case):
        at, path = rng.randrange(len(parents)), []
        while at >= 0:
            path.append(at)
            at = parents[at]
        paths.append(path[::-1])
    return paths


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, lengths = TYPES[case["dtype"]], _numbers(case["lengths"])
    total, n = sum(lengths), len(lengths)

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)

    st = dict(case=case, lengths=lengths)
    if case["kind"].startswith("recurrence"):
        channels = case["channels"]
        rate = torch.exp(torch.rand(channels, generator=g, device=DEVICE) * -math.log(1e-3) + math.log(1e-3))
        st |= dict(x=normal(total, channels), log_decay=(-rate * torch.sigmoid(normal(total, channels, dtype=torch.float32))).to(dt),
                   state=normal(n, channels, dtype=torch.float32) if case["carried"] else None)
        if case["kind"] == "recurrence_train":
            st["do"] = normal(total, channels)
            st["dfinal"] = normal(n, channels, dtype=torch.float32) if case["carried"] else None
    else:
        cached, hq, hk, d, page = _numbers(case["cached"]), case["heads"], case["kv_heads"], case["width"], case["page"]
        pages = [-(-(c + m) // page) for c, m in zip(cached, lengths)]
        pool, most = sum(pages) + 3, max(pages)
        order = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
        table = torch.zeros(n, most, device=DEVICE, dtype=torch.int32)
        at = 0
        for b, m in enumerate(pages):
            table[b, :m] = order[at:at + m]
            at += m
        st |= dict(k_pages=normal(pool, page, hk, d), v_pages=normal(pool, page, hk, d), table=table,
                   cached=torch.tensor(cached, device=DEVICE, dtype=torch.int32), parents=None)
        if case["tree"]:
            st["parents"] = torch.tensor(sum(_trees(case), []), device=DEVICE, dtype=torch.int32)
        if case["kind"] == "keep":
            paths = _paths(case)
            longest = max(len(p) for p in paths)
            st["kept"] = torch.tensor([p + [0] * (longest - len(p)) for p in paths], device=DEVICE, dtype=torch.int32)
            st["counts"] = torch.tensor([len(p) for p in paths], device=DEVICE, dtype=torch.int32)
        else:
            st["q"] = normal(total, hq, d)
        if case["kind"] == "append":
            st |= dict(k=normal(total, hk, d), v=normal(total, hk, d))
            if own:
                from f3m_b200 import paged
                st["rotation"] = paged.Rotation(case["rotated"], base=BASE, interleaved=case["interleaved"], device=DEVICE)
    if case["kind"] not in ("keep", "recurrence_step"):
        if own:
            from f3m_b200 import sequence
            st["plan"] = sequence.SequencePlan(lengths, device=DEVICE)
        else:
            lens = torch.tensor(lengths, device=DEVICE)
            first = torch.cumsum(lens, 0) - lens
            of = torch.repeat_interleave(torch.arange(n, device=DEVICE), lens)
            st |= dict(lens=lens, first=first, of=of, at=torch.arange(total, device=DEVICE) - first[of])
    return st


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _depths(st):
    """Tokens between each new token and its root"""
    if st["parents"] is None:
        return st["at"]
    up = torch.where(st["parents"] < 0, -1, st["parents"] + st["first"][st["of"]])
    depth = (up >= 0).long()
    for _ in range(max(st["lengths"]).bit_length()):      # twice as far each time
        above = up.clamp(min=0)
        depth, up = depth + torch.where(up < 0, 0, depth[above]), torch.where(up < 0, -1, up[above])
    return depth


def _ancestors(st):
    """(sequences, longest, longest): whether new token m is new token i or above it"""
    n, t = len(st["lengths"]), max(st["lengths"])
    i = torch.arange(t, device=DEVICE)
    if st["parents"] is None:
        return (i[None, :] <= i[:, None]).expand(n, t, t)
    reach = torch.eye(t, device=DEVICE).repeat(n, 1, 1)
    parent = torch.full((n, t), -1, device=DEVICE, dtype=torch.long)
    parent[st["of"], st["at"]] = st["parents"].long()
    reach += (parent[:, :, None] == i) * 1.0
    for _ in range(max(1, (t - 1).bit_length())):
        reach = ((reach @ reach) > 0).float()
    return reach > 0


def _plain_append(st):
    case, page = st["case"], st["case"]["page"]
    slot = st["cached"][st["of"]].long() + st["at"]
    pos = st["cached"][st["of"]].long() + _depths(st)
    half = case["rotated"] // 2
    freq = torch.exp(torch.arange(half, device=DEVICE, dtype=torch.float64) * (-math.log(BASE) / half))
    angle = pos[:, None].double() * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotate(x):
        y, r = x.float(), case["rotated"]
        if case["interleaved"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            y = torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), y[..., r:]], -1)
        else:
            a, b = y[..., :half], y[..., half:r]
            y = torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., r:]], -1)
        return y.to(x.dtype)

    pg = st["table"][st["of"], slot // page].long()
    st["k_pages"][pg, slot % page] = rotate(st["k"])
    st["v_pages"][pg, slot % page] = st["v"]
    return rotate(st["q"]), st["k_pages"], st["v_pages"]


def _plain_attention(st):
    case, q = st["case"], st["q"]
    n, t, hk, hq, d = len(st["lengths"]), max(st["lengths"]), case["kv_heads"], case["heads"], case["width"]
    longest = max(c + m for c, m in zip(_numbers(case["cached"]), st["lengths"]))
    slot = torch.arange(longest, device=DEVICE)
    pg = st["table"][:, slot // case["page"]].long()
    kf, vf = (st[x][pg, slot % case["page"]].float().transpose(1, 2) for x in ("k_pages", "v_pages"))      # (n, hk, slots, d)
    qf = torch.zeros(n, t, hq, d, device=DEVICE)
    qf[st["of"], st["at"]] = q.float() * d ** -0.5
    s = qf.reshape(n, t, hk, -1, d).permute(0, 2, 3, 1, 4).flatten(2, 3) @ kf.transpose(-1, -2)              # (n, hk, group t, slots)
    depth = torch.zeros(n, t, device=DEVICE, dtype=torch.long)
    depth[st["of"], st["at"]] = _depths(st)
    length, w = st["cached"].long(), case["window"] or 1 << 40
    at = slot[None] - length[:, None]                                                                        # the slot's new token
    new = ((at >= 0) & (at < st["lens"][:, None]))[:, None]
    m = at.clamp(0, t - 1)
    above = _ancestors(st).gather(2, m[:, None].expand(n, t, longest))
    key_pos = torch.where(at < 0, slot[None], length[:, None] + depth.gather(1, m))
    apart = (length[:, None] + depth)[:, :, None] - key_pos[:, None]
    seen = ((at < 0)[:, None] | (new & above)) & ((apart < w) | (key_pos < case["sinks"])[:, None])         # (n, t, slots)
    s = s.reshape(n, hk, -1, t, longest).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = s.sub_(top).exp_()
    o = (p.flatten(2, 3) @ vf).reshape(n, hk, -1, t, d) / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(n, t, hq, d)[st["of"], st["at"]].to(q.dtype)


def _plain_keep(st):
    page, kept = st["case"]["page"], st["kept"].long()
    j, rows = torch.arange(kept.shape[1], device=DEVICE)[None], torch.arange(kept.shape[0], device=DEVICE)[:, None]
    there = j < st["counts"][:, None]
    length = st["cached"].long()[:, None]
    to = torch.where(there, length + j, length)       # behind a path's end its first token's place, with what that gets
    source = torch.where(there, length + kept, length + kept[:, :1])
    a, b = st["table"][rows, source // page].long(), st["table"][rows, to // page].long()
    for x in ("k_pages", "v_pages"):
        st[x][b, to % page] = st[x][a, source % page]
    return st["k_pages"], st["v_pages"]


def _doubling(a, h):
    """h_t <- a_t h_(t-1) + h_t along the first axis, from pairs twice as far apart each time"""
    s = 1
    while s < a.shape[0]:
        h = torch.cat([h[:s], h[s:] + a[s:] * h[:-s]])
        a = torch.cat([a[:s], a[s:] * a[:-s]])
        s *= 2
    return h


def _plain_recurrence(st):
    """In 64 bits: a decay next to 1 that is rounded to 32 leaves sums of some thousand tokens 1e-5 off."""
    x, first, last = st["x"], st["first"], st["first"] + st["lens"] - 1
    a = torch.exp(st["log_decay"].double().clamp(max=0))
    h, inner = x.double(), a.clone()
    if st["state"] is not None:
        h[first] += a[first] * st["state"]
    inner[first] = 0        # nothing of the sequence before
    h = _doubling(inner, h)
    if "do" not in st:
        return h.to(x.dtype), h[last].float()
    g = st["do"].double()
    if st["dfinal"] is not None:
        g[last] += st["dfinal"]
    nxt = torch.cat([inner[1:], inner[:1] * 0])     # a_(t+1), 0 behind a sequence's last token
    g = _doubling(nxt.flip(0), g.flip(0)).flip(0)
    before = torch.cat([h[:1] * 0, h[:-1]])
    before[first] = st["state"].double() if st["state"] is not None else 0.0
    return h.to(x.dtype), h[last].float(), g.to(x.dtype), (g * a * before).to(x.dtype), (a[first] * g[first]).float()


def _run_plain(st):
    kind = st["case"]["kind"]
    if kind == "append":
        return _plain_append(st)
    if kind == "attention":
        return _plain_attention(st)
    if kind == "keep":
        return _plain_keep(st)
    if kind == "recurrence_step":
        st["state"].mul_(torch.exp(st["log_decay"].float().clamp(max=0))).add_(st["x"])
        return st["state"].to(st["x"].dtype), st["state"]
    return _plain_recurrence(st)


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------------
def _run_own(st):
    from f3m_b200 import paged, sequence
    case, kind = st["case"], st["case"]["kind"]
    if kind == "append":
        q = paged.paged_append(st["plan"], st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["cached"], rotation=st["rotation"],
                               parents=st["parents"], q=st["q"])
        return q, st["k_pages"], st["v_pages"]
    if kind == "attention":
        return paged.paged_attention(st["plan"], st["q"], st["k_pages"], st["v_pages"], st["table"], st["cached"], window=case["window"] or None,
                                     sinks=case["sinks"], parents=st["parents"])
    if kind == "keep":
        paged.paged_keep(st["k_pages"], st["v_pages"], st["table"], st["cached"], st["kept"], st["counts"])
        return st["k_pages"], st["v_pages"]
    if kind == "recurrence_step":
        return sequence.gated_recurrence_step(st["x"], st["log_decay"], st["state"]), st["state"]
    out, final = sequence.gated_recurrence(st["plan"], st["x"], st["log_decay"], st["state"])
    if kind == "recurrence_prompt":
        return out, final
    return (out, final) + tuple(sequence.gated_recurrence_grad(st["plan"], st["log_decay"], out, st["do"], st["state"], st["dfinal"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_depths(case):
    if not case["tree"]:
        return [list(range(n)) for n in _numbers(case["lengths"])]
    depths = []
    for parents in _trees(case):
        d = []
        for p in parents:
            d.append(0 if p < 0 else d[p] + 1)
        depths.append(d)
    return depths


def _slots(case, st, b, slots):
    """Rows of the pages, as one axis, that hold these slots of a sequence"""
    slots = torch.as_tensor(slots, device=DEVICE)
    return st["table"][b].long()[slots // case["page"]] * case["page"] + slots % case["page"]


def _exact_append(case, st):
    r, half, r0 = case["rotated"], case["rotated"] // 2, 0
    x, y = (torch.arange(0, r, 2), torch.arange(1, r, 2)) if case["interleaved"] else (torch.arange(half), torch.arange(half, r))
    turn = torch.tensor([BASE ** (-i / half) for i in range(half)], dtype=torch.float64, device=DEVICE)
    q, k, v = (st[i].double() for i in "qkv")
    kp, vp = st["k_pages"].double(), st["v_pages"].double()
    for b, (length, cached, depths) in enumerate(zip(st["lengths"], _numbers(case["cached"]), _exact_depths(case))):
        z = torch.polar(torch.ones(length, half, device=DEVICE, dtype=torch.float64), (cached + torch.tensor(depths, device=DEVICE))[:, None] * turn)[:, None]
        for a in (q, k):
            part = a[r0:r0 + length]
            w = torch.complex(part[..., x], part[..., y]) * z
            part[..., x], part[..., y] = w.real, w.imag
        rows = _slots(case, st, b, list(range(cached, cached + length)))
        kp.flatten(0, 1)[rows], vp.flatten(0, 1)[rows] = k[r0:r0 + length], v[r0:r0 + length]
        r0 += length
    return q, kp, vp


def _exact_attention(case, st):
    q, r0 = st["q"].double(), 0
    out, group, w = torch.zeros_like(q), case["heads"] // case["kv_heads"], case["window"] or 1 << 40
    trees = _trees(case) if case["tree"] else None
    for b, (length, cached, depths) in enumerate(zip(st["lengths"], _numbers(case["cached"]), _exact_depths(case))):
        rows = _slots(case, st, b, list(range(cached + length)))
        k, v = (st[x].flatten(0, 1)[rows] for x in ("k_pages", "v_pages"))
        pos = torch.tensor(list(range(cached)) + [cached + d for d in depths], device=DEVICE)
        hidden = torch.ones(length, length, dtype=torch.bool)
        for i in range(length):
            if trees is None:
                hidden[i, :i + 1] = False
            else:
                hidden[i] = hidden[trees[b][i]] if trees[b][i] >= 0 else True
                hidden[i, i] = False
        apart = pos[cached:, None] - pos[None]
        hidden = torch.cat([torch.zeros(length, cached, dtype=torch.bool, device=DEVICE), hidden.to(DEVICE)], 1) | ((apart >= w) & (pos >= case["sinks"]))
        for h in range(case["heads"]):
            kh, vh = k[:, h // group].double(), v[:, h // group].double()
            for i in range(0, length, 512):
                s = (q[r0 + i:r0 + min(i + 512, length), h] @ kh.t() * case["width"] ** -0.5).masked_fill(hidden[i:i + 512], -math.inf)
                out[r0 + i:r0 + min(i + 512, length), h] = torch.softmax(s, 1) @ vh
        r0 += length
    return out


def _exact_keep(case, st):
    kp, vp = st["k_pages"].double(), st["v_pages"].double()
    for b, (cached, path) in enumerate(zip(_numbers(case["cached"]), _paths(case))):
        to, source = _slots(case, st, b, [cached + j for j in range(len(path))]), _slots(case, st, b, [cached + m for m in path])
        for x in (kp, vp):
            x.flatten(0, 1)[to] = x.flatten(0, 1)[source].clone()
    return kp, vp


def _exact_recurrence(case, st):
    """Token by token, all sequences at once"""
    n, longest = len(st["lengths"]), max(st["lengths"])
    first = [sum(st["lengths"][:b]) for b in range(n)]
    x = st["x"].double()
    a = torch.exp(torch.minimum(st["log_decay"].double(), torch.zeros((), device=DEVICE, dtype=torch.float64)))
    state = st["state"].double() if st["state"] is not None else torch.zeros(n, x.shape[1], device=DEVICE, dtype=torch.float64)
    out, before = torch.empty_like(x), torch.empty_like(x)
    by_length = sorted(range(n), key=lambda b: -st["lengths"][b])       # those still going on are the first ones
    start, order = torch.tensor([first[b] for b in by_length], device=DEVICE), torch.tensor(by_length, device=DEVICE)
    going = [sum(m > t for m in st["lengths"]) for t in range(longest)]
    h = state[order]
    for t, m in enumerate(going):
        at = start[:m] + t
        before[at] = h[:m]
        h[:m] = a[at] * h[:m] + x[at]
        out[at] = h[:m]
    finals = torch.empty_like(h)
    finals[order] = h
    if case["kind"] == "recurrence_prompt":
        return out, finals
    dx, g = st["do"].double(), torch.zeros_like(h)
    if st["dfinal"] is not None:
        g = st["dfinal"].double()[order]
    for t in range(longest - 1, -1, -1):
        m = going[t]
        at = start[:m] + t
        dx[at] += g[:m]
        g[:m] = a[at] * dx[at]
    dstate = torch.empty_like(g)
    dstate[order] = g
    return out, finals, dx, dx * a * before, dstate


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "append":
        return _exact_append(case, st)
    if kind == "attention":
        return _exact_attention(case, st)
    if kind == "keep":
        return _exact_keep(case, st)
    if kind == "recurrence_step":
        h = st["state"].double() * torch.exp(st["log_decay"].double()) + st["x"].double()
        return h, h
    return _exact_recurrence(case, st)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    lengths = _numbers(case["lengths"])
    total, n, size = sum(lengths), len(lengths), 4 if case["dtype"] == "fp32" else 2
    if case["kind"].startswith("recurrence"):
        channels = case["channels"]
        if case["kind"] == "recurrence_step":
            return {"bytes": n * channels * (3 * size + 8), "flops": 2 * n * channels}
        states = 4 * n * channels * (2 if case["carried"] else 1)
        if case["kind"] == "recurrence_prompt":
            return {"bytes": 3 * size * total * channels + states, "flops": 2 * total * channels}
        # the gradients: log_decay, out and dout in, dx and dlog_decay out
        return {"bytes": 8 * size * total * channels + 2 * states, "flops": 6 * total * channels}
    hq, hk, d, cached = case["heads"], case["kv_heads"], case["width"], _numbers(case["cached"])
    if case["kind"] == "append":
        return {"bytes": 2 * size * total * d * (hq + 2 * hk) + 8 * n, "flops": 3 * total * case["rotated"] * (hq + hk)}
    if case["kind"] == "keep":
        moved = sum(sum(m != j for j, m in enumerate(p)) for p in _paths(case))
        return {"bytes": 4 * size * moved * hk * d + 8 * n + 4 * sum(len(p) for p in _paths(case)), "flops": 0}
    w, sk, pairs, keys = case["window"] or 1 << 40, case["sinks"], 0, 0
    for length, c, depths in zip(lengths, cached, _exact_depths(case)):
        for i, dep in enumerate(depths):
            lo = max(0, c + dep - w + 1)
            before = c - min(lo, c) + min(sk, lo, c)
            among = min(dep + 1, w) + max(0, min(sk, lo) - c)
            pairs += before + among
        lo = max(0, c + min(depths) - w + 1)
        keys += c - min(lo, c) + min(sk, lo, c) + length
    return {"bytes": 2 * size * keys * hk * d + 2 * size * total * hq * d + 8 * n, "flops": 4 * pairs * hq * d}
