"""Performance cases of the kernel products over sequences: window attention and attention with a decay.

A case is a dict of plain values; `kind` names what is timed:

  window_prompt   window_attention: a batch of sequences, packed, as a prompt is read
  window_train    the same and its gradients
  window_step     window_attention_step: one new token of each sequence against its cache
  decay_prompt    decay_attention: outputs and the state behind the last token
  decay_train     the same and its gradients, the states' among them
  decay_step      decay_attention_step: one new token of each sequence, state updated in place

Sequences are packed: q, k, v are (tokens, heads, width) arrays whose rows are the sequences one after the other.  `lengths` is
a text of their lengths.  Inputs are standard normal, as behind a norm; a head's decay is exp(-2^(-8 (h + 1) / heads)), the
usual geometric series of slopes.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _window(name, kind, dtype, heads, kv_heads, width, window, sinks, lengths, cache=0):
    c = dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, width=width, window=window, sinks=sinks,
             lengths=",".join(str(n) for n in lengths), cache=cache)
    return dict(c, name=name) if name else c


def _decay(name, kind, dtype, heads, width_k, width_v, lengths, carried):
    c = dict(kind=kind, dtype=dtype, heads=heads, width_k=width_k, width_v=width_v, lengths=",".join(str(n) for n in lengths),
             carried=carried)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the smallest prompt: one short question, odd length, few heads; latency counts
        _window("window_prompt_short", "window_prompt", "fp16", 8, 2, 64, 128, 4, [129]),
        # prompts of a batch of requests as they come, one of a single token among them
        _window("window_prompt_ragged", "window_prompt", "bf16", 32, 8, 128, 1024, 4, [4096, 1021, 1, 2500, 57, 333, 1600, 513]),
        # one long document
        _window("window_prompt_long", "window_prompt", "bf16", 16, 4, 128, 4096, 16, [16384]),
        # a training step on documents packed to one row
        _window("window_train_packed", "window_train", "bf16", 16, 4, 64, 512, 8, [2048, 1500, 777, 3000, 867]),
        # the same at the width of the larger models, one head of keys for each of queries
        _window("window_train_wide", "window_train", "fp16", 8, 8, 128, 2048, 0, [4096, 4000]),
        # one conversation, one token
        _window("window_step_one", "window_step", "bf16", 8, 2, 64, 1024, 4, [1500], cache=2048),
        # a serving batch behind conversations of many lengths
        _window("window_step_batch", "window_step", "bf16", 32, 8, 128, 4096, 4,
                [16384 - 509 * (i % 31) - 37 * i for i in range(31)] + [2], cache=16384),
        # a short prompt, odd length
        _decay("decay_prompt_short", "decay_prompt", "fp16", 8, 64, 64, [129], False),
        # prompts of a batch of requests
        _decay("decay_prompt_ragged", "decay_prompt", "bf16", 32, 128, 128, [8192, 2021, 1, 5000, 57, 333, 3200, 1025], True),
        # one long document on few heads: the work is split over its length
        _decay("decay_prompt_long", "decay_prompt", "bf16", 8, 128, 128, [65536], False),
        # a training step on packed documents
        _decay("decay_train_packed", "decay_train", "bf16", 16, 128, 128, [4096, 1500, 777, 5000, 1011], True),
        # a serving batch
        _decay("decay_step_batch", "decay_step", "bf16", 32, 128, 128, [1] * 64, True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("window_prompt", "window_train", "window_step", "decay_prompt", "decay_train", "decay_step"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind.startswith("window"):
        kv = rng.choice((1, 2, 4, 8))
        heads, width = kv * rng.choice((1, 2, 4, 8)), rng.choice((32, 64, 80, 96, 128))
        sinks = rng.choice((0, 1, 4, 16, rng.randint(2, 200)))
        if kind == "window_step":
            cache = _log_uniform(rng, 64, 32768)
            n = _log_uniform(rng, 1, max(1, min(128, (1 << 19) // cache)))
            window = rng.choice((cache, _log_uniform(rng, 16, cache)))
            lengths = [_log_uniform(rng, 1, cache) if rng.random() < 0.3 else rng.randint(max(1, cache // 2), cache) for _ in range(n)]
            return _window("", kind, dtype, heads, kv, width, window, sinks, lengths, cache)
        top = 8192 if kind == "window_prompt" else 4096
        longest = _log_uniform(rng, 16, top)
        # the plain form holds heads * sequences * longest^2 numbers: no more than the largest listed case's
        room = int((2e9 if kind == "window_prompt" else 5e8) // (heads * longest * longest))
        n = rng.randint(1, max(1, min(8, room)))
        lengths = [longest] + [_log_uniform(rng, 1, longest) for _ in range(n - 1)]
        return _window("", kind, dtype, heads, kv, width, _log_uniform(rng, 8, 4096), sinks, lengths)
    heads = rng.choice((1, 2, 4, 8, 12, 16, 32))
    width_k, width_v = rng.choice((32, 64, 96, 128)), rng.choice((32, 64, 96, 128))
    if kind == "decay_step":
        return _decay("", kind, dtype, heads, width_k, width_v, [1] * _log_uniform(rng, 1, 64), True)
    longest = _log_uniform(rng, 16, 32768 if kind == "decay_prompt" else 8192)
    n = rng.randint(1, max(1, min(8, (1 << 19) // (heads * longest))))
    lengths = [longest] + [_log_uniform(rng, 1, longest) for _ in range(n - 1)]
    return _decay("", kind, dtype, heads, width_k, width_v, lengths, rng.random() < 0.5)


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------------------------------------
class _Packing:
    """Where the tokens of packed sequences lie in a padded (sequences, longest) array, and back; `order` -1 from the end."""

    def __init__(self, lengths, device):
        n, longest = len(lengths), max(lengths)
        lens = torch.tensor(lengths, device=device)
        first = torch.cumsum(lens, 0) - lens
        at = torch.arange(longest, device=device)
        self.lens, self.n, self.longest, self.total = lens, n, longest, sum(lengths)
        self.there = at[None, :] < lens[:, None]
        last = self.total - 1
        self.forward = (first[:, None] + at).clamp(max=last)
        self.backward = (first[:, None] + lens[:, None] - 1 - at).clamp(0, last)
        self.of = torch.repeat_interleave(torch.arange(n, device=device), lens)
        self.pos = torch.arange(self.total, device=device) - first[self.of]
        self.rpos = lens[self.of] - 1 - self.pos

    def pad(self, x, back=False):
        """(tokens, heads, width) -> (sequences, heads, longest, width), zero behind the last token, in 32 bits."""
        y = x[self.backward if back else self.forward].float()
        return (y * self.there[:, :, None, None]).transpose(1, 2)

    def unpad(self, y, back=False):
        return y[self.of, :, self.rpos if back else self.pos]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, lengths = TYPES[case["dtype"]], _lengths(case)
    total, n = sum(lengths), len(lengths)

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)

    st = dict(case=case, lengths=lengths)
    if case["kind"] == "window_step":
        hq, hk, d = case["heads"], case["kv_heads"], case["width"]
        st |= dict(q=normal(n, hq, d), k=normal(n, case["cache"], hk, d), v=normal(n, case["cache"], hk, d),
                   lens=torch.tensor(lengths, device=DEVICE, dtype=torch.int32))
    elif case["kind"].startswith("window"):
        hq, hk, d = case["heads"], case["kv_heads"], case["width"]
        st |= dict(q=normal(total, hq, d), k=normal(total, hk, d), v=normal(total, hk, d))
        if case["kind"] == "window_train":
            st["do"] = normal(total, hq, d)
    else:
        h, dk, dv = case["heads"], case["width_k"], case["width_v"]
        st |= dict(q=normal(total, h, dk), k=normal(total, h, dk), v=normal(total, h, dv),
                   log_decay=-torch.exp2(-8.0 * torch.arange(1, h + 1, device=DEVICE, dtype=torch.float32) / h))
        st["state"] = normal(n, h, dk, dv, dtype=torch.float32) if case["carried"] else None
        if case["kind"] == "decay_train":
            st["do"] = normal(total, h, dv)
            st["dfinal"] = normal(n, h, dk, dv, dtype=torch.float32) if case["carried"] else None
    if not case["kind"].endswith("step"):
        if own:
            from f3m_b200 import sequence
            st["plan"] = sequence.SequencePlan(lengths, device=DEVICE)
        else:
            st["packing"] = _Packing(lengths, DEVICE)
    return st


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _scores(case, pk, q, k):
    """exponents, -inf where a key is not visible: (sequences, kv_heads, group, longest, longest)"""
    n, hk, d, t = pk.n, case["kv_heads"], case["width"], pk.longest
    s = (pk.pad(q) * d ** -0.5).reshape(n, hk, -1, t, d) @ pk.pad(k).reshape(n, hk, 1, t, d).transpose(-1, -2)
    i, j = torch.arange(t, device=DEVICE)[:, None], torch.arange(t, device=DEVICE)[None, :]
    seen = (j <= i) & ((i - j < case["window"]) | (j < case["sinks"]))
    return s.masked_fill_(~seen, -math.inf)


def _plain_window(case, pk, q, k, v, do=None):
    n, hk, hq, d, t = pk.n, case["kv_heads"], case["heads"], case["width"], pk.longest
    s = _scores(case, pk, q, k)
    top = s.amax(-1, keepdim=True)
    p = (s - top).exp_()
    del s
    total = p.sum(-1, keepdim=True)
    vf = pk.pad(v).reshape(n, hk, 1, t, d)
    o = (p @ vf) / total
    out = pk.unpad(o.reshape(n, hq, t, d)).to(q.dtype)
    lse = pk.unpad((top + total.log()).reshape(n, hq, t, 1))[:, :, 0].t().contiguous()
    if do is None:
        return out, lse
    p /= total
    g = pk.pad(do).reshape(n, hk, -1, t, d)
    dv = (p.transpose(-1, -2) @ g).sum(2)
    ds = p * (g @ vf.transpose(-1, -2) - (g * o).sum(-1, keepdim=True)) * d ** -0.5
    dq = ds @ pk.pad(k).reshape(n, hk, 1, t, d)
    dk = (ds.transpose(-1, -2) @ pk.pad(q).reshape(n, hk, -1, t, d)).sum(2)
    return out, lse, pk.unpad(dq.reshape(n, hq, t, d)).to(q.dtype), pk.unpad(dk).to(k.dtype), pk.unpad(dv).to(v.dtype)


def _plain_window_step(case, q, k, v, lens):
    n, hk, d, w, sk = q.shape[0], case["kv_heads"], case["width"], min(case["window"], k.shape[1]), case["sinks"]
    lens = lens.long()
    back = lens[:, None] - 1 - torch.arange(w, device=DEVICE)          # the window, newest first
    first = torch.arange(sk, device=DEVICE).expand(n, sk)              # the sinks, those that the window does not hold
    at = torch.cat([back, first], 1)
    seen = torch.cat([back >= 0, (first < lens[:, None]) & (lens[:, None] - 1 - first >= w)], 1)
    rows = torch.arange(n, device=DEVICE)[:, None]
    at = at.clamp(0, k.shape[1] - 1)
    kf, vf = k[rows, at].float().transpose(1, 2), v[rows, at].float().transpose(1, 2)      # (n, hk, keys, d)
    s = (q.float() * d ** -0.5).reshape(n, hk, -1, d) @ kf.transpose(-1, -2)
    s = s.masked_fill_(~seen[:, None, None, :], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    o = (p @ vf) / p.sum(-1, keepdim=True)
    return o.reshape(q.shape).to(q.dtype)


CHUNK = 128


def _power(log_decay, n):
    """decay^n for whole n >= 0, by head: (heads, *n.shape)"""
    return torch.exp(log_decay.double().reshape(-1, *[1] * n.dim()) * n.double()).float()


def _plain_decay(log_decay, q, k, v, start, undecayed=False):
    """o_i = sum_(j <= i) decay^(i - j) (q_i . k_j) v_j + decay^(i + 1) q_i start on padded (sequences, heads, longest, width)
    arrays; with `undecayed` the start enters as decay^i."""
    n, h, t, dk = q.shape
    dv, nc = v.shape[-1], -(-t // CHUNK)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, nc * CHUNK - t)).reshape(n, h, nc, CHUNK, -1) for x in (q, k, v))
    i = torch.arange(CHUNK, device=DEVICE)
    apart = i[:, None] - i[None, :]
    inner = _power(log_decay, apart.clamp(min=0)) * (apart >= 0)
    o = ((q @ k.transpose(-1, -2)) * inner[:, None]) @ v
    made = (k * _power(log_decay, CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2) @ v           # (n, h, nc, dk, dv)
    a = torch.arange(nc, device=DEVICE)
    gone = a[:, None] - 1 - a[None, :]
    carry = _power(log_decay, gone.clamp(min=0) * CHUNK) * (gone >= 0)
    before = (carry @ made.reshape(n, h, nc, dk * dv)).reshape(n, h, nc, dk, dv)
    o += (q * _power(log_decay, i + 1)[:, None, :, None]) @ before
    if start is not None:
        steps = (torch.arange(nc * CHUNK, device=DEVICE) + (0 if undecayed else 1)).reshape(nc, CHUNK)
        o += (q * _power(log_decay, steps)[..., None]) @ start[:, :, None]
    return o.reshape(n, h, nc * CHUNK, dv)[:, :, :t]


def _plain_last(log_decay, k, v, lens, start, more=0):
    """sum_j decay^(length - 1 - j + more) k_j v_j^T + decay^length start"""
    left = lens[:, None] - 1 - torch.arange(k.shape[2], device=DEVICE)[None, :]
    w = _power(log_decay, left.clamp(min=0) + more).transpose(0, 1)[..., None]
    last = (k * w).transpose(-1, -2) @ v
    return last if start is None else last + _power(log_decay, lens).t()[..., None, None] * start


def _plain_decay_attention(pk, q, k, v, log_decay, start, do=None, dfinal=None):
    scale = q.shape[-1] ** -0.5
    qf, kf, vf = pk.pad(q) * scale, pk.pad(k), pk.pad(v)
    out = pk.unpad(_plain_decay(log_decay, qf, kf, vf, start)).to(q.dtype)
    final = _plain_last(log_decay, kf, vf, pk.lens, start)
    if do is None:
        return out, final
    gf = pk.pad(do)
    dq = _plain_decay(log_decay, gf, vf, kf, None if start is None else start.transpose(-1, -2)) * scale
    qb, kb, vb, gb = pk.pad(q, True) * scale, pk.pad(k, True), pk.pad(v, True), pk.pad(do, True)
    dk = _plain_decay(log_decay, vb, gb, qb, None if dfinal is None else dfinal.transpose(-1, -2), True)
    dv = _plain_decay(log_decay, kb, qb, gb, dfinal, True)
    dstart = _plain_last(log_decay, qb, gb, pk.lens, dfinal, 1)
    return (out, final, pk.unpad(dq).to(q.dtype), pk.unpad(dk, True).to(k.dtype), pk.unpad(dv, True).to(v.dtype), dstart)


def _plain_decay_step(q, k, v, log_decay, state):
    state.mul_(torch.exp(log_decay)[:, None, None]).add_(k.float()[..., None] * v.float()[..., None, :])
    o = ((q.float() * q.shape[-1] ** -0.5)[..., None, :] @ state)[..., 0, :]
    return o.to(q.dtype), state


def _run_plain(st):
    case, kind = st["case"], st["case"]["kind"]
    if kind == "window_step":
        return _plain_window_step(case, st["q"], st["k"], st["v"], st["lens"])
    if kind.startswith("window"):
        return _plain_window(case, st["packing"], st["q"], st["k"], st["v"], st.get("do"))
    if kind == "decay_step":
        return _plain_decay_step(st["q"], st["k"], st["v"], st["log_decay"], st["state"])
    return _plain_decay_attention(st["packing"], st["q"], st["k"], st["v"], st["log_decay"], st["state"], st.get("do"), st.get("dfinal"))


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------------
def _run_own(st):
    from f3m_b200 import sequence as sq
    case, kind = st["case"], st["case"]["kind"]
    q, k, v = st["q"], st["k"], st["v"]
    if kind == "window_step":
        return sq.window_attention_step(q, k, v, st["lens"], case["window"], case["sinks"])
    if kind.startswith("window"):
        out, lse = sq.window_attention(st["plan"], q, k, v, case["window"], case["sinks"])
        if kind == "window_prompt":
            return out, lse
        return (out, lse) + tuple(sq.window_attention_grad(st["plan"], q, k, v, out, lse, st["do"], case["window"], case["sinks"]))
    if kind == "decay_step":
        return sq.decay_attention_step(q, k, v, st["log_decay"], st["state"]), st["state"]
    out, final = sq.decay_attention(st["plan"], q, k, v, st["log_decay"], st["state"])
    if kind == "decay_prompt":
        return out, final
    return (out, final) + tuple(sq.decay_attention_grad(st["plan"], q, k, v, st["log_decay"], st["do"], st["state"], st["dfinal"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_window(case, st):
    """Sequence by sequence, head by head, block of queries by block of queries, over the keys from the first to the last seen."""
    grads = case["kind"] == "window_train"
    group, w, sk, scale = case["heads"] // case["kv_heads"], case["window"], case["sinks"], case["width"] ** -0.5
    q, k, v = (st[x].double() for x in "qkv")
    out, lse = torch.empty_like(q), torch.empty(q.shape[1], q.shape[0], device=DEVICE, dtype=torch.float64)
    do = st["do"].double() if grads else None
    dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v)) if grads else (None,) * 3
    r0 = 0
    for length in st["lengths"]:
        for b0 in range(0, length, 2048):
            b1 = min(length, b0 + 2048)
            lo = max(0, b0 - w + 1)
            keys = torch.cat([torch.arange(0, min(sk, lo), device=DEVICE), torch.arange(lo, b1, device=DEVICE)])
            i = torch.arange(b0, b1, device=DEVICE)[:, None]
            hidden = (keys[None] > i) | ((i - keys[None] >= w) & (keys[None] >= sk))
            for h in range(case["heads"]):
                qa, ka, va = q[r0 + b0:r0 + b1, h], k[r0 + keys, h // group], v[r0 + keys, h // group]
                s = (qa @ ka.t() * scale).masked_fill(hidden, -math.inf)
                z = torch.logsumexp(s, 1)
                p = torch.exp(s - z[:, None])
                out[r0 + b0:r0 + b1, h], lse[h, r0 + b0:r0 + b1] = p @ va, z
                if grads:
                    ga = do[r0 + b0:r0 + b1, h]
                    e = ga @ va.t()
                    e = p * (e - (p * e).sum(1, keepdim=True)) * scale
                    dq[r0 + b0:r0 + b1, h] = e @ ka
                    dk[:, h // group].index_add_(0, r0 + keys, e.t() @ qa)
                    dv[:, h // group].index_add_(0, r0 + keys, p.t() @ ga)
        r0 += length
    return (out, lse, dq, dk, dv) if grads else (out, lse)


def _exact_window_step(case, st):
    group, w, sk = case["heads"] // case["kv_heads"], case["window"], case["sinks"]
    out = torch.zeros(st["q"].shape, device=DEVICE, dtype=torch.float64)
    for b, length in enumerate(st["lengths"]):
        lo = max(0, length - w)
        k, v = (torch.cat([st[x][b, :min(sk, lo)], st[x][b, lo:length]]).double().repeat_interleave(group, 1) for x in "kv")
        p = torch.softmax(torch.einsum("hd,khd->hk", st["q"][b].double(), k) * case["width"] ** -0.5, 1)
        out[b] = torch.einsum("hk,khd->hd", p, v)
    return out


def _exact_decay(case, st):
    """The recurrence S <- decay S + k v^T, o = q S, whole blocks of it at a time, and the adjoint recurrence from the end."""
    grads, scale, ld = case["kind"] == "decay_train", case["width_k"] ** -0.5, st["log_decay"].double()
    q, k, v = (st[x].double().transpose(0, 1) for x in "qkv")          # (heads, tokens, width)
    q = q * scale
    do = st["do"].double().transpose(0, 1) if grads else None
    out = torch.empty_like(v)
    dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
    finals, dstarts, r0, block = [], [], 0, 512
    for b, length in enumerate(st["lengths"]):
        S = st["state"][b].double() if st["state"] is not None else torch.zeros(q.shape[0], q.shape[2], v.shape[2], device=DEVICE, dtype=torch.float64)
        for a in range(0, length, block):
            m = min(block, length - a)
            at, i = slice(r0 + a, r0 + a + m), torch.arange(m, device=DEVICE, dtype=torch.float64)
            L = torch.exp(ld[:, None, None] * (i[:, None] - i[None, :]).clamp(min=0)).tril()
            since = torch.exp(ld[:, None, None] * (i + 1)[:, None])
            till = torch.exp(ld[:, None, None] * (m - 1 - i)[:, None])
            out[:, at] = (L * (q[:, at] @ k[:, at].mT)) @ v[:, at] + since * (q[:, at] @ S)
            if grads:
                dq[:, at] = ((L * (do[:, at] @ v[:, at].mT)) @ k[:, at] + since * (do[:, at] @ S.mT)) * scale
            S = torch.exp(ld * m)[:, None, None] * S + (till * k[:, at]).mT @ v[:, at]
        finals.append(S)
        if grads:
            # D is the gradient of the state behind the block's last token
            D = st["dfinal"][b].double() if st["dfinal"] is not None else torch.zeros_like(S)
            for a in reversed(range(0, length, block)):
                m = min(block, length - a)
                at, i = slice(r0 + a, r0 + a + m), torch.arange(m, device=DEVICE, dtype=torch.float64)
                L = torch.exp(ld[:, None, None] * (i[:, None] - i[None, :]).clamp(min=0)).tril()
                since = torch.exp(ld[:, None, None] * (i + 1)[:, None])
                till = torch.exp(ld[:, None, None] * (m - 1 - i)[:, None])
                dk[:, at] = (L * (do[:, at] @ v[:, at].mT)).mT @ q[:, at] + till * (v[:, at] @ D.mT)
                dv[:, at] = (L * (q[:, at] @ k[:, at].mT)).mT @ do[:, at] + till * (k[:, at] @ D)
                D = torch.exp(ld * m)[:, None, None] * D + (since * q[:, at]).mT @ do[:, at]
            dstarts.append(D)
        r0 += length
    out, finals = out.transpose(0, 1).contiguous(), torch.stack(finals)
    if not grads:
        return out, finals
    return (out, finals) + tuple(x.transpose(0, 1).contiguous() for x in (dq, dk, dv)) + (torch.stack(dstarts),)


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "window_step":
        return _exact_window_step(case, st)
    if kind.startswith("window"):
        return _exact_window(case, st)
    if kind == "decay_step":
        S = st["state"].double() * torch.exp(st["log_decay"].double())[:, None, None] + torch.einsum("bhk,bhv->bhkv", st["k"].double(), st["v"].double())
        return torch.einsum("bhk,bhkv->bhv", st["q"].double(), S) * case["width_k"] ** -0.5, S
    return _exact_decay(case, st)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def _seen(case, length):
    """(query, key) pairs of one sequence"""
    w, sk = case["window"], case["sinks"]
    near = sum(min(i + 1, w) for i in range(length)) if length <= w else w * (w + 1) // 2 + (length - w) * w
    far = sum(min(sk, i + 1 - w) for i in range(w, length)) if sk and length > w else 0
    return near + far


def work(case):
    lengths, kind = _lengths(case), case["kind"]
    total, n = sum(lengths), len(lengths)
    if kind == "window_step":
        hq, hk, d = case["heads"], case["kv_heads"], case["width"]
        keys = sum(min(x, case["window"]) + max(0, min(case["sinks"], x - case["window"])) for x in lengths)
        return {"bytes": 2 * (2 * keys * hk * d + 2 * n * hq * d) + 4 * n, "flops": 4 * keys * hq * d}
    if kind.startswith("window"):
        hq, hk, d = case["heads"], case["kv_heads"], case["width"]
        pairs = sum(_seen(case, x) for x in lengths)
        nbytes = 2 * total * d * (2 * hq + 2 * hk) + 4 * total * hq
        if kind == "window_train":      # and dout, dq, dk, dv; the gradients take five products to the forward's two
            nbytes += 2 * total * d * (2 * hq + 2 * hk)
        return {"bytes": nbytes, "flops": pairs * hq * d * (14 if kind == "window_train" else 4)}
    h, dk, dv = case["heads"], case["width_k"], case["width_v"]
    state = 4 * n * h * dk * dv
    if kind == "decay_step":
        return {"bytes": 2 * n * h * (2 * dk + 2 * dv) + 2 * state, "flops": 5 * n * h * dk * dv}
    nbytes = 2 * total * h * (2 * dk + 2 * dv) + state * (2 if case["carried"] else 1)
    flops = 4 * total * h * dk * dv     # the recurrence: state and output, a multiply-add each by entry of the state
    if kind == "decay_train":
        nbytes += 2 * total * h * (2 * dk + 2 * dv) + state * (2 if case["carried"] else 1)
        flops *= 3
    return {"bytes": nbytes, "flops": flops}
