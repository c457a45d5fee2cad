"""Cases and plain forms of the quantised paged KV cache operators.

The cache of one layer holds keys and values in 8 or 4 bits, one group per
(token, KV head), in pages of `page` tokens:

    codes   [pages][kv_heads][page][head_dim * bits / 8]  bytes, LSB first
    scales  [pages][kv_heads][page][1]  8 bits: scale
            [pages][kv_heads][page][2]  4 bits: scale, zero

    8 bits: scale = fl32(max|x| / 127),        value = scale * (code - 128)
    4 bits: scale = fl32((max x - min x) / 15), zero = fl32(min x + 8 * scale),
            value = zero + scale * (code - 8)

with code the nearest integer (ties to even).  The operators: new tokens are
quantised as they are written and read back (`append`), and a chunk of new
tokens, or a single one, attends over the paged cache (`attend`): key j is
visible to the query at position i when j <= i and (window == 0 or
j > i - window or j < sinks).

`own` false: the operators as elementary torch operations.  `own` true: the
framework's calls.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(name, kind, seqs, q, kv, heads, kv_heads, dim, bits_k, bits_v, dtype, page=16, window=0, sinks=0,
          singles=0):
    """q and kv: (smallest, largest) new tokens and cache lengths (the new
    tokens among them) of the batch's sequences; `singles` of them bring one
    token."""
    c = dict(kind=kind, seqs=seqs, q_lo=q[0], q_hi=q[1], kv_lo=kv[0], kv_hi=kv[1], heads=heads, kv_heads=kv_heads,
             dim=dim, bits_k=bits_k, bits_v=bits_v, dtype=dtype, page=page, window=window, sinks=sinks,
             singles=singles)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decode token of the engine's own type into one layer's cache
        _case("append_one_f32", "append", 1, (1, 1), (578, 578), 32, 8, 128, 8, 8, "f32"),
        # one decode step of 64 requests
        _case("append_decode64_4bit", "append", 64, (1, 1), (1024, 8192), 32, 8, 128, 4, 4, "bf16"),
        # prompts of four requests, the largest write
        _case("append_prompts", "append", 4, (4097, 12000), (4097, 12000), 32, 8, 128, 8, 8, "bf16"),
        # ragged chunks, half-width heads, keys and values in different widths
        _case("append_ragged_d64", "append", 7, (1, 2500), (13, 5003), 12, 4, 64, 8, 4, "f16", page=32),
        # one request's decode step behind a 512-token prompt: latency
        _case("decode_one", "attend", 1, (1, 1), (577, 577), 32, 8, 128, 8, 8, "bf16"),
        # continuous decode of 64 requests over 4-bit pages
        _case("decode_64", "attend", 64, (1, 1), (1024, 8192), 32, 8, 128, 4, 4, "bf16"),
        # one request far into its context
        _case("decode_long", "attend", 1, (1, 1), (131071, 131071), 64, 8, 128, 8, 8, "f16"),
        # decode with a sliding window and a few first tokens kept visible
        _case("decode_window_f32", "attend", 32, (1, 1), (700, 32768), 12, 4, 64, 8, 4, "f32", page=32, window=1024,
              sinks=4),
        # a 4096-token prompt at once
        _case("prompt_4096", "attend", 1, (4096, 4096), (4096, 4096), 32, 8, 128, 8, 8, "bf16"),
        # chunks of three prompts behind long cached contexts
        _case("chunk_behind_context", "attend", 3, (300, 1024), (5000, 16001), 64, 8, 128, 4, 4, "bf16", page=64),
        # a long prompt under a sliding window with sinks, the largest score matrix
        _case("prompt_window", "attend", 1, (8192, 8192), (8192, 8192), 32, 8, 128, 8, 4, "f16", window=1024,
              sinks=4),
        # the tiny configuration's heads: decode steps and chunks in one batch
        _case("mixed_tiny_f32", "attend", 16, (33, 512), (40, 2000), 8, 4, 32, 8, 8, "f32", singles=10),
    ]


def _lens(case):
    """(new tokens, cache length) of each sequence, spread over the case's range."""
    n = case["seqs"]
    out = []
    for b in range(n):
        f = b / (n - 1) if n > 1 else 1.0
        g = (b * 7 % n) / (n - 1) if n > 1 else 1.0  # another order, so that long chunks meet short contexts
        q = 1 if b < case["singles"] else round(case["q_lo"] + (case["q_hi"] - case["q_lo"]) * f)
        kv = round(case["kv_lo"] + (case["kv_hi"] - case["kv_lo"]) * g)
        out.append((q, max(kv, q)))
    return out


def _pairs(q, kv, window, sinks):
    """Visible (query, key) pairs of q new tokens at the end of kv."""
    if window == 0:
        return q * kv - q * (q - 1) // 2
    total = 0
    for i in range(kv - q, kv):
        lo = max(0, i - window + 1)
        total += i - lo + 1 + min(sinks, lo)
    return total


def _read(q, kv, window, sinks):
    """Keys that at least one of the q queries sees."""
    if window == 0:
        return kv
    lo = max(0, kv - q - window + 1)
    return kv - lo + min(sinks, lo)


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        heads, kv_heads, dim = rng.choice([(8, 4, 32), (32, 8, 128), (64, 8, 128), (12, 4, 64), (16, 16, 64),
                                           (40, 8, 128), (16, 1, 128), (6, 2, 32), (24, 8, 64)])
        bits_k, bits_v = rng.choice([8, 4]), rng.choice([8, 4])
        dtype, page = rng.choice(list(DTYPES)), rng.choice([16, 32, 64, 128])
        kind = rng.choice(["append", "decode", "chunk", "mixed"])
        window, sinks = (0, 0) if rng.random() < 0.5 else (log_int(33, 5000), rng.choice([0, 1, 4, 67]))
        singles = 0
        if kind == "decode":
            seqs, q = log_int(1, 96), (1, 1)
            kv_hi = log_int(40, 100000)
        elif kind == "append":
            seqs, q_hi = log_int(1, 64), log_int(1, 12000)
            q = (max(1, q_hi // rng.randint(1, 9)), q_hi)
            kv_hi = log_int(q_hi, max(q_hi, 16000))
        else:
            seqs, q_hi = log_int(1, 12), log_int(2, 6000)
            q = (max(1, q_hi // rng.randint(1, 9)), q_hi)
            kv_hi = log_int(q_hi, max(q_hi, 40000))
            if kind == "mixed":
                seqs += 1
                singles = rng.randint(1, seqs - 1)
        kv = (max(1, kv_hi // rng.randint(1, 9)), kv_hi)
        case = _case(None, "append" if kind == "append" else "attend", seqs, q, kv, heads, kv_heads, dim, bits_k,
                     bits_v, dtype, page, 0 if kind == "append" else window, 0 if kind == "append" else sinks, singles)
        lens = _lens(case)
        # no more than the largest listed cases: score matrix, cache and new tokens
        if (seqs * max(n for n, _ in lens) * heads * max(t for _, t in lens) <= 8192 * 8192 * 32
                and seqs * max(t for _, t in lens) * kv_heads * dim <= 64 * 8192 * 8 * 128
                and (kind != "append" or sum(n for n, _ in lens) * kv_heads * dim <= 32194 * 8 * 128)):
            return case


def work(case):
    lens, e = _lens(case), DTYPES[case["dtype"]].itemsize
    hkv, d = case["kv_heads"], case["dim"]
    # one (token, head) of the cache: codes, scales (and zeros)
    cached = sum(d * b // 8 + (4 if b == 8 else 8) for b in (case["bits_k"], case["bits_v"]))
    if case["kind"] == "append":
        n = sum(q for q, _ in lens) * hkv
        # new rows read, cache written; cache read back, values written
        return {"bytes": n * (2 * 2 * d * e + 2 * cached), "flops": n * 2 * d * 6}
    w, s = case["window"], case["sinks"]
    rows = sum(q for q, _ in lens) * case["heads"] * d * e
    pages = sum(-(-_read(q, t, w, s) // case["page"]) for q, t in lens)
    return {"bytes": sum(_read(q, t, w, s) for q, t in lens) * hkv * cached + 2 * rows + 4 * pages,
            "flops": 4 * d * case["heads"] * sum(_pairs(q, t, w, s) for q, t in lens)}


def _random_cache(g, pages, hkv, page, d, bits):
    """A side of the cache as earlier tokens left it: normal values around per-channel offsets."""
    x = torch.randn((pages, hkv, page, d), generator=g, device="cuda")
    x += torch.randn((hkv, 1, d), generator=g, device="cuda")
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    if bits == 8:
        scale = torch.maximum(hi, -lo) / 127
        codes = x.div_(scale).round_().add_(128).to(torch.uint8)
        return codes, scale
    scale = (hi - lo) / 15
    codes = x.sub_(lo).div_(scale).round_().to(torch.uint8)
    codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return codes, torch.cat([scale, lo + 8 * scale], -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    lens, dt, d, hkv, page = _lens(case), DTYPES[case["dtype"]], case["dim"], case["kv_heads"], case["page"]
    n = sum(q for q, _ in lens)
    per = max(-(-t // page) for _, t in lens)
    need = [-(-t // page) for _, t in lens]
    pages = sum(need) + 3
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.zeros((len(lens), per), dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = ids[at:at + k]
        at += k
    starts = [0]
    for q, _ in lens:
        starts.append(starts[-1] + q)
    k_codes, k_scales = _random_cache(g, pages, hkv, page, d, case["bits_k"])
    v_codes, v_scales = _random_cache(g, pages, hkv, page, d, case["bits_v"])
    state = dict(case=case, k_codes=k_codes, k_scales=k_scales, v_codes=v_codes, v_scales=v_scales,
                 q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 kv_len=torch.tensor([t for _, t in lens], dtype=torch.int32, device="cuda"),
                 page_table=table.cuda(), max_q=max(q for q, _ in lens), max_kv=max(t for _, t in lens))
    if case["kind"] == "append":
        for x in ("k", "v"):
            new = torch.randn((n, hkv, d), generator=g, device="cuda")
            new += torch.randn((hkv, d), generator=g, device="cuda")
            state[x] = new.to(dt)
    else:
        state["q"] = (1.5 * torch.randn((n, case["heads"], d), generator=g, device="cuda")).to(dt)
    return state


_backend = None


def _handles(state):
    """The cache and batch handles that a program keeps beside its buffers."""
    global _backend
    from nexus_b200 import CudaBackend, KvBatch, PagedKvCache
    if _backend is None:
        _backend = CudaBackend(device=0)
    if "cache" not in state:
        state["cache"] = PagedKvCache(_backend, state["k_codes"], state["k_scales"], state["v_codes"],
                                      state["v_scales"])
        state["batch"] = KvBatch(state["q_start"], state["kv_len"], state["page_table"], state["max_q"],
                                 state["max_kv"])
    return state["cache"], state["batch"]


def _rows(state):
    """(sequence, position) of every new token."""
    start, kv = state["q_start"].long(), state["kv_len"].long()
    new = start[1:] - start[:-1]
    seq = torch.repeat_interleave(torch.arange(len(kv), device="cuda"), new)
    pos = kv[seq] - new[seq] + torch.arange(len(seq), device="cuda") - start[seq]
    return seq, pos


def _quantise(x, bits):
    """Codes and scales of groups over the last axis; quotients in 64 bits,
    so that a scale is rounded once and a code at the border between two is
    the nearer one."""
    x = x.float()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    if bits == 8:
        scale = (torch.maximum(hi, -lo).double() / 127).float()
        zero, top, mid = torch.zeros_like(scale), 127, 128
    else:
        scale = ((hi - lo).double() / 15).float()
        zero, top, mid = lo + 8 * scale, 7, 8
    quotient = (x.double() - zero.double()) / torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    codes = quotient.round().clamp(-top if bits == 8 else -8, top).add(mid).to(torch.uint8)
    if bits == 8:
        return codes, scale
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.cat([scale, zero], -1)


def _values(codes, scales, bits):
    """The 32-bit values that codes and scales stand for, each rounded once."""
    if bits == 8:
        return (codes.float() - 128) * scales
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double() - 8
    return (scales[..., 1:].double() + scales[..., :1].double() * c).float()


def _plain_append(state):
    case, page = state["case"], state["case"]["page"]
    seq, pos = _rows(state)
    at = state["page_table"].long()[seq, pos // page], slice(None), pos % page
    out = {}
    for x in ("k", "v"):
        bits = case["bits_" + x]
        codes, scales = _quantise(state[x], bits)
        state[x + "_codes"][at] = codes
        state[x + "_scales"][at] = scales
        out[x] = _values(state[x + "_codes"][at], state[x + "_scales"][at], bits).to(state[x].dtype)
    return out


def _plain_attend(state):
    case, q = state["case"], state["q"].float()
    hkv, d, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // hkv
    seq, pos = _rows(state)
    row = torch.arange(len(seq), device="cuda") - state["q_start"].long()[seq]
    table, n_seqs, max_q = state["page_table"].long(), len(state["kv_len"]), state["max_q"]
    # [sequences][kv heads][tokens][dim]
    k, v = (_values(state[x + "_codes"][table], state[x + "_scales"][table], case["bits_" + x]).transpose(1, 2)
            .flatten(2, 3) for x in ("k", "v"))
    padded = q.new_zeros((n_seqs, max_q, hkv, group, d))
    padded[seq, row] = q.view(-1, hkv, group, d)
    at = torch.full((n_seqs, max_q), -1, device="cuda")
    at[seq, row] = pos
    s = torch.matmul(padded.permute(0, 2, 3, 1, 4).flatten(2, 3), k.transpose(2, 3)).mul_(1 / math.sqrt(d))
    s = s.view(n_seqs, hkv, group, max_q, -1)
    key = torch.arange(s.shape[-1], device="cuda")
    seen = key <= at[:, :, None]
    if case["window"]:
        seen &= (key > at[:, :, None] - case["window"]) | (key < case["sinks"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).view(n_seqs, hkv, group, max_q, d) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4)[seq, row].flatten(1, 2).to(state["q"].dtype)


def run(state):
    if state["case"]["kind"] == "append":
        if own:
            cache, batch = _handles(state)
            cache.append(batch, state["k"], state["v"])
            k, v = cache.read(batch, state["k"].shape[0], dtype=state["k"].dtype)
            return {"k": k, "v": v}
        return _plain_append(state)
    if own:
        cache, batch = _handles(state)
        return cache.attention(batch, state["q"], window=state["case"]["window"], sinks=state["case"]["sinks"])
    return _plain_attend(state)


def exact(case, seed):
    """The definition in 64 bits, sequence by sequence and head by head."""
    state = prepare(case, seed)
    if case["kind"] == "append":
        out = {}
        for x in ("k", "v"):
            t = state[x].double()
            if case["bits_" + x] == 8:
                step = (t.abs().max(-1, keepdim=True).values / 127).float().double()
                out[x] = step * torch.nan_to_num(t / step).round()
            else:
                low, high = t.min(-1, keepdim=True).values, t.max(-1, keepdim=True).values
                # the range is a 32-bit difference and the zero a 32-bit number, as the cache holds them
                step = ((high - low).float().double() / 15).float().double()
                zero = (low + 8 * step).float().double()
                out[x] = zero + step * torch.nan_to_num((t - zero) / step).round()
        return out
    lens, page, hkv = _lens(case), case["page"], case["kv_heads"]
    group, d, result, at = case["heads"] // hkv, case["dim"], [], 0
    for b, (n, kv) in enumerate(lens):
        ids = state["page_table"][b, :-(-kv // page)].long()
        heads = []
        key = torch.arange(kv, device="cuda")[None]
        i = torch.arange(kv - n, kv, device="cuda")[:, None]
        hidden = key > i
        if case["window"]:
            hidden |= (key <= i - case["window"]) & (key >= case["sinks"])
        for h in range(hkv):
            side = []
            for x in ("k", "v"):
                codes, sc = state[x + "_codes"][ids, h].reshape(-1, state[x + "_codes"].shape[-1])[:kv], \
                    state[x + "_scales"][ids, h].reshape(-1, state[x + "_scales"].shape[-1])[:kv].double()
                if case["bits_" + x] == 8:
                    side.append(sc * (codes.double() - 128))
                else:
                    nib = torch.empty((kv, d), dtype=torch.float64, device="cuda")
                    nib[:, 0::2], nib[:, 1::2] = (codes % 16).double(), (codes // 16).double()
                    side.append(sc[:, 1:] + sc[:, :1] * (nib - 8))
            per_head = []
            for qh in range(h * group, (h + 1) * group):
                score = state["q"][at:at + n, qh].double() @ side[0].T / math.sqrt(d)
                per_head.append(torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ side[1])
            heads.append(torch.stack(per_head, 1))
        result.append(torch.cat(heads, 1))
        at += n
    return torch.cat(result)
