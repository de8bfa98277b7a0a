"""Linear attention with a decay for each head, and the rotation of queries and keys, measured through the public API.

Linear attention. With lambda = exp(-decay[h]) a head of queries holds a state of Dk x Dv values,

    S_t = lambda S_{t-1} + k_t v_t^T,     o_t = scale q_t^T S_t = scale sum_{s<=t} lambda^(t-s) (q_t . k_s) v_s,

and several heads of queries may share one head of keys and values. Five operators:

  train   linear_attn_func / linear_attn_varlen_func and their backward pass: dense and packed batches
  prompt  linear_attn_func / linear_attn_varlen_func, an initial state in and the final state out
  step    linear_attn_with_state: one new token or a few, the states of a pool updated in place
  rotary  flash_attn_rotary_func: queries and keys of a padded or packed batch rotated by the rows of two
          tables at each token's position, and (training) the gradients rotated back
  tables  flash_attn_rotary_tables: the cosines and sines of all positions, frequencies scaled for contexts
          longer than the trained ones

Queries and keys are SiLU(N(0, 1)), values N(0, 1), as the projections of such layers have them; the
decays are 2^(-8 i / H), i = 1..H, those of the linear biases that flash_attn_func takes (memories of
one token to hundreds), over `slow` (1: as they are; 16: contexts of thousands).
"""
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(ROOT, "flash-attention-rdna2_amd")

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _case(name, op, dtype, **kw):
    """A case with every field present: sequences of lo..hi tokens (packed) or hi (padded), hq / hk heads of dk
    (queries, keys) and dv (values) columns. rotary: dk the head dim, rd the rotated part, positions from up to
    `past`; tables: hi rows of rd / 2 values."""
    c = {"op": op, "dtype": dtype, "batch": 1, "lo": 1, "hi": 1, "packed": False, "hq": 1, "hk": 1, "dk": 128, "dv": 128,
         "slow": 1, "carry": False, "rd": 0, "interleaved": False, "past": 0, "grad": False, "factor": 1.0, "trained": 0}
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # A training step's layer on the batch of the benchmark's backward (B 2, S 4096, 32 heads of 128).
        _case("train_dense", "train", "bf16", batch=2, hi=4096, hq=32, hk=32),
        # Training on packed documents of unequal lengths, small heads.
        _case("train_packed", "train", "fp16", batch=24, lo=64, hi=2048, packed=True, hq=16, hk=16, dk=64, dv=64),
        # A small layer kept in 32 bits, keys and values shared by four heads of queries, values wider than keys.
        _case("train_shared_fp32", "train", "fp32", batch=2, hi=1000, hq=16, hk=4, dk=64, dv=128),
        # One long document read in one go; its final state is what the answer goes on from.
        _case("prompt_long", "prompt", "bf16", batch=1, hi=32768, hq=32, hk=32, slow=16),
        # The next chunks of eight requests' prompts, packed, behind states of what came before.
        _case("prompt_packed", "prompt", "bf16", batch=8, lo=16, hi=2048, packed=True, hq=32, hk=8, carry=True),
        # One request being answered: latency.
        _case("step_one", "step", "bf16", batch=1, hq=32, hk=32),
        # A serving batch in flight.
        _case("step_batch", "step", "bf16", batch=48, hq=64, hk=64, slow=16),
        # Four drafted tokens of eight requests, wide heads.
        _case("step_draft", "step", "fp16", batch=8, hi=4, hq=16, hk=4, dk=256, dv=256),
        # The queries and keys of a training step's exact attention, and their gradients.
        _case("rotary_train", "rotary", "bf16", batch=2, hi=4096, hq=32, hk=8, rd=128, grad=True),
        # One decoding step's new token of 48 requests, a quarter of each head rotated: latency.
        _case("rotary_step", "rotary", "fp16", batch=48, hi=1, hq=64, hk=8, rd=32, interleaved=True, past=8000),
        # Tables for four times the trained context.
        _case("tables_long", "tables", "fp32", hi=131072, rd=128, factor=4.0, trained=32768),
        # Tables of a short context, unscaled: the smallest work.
        _case("tables_short", "tables", "fp32", hi=2048, rd=64),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above."""
    op = rng.choice(["train"] * 3 + ["prompt"] * 2 + ["step"] * 3 + ["rotary"] * 2 + ["tables"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    hk = rng.choice([1, 2, 4, 8, 16, 32])
    hq = hk * rng.choice([1, 1, 1, 2, 4])
    wide = [32, 64, 80, 96, 128, 128, 192, 256]
    dk = rng.choice(wide)
    dv = rng.choice([dk, dk, rng.choice(wide)])
    kw = {"hq": hq, "hk": hk, "dk": dk, "dv": dv, "slow": rng.choice([1, 1, 4, 16])}
    if op in ("train", "prompt"):
        hi = _log_int(rng, 16, 4096 if op == "train" else 32768)
        room = (1 << 25) // (hq * max(dk, dv) * (2 if dtype == "fp32" else 1))         # tokens
        hi = min(hi, room)
        kw.update(batch=_log_int(rng, 1, max(1, min(24, room // hi))), hi=hi, packed=rng.random() < 0.6)
        kw.update(lo=max(1, hi // 32) if kw["packed"] else hi, carry=op == "prompt" and rng.random() < 0.6)
    elif op == "step":
        kw.update(hi=rng.choice([1, 1, 1, rng.randint(2, 8)]), batch=_log_int(rng, 1, max(1, min(64, 48 * 64 * 16384 // (hq * dk * dv)))))
        kw["lo"] = kw["hi"]
    elif op == "rotary":
        rd = rng.choice([dk, dk, dk // 2, 16 * rng.randint(1, dk // 16)])
        hi = rng.choice([1, _log_int(rng, 2, 8192)])
        kw.update(hi=hi, batch=_log_int(rng, 1, max(1, min(64, (1 << 25) // (hi * hq * dk)))), packed=rng.random() < 0.5, rd=rd,
                  interleaved=rng.random() < 0.5, past=rng.choice([0, _log_int(rng, 16, 30000)]), grad=rng.random() < 0.6, dv=dk)
        kw["lo"] = max(1, hi // 16) if kw["packed"] else hi
    else:
        scaled = rng.random() < 0.7
        kw = {"hi": _log_int(rng, 512, 131072), "rd": 2 * rng.randint(8, 64), "factor": rng.choice([2.0, 4.0, 8.0, 2.5]) if scaled else 1.0,
              "trained": rng.choice([0, 4096, 8192, 32768]) if scaled else 0}
        dtype = "fp32"
    return _case(None, op, dtype, **kw)


# ----------------------------------------------------------------------------- sizes of a case
def _lengths(case):
    """The sequences' token counts, the same for every seed; the longest is hi."""
    if not case["packed"]:
        return [case["hi"]] * case["batch"]
    r = random.Random(11)
    v = [r.randint(min(case["lo"], case["hi"]), case["hi"]) for _ in range(case["batch"])]
    v[r.randrange(len(v))] = case["hi"]
    return v


def work(case):
    """Linear attention by its recurrence: 4 Dk Dv operations per token and head (the state's update, the output),
    10 more for the gradients (the state again, its gradient, dq, dk, dv). Bytes: every input read and every
    output written once."""
    n, b, e = sum(_lengths(case)), case["batch"], 4 if case["dtype"] == "fp32" else 2
    hq, hk, dk, dv, op = case["hq"], case["hk"], case["dk"], case["dv"], case["op"]
    if op == "tables":
        return {"bytes": 4 * case["hi"] * case["rd"], "flops": 2 * case["hi"] * case["rd"]}
    if op == "rotary":
        times = 2 if case["grad"] else 1
        rows = (case["past"] + case["hi"]) if n > case["past"] + case["hi"] else n
        return {"bytes": times * 2 * e * n * (hq + hk) * dk + 4 * rows * case["rd"], "flops": times * 3 * n * (hq + hk) * case["rd"]}
    rows = e * n * (hq * (dk + dv) + hk * (dk + dv))
    if op == "train":          # q, k, v and dout read, out and the gradients written
        return {"bytes": 2 * rows, "flops": 14 * n * hq * dk * dv}
    state = 4 * b * hq * dk * dv
    return {"bytes": rows + state * (2 if case["carry"] or op == "step" else 1), "flops": 4 * n * hq * dk * dv}


# ----------------------------------------------------------------------------- inputs
def _cu(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    """What a program holds before the call: activations, decays, states and their slots, tables and lengths."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, b, hq, hk, dk, dv = _DT[case["dtype"]], case["batch"], case["hq"], case["hk"], case["dk"], case["dv"]
    s = {"case": case, "max_n": case["hi"]}
    if case["op"] == "tables":
        # A base of its own for every seed: the tables have no other input.
        s["base"] = 10000.0 + 1000.0 * (seed % 97)
        return s
    lens = _lengths(case)
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    rows = (sum(lens),) if case["packed"] else (b, case["hi"])
    s["cu"] = _cu(lens) if case["packed"] else None
    if case["op"] == "rotary":
        # Queries and keys are columns of one projection's output.
        x = rand(*rows, hq + 2 * hk, dk).to(dt)
        s["q"], s["k"] = x[..., :hq, :], x[..., hq:hq + hk, :]
        pos = torch.arange(case["past"] + case["hi"], device="cuda", dtype=torch.float64)[:, None]
        freq = 10000.0 ** (-torch.arange(0, case["rd"], 2, device="cuda", dtype=torch.float64) / case["rd"])
        s["cos"], s["sin"] = torch.cos(pos * freq).float(), torch.sin(pos * freq).float()
        s["start"] = torch.randint(0, case["past"] + 1, (b,), generator=gen, device="cuda", dtype=torch.int32) if case["past"] else None
        if case["grad"]:
            s["q"].requires_grad_(), s["k"].requires_grad_()
            s["dq"], s["dk"] = rand(*rows, hq, dk).to(dt), rand(*rows, hk, dk).to(dt)
        return s
    silu = lambda x: x * torch.sigmoid(x)
    s["q"], s["k"], s["v"] = silu(rand(*rows, hq, dk)).to(dt), silu(rand(*rows, hk, dk)).to(dt), rand(*rows, hk, dv).to(dt)
    s["decay"] = torch.exp2(-8.0 * torch.arange(1, hq + 1, device="cuda") / hq) / case["slow"]
    if case["op"] == "train":
        s["dout"] = rand(*rows, hq, dv).to(dt)
        for x in ("q", "k", "v"):
            s[x].requires_grad_()
    if case["carry"]:
        s["first"] = 4 * rand(b, hq, dk, dv)
    if case["op"] == "step":
        # A pool of states with a few slots to spare, the requests in any order.
        s["pool"] = 4 * rand(b + 3, hq, dk, dv)
        s["idx"] = torch.randperm(b + 3, generator=gen, device="cuda")[:b].to(torch.int32)
    return s


# ----------------------------------------------------------------------------- one pass
def run(state):
    """One call of an operator, and what it gives."""
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import fable_attn as fa
    case, op = s["case"], s["case"]["op"]
    if op == "tables":
        return fa.flash_attn_rotary_tables(case["hi"], case["rd"], base=s["base"], factor=case["factor"],
                                           original_seqlen=case["trained"] or None, device="cuda")
    if op == "rotary":
        q, k = fa.flash_attn_rotary_func(s["q"], s["k"], s["cos"], s["sin"], rotary_interleaved=case["interleaved"],
                                         rotary_seqlens=s["start"], cu_seqlens=s["cu"])
        if not case["grad"]:
            return q, k
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if op == "step":
        out = fa.linear_attn_with_state(s["q"], s["k"], s["v"], s["pool"], s["decay"], state_idx=s["idx"])
        return {"out": out, "state": s["pool"]}
    more = {"initial_state": s.get("first"), "return_final_state": True} if op == "prompt" else {}
    if case["packed"]:
        out = fa.linear_attn_varlen_func(s["q"], s["k"], s["v"], s["cu"], s["max_n"], s["decay"], **more)
    else:
        out = fa.linear_attn_func(s["q"], s["k"], s["v"], s["decay"], **more)
    if op == "prompt":
        return {"out": out[0], "state": out[1]}
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


# -- the plain form
def _padded(s, x, heads):
    """x as (batch, heads, rows, d) in 32 bits, zeros behind each sequence's end; each head repeated to `heads`."""
    x = x.detach().float()
    if s["cu"] is not None:
        cu = s["cu"].long()
        t = torch.arange(s["max_n"], device="cuda")
        row = cu[:-1, None] + t
        x = x[row.clamp_max(x.shape[0] - 1)] * (row < cu[1:, None])[..., None, None]
    x = x.transpose(1, 2)
    return x.repeat_interleave(heads // x.shape[1], dim=1) if x.shape[1] != heads else x


def _rows(s, x):
    """(batch, heads, rows, d) as the call's outputs are laid out."""
    x = x.transpose(1, 2)
    if s["cu"] is None:
        return x
    row = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    return x[seq, row - s["cu"].long()[seq]]


def _powers(decay, n):
    """lambda^n for whole n (of any shape), per head: (heads, ...) in 32 bits, from exponents in 64."""
    return torch.exp(-decay.double().view(-1, *[1] * n.dim()) * n.double()).float()


def _mix(x, y, z, decay, scale, first=None):
    """scale sum_{s<=t} lambda^(t-s) (x_t . y_s) z_s, (batch, heads, rows, d) each, by chunks of 128 rows whose
    states are summed by one product over all chunks; first: the state before row 0."""
    b, h, n, a = x.shape
    c = min(128, n)
    m = -(-n // c)
    cut = lambda u: torch.nn.functional.pad(u, (0, 0, 0, m * c - n)).view(b, h, m, c, u.shape[-1])
    xs, ys, zs = cut(x), cut(y), cut(z)
    i, j = torch.arange(c, device="cuda"), torch.arange(m, device="cuda")
    inside = _powers(decay, (i[:, None] - i).clamp_min(0)).tril_()[:, None]                        # (h, 1, c, c)
    out = torch.matmul(torch.matmul(xs, ys.transpose(-1, -2).contiguous()).mul_(inside), zs)
    if m > 1:
        part = torch.matmul((ys * _powers(decay, c - 1 - i)[:, None, :, None]).transpose(-1, -2).contiguous(), zs)
        over = _powers(decay, (c * (j[:, None] - 1 - j)).clamp_min(0)).tril_(-1)                   # (h, m, m)
        state = torch.matmul(over.expand(b, h, m, m).contiguous(), part.view(b, h, m, -1)).view_as(part)
        out += torch.matmul(xs * _powers(decay, i + 1)[:, None, :, None], state)
    out = out.view(b, h, m * c, -1)[:, :, :n]
    if first is not None:
        out = out + torch.matmul(x * _powers(decay, torch.arange(1, n + 1, device="cuda"))[..., None], first)
    return out * scale


def _final(s, k, v, decay, first):
    """The state behind each sequence's last token."""
    n = s["lens"]
    left = n[:, None] - 1 - torch.arange(k.shape[2], device="cuda")                                # (batch, rows)
    w = _powers(decay, left.clamp_min(0)).transpose(0, 1) * (left >= 0)[:, None]
    state = torch.matmul((k * w[..., None]).transpose(-1, -2).contiguous(), v)
    if first is not None:
        state = state + first * _powers(decay, n).transpose(0, 1)[..., None, None]
    return state


def _turned(s, x):
    """x (rows.., heads, d), its first rd columns turned by (cos, sin) of each row's position."""
    case = s["case"]
    if s["cu"] is None:
        pos = torch.arange(s["max_n"], device="cuda").expand(case["batch"], -1)
        pos = pos if s["start"] is None else pos + s["start"].long()[:, None]
    else:
        row = torch.arange(x.shape[0], device="cuda")
        seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
        pos = row - s["cu"].long()[seq]
        pos = pos if s["start"] is None else pos + s["start"].long()[seq]
    return pos


def _rotate(x, c, w, rd, interleaved):
    """The first rd columns of x turned by (c, w), in 32 bits."""
    out, y = x.detach().float().clone(), x.detach()[..., :rd].float()
    if interleaved:
        a, b = y[..., 0::2], y[..., 1::2]
        out[..., :rd] = torch.stack((a * c - b * w, b * c + a * w), -1).flatten(-2)
    else:
        a, b = y.chunk(2, -1)
        out[..., :rd] = torch.cat((a * c - b * w, b * c + a * w), -1)
    return out.to(x.dtype)


def _frequencies(case, base):
    """The angle per position of each pair of columns, in 64 bits. With a factor f and the trained length n, a pair
    that turns r times over n positions keeps the share clamp((r - 1) / 31, 0, 1) of its frequency, and the rest of
    it is divided by f; without a trained length all are divided by f."""
    freq = base ** (-torch.arange(0, case["rd"], 2, device="cuda", dtype=torch.float64) / case["rd"])
    if case["factor"] == 1.0:
        return freq
    keep = ((case["trained"] * freq / (2 * math.pi) - 1) / 31).clamp(0, 1) if case["trained"] else torch.zeros_like(freq)
    return freq * (keep + (1 - keep) / case["factor"])


def _run_plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "tables":
        angle = torch.arange(case["hi"], device="cuda", dtype=torch.float64)[:, None] * _frequencies(case, s["base"])
        return angle.cos().float(), angle.sin().float()
    if op == "rotary":
        pos = _turned(s, s["q"])
        c, w, more = s["cos"][pos].unsqueeze(-2), s["sin"][pos].unsqueeze(-2), (case["rd"], case["interleaved"])
        q, k = _rotate(s["q"], c, w, *more), _rotate(s["k"], c, w, *more)
        if not case["grad"]:
            return q, k
        return {"q": q, "k": k, "dq": _rotate(s["dq"], c, -w, *more), "dk": _rotate(s["dk"], c, -w, *more)}
    hq, hk, dt, scale, decay = case["hq"], case["hk"], _DT[case["dtype"]], case["dk"] ** -0.5, s["decay"]
    if op == "step":
        s["cu"] = None
    q, k, v = _padded(s, s["q"], hq), _padded(s, s["k"], hq), _padded(s, s["v"], hq)
    s["lens"] = (s["cu"][1:] - s["cu"][:-1]).long() if s["cu"] is not None else torch.full((case["batch"],), s["max_n"], device="cuda")
    first = s["pool"][s["idx"].long()] if op == "step" else s.get("first")
    out = _rows(s, _mix(q, k, v, decay, scale, first)).to(dt)
    if op == "step":
        s["pool"][s["idx"].long()] = _final(s, k, v, decay, first)
        return {"out": out, "state": s["pool"]}
    if op == "prompt":
        return {"out": out, "state": _final(s, k, v, decay, first)}
    do = _padded(s, s["dout"], hq)
    back = lambda x: x.flip(2)                                             # the sums over later rows: time reversed
    shared = lambda x: _rows(s, x.view(case["batch"], hk, hq // hk, *x.shape[2:]).sum(2)).to(dt)
    dq = _rows(s, _mix(do, v, k, decay, scale)).to(dt)
    dv = shared(back(_mix(back(k), back(q), back(do), decay, scale)))
    dk = shared(back(_mix(back(v), back(do), back(q), decay, scale)))
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


# ----------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """What run gives for these inputs, by the definitions in 64 bits."""
    def scan(q, k, v, lam, scale, lens, state):
        """The recurrence, token by token, over (batch, rows, heads, d): outputs and the final state; a sequence's state
        stands still past its end."""
        out = torch.zeros(*q.shape[:3], v.shape[-1], dtype=torch.float64, device="cuda")
        for t in range(q.shape[1]):
            new = state * lam + k[:, t, :, :, None] * v[:, t, :, None, :]
            state = new if lens is None else torch.where((t < lens)[:, None, None, None], new, state)
            out[:, t] = scale * (q[:, t, :, None, :] @ state)[..., 0, :]
        return out, state

    def scan_back(q, k, v, dout, lam, scale):
        """dq, dk, dv of the recurrence: the state S in order, and its gradient G_t = lambda G_{t+1} + scale q_t dout_t^T
        from the last token on (rows behind a sequence's end are zeros). dq_t = scale S_t dout_t, dk_t = G_t v_t,
        dv_t = G_t^T k_t."""
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        shape = (q.shape[0], q.shape[2], q.shape[3], v.shape[3])
        state = torch.zeros(shape, dtype=torch.float64, device="cuda")
        for t in range(q.shape[1]):
            state = state * lam + k[:, t, :, :, None] * v[:, t, :, None, :]
            dq[:, t] = scale * (state @ dout[:, t, :, :, None])[..., 0]
        state.zero_()
        for t in reversed(range(q.shape[1])):
            state = state * lam + scale * q[:, t, :, :, None] * dout[:, t, :, None, :]
            dk[:, t] = (state @ v[:, t, :, :, None])[..., 0]
            dv[:, t] = (k[:, t, :, None, :] @ state)[..., 0, :]
        return dq, dk, dv

    s, op = prepare(case, seed), case["op"]
    with torch.no_grad():
        if op == "tables":
            return _exact_tables(case, s["base"])
        if op == "rotary":
            return _exact_rotary(case, s)
        lens = _lengths(case)
        start = [sum(lens[:i]) for i in range(len(lens))]

        def wide(x, heads):
            x = x.detach().double()
            if case["packed"]:
                full = torch.zeros(case["batch"], case["hi"], *x.shape[1:], dtype=torch.float64, device="cuda")
                for i, n in enumerate(lens):
                    full[i, :n] = x[start[i]:start[i] + n]
                x = full
            return x[:, :, [h * x.shape[2] // heads for h in range(heads)]]

        def narrow(x):
            return torch.cat([x[i, :n] for i, n in enumerate(lens)]) if case["packed"] else x

        hq, hk, dk, dv = case["hq"], case["hk"], case["dk"], case["dv"]
        q, k, v = wide(s["q"], hq), wide(s["k"], hq), wide(s["v"], hq)
        lam = torch.exp(-s["decay"].double())[:, None, None]
        scale = 1.0 / math.sqrt(dk)
        if op == "step":
            state = s["pool"][s["idx"].long()].double()
        else:
            state = s["first"].double() if case["carry"] else torch.zeros(case["batch"], hq, dk, dv, dtype=torch.float64, device="cuda")
        n = torch.tensor(lens, device="cuda") if case["packed"] else None
        out, state = scan(q, k, v, lam, scale, n, state)
        if op == "step":
            pool = s["pool"].double()
            pool[s["idx"].long()] = state
            return {"out": out, "state": pool}
        if op == "prompt":
            return {"out": narrow(out), "state": state}
        gq, gk, gv = scan_back(q, k, v, wide(s["dout"], hq), lam, scale)
        fold = lambda x: torch.stack([x[:, :, h * (hq // hk):(h + 1) * (hq // hk)].sum(2) for h in range(hk)], 2)
        return {"out": narrow(out), "dq": narrow(gq), "dk": narrow(fold(gk)), "dv": narrow(fold(gv))}


def _exact_tables(case, base):
    def freq(i):
        f = math.exp(-2 * i / case["rd"] * math.log(base))
        if case["factor"] == 1.0:
            return f
        turns = case["trained"] * f / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1) / 31)) if case["trained"] else 0.0
        return f * keep + f / case["factor"] * (1 - keep)

    pos = torch.arange(case["hi"], dtype=torch.float64, device="cuda")
    angle = torch.outer(pos, torch.tensor([freq(i) for i in range(case["rd"] // 2)], dtype=torch.float64, device="cuda"))
    return torch.cos(angle), torch.sin(angle)


def _exact_rotary(case, s):
    """Pairs of columns as complex numbers, turned by cos + i sin (gradients by the conjugate)."""
    rd, lens = case["rd"], _lengths(case)
    first = s["start"].tolist() if s["start"] is not None else [0] * case["batch"]
    pos = torch.cat([torch.arange(n) + p for n, p in zip(lens, first)]).cuda()
    turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]

    def of(x, w):
        y = x.detach().double().reshape(-1, *x.shape[-2:]).clone()
        one, two = (slice(0, rd, 2), slice(1, rd, 2)) if case["interleaved"] else (slice(0, rd // 2), slice(rd // 2, rd))
        z = torch.complex(y[..., one].contiguous(), y[..., two].contiguous()) * w
        y[..., one], y[..., two] = z.real, z.imag
        return y.view(x.shape)

    if not case["grad"]:
        return of(s["q"], turn), of(s["k"], turn)
    back = turn.conj().resolve_conj()
    return {"q": of(s["q"], turn), "k": of(s["k"], turn), "dq": of(s["dq"], back), "dk": of(s["dk"], back)}
