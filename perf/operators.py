"""Measured cases of the block operators: a matrix product with its epilogue, rotary positions, per-head
norms with the rotation, and attention over selected key blocks.

``run`` computes each operator from elementary torch operations in 32 bits (64 where 32 lose what matters:
the angles of far positions, the scores that pick blocks), or, with ``own``, through this package's
entry points.  ``exact`` is the definition in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HEAD = 64  # channels of an attention head


def listed():
    return [
        # one token through the first feed-forward product (2048 -> 4 * 2048, tanh GELU)
        dict(name="linear token", op="linear", dtype="bf16", rows=1, n=8192, k=2048, activation="gelu_tanh",
             bias=True, gate=0, residual=False),
        # a ragged handful of rows, sizes that are no multiple of a tile, FP16
        dict(name="linear ragged", op="linear", dtype="fp16", rows=77, n=1999, k=1048, activation="silu",
             bias=True, gate=0, residual=True),
        # second feed-forward product of one eighth of a clip: gated residual of the block's output
        dict(name="linear residual", op="linear", dtype="bf16", rows=8160, n=2048, k=8192, activation="none",
             bias=True, gate=2, residual=True),
        # first feed-forward product of two clips of 16 x 34 x 60 latent tokens
        dict(name="linear clip", op="linear", dtype="bf16", rows=65280, n=8192, k=2048, activation="gelu_tanh",
             bias=True, gate=0, residual=False),
        # single tokens of 16 sequences, far into a stretched context, grouped key heads
        dict(name="rotary token", op="rotary", dtype="fp16", batch=16, seq=1, heads=32, kv_heads=8, dim=128,
             rotary_dim=128, layout="half", scaling="yarn", axes=1, start=900001, inverse=False),
        # odd length, part of the head, 32-bit values, the transposed direction
        dict(name="rotary partial", op="rotary", dtype="fp32", batch=2, seq=1777, heads=12, kv_heads=12, dim=80,
             rotary_dim=32, layout="interleaved", scaling="ntk", axes=1, start=70000, inverse=True),
        # two clips: frame, row and column positions
        dict(name="rotary clip", op="rotary", dtype="bf16", batch=2, seq=32640, heads=32, kv_heads=32, dim=64,
             rotary_dim=64, layout="interleaved", scaling="none", axes=3, start=0, inverse=False),
        # single token of one sequence: norms and rotation before attention
        dict(name="head norm token", op="norm", dtype="bf16", batch=1, seq=1, heads=32, kv_heads=32, dim=64,
             rotary_dim=64, layout="half", scaling="linear", axes=1, start=32639),
        # two clips, queries and keys inside the interleaved projection buffer
        dict(name="head norm clip", op="norm", dtype="bf16", batch=2, seq=32640, heads=32, kv_heads=32, dim=64,
             rotary_dim=64, layout="half", scaling="none", axes=3, start=0),
        # one new token of four sequences against long key/value buffers whose block means are kept
        dict(name="blocks token", op="blocks", dtype="bf16", batch=4, q_len=1, kv_len=32640, heads=32, kv_heads=32,
             topk=32, query_block=1, key_block=64, lengths=True, pooled=True),
        # ragged batch, grouped key heads, one sequence without keys, FP16
        dict(name="blocks ragged", op="blocks", dtype="fp16", batch=3, q_len=2005, kv_len=2005, heads=8, kv_heads=2,
             topk=5, query_block=128, key_block=128, lengths=True, pooled=False),
        # a clip of 16 x 34 x 60 latent tokens attending an eighth of its keys
        dict(name="blocks clip", op="blocks", dtype="bf16", batch=1, q_len=32640, kv_len=32640, heads=32, kv_heads=32,
             topk=64, query_block=128, key_block=64, lengths=False, pooled=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "rotary", "norm", "blocks"])
    if op == "linear":
        n, k = _log(rng, 64, 8192), 8 * _log(rng, 16, 1024)
        rows = _log(rng, 1, min(65280, int(1.0e12 / (n * k))))
        gate = rng.choice([0, 0, 1])
        return dict(op=op, dtype=rng.choice(["bf16", "fp16"]), rows=rows, n=n, k=k,
                    activation=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                    bias=rng.random() < 0.7, gate=gate, residual=rng.random() < 0.5)
    if op in ("rotary", "norm"):
        dim = rng.choice([40, 64, 64, 80, 96, 128, 128])
        axes = rng.choice([1, 1, 3])
        rotary_dim = dim if axes == 3 else rng.choice([dim, dim, 2 * rng.randint(2, dim // 2)])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4])
        batch = _log(rng, 1, 16)
        seq = _log(rng, 1, min(32640, 2 ** 27 // (batch * (heads + kv_heads) * dim)))
        case = dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), batch=batch, seq=seq, heads=heads,
                    kv_heads=kv_heads, dim=dim, rotary_dim=rotary_dim, layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), axes=axes,
                    start=rng.choice([0, _log(rng, 1, 4000000)]))
        if op == "rotary":
            case["inverse"] = rng.random() < 0.3
        return case
    key_block = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4])
    if rng.random() < 0.4:
        kv_len = _log(rng, 1, 65536)
        batch = _log(rng, 1, 16)
        return dict(op=op, dtype=rng.choice(["bf16", "fp16"]), batch=batch, q_len=rng.choice([1, 1, 1, rng.randint(2, 9)]),
                    kv_len=kv_len, heads=heads, kv_heads=kv_heads, topk=rng.randint(1, 64 if key_block == 64 else 32),
                    query_block=1, key_block=key_block, lengths=rng.random() < 0.5, pooled=rng.random() < 0.7)
    kv_len = _log(rng, 1, 16384)
    batch = _log(rng, 1, 4)
    return dict(op=op, dtype=rng.choice(["bf16", "fp16"]), batch=batch, q_len=kv_len if rng.random() < 0.7 else _log(rng, 1, 8192),
                kv_len=kv_len, heads=heads, kv_heads=kv_heads, topk=rng.randint(1, 64 if key_block == 64 else 32),
                query_block=128, key_block=key_block, lengths=rng.random() < 0.5, pooled=rng.random() < 0.2)


# ------------------------------------------------------------------ inputs
def _scaling(name, dim):
    return {"none": None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 8.0},
            "yarn": {"type": "yarn", "factor": 16.0, "original_length": 65536}}[name]


def _axes_dim(case):
    if case["axes"] == 1:
        return None
    # channels of frame, row and column: even parts of the rotated width
    part = case["rotary_dim"] // 6 * 2
    return (case["rotary_dim"] - 2 * part, part, part)


def _frequencies(case, device):
    """Angle per position step of every rotated pair, 64 bits, and the factor on cosine and sine."""
    scaling, theta, amplitude, parts = _scaling(case["scaling"], case["dim"]), 10000.0, 1.0, []
    for dim in _axes_dim(case) or (case["rotary_dim"],):
        i = torch.arange(0, dim, 2, dtype=torch.float64, device=device)
        if case["scaling"] == "ntk":
            parts.append((theta * scaling["factor"] ** (dim / (dim - 2))) ** (-i / dim))
            continue
        f = theta ** (-i / dim)
        if case["scaling"] == "linear":
            f = f / scaling["factor"]
        elif case["scaling"] == "yarn":
            turn = lambda beta: dim * math.log(scaling["original_length"] / (beta * 2 * math.pi)) / (2 * math.log(theta))
            low, high = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), dim - 1)
            ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
            f = f / scaling["factor"] * ramp + f * (1 - ramp)
            amplitude = 0.1 * math.log(scaling["factor"]) + 1.0
        parts.append(f)
    return torch.cat(parts), amplitude


def _positions(case, device):
    batch, seq, start = case["batch"], case["seq"], case["start"]
    s = torch.arange(seq, device=device)
    if case["axes"] == 3:  # raster order of a latent grid 60 wide and 34 high
        return torch.stack([s // (34 * 60) + start, s // 60 % 34, s % 60]).to(torch.int32)
    # sequences of a batch stand at different places
    return s + start + 37 * torch.arange(batch, device=device)[:, None]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = DTYPES[case["dtype"]], case["op"]
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    state = {"case": case}
    if op == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        state["x"] = randn(m, k).to(dtype)
        state["weight"] = (randn(n, k) * k ** -0.5).to(dtype)
        state["bias"] = (randn(n) * 0.5).to(dtype) if case["bias"] else None
        state["gate"] = randn(case["gate"], n).to(dtype) if case["gate"] else None
        state["residual"] = randn(m, n).to(dtype) if case["residual"] else None
        return state
    if op in ("rotary", "norm"):
        b, s, h, kvh, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"]
        # queries and keys as views of the projection's buffer (queries | keys | values of each token)
        buffer = torch.empty(b, s, (h + 2 * kvh) * d, device="cuda", dtype=dtype)
        buffer.normal_(generator=g)
        state["query"] = buffer[..., :h * d].unflatten(-1, (h, d))
        state["key"] = buffer[..., h * d:(h + kvh) * d].unflatten(-1, (kvh, d))
        state["positions"] = _positions(case, "cuda")
        state["frequencies"], state["amplitude"] = _frequencies(case, "cuda")
        if op == "norm":
            state["norms"] = [torch.nn.RMSNorm(d, eps=1e-6, device="cuda", dtype=dtype).requires_grad_(False)
                              for _ in range(2)]
            for norm in state["norms"]:
                norm.weight.copy_(1 + 0.3 * randn(d))
        if own:
            from eraserdit_b200.rotary import RotaryPositions
            state["rotary"] = RotaryPositions(d, rotary_dim=case["rotary_dim"], layout=case["layout"],
                                              scaling=_scaling(case["scaling"], d), axes_dim=_axes_dim(case))
        return state
    b, h, kvh, kb = case["batch"], case["heads"], case["kv_heads"], case["key_block"]
    sq, sk = case["q_len"], case["kv_len"]
    nblocks = -(-sk // kb)
    # keys and queries vary from token to token around what their part of the sequence shares
    shared = randn(b, nblocks, kvh, HEAD).repeat_interleave(kb, 1)[:, :sk]
    state["key"] = (randn(b, sk, kvh, HEAD) + 0.5 * shared).to(dtype)
    state["value"] = randn(b, sk, kvh, HEAD).to(dtype)
    q_shared = randn(b, -(-sq // 128), h, HEAD).repeat_interleave(128, 1)[:, :sq]
    state["query"] = (randn(b, sq, h, HEAD) + 0.5 * q_shared).to(dtype)
    state["lengths"] = None
    if case["lengths"]:
        # the first sequence is full, the second (where there are three) empty, the others in between
        lengths = [sk] + [0] * (b > 2) + [max(1, sk * 3 // 8 + 11 * i) for i in range(b)]
        state["lengths"] = torch.tensor([min(n, sk) for n in lengths[:b]], dtype=torch.int32, device="cuda")
    state["pool"] = _block_means(state["key"], kb, state["lengths"]) if case["pooled"] else None
    return state


# -------------------------------------------------------------- plain forms
def _block_means(key, key_block, lengths):
    """[B, Hkv, blocks, 64] means of each block's valid keys in 64 bits (0 for a block without one)."""
    b, sk, kvh, d = key.shape
    n = -(-sk // key_block)
    valid = torch.arange(sk, device=key.device) < (lengths[:, None] if lengths is not None else sk)
    k = key.double().masked_fill(~valid.expand(b, sk)[:, :, None, None], 0)
    k = torch.nn.functional.pad(k, (0, 0, 0, 0, 0, n * key_block - sk))
    count = torch.nn.functional.pad(valid.expand(b, sk).double(), (0, n * key_block - sk)).view(b, n, key_block).sum(-1)
    return (k.view(b, n, key_block, kvh, d).sum(2) / count.clamp(min=1)[:, :, None, None]).permute(0, 2, 1, 3).contiguous()


def _activate(y, name):
    if name == "relu":
        return y.clamp(min=0)
    if name == "silu":
        return y / (1 + torch.exp(-y))
    if name == "gelu":
        return 0.5 * y * (1 + torch.erf(y * 2 ** -0.5))
    if name == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y * y * y)))
    return y


def _plain_linear(state):
    x, case = state["x"], state["case"]
    y = x.float() @ state["weight"].float().T
    if state["bias"] is not None:
        y = y + state["bias"].float()
    y = _activate(y, case["activation"])
    if state["gate"] is not None:
        y = (y.view(case["gate"], -1, case["n"]) * state["gate"].float()[:, None]).view(y.shape)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(x.dtype)


def _plain_rotate(x, state):
    """The rotation of 32-bit [B, S, H, D]."""
    case = state["case"]
    half, pos = case["rotary_dim"] // 2, state["positions"]
    if case["axes"] == 3:
        widths = torch.tensor([w // 2 for w in _axes_dim(case)], device=pos.device)
        axis = torch.repeat_interleave(torch.arange(3, device=pos.device), widths, output_size=half)
        pos = pos[axis].T  # [S, pairs]
    else:
        pos = pos[..., None]
    angle = pos.double() * state["frequencies"]
    c = (angle.cos() * state["amplitude"]).float().unsqueeze(-2)
    s = (angle.sin() * state["amplitude"]).float().unsqueeze(-2)
    if case.get("inverse"):
        s = -s
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if case["layout"] == "half":
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_norm(x, norm):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.float()


def _plain_blocks(state):
    case, q, k, v = state["case"], state["query"], state["key"], state["value"]
    b, sq, h, d = q.shape
    sk, kvh, kb, qb = k.shape[1], k.shape[2], case["key_block"], case["query_block"]
    n, groups = -(-sk // kb), -(-sq // qb)
    pool = state["pool"] if state["pool"] is not None else _block_means(k, kb, state["lengths"])
    lengths = state["lengths"] if state["lengths"] is not None else torch.full((b,), sk, device=q.device)
    qp = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, groups * qb - sq)).view(b, groups, qb, h, d).permute(0, 3, 1, 2, 4)
    count = (sq - qb * torch.arange(groups, device=q.device)).clamp(max=qb)
    score = (qp.double().sum(3) / count[:, None]) @ pool.repeat_interleave(h // kvh, 1).transpose(-1, -2)
    blocks = (lengths + kb - 1) // kb  # blocks with a valid key
    score = score.masked_fill(torch.arange(n, device=q.device) >= blocks[:, None, None, None], -math.inf)
    take = min(case["topk"], n)
    chosen = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :take]
    kept = torch.arange(take, device=q.device) < blocks[:, None, None, None]
    chosen = torch.where(kept, chosen, n).sort(-1).values  # [B, H, groups, take], n where there is none
    real = (chosen < n)
    at = chosen.clamp(max=n - 1)
    bi = torch.arange(b, device=q.device)[:, None, None, None]
    hi = (torch.arange(h, device=q.device) // (h // kvh))[None, :, None, None]
    rows = lambda t: torch.nn.functional.pad(t, (0, 0, 0, 0, 0, n * kb - sk)).view(b, n, kb, kvh, d)
    valid = (at[..., None] * kb + torch.arange(kb, device=q.device) < lengths[:, None, None, None, None]) & real[..., None]
    valid = valid.flatten(-2)[:, :, :, None, :]
    s = qp.float() @ rows(k)[bi, at, :, hi].float().flatten(3, 4).transpose(-1, -2)
    s = s.mul_(HEAD ** -0.5).masked_fill_(~valid, -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ rows(v)[bi, at, :, hi].float().flatten(3, 4)) / total.clamp(min=1e-30)
    o = o.permute(0, 2, 3, 1, 4).reshape(b, groups * qb, h, d)[:, :sq].to(q.dtype)
    chosen = torch.where(real, chosen, -1).to(torch.int32)
    if take < case["topk"]:
        chosen = torch.nn.functional.pad(chosen, (0, case["topk"] - take), value=-1)
    return o, chosen


# ------------------------------------------------------------------- a pass
def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        if op == "linear":
            from eraserdit_b200.linear import linear_act
            return linear_act(state["x"], state["weight"], state["bias"], activation=case["activation"],
                              gate=state["gate"], residual=state["residual"])
        if op == "rotary":
            from eraserdit_b200.rotary import apply_rotary
            return apply_rotary(state["query"], state["key"], state["rotary"], state["positions"],
                                inverse=case["inverse"])
        if op == "norm":
            from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
            return apply_fused_qk_head_rmsnorm_rotary(state["query"], state["key"], *state["norms"],
                                                      state["rotary"], state["positions"])
        from eraserdit_b200.block_topk import block_topk_attention
        return block_topk_attention(state["query"], state["key"], state["value"], HEAD ** -0.5, case["topk"],
                                    query_block=case["query_block"], key_block=case["key_block"],
                                    key_lengths=state["lengths"], key_pool=state["pool"], return_selection=True)
    if op == "linear":
        return _plain_linear(state)
    if op == "rotary":
        return tuple(_plain_rotate(x.float(), state).to(x.dtype) for x in (state["query"], state["key"]))
    if op == "norm":
        return tuple(_plain_rotate(_plain_norm(x, norm), state).to(x.dtype)
                     for x, norm in zip((state["query"], state["key"]), state["norms"]))
    return _plain_blocks(state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        values = m * k + n * k + m * n * (2 if case["residual"] else 1) + n * (case["gate"] + bool(case["bias"]))
        return {"bytes": values * size, "flops": 2 * m * n * k}
    if case["op"] in ("rotary", "norm"):
        values = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * values * size, "flops": values * (3 if case["op"] == "rotary" else 6)}
    b, h, kvh, kb = case["batch"], case["heads"], case["kv_heads"], case["key_block"]
    sq, sk = case["q_len"], case["kv_len"]
    lengths = [sk] + [0] * (b > 2) + [min(sk, max(1, sk * 3 // 8 + 11 * i)) for i in range(b)]
    lengths = lengths[:b] if case["lengths"] else [sk] * b
    groups, n = -(-sq // case["query_block"]), -(-sk // kb)
    keys = [min(x, case["topk"] * kb) for x in lengths]  # attended by each query
    flops = sum(4 * sq * h * x * HEAD + 2 * groups * h * -(-y // kb) * HEAD for x, y in zip(keys, lengths))
    # keys: all of them for the scores, or the kept means and the blocks attended; values: the blocks attended
    touched = sum(min(y, groups * (h // kvh) * x) * kvh * HEAD for x, y in zip(keys, lengths))
    reads = (touched if case["pooled"] else sum(lengths) * kvh * HEAD) + touched
    data = 2 * (2 * b * sq * h * HEAD + reads) + 4 * b * h * groups * case["topk"]
    return {"bytes": data + (8 * b * kvh * n * HEAD if case["pooled"] else 0), "flops": flops}


# ------------------------------------------------- the definitions in 64 bits
def _exact_activate(y, name):
    if name == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if name == "silu":
        return y * torch.sigmoid(y)
    if name == "gelu":
        return torch.special.ndtr(y) * y
    if name == "gelu_tanh":  # (1 + tanh(u)) / 2 = sigmoid(2 u)
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return y


def _exact_linear(state):
    case = state["case"]
    y = torch.nn.functional.linear(state["x"].double(), state["weight"].double(),
                                   None if state["bias"] is None else state["bias"].double())
    y = _exact_activate(y, case["activation"])
    if state["gate"] is not None:
        y *= state["gate"].double().repeat_interleave(case["rows"] // case["gate"], 0)
    return y if state["residual"] is None else y + state["residual"].double()


def _exact_rotate(x, state):
    """Pairs as complex numbers, turned by the angle of each token and pair."""
    case = state["case"]
    frequencies, amplitude = _frequencies(case, x.device)
    widths = [w // 2 for w in _axes_dim(case) or (case["rotary_dim"],)]
    pos = state["positions"].double()
    per_axis = pos.unbind(0) if case["axes"] == 3 else [pos]
    angle = torch.cat([p[..., None] * f for p, f in zip(per_axis, frequencies.split(widths))], -1)
    turn = torch.polar(torch.full_like(angle, amplitude), -angle if case.get("inverse") else angle).unsqueeze(-2)
    y, r = x.double().clone(), case["rotary_dim"]
    pairs = y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" else \
        y[..., :r].unflatten(-1, (r // 2, 2))
    z = torch.view_as_real(torch.complex(pairs[..., 0].contiguous(), pairs[..., 1].contiguous()) * turn)
    y[..., :r] = (z.transpose(-1, -2) if case["layout"] == "half" else z).flatten(-2)
    return y


def _exact_blocks(state):
    """Dense attention of each sequence and head under the mask that the scores' ranks give."""
    case, q, k, v = state["case"], state["query"], state["key"], state["value"]
    b, sq, h, d = q.shape
    sk, kb, qb, topk = k.shape[1], case["key_block"], case["query_block"], case["topk"]
    per = h // k.shape[2]
    out = torch.zeros(b, sq, h, d, dtype=torch.float64, device=q.device)
    picked = torch.full((b, h, -(-sq // qb), topk), -1, dtype=torch.int32, device=q.device)
    for i in range(b):
        length = sk if state["lengths"] is None else int(state["lengths"][i])
        if length == 0:
            continue
        ends = torch.arange(kb, length + kb, kb).clamp(max=length).tolist()
        for j in range(h):
            kf, vf = k[i, :length, j // per].double(), v[i, :length, j // per].double()
            qf = q[i, :, j].double()
            means = torch.stack([p.mean(0) for p in kf.split(kb)])
            q_means = qf if qb == 1 else torch.stack([p.mean(0) for p in qf.split(qb)])
            score = q_means @ means.T
            n = len(ends)
            rank = (score[:, None, :] > score[:, :, None]).sum(-1)
            earlier = torch.ones(n, n, dtype=torch.bool, device=q.device).tril(-1)
            rank += ((score[:, None, :] == score[:, :, None]) & earlier).sum(-1)
            keep = rank < topk
            where = keep.nonzero()[:, 1].view(keep.shape[0], -1)
            picked[i, j, :, :where.shape[1]] = where.int()
            for at in range(0, sq, 8192):
                rows = torch.arange(at, min(sq, at + 8192), device=q.device)
                mask = keep.repeat_interleave(kb, 1)[:, :length][rows // qb]
                logits = (qf[rows] @ kf.T * HEAD ** -0.5).masked_fill_(~mask, -math.inf)
                out[i, rows, j] = torch.softmax(logits, -1) @ vf
    return out, picked


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(state)
    if case["op"] == "rotary":
        return tuple(_exact_rotate(x, state) for x in (state["query"], state["key"]))
    if case["op"] == "norm":
        normed = [x.double() / torch.sqrt(x.double().pow(2).mean(-1, keepdim=True) + norm.eps) * norm.weight.double()
                  for x, norm in zip((state["query"], state["key"]), state["norms"])]
        return tuple(_exact_rotate(x, state) for x in normed)
    return _exact_blocks(state)
