"""What stands between two graph convolutions, as measured cases: layer norm, dropout from a counter-based generator,
and both with the ReLU between them.  Every operator works on a matrix with one row per node.

    layer norm   m = mean(x), v = mean((x - m)^2), h = (x - m) / sqrt(v + eps), y = h * weight + bias     (of each row)
    dropout      y = x * 65536 / (65536 - t) where u >= t, else 0;  t = floor(65536 p + 1/2)
    tail         y = dropout(max(layer_norm(x), 0))

u is a 16-bit number per element: the columns of a row are taken in groups of eight (the last one may be shorter),
group i = row * ceil(cols / 8) + column // 8 is the low half of the 128-bit counter of Philox4x32 (Salmon, Moraes, Dror,
Shaw 2011) with seven rounds, the offset its high half, the seed its key, and field column % 8 of the four words (low
half of a word first) is the element's."""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
WORD = 0xFFFFFFFF


def _case(name, op, rows, cols, x="f32", y=None, train=True, p=0.0, pitch=0):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "x": x, "y": y or x, "train": train, "p": p,
            "pitch": max(pitch, cols)}


def listed():
    return [
        # the smallest graph's features, 32 wide: forward and backward are a matter of launches
        _case("dropout_16384x32_f32", "dropout", 16384, 32, p=0.5),
        # 2.4 million nodes with 100 features, packed rows
        _case("dropout_2400000x100_f32", "dropout", 2400000, 100, p=0.2),
        # the mixed-precision training step's hidden rows
        _case("dropout_4194304x256_bf16", "dropout", 4194304, 256, "bf16", p=0.5),
        # one node asked for by a serving program: no gradient
        _case("norm_1x256_f32", "norm", 1, 256, train=False),
        # hidden rows of a two-layer network at inference
        _case("norm_262144x256_f32", "norm", 262144, 256, train=False),
        # 47 columns in rows of 48, as the aggregation of 2.4 million nodes may leave them
        _case("norm_train_2400000x47_f32", "norm", 2400000, 47, pitch=48),
        # a million nodes at hidden width 64, mixed precision
        _case("norm_train_1048576x64_bf16", "norm", 1048576, 64, "bf16"),
        # wide node features (text, bags of words): an odd number of nodes and of columns
        _case("norm_train_20011x4099_bf16", "norm", 20011, 4099, "bf16"),
        # the training command's default: 16 hidden units on the smallest graph
        _case("tail_train_16384x16_f32", "tail", 16384, 16, p=0.5),
        # an odd number of nodes, 100 hidden units, a low rate
        _case("tail_train_1000003x100_f32", "tail", 1000003, 100, p=0.1),
        # float32 out of the convolution, bfloat16 into the next one
        _case("tail_train_262144x256_f32_bf16", "tail", 262144, 256, "f32", "bf16", p=0.5),
        # the mixed-precision training step on 4 million nodes
        _case("tail_train_4194304x256_bf16", "tail", 4194304, 256, "bf16", p=0.5),
    ]


def draw(rng):
    op = rng.choice(["dropout", "norm", "tail"])
    x = rng.choice(["f32", "bf16"])
    y = x if op == "dropout" else rng.choice(["f32", "bf16"])
    cols = int(round(math.exp(rng.uniform(math.log(16), math.log(4608)))))
    most = min(4194304, (1 << (29 if "f32" in (x, y) else 30)) // cols)
    rows = int(round(math.exp(rng.uniform(0.0, math.log(most)))))
    pitch = cols + rng.choice([0, 0, 1, (-cols) % 8])
    return _case(None, op, rows, cols, x, y, op != "norm" or rng.random() < 0.7,
                 0.0 if op == "norm" else rng.choice([0.1, 0.2, 0.5, 0.75, rng.uniform(0.02, 0.9)]), pitch) | {"salt": rng.randrange(1 << 30)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed((seed * 1000003 + case.get("salt", 0)) % (1 << 62))
    n, f = case["rows"], case["cols"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    # rows out of an aggregation: their spread goes with the node's degree, their columns have means of their own
    spread = torch.exp(0.5 * normal(n, 1))
    x = torch.empty((n, case["pitch"]), dtype=TYPES[case["x"]], device="cuda")[:, :f]
    x.copy_(normal(n, f).mul_(spread).add_(normal(1, f), alpha=0.3))
    state = {"case": case, "x": x.requires_grad_(case["train"])}
    if case["train"]:
        state["dy"] = normal(n, f).to(TYPES[case["y"]])
    if case["op"] != "dropout":
        state["weight"] = (1.0 + 0.2 * normal(f)).requires_grad_(case["train"])
        state["bias"] = (0.2 * normal(f)).requires_grad_(case["train"])
    if case["p"]:
        state["rng"] = torch.randint(0, 1 << 62, (2,), device="cuda", generator=gen)
    return state


def _round(c, key):
    a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57     # wraps at 64 bits; the bits are those of the unsigned product
    return ((b >> 32) & WORD) ^ c[1] ^ key[0], b & WORD, ((a >> 32) & WORD) ^ c[3] ^ key[1], a & WORD


def _kept(case, rng):
    n, f = case["rows"], case["cols"]
    groups = -(-f // 8)
    i = torch.arange(n * groups, device=rng.device)
    seed, offset = torch.stack([rng & WORD, (rng >> 32) & WORD], 1)
    step = torch.tensor([0x9E3779B9, 0xBB67AE85]).to(rng.device, non_blocking=True)
    keys = (seed + torch.arange(7, device=rng.device)[:, None] * step) & WORD
    k0, k1, k2, k3, k4, k5, k6 = keys
    c = _round((i & WORD, i >> 32, offset[0], offset[1]), k0)
    c = _round(_round(_round(c, k1), k2), k3)
    c = _round(_round(_round(c, k4), k5), k6)
    t = int(case["p"] * 65536 + 0.5)
    low, high = (torch.stack([w & 0xFFFF for w in c], 1) >= t, torch.stack([w >> 16 for w in c], 1) >= t)
    return torch.stack([low, high], 2).view(n, groups * 8)[:, :f], 65536 / (65536 - t)


def _plain_dropout(s):
    case = s["case"]
    kept, scale = _kept(case, s["rng"])
    y = torch.where(kept, s["x"].detach().float() * scale, 0.0).to(TYPES[case["y"]])
    if not case["train"]:
        return {"y": y}
    return {"y": y, "dx": torch.where(kept, s["dy"].float() * scale, 0.0).to(TYPES[case["x"]])}


def _plain_norm(s):
    case, tail = s["case"], s["case"]["op"] == "tail"
    x, w, b = s["x"].detach().float(), s["weight"].detach(), s["bias"].detach()
    h = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    h = h * r
    y = h * w + b
    if tail:
        kept, scale = _kept(case, s["rng"])
        y = torch.where(kept, torch.clamp(y, min=0.0) * scale, 0.0)
    y = y.to(TYPES[case["y"]])
    if not case["train"]:
        return {"y": y}
    d = s["dy"].float()
    if tail:
        # the ReLU's gate is a border: 64 bits
        e = x.double()
        e = e - e.mean(1, keepdim=True)
        e = e / torch.sqrt((e * e).mean(1, keepdim=True) + EPS)
        d = torch.where(kept & (e * w.double() + b.double() > 0), d * scale, 0.0)
        del e, kept
    g = d * w
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(TYPES[case["x"]]), "dweight": (d * h).sum(0), "dbias": d.sum(0)}


def _own(s):
    from artifact_amd.row_ops import dropout, layer_norm

    case = s["case"]
    if case["op"] == "dropout":
        y = dropout(s["x"], case["p"], s["rng"])
        of = {"dx": s["x"]}
    else:
        y = layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, relu=case["op"] == "tail", dropout=case["p"],
                       rng=s.get("rng"), out_dtype=TYPES[case["y"]])
        of = {"dx": s["x"], "dweight": s["weight"], "dbias": s["bias"]}
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, list(of.values()), s["dy"])
    return {"y": y.detach()} | dict(zip(of, grads))


def run(state):
    if own:
        return _own(state)
    return _plain_dropout(state) if state["case"]["op"] == "dropout" else _plain_norm(state)


def work(case):
    n, f = case["rows"], case["cols"]
    sx, sy = TYPES[case["x"]].itemsize, TYPES[case["y"]].itemsize
    norm = case["op"] != "dropout"
    params = 8 * f if norm else 0
    bytes_ = n * f * (sx + sy) + params
    flops = n * f * ((8 if norm else 0) + (2 if case["p"] else 0))
    if case["train"]:
        bytes_ += n * f * (sx + sy) + params
        flops += n * f * ((13 if norm else 0) + (2 if case["p"] else 0))
    return {"bytes": bytes_, "flops": flops}


def _words(group, seed, offset):
    """Philox4x32, seven rounds, for a vector of group numbers: products from 16-bit halves, key and offset as whole numbers."""
    def product(v, m):
        ml, mh = m & 0xFFFF, m >> 16
        vl, vh = v & 0xFFFF, v >> 16
        mid = vh * ml + (vl * ml >> 16)
        cross = vl * mh + (mid & 0xFFFF)
        return vh * mh + (mid >> 16) + (cross >> 16), ((cross & 0xFFFF) << 16) | (vl * ml & 0xFFFF)

    x = [group & WORD, group >> 32, torch.full_like(group, offset & WORD), torch.full_like(group, offset >> 32 & WORD)]
    key = [seed & WORD, seed >> 32 & WORD]
    for _ in range(7):
        (h0, l0), (h1, l1) = product(x[0], 0xD2511F53), product(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ key[0], l1, h0 ^ x[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) & WORD, (key[1] + 0xBB67AE85) & WORD]
    return x


def exact(case, seed):
    s = prepare(case, seed)
    n, f, p, tail = case["rows"], case["cols"], case["p"], case["op"] == "tail"
    groups, column = (f + 7) // 8, torch.arange(f, device="cuda")
    if p:
        t = math.floor(p * 65536 + 0.5)
        key, offset = (int(v) for v in s["rng"].tolist())
    parts, dw, db = [], 0.0, 0.0
    step = max(1, (1 << 24) // f)
    for r0 in range(0, max(n, 1), step):
        x = s["x"].detach()[r0:r0 + step].double()
        rows = torch.arange(r0, r0 + len(x), device="cuda")
        factor = torch.ones_like(x)
        if p:
            words = torch.stack(_words((rows[:, None] * groups + torch.arange(groups, device="cuda")).flatten(), key, offset), -1)
            field = words.view(len(x), groups * 4)[:, column // 2] >> (16 * (column % 2)) & 0xFFFF
            factor = (field >= t) * (65536.0 / (65536 - t))
            del words, field
        if case["op"] == "dropout":
            part = [x * factor]
            if case["train"]:
                part.append(s["dy"][r0:r0 + step].double() * factor)
            parts.append(part)
            continue
        w, b = s["weight"].detach().double(), s["bias"].detach().double()
        mean = x.sum(1, keepdim=True) / f
        std = torch.sqrt(((x - mean) ** 2).sum(1, keepdim=True) / f + EPS)
        h = (x - mean) / std
        y = h * w + b
        if tail:
            factor = factor * (y > 0)
            y = y * factor
        part = [y]
        if case["train"]:
            up = s["dy"][r0:r0 + step].double() * factor
            dw, db = dw + (up * h).sum(0), db + up.sum(0)
            dh = up * w
            part.append((dh - dh.sum(1, keepdim=True) / f - h * ((dh * h).sum(1, keepdim=True) / f)) / std)
        parts.append(part)
    whole = [torch.cat(column_of) for column_of in zip(*parts)]
    answer = {"y": whole[0]}
    if case["train"]:
        answer["dx"] = whole[1]
        if case["op"] != "dropout":
            answer |= {"dweight": dw, "dbias": db}
    return answer
