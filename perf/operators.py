"""AdamW steps over many tensors (states in fp32 or in 8 bits) and the global gradient norm: what they are timed on.

A case is a dict of plain values.  `prepare` makes what a training program holds between backward() and step(): parameters,
gradients, optimizer states in mid-training.  `run` is one call: `optimizer.step()` of `came_b200.AdamW` / `AdamW8bit`, or
`came_b200.clip_grad_norm_`; where `own` is false the same in elementary torch operations.

Operators (`"op"`): adamw (states fp32), adamw8 (states float8 with a power-of-two scale, itself in
8 bits, for each 256 elements), clip (norm, gradients scaled in place).
Parameter sets (`"set"`):

    decoder   embedding and head [vocab, hidden], per layer q, o [hidden, hidden], k, v [hidden, kv], gate, up [hidden, ffn],
              down [ffn, hidden] and two norm vectors
    adapter   pairs of low-rank factors [rank, width], [width, rank]
    conv      3 x 3 and 1 x 1 convolution kernels over a pyramid of widths, each with a bias
    dense     one matrix and its bias
    odd       an embedding, a head stored [hidden, vocab] and two feed-forward matrices whose sizes are no multiple of 8
"""
import math

import torch

own = False

LR, WD, BETAS, EPS = 2e-4, 1e-2, (0.9, 0.999), 1e-8
BLOCK = 256
PAST = 100               # steps that the states have behind them
ALIGN = 512              # bytes: what the allocator gives a tensor of its own
M32 = 0xFFFFFFFF


def listed():
    return [
        # the smallest call: a classifier on frozen features, where launches and the host are all there is
        dict(name="probe-fp32", op="adamw", set="dense", rows=100, cols=512, dtype="float32"),
        # low-rank fine-tuning with the usual clip: hundreds of small thin matrices
        dict(name="adapter-bf16-clip", op="adamw", set="adapter", modules=264, rank=16, width=640, dtype="bfloat16", max_norm=1.0),
        # sizes that suit no vector width, packed into one flat buffer (no tensor starts on a 16-byte boundary), loss scaling
        dict(name="odd-packed-fp16", op="adamw", set="odd", vocab=50257, hidden=770, ffn=3083, dtype="float16", grad_scale=1.0 / 1024,
             packed=True),
        # a mid-size language model in fp32; gradients are dropped and made anew at every step
        dict(name="mid-lm-fp32-moved", op="adamw", set="decoder", vocab=32000, hidden=1024, kv=256, ffn=2816, layers=12, dtype="float32",
             moved=True),
        # a 1.3 B parameter model with a clip
        dict(name="llama1b-bf16-clip", op="adamw", set="decoder", vocab=32000, hidden=2048, kv=2048, ffn=5632, layers=22, dtype="bfloat16",
             max_norm=1.0),
        # 8-bit states: the smallest call
        dict(name="probe-bf16-8bit", op="adamw8", set="dense", rows=1000, cols=768, dtype="bfloat16"),
        # a small language model whose whole step, clip included, is replayed as a CUDA graph
        dict(name="small-lm-bf16-8bit-clip-graph", op="adamw8", set="decoder", vocab=8000, hidden=512, kv=512, ffn=1408, layers=8,
             dtype="bfloat16", max_norm=1.0, graph=True),
        # a convolutional network in fp16 with loss scaling: thousands of short blocks, biases, tensors of four dimensions
        dict(name="conv-fp16-8bit", op="adamw8", set="conv", width=320, levels=3, blocks=2, dtype="float16", grad_scale=1.0 / 1024),
        # fp32 weights whose sizes are no multiple of a block
        dict(name="odd-fp32-8bit", op="adamw8", set="odd", vocab=50257, hidden=770, ffn=3083, dtype="float32"),
        # the 1.3 B parameter model
        dict(name="llama1b-bf16-8bit", op="adamw8", set="decoder", vocab=32000, hidden=2048, kv=2048, ffn=5632, layers=22, dtype="bfloat16"),
        # the norm of a fine-tuning step (below the limit, as in most steps)
        dict(name="adapter-bf16-norm", op="clip", set="adapter", modules=264, rank=16, width=640, dtype="bfloat16", max_norm=1e4),
        # the norm of the 1.3 B parameter model
        dict(name="llama1b-bf16-norm", op="clip", set="decoder", vocab=32000, hidden=2048, kv=2048, ffn=5632, layers=22, dtype="bfloat16",
             max_norm=1e4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step=64, odd=0.3):
    n = _log(rng, lo, hi)
    return n if rng.random() < odd else max(step, n // step * step)


def draw(rng):
    case = dict(op=rng.choice(["adamw", "adamw", "adamw8", "adamw8", "clip"]), set=rng.choice(["decoder", "decoder", "adapter", "conv", "dense", "odd"]),
                dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
    kind = case["set"]
    if kind == "decoder":
        hidden = _size(rng, 64, 2048)
        case.update(vocab=_log(rng, 500, 32000), hidden=hidden, kv=hidden if rng.random() < 0.5 else max(32, hidden // 4),
                    ffn=_size(rng, 2 * hidden, 4 * hidden, 64, 0.2))
        most = max(1, 400_000_000 // (hidden * (2 * hidden + 2 * case["kv"] + 3 * case["ffn"])))
        case["layers"] = _log(rng, 1, min(24, most))
    elif kind == "adapter":
        case.update(modules=_log(rng, 8, 300), rank=rng.choice([3, 4, 8, 16, 32, 64]), width=_size(rng, 100, 2000))
    elif kind == "conv":
        case.update(width=_size(rng, 8, 320, 32), levels=rng.randint(1, 3), blocks=rng.randint(1, 3))
    elif kind == "dense":
        case.update(rows=_log(rng, 1, 8192), cols=_log(rng, 16, 8192))
    else:
        case.update(vocab=_log(rng, 1000, 50257), hidden=_log(rng, 129, 1100), ffn=_log(rng, 500, 4400))
    if case["op"] == "clip":
        case["max_norm"] = rng.choice([0.5, 1.0, 10.0, 1e4])
    elif rng.random() < 0.4:
        case["max_norm"] = rng.choice([0.5, 1.0, 10.0])
    if case["op"] != "clip" and case["dtype"] == "float16" and rng.random() < 0.6:
        case["grad_scale"] = 1.0 / 1024
    if kind in ("odd", "dense") and rng.random() < 0.4:
        case["packed"] = True
    if case["op"] != "clip" and rng.random() < 0.25:
        case["graph"] = True
    elif rng.random() < 0.25:
        case["moved"] = True
    return case


def _shapes(case):
    kind = case["set"]
    if kind == "decoder":
        h, kv, f = case["hidden"], case["kv"], case["ffn"]
        out = [(case["vocab"], h)]
        for _ in range(case["layers"]):
            out += [(h, h), (h, kv), (h, kv), (h, h), (h, f), (h, f), (f, h), (h,), (h,)]
        return out + [(h,), (case["vocab"], h)]
    if kind == "adapter":
        out = []
        for i in range(case["modules"]):
            w = case["width"] * (1 + i % 2)
            out += [(case["rank"], w), (w, case["rank"])]
        return out
    if kind == "conv":
        out, c_in = [], 4
        for level in range(case["levels"]):
            c = case["width"] << level
            out += [(c, c_in, 3, 3), (c,)]
            for _ in range(case["blocks"]):
                out += [(c, c, 3, 3), (c,), (c, c, 1, 1), (c,)]
            c_in = c
        return out
    if kind == "dense":
        return [(case["rows"], case["cols"]), (case["rows"],)]
    v, h, f = case["vocab"], case["hidden"], case["ffn"]
    return [(v, h), (h, f), (f,), (f, h), (h,), (h, v)]


def _flat(shapes, dtype, device, packed=False):
    """One buffer and a view of it for each shape, every view on an allocation boundary unless they are packed."""
    step = 1 if packed else ALIGN // torch.empty(0, dtype=dtype).element_size()
    at, places = (3 if packed else 0), []
    for s in shapes:
        places.append(at)
        at += -(-math.prod(s) // step) * step
    buf = torch.zeros(at, dtype=dtype, device=device)
    return buf, [buf[i: i + math.prod(s)].view(s) for i, s in zip(places, shapes)]


def _blocks(n):
    return -(-n // BLOCK)


def _power_of_two(x, top):
    """2^(exponent of x - top), as a block's scale is: x its largest magnitude."""
    e = torch.frexp(x)[1] - 1 - top
    return torch.where(x > 0, torch.ldexp(torch.ones_like(x), e.clamp(-126, 127)), torch.full_like(x, 2.0 ** -126))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dtype, shapes, packed = getattr(torch, case["dtype"]), _shapes(case), case.get("packed", False)
    st = dict(case=case, shapes=shapes, turn=0)
    # gradients N(0, 1) times a scale of the tensor's own, times the loss scale; moments as of an average over such gradients
    scales = [10.0 ** float(x) for x in torch.empty(len(shapes)).uniform_(-5, -2, generator=host)]
    loss_scale = 1.0 / case.get("grad_scale", 1.0)
    st["grads"] = []
    for _ in range(2 if case.get("moved") else 1):
        buf, views = _flat(shapes, dtype, dev, packed)
        for g, sc in zip(views, scales):
            g.copy_(torch.randn(g.shape, generator=gen, device=dev).mul_(sc * loss_scale))
        st["grads"].append((buf, views))
    st["p_buf"], st["p"] = _flat(shapes, dtype, dev, packed)
    for p in st["p"]:
        p.copy_(torch.randn(p.shape, generator=gen, device=dev).mul_(0.02))
    if case["op"] != "clip":
        st["steps"] = torch.full((len(shapes),), float(PAST), device=dev)
        if case["op"] == "adamw":
            for k in ("m", "v"):
                st[k + "_buf"], st[k] = _flat(shapes, torch.float32, dev)
        else:
            for k, dt in (("m", torch.float8_e4m3fn), ("v", torch.float8_e5m2)):
                st[k + "_buf"], st[k] = _flat(shapes, dt, dev)
                st[k + "_scale_buf"], st[k + "_scale"] = _flat([(_blocks(math.prod(s)),) for s in shapes], torch.float8_e8m0fnu, dev)
        for i, (s, sc) in enumerate(zip(shapes, scales)):
            m = torch.randn(s, generator=gen, device=dev).mul_(0.23 * sc)
            v = torch.rand(s, generator=gen, device=dev).add_(0.5).mul_(0.1 * sc * sc)
            for k, x, top in (("m", m, 7), ("v", v, 14)):
                if case["op"] == "adamw":
                    st[k][i].copy_(x)
                else:
                    b = _in_blocks(x)
                    scale = _power_of_two(b.abs().amax(1, keepdim=True), top)
                    st[k + "_scale"][i].copy_(scale[:, 0])
                    st[k][i].copy_((b / scale).reshape(-1)[: x.numel()].view(s))
    if own:
        # what the program keeps: the parameters with their gradients, and the optimizer over them
        st["params"] = [torch.nn.Parameter(p) for p in st["p"]]
        for p, g in zip(st["params"], st["grads"][0][1]):
            p.grad = g
        if case["op"] != "clip":
            _optimizer(case, st)
    return st


def _optimizer(case, st):
    import came_b200
    cls = came_b200.AdamW if case["op"] == "adamw" else came_b200.AdamW8bit
    opt = st["opt"] = cls(st["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, max_grad_norm=case.get("max_norm"))
    if "grad_scale" in case:
        opt.param_groups[0]["grad_scale"] = case["grad_scale"]
    opt.prime_for_cuda_graph()
    for i, p in enumerate(st["params"]):      # the states of a checkpoint, in flat buffers
        s = opt.state[p]
        s["step"] = st["steps"][i]
        if case["op"] == "adamw":
            s["exp_avg"], s["exp_avg_sq"] = st["m"][i], st["v"][i]
        else:
            s["exp_avg_q"], s["exp_avg_scale"], s["exp_avg_sq_q"], s["exp_avg_sq_scale"] = (
                st["m"][i], st["m_scale"][i], st["v"][i], st["v_scale"][i])
    opt.prime_for_cuda_graph()
    if case.get("graph"):
        torch.cuda.synchronize()
        st["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(st["graph"]):
            opt.step()


def run(state):
    case, st = state["case"], state
    if len(st["grads"]) > 1:      # gradients that backward() has put elsewhere than at the last step
        st["turn"] ^= 1
        if own:
            for p, g in zip(st["params"], st["grads"][st["turn"]][1]):
                p.grad = g
    grads_buf, grads = st["grads"][st["turn"]]
    if case["op"] == "clip":
        if own:
            import came_b200
            norm = came_b200.clip_grad_norm_(st["params"], case["max_norm"])
        else:
            norm = _plain_clip(grads, case["max_norm"])
        return {"norm": norm, "grads": grads_buf}
    norm = None
    if own:
        if "graph" in st:
            st["graph"].replay()
        else:
            st["opt"].step()
        if "max_norm" in case:
            norm = st["opt"].grad_norm
    else:
        norm = _plain_step(case, st, grads)
    out = {"params": st["p_buf"], "exp_avg": st["m_buf"], "exp_avg_sq": st["v_buf"], "steps": st["steps"]}
    if case["op"] == "adamw8":
        out.update(exp_avg_scale=st["m_scale_buf"], exp_avg_sq_scale=st["v_scale_buf"])
    if norm is not None:
        out["norm"] = norm
    return out


# ---- plain form ------------------------------------------------------------------------------------------------------

def _plain_norm(grads, scale=1.0):
    """Square root of the sum of all squares; the long sum in 64 bits."""
    total = torch.stack([g.double().mul(scale).square().sum() for g in grads]).sum()
    return total.sqrt()


def _coefficient(norm, max_norm):
    return torch.clamp(max_norm / (norm + 1e-6), max=1.0)


def _plain_clip(grads, max_norm):
    norm = _plain_norm(grads)
    c = _coefficient(norm, max_norm).float()
    for g in grads:
        g.copy_(g.float() * c)
    return norm.float()


def _in_blocks(x):
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _mix32(x):
    """A hash of 32-bit numbers (held in int64): xor-shifts and multiplications."""
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & M32
    x = ((x ^ (x >> 15)) * 0x846CA68B) & M32
    return x ^ (x >> 16)


def _random_bits(n, t, device):
    """32 bits for each flat element of a tensor at its step t (a tensor)."""
    e = torch.arange(n, dtype=torch.int64, device=device)
    key = _mix32(t.to(torch.int64) & M32)
    h = _mix32(((e >> 3) + key) & M32)
    return (h * (((2 * (e & 7) + 1) * 0x9E3779B1) & M32)) & M32


def _encode(x, r, top, bits, dtype, floor):
    """(codes, scales) of blocks x [n, 256]: stochastic rounding by adding r below the last bit that is kept."""
    a = x.abs().amax(1, keepdim=True)
    scale = _power_of_two(a, top)
    y = x / scale
    if floor:
        y = torch.where(a > 0, y.clamp(min=floor), y)
    y = ((y.view(torch.int32) + r) & ~((1 << bits) - 1)).view(torch.float32)
    return y.to(dtype), scale[:, 0]


def _plain_step(case, st, grads):
    gs = case.get("grad_scale", 1.0)
    norm, c = None, torch.tensor(gs, device=grads[0].device)
    if "max_norm" in case:
        norm = _plain_norm(grads, gs)
        c = (_coefficient(norm, case["max_norm"]) * gs).float()
        norm = norm.float()
    st["steps"].add_(1)
    t = st["steps"].double()
    # 64 bits: 1 - beta^t loses what t = 1 leaves of it in 32
    size = (LR / (1.0 - BETAS[0] ** t)).float()
    root = (1.0 / (1.0 - BETAS[1] ** t).sqrt()).float()
    for i, (p, g) in enumerate(zip(st["p"], grads)):
        g32 = g.float() * c
        if case["op"] == "adamw":
            m, v = st["m"][i], st["v"][i]
        else:
            n = p.numel()
            m, v = ((_in_blocks(st[k][i].float()) * st[k + "_scale"][i].float()[:, None]).reshape(-1)[:n].view(p.shape) for k in ("m", "v"))
        m = m * BETAS[0] + g32 * (1.0 - BETAS[0])
        v = v * BETAS[1] + g32 * g32 * (1.0 - BETAS[1])
        p.copy_(p.float() * (1.0 - LR * WD) - size[i] * (m / (v.sqrt() * root[i] + EPS)))
        if case["op"] == "adamw":
            st["m"][i].copy_(m)
            st["v"][i].copy_(v)
        else:
            h = _in_blocks(_random_bits(n, st["steps"][i], p.device))
            qm, sm = _encode(_in_blocks(m), (h & 0xFFFFF).int(), 7, 20, torch.float8_e4m3fn, None)
            qv, sv = _encode(_in_blocks(v), (h >> 11).int(), 14, 21, torch.float8_e5m2, 2.0 ** -16)
            st["m"][i].copy_(qm.reshape(-1)[:n].view(p.shape))
            st["v"][i].copy_(qv.reshape(-1)[:n].view(p.shape))
            st["m_scale"][i].copy_(sm)
            st["v_scale"][i].copy_(sv)
    return norm


# ---- 64 bits ---------------------------------------------------------------------------------------------------------

def _exact_round(x, r, drop, top, floor):
    """A tensor's value after stochastic rounding to a float8 grid, from the definition: (values, scales)."""
    n = x.numel()
    full = torch.zeros(_blocks(n) * BLOCK, dtype=torch.float64, device=x.device)
    full[:n] = x.reshape(-1)
    full = full.view(-1, BLOCK)
    big = full.abs().max(dim=1).values
    k = torch.floor(torch.log2(big.clamp(min=2.0 ** -1000))) - top
    scale = torch.pow(2.0, k.clamp(-126, 127))
    y = full / scale[:, None]
    if floor:
        y = torch.where(big[:, None] > 0, torch.maximum(y, torch.full_like(y, floor)), y)
    a = y.abs()
    ulp = torch.pow(2.0, torch.floor(torch.log2(a.clamp(min=2.0 ** -120))) - (23 - drop))
    frac = torch.zeros(full.numel(), dtype=torch.float64, device=x.device)
    frac[:n] = r / 2.0 ** drop
    q = torch.floor(a / ulp + frac.view(-1, BLOCK)) * ulp
    least = 2.0 ** -9 if top == 7 else 2.0 ** -16      # subnormal spacing of the format
    q = torch.where(q < least * 2.0 ** (23 - drop), torch.round(q / least) * least, q) * torch.sign(y)
    return q.reshape(-1)[:n].view(x.shape), scale


def _exact_bits(n, t, device):
    group = torch.arange(-(-n // 8), dtype=torch.int64, device=device)

    def mixed(x):
        for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
            x = torch.remainder(torch.bitwise_xor(x, torch.div(x, 1 << shift, rounding_mode="floor")) * factor, 1 << 32)
        return torch.bitwise_xor(x, torch.div(x, 1 << 16, rounding_mode="floor"))

    key = mixed(torch.tensor(t, dtype=torch.int64, device=device))
    h = mixed(torch.remainder(group + key, 1 << 32))[:, None]
    odd = torch.tensor([(0x9E3779B1 * (2 * j + 1)) % (1 << 32) for j in range(8)], dtype=torch.int64, device=device)
    return torch.bitwise_and(h * odd[None, :], M32).reshape(-1)[:n]


def exact(case, seed):
    st = prepare(case, seed)
    turn = 1 if len(st["grads"]) > 1 else 0
    dev, gs, limit = st["p_buf"].device, case.get("grad_scale", 1.0), case.get("max_norm")
    total = torch.zeros((), dtype=torch.float64, device=dev)
    grads = st["grads"][turn][1]
    for g in grads:
        total += torch.linalg.vector_norm(g.double()) ** 2
    norm = torch.sqrt(total) * gs
    factor = gs * (min(1.0, limit / (float(norm) + 1e-6)) if limit is not None else 1.0)
    if case["op"] == "clip":
        return {"norm": norm, "grads": st["grads"][turn][0].double() * factor}
    out = {"params": torch.zeros_like(st["p_buf"], dtype=torch.float64), "steps": st["steps"].double() + 1}
    t = PAST + 1
    names = {"m": "exp_avg", "v": "exp_avg_sq"}
    for k in ("m", "v"):
        out[names[k]] = torch.zeros(st[k + "_buf"].shape, dtype=torch.float64, device=dev)
        if case["op"] == "adamw8":
            out[names[k] + "_scale"] = st[k + "_scale_buf"].float().double()

    def place(buf, like, view, x):
        start = (view.data_ptr() - like.data_ptr()) // like.element_size()
        buf[start: start + x.numel()] = x.reshape(-1)

    for i, g in enumerate(grads):
        g = g.double() * factor
        old = {}
        for k in ("m", "v"):
            x = st[k][i].to(torch.float64) if case["op"] == "adamw" else st[k][i].float().double()
            if case["op"] == "adamw8":
                x = (x.reshape(-1) * st[k + "_scale"][i].float().double().repeat_interleave(BLOCK)[: x.numel()]).view(x.shape)
            old[k] = x
        m = old["m"] + (1.0 - BETAS[0]) * (g - old["m"])
        v = old["v"] + (1.0 - BETAS[1]) * (g ** 2 - old["v"])
        m_hat, v_hat = m / (1.0 - BETAS[0] ** t), v / (1.0 - BETAS[1] ** t)
        p = st["p"][i].double()
        place(out["params"], st["p_buf"], st["p"][i], p - LR * WD * p - LR * m_hat / (torch.sqrt(v_hat) + EPS))
        if case["op"] == "adamw":
            place(out["exp_avg"], st["m_buf"], st["m"][i], m)
            place(out["exp_avg_sq"], st["v_buf"], st["v"][i], v)
            continue
        h = _exact_bits(m.numel(), t, dev)
        for k, x, r, drop, top, floor in (("m", m, h % (1 << 20), 20, 7, None),
                                          ("v", v, torch.div(h, 2048, rounding_mode="floor"), 21, 14, 2.0 ** -16)):
            q, scale = _exact_round(x, r.double(), drop, top, floor)
            place(out[names[k]], st[k + "_buf"], st[k][i], q)
            place(out[names[k] + "_scale"], st[k + "_scale_buf"], st[k + "_scale"][i], scale)
    if limit is not None:
        out["norm"] = norm
    return out


def work(case):
    """Compulsory bytes and operations of a pass: every input read once, every output written once.  A norm in front of a step reads
    the gradients once more: no element can be stepped before the last one has been seen.  Clip: below the limit."""
    esz = 4 if case["dtype"] == "float32" else 2
    n = float(sum(math.prod(s) for s in _shapes(case)))
    blocks = float(sum(_blocks(math.prod(s)) for s in _shapes(case)))
    if case["op"] == "clip":
        return {"bytes": n * esz, "flops": 2.0 * n}
    nbytes = n * 3 * esz + (16.0 * n if case["op"] == "adamw" else 4.0 * n + 4.0 * blocks)
    flops = (14.0 if case["op"] == "adamw" else 40.0) * n
    if "max_norm" in case:
        nbytes, flops = nbytes + n * esz, flops + 2.0 * n
    return {"bytes": nbytes, "flops": flops}
