"""Cases of the operators on 8-bit floating-point blocks: quantising with a scale for each block of 128, reading such a
matrix back, the matrix product of two of them, and that product grouped by expert with ragged sizes.

Sizes are those of the Llama-2-7B-shaped and Llama-3-70B-shaped weight sets that `bench.py` folds (4096, 11008, 8192,
1024), or generic ones where a mixture of experts or a ragged batch is meant. A matrix [rows, cols] of 8-bit floats
has scales of its own: one for each run of 128 columns of a row ("token" blocks, what a product multiplies), or one for each
block of 128 rows by 128 columns ("weight" blocks)."""
import functools
import math

import torch

own = False  # True: run() calls the library's operators; False: their plain form in elementary torch operations

DEV = "cuda"
BLOCK = 128
CODE = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SMALLEST_SCALE = 2.0 ** -126  # the scale of a block of zeros


# ---- cases -------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decoded token's activations in front of a projection: a call of a few microseconds
        {"name": "quantize_token", "op": "quantize", "rows": 1, "cols": 4096, "blocks": "token", "src": "bf16", "code": "e4m3"},
        # the activations of a long prompt in front of the down projection
        {"name": "quantize_prompt", "op": "quantize", "rows": 8192, "cols": 11008, "blocks": "token", "src": "bf16", "code": "e4m3"},
        # folding an up projection's fp16 weights
        {"name": "quantize_weight", "op": "quantize", "rows": 11008, "cols": 4096, "blocks": "weight", "src": "f16", "code": "e4m3"},
        # reading a folded weight back, to compare it or to run it where 8-bit products are not wanted
        {"name": "dequantize_weight", "op": "dequantize", "rows": 11008, "cols": 4096, "blocks": "weight", "code": "e4m3", "out": "f16"},
        # gradients or statistics kept in the wide-range type, read back in full precision; ragged both ways
        {"name": "dequantize_ragged", "op": "dequantize", "rows": 1003, "cols": 1111, "blocks": "token", "code": "e5m2", "out": "f32"},
        # one token through an up projection: the weights are read once, nothing else counts
        {"name": "matmul_token", "op": "matmul", "m": 1, "n": 11008, "k": 4096, "x": "e4m3", "w": "e4m3", "out": "bf16"},
        # a serving batch through a down projection: long sums, few rows
        {"name": "matmul_batch", "op": "matmul", "m": 48, "n": 4096, "k": 11008, "x": "e4m3", "w": "e4m3", "out": "bf16"},
        # nothing a multiple of anything: a ragged prompt through a layer of odd width, types mixed
        {"name": "matmul_ragged", "op": "matmul", "m": 777, "n": 1501, "k": 1000, "x": "e5m2", "w": "e4m3", "out": "f16"},
        # a prompt through an up projection: arithmetic bound
        {"name": "matmul_prompt", "op": "matmul", "m": 4096, "n": 11008, "k": 4096, "x": "e4m3", "w": "e4m3", "out": "bf16"},
        # a few tokens spread over many experts: most experts see one token or none
        {"name": "grouped_token", "op": "grouped", "m": 32, "pad": 0, "experts": 64, "n": 1024, "k": 2048, "x": "e4m3", "w": "e4m3", "out": "bf16"},
        # a small batch over few experts of odd width, with rows behind the last expert's that stay as they are
        {"name": "grouped_ragged", "op": "grouped", "m": 901, "pad": 123, "experts": 7, "n": 1410, "k": 1000, "x": "e4m3", "w": "e4m3", "out": "f16"},
        # a prompt's tokens routed over the experts of a layer
        {"name": "grouped_prompt", "op": "grouped", "m": 8192, "pad": 0, "experts": 32, "n": 4096, "k": 2048, "x": "e4m3", "w": "e4m3", "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "dequantize", "matmul", "grouped"])
    code = rng.choice(["e4m3", "e4m3", "e5m2"])
    if op in ("quantize", "dequantize"):
        cols = _log(rng, 1, 16384)
        rows = _log(rng, 1, min(32768, 8192 * 11008 // cols))
        c = {"op": op, "rows": rows, "cols": cols, "blocks": rng.choice(["token", "weight"]), "code": code}
        c["src" if op == "quantize" else "out"] = rng.choice(["f32", "f16", "bf16"])
        return c
    types = {"x": code, "w": rng.choice(["e4m3", "e4m3", "e5m2"]), "out": rng.choice(["bf16", "f16"])}
    k = _log(rng, 16, 11008)
    if op == "matmul":
        n = _log(rng, 1, 11008)
        return {"op": op, "m": _log(rng, 1, min(8192, 4096 * 11008 * 4096 // (n * k))), "n": n, "k": k, **types}
    experts = rng.randint(1, 64)
    n = _log(rng, 1, min(8192, 32 * 4096 * 2048 // (experts * min(k, 2048))))
    k = min(k, 32 * 4096 * 2048 // (experts * n))
    m = _log(rng, 1, max(2, min(8192, 8192 * 4096 * 2048 // (n * k))))
    return {"op": op, "m": m, "pad": rng.choice([0, 0, rng.randint(1, 200)]), "experts": experts, "n": n, "k": max(16, k), **types}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _ld(cols):
    return -(-cols // 16) * 16  # rows of 8-bit codes start on 16-byte boundaries


def _values(g, shape, sigma, outliers):
    """Bell-shaped values with an outlier every thousand elements, 20 times as large, as the weight sets have them."""
    x = torch.randn(shape, generator=g, device=DEV) * sigma
    if outliers:
        x = torch.where(torch.rand(shape, generator=g, device=DEV) < 1e-3, x * 20, x)
    return x


def _padded(x, rows):
    r, c = x.shape[-2:]
    return torch.nn.functional.pad(x, (0, -c % BLOCK, 0, -r % rows))


def _quantized(x, rows, code):
    """(codes [..., rows, cols], scales [..., row blocks, column blocks]) of x."""
    r, c = x.shape[-2:]
    p = _padded(x.float(), rows)
    b = p.reshape(*p.shape[:-2], p.shape[-2] // rows, rows, p.shape[-1] // BLOCK, BLOCK)
    scale = (b.abs().amax((-3, -1)) / LARGEST[code]).clamp_min(SMALLEST_SCALE)
    q = b * (1.0 / scale)[..., :, None, :, None]
    q = q.clamp(-LARGEST[code], LARGEST[code]).reshape(p.shape)[..., :r, :c]
    return q.to(CODE[code]), scale


def _made(g, shape, rows, code, sigma, outliers):
    """A matrix (or a stack of them) of 8-bit floats in memory as a program keeps it: codes with padded rows, scales. The
    scales of token blocks lie column block by column block, so that the rows of a tile are neighbours."""
    codes, scales = _quantized(_values(g, shape, sigma, outliers), rows, code)
    buf = torch.zeros(*shape[:-1], _ld(shape[-1]), dtype=torch.uint8, device=DEV)
    buf[..., :shape[-1]] = codes.view(torch.uint8)
    return buf, (scales.transpose(-1, -2) if rows == 1 else scales).contiguous()


def _counts(case, seed):
    """How many rows each expert gets: experts differ in how often they are chosen, some get none."""
    g = torch.Generator().manual_seed(seed)
    chosen = torch.multinomial(_popularity(case["experts"]), case["m"], True, generator=g)
    return torch.bincount(chosen, minlength=case["experts"])


def _popularity(experts):
    return 1.0 / (torch.arange(experts, dtype=torch.float64) + 8.0)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["op"] in ("quantize", "dequantize"):
        s["block_rows"] = rows = 1 if case["blocks"] == "token" else BLOCK
        shape = (case["rows"], case["cols"])
        row_blocks, col_blocks = -(-shape[0] // rows), -(-shape[1] // BLOCK)
    if case["op"] == "quantize":
        s["base"] = _values(g, shape, 0.02 if rows > 1 else 1.0, True).to(FLOAT[case["src"]])
        s["codes"] = torch.empty(shape[0], _ld(shape[1]), dtype=torch.uint8, device=DEV)
        s["scales"] = torch.empty((col_blocks, row_blocks) if rows == 1 else (row_blocks, col_blocks), device=DEV)
    elif case["op"] == "dequantize":
        s["codes"], s["scales"] = _made(g, shape, rows, case["code"], 0.02, True)
        s["dst"] = torch.empty(shape, dtype=FLOAT[case["out"]], device=DEV)
    else:
        experts = case.get("experts", 0)
        rows = case["m"] + case.get("pad", 0)
        s["xc"], s["xs"] = _made(g, (rows, case["k"]), 1, case["x"], 1.0, True)
        s["wc"], s["ws"] = _made(g, ((experts,) if experts else ()) + (case["n"], case["k"]), BLOCK, case["w"], 0.02, True)
        s["dst"] = torch.randn(rows, case["n"], generator=g, device=DEV).to(FLOAT[case["out"]])
        if experts:
            counts = _counts(case, seed)
            s["most"] = int(counts.max())
            s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(DEV)
    if own:
        _handles(s)
    return s


# ---- the library's operators -------------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _context(device, stream):
    from vpux_plugin_b200.lib import Library
    return Library(device=device, stream=stream or 1, pipelined=True)  # 1 is the handle of the legacy default stream


def _library(device):
    """The context of torch's current stream on `device`: its calls line up with what torch enqueues there. (The handle is
    asked for as compiled graphs do it; the stream object of torch.cuda.current_stream() costs as much as a small call.)"""
    return _context(device, torch._C._cuda_getCurrentRawStream(device))


def _matrix(codes, scales, cols, rows, code):
    from vpux_plugin_b200 import abi
    dtype = abi.VF_DT_F8E4M3FN if code == "e4m3" else abi.VF_DT_F8E5M2
    token = rows == 1
    return abi.block_matrix(codes.data_ptr(), scales.data_ptr(), dtype, rows, codes.shape[-2], cols, ld=codes.shape[-1],
                            count=codes.shape[0] if codes.dim() == 3 else 1,
                            scale_row_stride=1 if token else scales.shape[-1], scale_col_stride=scales.shape[-1] if token else 1)


def _handles(s):
    """What a program keeps next to its buffers: the descriptors of its matrices. The context that it calls is made here too."""
    from vpux_plugin_b200 import abi
    s["device"] = torch.cuda.current_device()
    _library(s["device"])
    dt = {"f32": abi.VF_DT_F32, "f16": abi.VF_DT_F16, "bf16": abi.VF_DT_BF16}
    if s["op"] in ("quantize", "dequantize"):
        s["matrix"] = _matrix(s["codes"], s["scales"], s["cols"], s["block_rows"], s["code"])
    if s["op"] == "quantize":
        s["content"], s["keep"] = abi.make_content(abi.TType(list(s["base"].shape), dt[s["src"]]), None, mem_kind=abi.VF_MEM_DEVICE,
                                                   ptr=s["base"].data_ptr(), nbytes=s["base"].nbytes)
    else:
        s["out_dtype"] = dt[s["out"]]
    if s["op"] in ("matmul", "grouped"):
        s["xm"] = _matrix(s["xc"], s["xs"], s["k"], 1, s["x"])
        s["wm"] = _matrix(s["wc"], s["ws"], s["k"], BLOCK, s["w"])


def _own(s):
    lib = _library(s["device"])
    if s["op"] == "quantize":
        lib.quantize_blocks(s["content"], s["matrix"])
        return {"codes": s["codes"].view(CODE[s["code"]])[:, :s["cols"]], "scales": s["scales"]}
    dst = s["dst"]
    if s["op"] == "dequantize":
        lib.dequantize_blocks(s["matrix"], dst.data_ptr(), s["out_dtype"], dst.nbytes)
    elif s["op"] == "matmul":
        lib.matmul_blocks(s["xm"], s["wm"], dst.data_ptr(), s["out_dtype"], dst.nbytes)
    else:
        lib.matmul_blocks_grouped(s["xm"], s["wm"], s["offsets"].data_ptr(), dst.data_ptr(), s["out_dtype"], dst.nbytes)
    return dst


# ---- the plain form ----------------------------------------------------------------------------------------------------

def _floats(codes, scales, cols, rows, code):
    """The fp32 values of a matrix of 8-bit floats: code times its block's scale."""
    v = codes.view(CODE[code])[..., :cols].float()
    if rows == 1:
        scales = scales.transpose(-1, -2)
    scales = scales.repeat_interleave(rows, -2)[..., :v.shape[-2], :].repeat_interleave(BLOCK, -1)[..., :cols]
    return v * scales


def _plain(s):
    if s["op"] == "quantize":
        q, scale = _quantized(s["base"], s["block_rows"], s["code"])
        return {"codes": q, "scales": (scale.transpose(-1, -2) if s["block_rows"] == 1 else scale).contiguous()}
    if s["op"] == "dequantize":
        return _floats(s["codes"], s["scales"], s["cols"], s["block_rows"], s["code"]).to(FLOAT[s["out"]])
    x = _floats(s["xc"], s["xs"], s["k"], 1, s["x"])
    w = _floats(s["wc"], s["ws"], s["k"], BLOCK, s["w"])
    if s["op"] == "matmul":
        return (x @ w.T).to(FLOAT[s["out"]])
    # every expert's rows, padded to the longest one's, as one batch of products
    first, last = s["offsets"][:-1, None], s["offsets"][1:, None]
    at = first + torch.arange(max(1, s["most"]), device=DEV)[None]
    mine = at < last
    y = x[at.clamp_max(x.shape[0] - 1)] @ w.transpose(1, 2)
    out = s["dst"].clone()
    out[at[mine]] = y[mine].to(out.dtype)
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    col_blocks = -(-case.get("cols", case.get("k", 0)) // BLOCK)
    if case["op"] in ("quantize", "dequantize"):
        n = case["rows"] * case["cols"]
        row_blocks = case["rows"] if case["blocks"] == "token" else -(-case["rows"] // BLOCK)
        wide = SIZE[case["src" if case["op"] == "quantize" else "out"]]
        return {"bytes": n * (1 + wide) + 4 * row_blocks * col_blocks, "flops": n * (2 if case["op"] == "quantize" else 1)}
    m, n, k = case["m"], case["n"], case["k"]
    used = 1.0
    if case["op"] == "grouped":  # the experts that get a row, on average over the routing
        p = _popularity(case["experts"])
        used = float((1 - (1 - p / p.sum()) ** m).sum())
    return {"bytes": m * (k + 4 * col_blocks) + used * (n * k + 4 * -(-n // BLOCK) * col_blocks) + m * n * SIZE[case["out"]],
            "flops": 2.0 * m * n * k}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------

def _table(code):
    """The values of the 256 codes, from the format: sign, exponent field, mantissa field."""
    exp_bits, man_bits = (4, 3) if code == "e4m3" else (5, 2)
    bias = 2 ** (exp_bits - 1) - 1
    out = []
    for b in range(256):
        e, m = (b >> man_bits) & (2 ** exp_bits - 1), b & (2 ** man_bits - 1)
        v = math.ldexp(m, 1 - bias - man_bits) if e == 0 else math.ldexp(2 ** man_bits + m, e - bias - man_bits)
        if code == "e5m2" and e == 31:
            v = math.nan if m else math.inf
        if code == "e4m3" and b & 127 == 127:
            v = math.nan
        out.append(-v if b & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device=DEV)


def _exact_values(codes, scales, cols, rows, code):
    v = _table(code)[codes[..., :cols].long()]
    sc = scales.double()
    r = torch.arange(v.shape[-2], device=DEV) // rows
    c = torch.arange(cols, device=DEV) // BLOCK
    return v * (sc[..., c, :][..., r].transpose(-1, -2) if rows == 1 else sc[..., r, :][..., c])


def _nearest(v, code):
    """v rounded to the nearest value of the 8-bit type, ties to the even mantissa; v is within its range."""
    man, least = (3, -6) if code == "e4m3" else (2, -14)
    step = torch.exp2(torch.frexp(v)[1].sub(1).clamp_min(least).double() - man)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x, rows = s["base"].double(), s["block_rows"]
        p = _padded(x, rows)
        top = p.abs().reshape(p.shape[0] // rows, rows, p.shape[1] // BLOCK, BLOCK).amax((1, 3)) / LARGEST[case["code"]]
        top = top.clamp_min(SMALLEST_SCALE)
        r, c = torch.arange(x.shape[0], device=DEV) // rows, torch.arange(x.shape[1], device=DEV) // BLOCK
        return {"codes": _nearest(x / top[r][:, c], case["code"]), "scales": top.T.contiguous() if rows == 1 else top}
    if case["op"] == "dequantize":
        return _exact_values(s["codes"], s["scales"], s["cols"], s["block_rows"], s["code"])
    x = _exact_values(s["xc"], s["xs"], s["k"], 1, s["x"])
    if case["op"] == "matmul":
        return x @ _exact_values(s["wc"], s["ws"], s["k"], BLOCK, s["w"]).T
    out, at = s["dst"].double(), s["offsets"].tolist()
    for e in range(case["experts"]):
        if at[e] < at[e + 1]:
            out[at[e]:at[e + 1]] = x[at[e]:at[e + 1]] @ _exact_values(s["wc"][e], s["ws"][e], s["k"], BLOCK, s["w"]).T
    return out
