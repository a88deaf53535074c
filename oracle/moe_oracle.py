"""CPU oracle for the DeepSeek-V2 MoE block -- TEST INFRASTRUCTURE ONLY.

Only ``tests/``, ``__graft_entry__.smoke()`` and ``bench.py``'s CPU-baseline leg (``cpu_baseline``
and ``--impl reference``) import this module, and only as the checker or as the timed CPU
baseline. The product path (``libuocr_moe.so`` and the ``unlimited-ocr-max_b200`` package)
never imports it and has no CPU fallback.

Parity is pinned: ``tests/test_oracle.py`` checks every function here against the golden
fixtures that ``tests/golden/make_golden.py`` generated by running the reference's own numpy
code (its quantiser, its kernel tests' reference functions, its float64 MoE reference).

Two kinds of functions:

* bit-exact fp32 orders (``route_fp32``, ``int8_qmv_base_order``, ``exp_f32``) live in
  ``moe_oracle.c`` and are called through ctypes; the CUDA kernels reproduce them bit for bit;
* float64 / numpy / torch restatements of the reference's math (``quantize_per_group``,
  ``dequant_bits``, ``qmv_ref64``, ``moe_layer_fp64``, the fp32 CPU paths used as the timed
  baseline), each citing the reference ``file:line`` it follows.
"""

from __future__ import annotations

import ctypes
import os
import subprocess
from dataclasses import dataclass
from pathlib import Path

import numpy as np

HERE = Path(__file__).resolve().parent
BUILD_DIR = HERE / "_build"
LIB_PATH = BUILD_DIR / "liboracle.so"

#: int8 quantisation group along K (model_config.py:52 INT8_GROUP_SIZE; tools/quantize_int8.py:144)
GROUP_SIZE = 128
QMAX = 127


# ---------------------------------------------------------------------------
# the C library
# ---------------------------------------------------------------------------


def build(force: bool = False) -> Path:
    """Compile ``moe_oracle.c`` into ``_build/liboracle.so`` (gcc, no fp contraction)."""
    src = HERE / "moe_oracle.c"
    if LIB_PATH.exists() and not force and LIB_PATH.stat().st_mtime >= src.stat().st_mtime:
        return LIB_PATH
    BUILD_DIR.mkdir(exist_ok=True)
    tmp = LIB_PATH.with_suffix(f".{os.getpid()}.tmp")
    cmd = ["gcc", "-O2", "-std=c11", "-ffp-contract=off", "-fno-fast-math", "-fPIC", "-shared", str(src), "-o", str(tmp), "-lm"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


_LIB = None


def lib() -> ctypes.CDLL:
    global _LIB
    if _LIB is None:
        path = build()
        L = ctypes.CDLL(str(path))
        P = ctypes.c_void_p
        I = ctypes.c_int
        L.oracle_route_fp32.argtypes = [P, I, I, P, P, I, I, P, P, P, P]
        L.oracle_route_fp32.restype = I
        L.oracle_int8_qmv.argtypes = [P, I, I, P, P, P, I, I, I, P]
        L.oracle_int8_qmv.restype = I
        L.oracle_exp_many.argtypes = [P, P, ctypes.c_long]
        L.oracle_exp_many.restype = None
        L.oracle_exp_f32.argtypes = [ctypes.c_float]
        L.oracle_exp_f32.restype = ctypes.c_float
        _LIB = L
    return _LIB


def _ptr(a: np.ndarray | None):
    return None if a is None else ctypes.c_void_p(a.ctypes.data)


# ---------------------------------------------------------------------------
# bf16 helpers (tests/_harness.py:36-50, unlimited_ocr_max/bf16.py:37-63)
# ---------------------------------------------------------------------------


def bf16_bits(values: np.ndarray) -> np.ndarray:
    """fp32 -> bf16 bit patterns (uint16), round to nearest even, computed in uint32."""
    bits = np.ascontiguousarray(values, dtype=np.float32).view(np.uint32)
    carry = ((bits & np.uint32(0xFFFF)) + ((bits >> 16) & np.uint32(1)) + np.uint32(0x7FFF)) >> 16
    return ((bits >> 16) + carry).astype(np.uint16)


def bf16_to_f32(bits: np.ndarray) -> np.ndarray:
    """bf16 bit patterns -> fp32 (exact)."""
    return (np.asarray(bits, dtype=np.uint16).astype(np.uint32) << np.uint32(16)).view(np.float32)


def clamp(e: int, num_experts: int) -> int:
    """An expert id as the kernels read it: clamped to [0, E) (kernels/moe_routing.mojo:36-44)."""
    return min(max(int(e), 0), num_experts - 1)


def rel_err(got: np.ndarray, ref: np.ndarray) -> float:
    """max|got-ref| / max|ref| in float64 (tests/_harness.py:53-60)."""
    g, r = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    denom = float(np.max(np.abs(r))) if r.size else 0.0
    if denom == 0.0:
        return float(np.max(np.abs(g))) if g.size else 0.0
    return float(np.max(np.abs(g - r)) / denom)


def cosine(a: np.ndarray, b: np.ndarray) -> float:
    a, b = np.asarray(a, np.float64).ravel(), np.asarray(b, np.float64).ravel()
    return float(a @ b / (np.linalg.norm(a) * np.linalg.norm(b)))


def rel_l2(got: np.ndarray, ref: np.ndarray) -> float:
    g, r = np.asarray(got, np.float64).ravel(), np.asarray(ref, np.float64).ravel()
    return float(np.linalg.norm(g - r) / max(np.linalg.norm(r), 1e-300))


# ---------------------------------------------------------------------------
# the int8 format (tools/quantize_int8.py:55-70, 298-329; kernels/moe_int8.mojo:43-50, 330-340)
# ---------------------------------------------------------------------------


def quantize_per_group(w: np.ndarray, group: int = GROUP_SIZE) -> tuple[np.ndarray, np.ndarray]:
    """``[..., N, K]`` fp32 -> ``(int8 [..., N, K], fp32 [..., N, K/group])``.

    amax = max|w_g| in fp32; scale = amax / 127 (an fp32 DIVISION), 1.0 for an all-zero group;
    q = clip(rint(w / scale), -127, 127) with rint half-to-even and a true division per element.
    """
    w = np.ascontiguousarray(w, dtype=np.float32)
    *lead, n, k = w.shape
    if k % group:
        raise ValueError(f"K={k} is not divisible by the group size {group}")
    if not np.isfinite(w).all():
        raise ValueError("weight holds NaN or Inf; refusing to quantise it")
    g = w.reshape(*lead, n, k // group, group)
    amax = np.maximum(g.max(axis=-1), -g.min(axis=-1))
    scales = np.where(amax == np.float32(0.0), np.float32(1.0), amax / np.float32(QMAX)).astype(np.float32)
    q = np.rint(g / scales[..., None])
    q = np.clip(q, -QMAX, QMAX).astype(np.int8).reshape(*lead, n, k)
    return q, scales


def dequant_bits(w: np.ndarray, scales: np.ndarray, idx: int) -> np.ndarray:
    """int8_dequant_expert's bits: bf16_RNE(fp32(q[e]) * scale[e, n, k // G]), e clamped."""
    e = clamp(idx, w.shape[0])
    gsize = w.shape[2] // scales.shape[2]
    prod = w[e].astype(np.float32) * np.repeat(scales[e].astype(np.float32), gsize, axis=1)
    return bf16_bits(prod)


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------


def exp_f32(x: np.ndarray) -> np.ndarray:
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    lib().oracle_exp_many(_ptr(x), _ptr(y), x.size)
    return y


@dataclass
class Routing:
    ids: np.ndarray  # int32 [T, k]
    weights: np.ndarray  # fp32 [T, k]
    logits: np.ndarray  # fp32 [T, E] (bias added)
    probs: np.ndarray  # fp32 [T, E]


def route_fp32(x: np.ndarray, router_bits: np.ndarray, bias: np.ndarray | None = None, topk: int = 6) -> Routing:
    """The bit-exact fp32 router (MoEGate.__call__, decoder.py:509-514) in this build's order.

    See moe_oracle.c for the order; the GPU router reproduces it bit for bit.
    """
    x = np.ascontiguousarray(x, dtype=np.float32)
    w = np.ascontiguousarray(router_bits, dtype=np.uint16)
    T, H = x.shape
    E = w.shape[0]
    b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
    ids = np.empty((T, topk), np.int32)
    wts = np.empty((T, topk), np.float32)
    logits = np.empty((T, E), np.float32)
    probs = np.empty((T, E), np.float32)
    rc = lib().oracle_route_fp32(_ptr(x), T, H, _ptr(w), _ptr(b), E, topk, _ptr(ids), _ptr(wts), _ptr(logits), _ptr(probs))
    if rc:
        raise ValueError("oracle_route_fp32: bad shape")
    return Routing(ids, wts, logits, probs)


def route_fp64(x: np.ndarray, router: np.ndarray, bias: np.ndarray | None = None, topk: int = 6):
    """float64 gate as the reference's fp64 test oracle computes it (tests/test_decoder_int8.py:720-727):
    softmax over all experts, ``argsort(-p, kind="stable")`` top-k (ties -> lowest index).

    Returns ``(ids [T,k], weights [T,k], margin [T])`` where margin = p_k - p_{k+1} (the gap
    between the last chosen and the first unchosen probability): a near-tie indicator.
    """
    xf = np.asarray(x, np.float64)
    wf = np.asarray(router, np.float64)
    logits = xf @ wf.T
    if bias is not None:
        logits = logits + np.asarray(bias, np.float64)
    p = np.exp(logits - logits.max(axis=1, keepdims=True))
    p /= p.sum(axis=1, keepdims=True)
    order = np.argsort(-p, axis=1, kind="stable")
    ids = order[:, :topk].astype(np.int32)
    wts = np.take_along_axis(p, ids, axis=1)
    nxt = np.take_along_axis(p, order[:, topk : topk + 1], axis=1)[:, 0] if p.shape[1] > topk else np.full(len(p), np.inf)
    return ids, wts, wts[:, -1] - nxt


# ---------------------------------------------------------------------------
# expert GEMVs (the reference's custom ops)
# ---------------------------------------------------------------------------


def int8_qmv_base_order(x: np.ndarray, ids: np.ndarray, w: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """moe_int8_qmv's exact bits (kernels/moe_int8.mojo:114-148), via the C oracle."""
    x = np.ascontiguousarray(x, np.float32)
    ids = np.ascontiguousarray(ids, np.int32)
    w = np.ascontiguousarray(w, np.int8)
    scales = np.ascontiguousarray(scales, np.float32)
    k, K = x.shape
    E, N, _ = w.shape
    out = np.empty((k, N), np.float32)
    rc = lib().oracle_int8_qmv(_ptr(x), k, K, _ptr(ids), _ptr(w), _ptr(scales), E, N, scales.shape[2], _ptr(out))
    if rc:
        raise ValueError("oracle_int8_qmv: K must be a multiple of the group count")
    return out


def bf16_qmv_ref64(x: np.ndarray, ids: np.ndarray, w_bits: np.ndarray) -> np.ndarray:
    """float64 moe_bf16_qmv contract, ids clamped (tests/test_kernels_bf16.py:118-122)."""
    xf, wf = np.asarray(x, np.float64), bf16_to_f32(w_bits).astype(np.float64)
    E = w_bits.shape[0]
    out = np.zeros((x.shape[0], w_bits.shape[1]), np.float64)
    for s in range(x.shape[0]):
        out[s] = wf[clamp(ids[s], E)] @ xf[s]
    return out


def int8_qmv_ref64(x: np.ndarray, ids: np.ndarray, w: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """float64 moe_int8_qmv contract, ids clamped (tests/test_kernels_int8.py:142-155)."""
    xf, wf, sf = (np.asarray(a, np.float64) for a in (x, w, scales))
    E, N, K = w.shape
    G = scales.shape[2]
    out = np.empty((x.shape[0], N), np.float64)
    for s in range(x.shape[0]):
        e = clamp(ids[s], E)
        gs = (wf[e] * xf[s]).reshape(N, G, K // G).sum(axis=2)
        out[s] = (sf[e] * gs).sum(axis=1)
    return out


def kblocked(w_bits: np.ndarray, kblock: int = 16) -> np.ndarray:
    """W [N, K] -> [K/16, N, 16] (weight_adapters.py:222-233)."""
    n, k = w_bits.shape
    return np.ascontiguousarray(w_bits.reshape(n, k // kblock, kblock).transpose(1, 0, 2))


# ---------------------------------------------------------------------------
# the MoE layer
# ---------------------------------------------------------------------------


@dataclass
class MoEConfig:
    """The MoE hyper-parameters of the reference decoder (model_config.py:66-173, decoder.py:533-554)."""

    hidden: int = 1280
    inter: int = 896  # moe_intermediate_size
    n_routed: int = 64
    n_shared: int = 2  # shared_experts_dim = n_shared * inter
    top_k: int = 6
    group: int = GROUP_SIZE

    @property
    def shared_dim(self) -> int:
        return self.n_shared * self.inter


@dataclass
class MoEWeights:
    """One layer's weights in the reference's declared layout (decoder.py:305-313, 269-271, 507).

    bf16 tensors are uint16 bit patterns. ``gate/up/down`` are the routed stacks
    ``[E, I, H]``/``[E, I, H]``/``[E, H, I]`` -- bf16 bits, or int8 with ``*_scales``.
    """

    router: np.ndarray  # bf16 [E, H]
    gate: np.ndarray
    up: np.ndarray
    down: np.ndarray
    shared_gate: np.ndarray  # bf16 [S*I, H]
    shared_up: np.ndarray  # bf16 [S*I, H]
    shared_down: np.ndarray  # bf16 [H, S*I]
    gate_scales: np.ndarray | None = None
    up_scales: np.ndarray | None = None
    down_scales: np.ndarray | None = None

    @property
    def int8(self) -> bool:
        return self.gate.dtype == np.int8

    def stack_f64(self, name: str) -> np.ndarray:
        """A routed stack's exact values in float64 (int8: q * scale, the kernels' association)."""
        w = getattr(self, name)
        if w.dtype == np.int8:
            s = getattr(self, f"{name}_scales").astype(np.float64)
            return w.astype(np.float64) * np.repeat(s, w.shape[2] // s.shape[2], axis=2)
        return bf16_to_f32(w).astype(np.float64)


def synth_weights(cfg: MoEConfig, seed: int, *, int8: bool = False, std: float = 0.02) -> MoEWeights:
    """Seeded synthetic weights: every matrix ~N(0, std) rounded to bf16; int8 stacks quantised
    from those bf16 values by :func:`quantize_per_group`."""
    rng = np.random.default_rng(seed)
    H, I, E, SI = cfg.hidden, cfg.inter, cfg.n_routed, cfg.shared_dim

    def mat(*shape):
        return bf16_bits((rng.standard_normal(shape, dtype=np.float32) * np.float32(std)))

    router = mat(E, H)
    gate, up, down = mat(E, I, H), mat(E, I, H), mat(E, H, I)
    sg, su, sd = mat(SI, H), mat(SI, H), mat(H, SI)
    w = MoEWeights(router, gate, up, down, sg, su, sd)
    if int8:
        for name in ("gate", "up", "down"):
            q, s = quantize_per_group(bf16_to_f32(getattr(w, name)), cfg.group)
            setattr(w, name, q)
            setattr(w, f"{name}_scales", s)
    return w


def rms_normalised(x: np.ndarray, eps: float = 1e-6) -> np.ndarray:
    """x / sqrt(mean(x^2) + eps) per row, gamma = 1 (RMSNorm with model_config.py:54's eps)."""
    x64 = np.asarray(x, np.float64)
    return (x64 / np.sqrt((x64 * x64).mean(axis=1, keepdims=True) + eps)).astype(np.float32)


def synth_hidden(T: int, H: int, seed: int) -> np.ndarray:
    rng = np.random.default_rng(seed)
    return rms_normalised(rng.standard_normal((T, H), dtype=np.float32))


def moe_layer_fp64(cfg: MoEConfig, w: MoEWeights, x: np.ndarray, ids: np.ndarray | None = None,
                   wts: np.ndarray | None = None, bias: np.ndarray | None = None) -> np.ndarray:
    """The MoE layer's exact math in float64 (tests/test_decoder_int8.py:720-732, decoder.py:641-667).

    Routing comes from ``ids``/``wts`` when given (e.g. the bit-exact fp32 routing, so a near-tie
    cannot flip an expert between the two sides); else from :func:`route_fp64`.
    """
    xf = np.asarray(x, np.float64)
    if ids is None:
        ids, wts, _ = route_fp64(x, bf16_to_f32(w.router), bias, cfg.top_k)
    wts = np.asarray(wts, np.float64)
    ids = np.asarray(ids)
    gate, up, down = (w.stack_f64(n) for n in ("gate", "up", "down"))
    silu = lambda a: a / (1.0 + np.exp(-a))  # noqa: E731
    # per (token, slot) expert outputs, computed expert by expert over the tokens that chose it
    y = np.zeros((xf.shape[0], ids.shape[1], xf.shape[1]))
    for e in np.unique(ids):
        tt, ss = np.nonzero(ids == e)
        xe = xf[tt]
        y[tt, ss] = (silu(xe @ gate[e].T) * (xe @ up[e].T)) @ down[e].T
    out = np.zeros_like(xf)
    for s in range(ids.shape[1]):
        out += wts[:, s : s + 1] * y[:, s]
    sg, su, sd = (bf16_to_f32(a).astype(np.float64) for a in (w.shared_gate, w.shared_up, w.shared_down))
    out += (silu(xf @ sg.T) * (xf @ su.T)) @ sd.T
    return out


# ---------------------------------------------------------------------------
# the reference's fp32 CPU paths (the timed CPU baseline), restated in torch fp32
# ---------------------------------------------------------------------------


class TorchCpuLayer:
    """One MoE layer's weights as fp32 torch CPU tensors, for the reference's fp32 CPU paths.

    bf16 weights are held as their exact fp32 values (the reference upcasts at run time,
    decoder.py:227-234); int8 stacks as int8 + fp32 scales.
    """

    def __init__(self, cfg: MoEConfig, w: MoEWeights):
        import torch

        self.cfg = cfg
        f = lambda a: torch.from_numpy(bf16_to_f32(a))  # noqa: E731
        self.router = f(w.router)
        self.int8 = w.int8
        if w.int8:
            self.q = {n: torch.from_numpy(getattr(w, n)) for n in ("gate", "up", "down")}
            self.s = {n: torch.from_numpy(getattr(w, f"{n}_scales")) for n in ("gate", "up", "down")}
        else:
            self.stk = {n: f(getattr(w, n)) for n in ("gate", "up", "down")}
        self.sg, self.su, self.sd = f(w.shared_gate), f(w.shared_up), f(w.shared_down)

    def gate(self, x, bias=None):
        import torch

        logits = x @ self.router.T
        if bias is not None:
            logits = logits + bias
        p = torch.softmax(logits, dim=-1)
        wts, ids = torch.topk(p, self.cfg.top_k, dim=-1)
        return ids, wts

    def expert_rows(self, name: str, x, e: int):
        """``x @ W[e].T`` for one routed stack (int8: sum_g scale * sum_{k in g} q * x)."""
        import torch

        if not self.int8:
            return x @ self.stk[name][e].T
        q, s = self.q[name][e], self.s[name][e]
        n, k = q.shape
        g = s.shape[1]
        parts = torch.einsum("ngc,tgc->tng", q.float().view(n, g, k // g), x.view(x.shape[0], g, k // g))
        return (parts * s).sum(-1)

    def shared(self, x):
        import torch

        return (torch.nn.functional.silu(x @ self.sg.T) * (x @ self.su.T)) @ self.sd.T

    def decode_rows(self, x, bias=None):
        """MoE.decode_rows (decoder.py:641-655): top-k per row, the row's six expert GEMVs
        (moe_*_qmv), the [B,1,6]@[B,6,H] mix (decoder.py:599-604), plus the shared experts."""
        import torch

        ids, wts = self.gate(x, bias)
        B = x.shape[0]
        rows = []
        for b in range(B):
            ys = []
            for s in range(self.cfg.top_k):
                e = int(ids[b, s])
                xb = x[b : b + 1]
                h = torch.nn.functional.silu(self.expert_rows("gate", xb, e)) * self.expert_rows("up", xb, e)
                ys.append(self.expert_rows("down", h, e))
            rows.append(wts[b : b + 1] @ torch.cat(ys))
        return torch.cat(rows) + self.shared(x)

    def prefill_dense(self, x, bias=None):
        """MoE.__call__ on CPU / int8 (decoder.py:556-584, 657-667): the dense [T,64] router
        matrix and the unfused 64-term chain over ascending expert index, every expert over
        every token, plus the shared experts."""
        import torch

        ids, wts = self.gate(x, bias)
        router = torch.zeros(x.shape[0], self.cfg.n_routed, dtype=x.dtype)
        router.scatter_(1, ids, wts)
        routed = None
        for j in range(self.cfg.n_routed):
            h = torch.nn.functional.silu(self.expert_rows("gate", x, j)) * self.expert_rows("up", x, j)
            term = router[:, j : j + 1] * self.expert_rows("down", h, j)
            routed = term if routed is None else routed + term
        return routed + self.shared(x)


# ---------------------------------------------------------------------------
# the no-repeat-n-gram guard (kernels/ngram_block.mojo:1-33, the reference's
# SlidingWindowNoRepeatNgramProcessor; its tests' oracle, tests/test_kernels_ngram.py:56-69)
# ---------------------------------------------------------------------------

#: the value a banned logit is set to (kernels/ngram_block.mojo:47)
NGRAM_BLOCKED = np.float32(-3.0e38)


def ngram_banned(sequence, ngram_size: int, window: int) -> set[int]:
    """The token ids banned after ``sequence``: every n-gram that starts inside the last ``window``
    positions and whose first n - 1 ids equal the sequence's last n - 1 bans its last id (n = 1:
    every id in the window). Nothing for n < 1 or a sequence shorter than n."""
    ids = [int(i) for i in sequence]
    if ngram_size < 1 or len(ids) < ngram_size:
        return set()
    first = max(0, len(ids) - window)
    last = len(ids) - ngram_size + 1
    prefix = tuple(ids[len(ids) - (ngram_size - 1):]) if ngram_size > 1 else ()
    out: set[int] = set()
    for start in range(first, last):
        gram = ids[start:start + ngram_size]
        if ngram_size == 1 or tuple(gram[:-1]) == prefix:
            out.add(gram[-1])
    return out


def ngram_block_rows(logits: np.ndarray, sequences, ngram_size: int, window: int) -> np.ndarray:
    """``logits [B, V]`` with row b's banned ids (for ``sequences[b]``) set to NGRAM_BLOCKED."""
    out = np.array(logits, dtype=np.float32, copy=True)
    for b, seq in enumerate(sequences):
        for tok in ngram_banned(seq, ngram_size, window):
            if 0 <= tok < out.shape[1]:
                out[b, tok] = NGRAM_BLOCKED
    return out


# ---------------------------------------------------------------------------
# paged decode attention (decoder.py:425-437; the page pool of kv_cache.py:1-40)
# ---------------------------------------------------------------------------


def paged_decode_attention_ref(q, k_new, v_new, pool, layer, lut, write_index, attend_len, scale):
    """float64 restatement: store k_new[b] / v_new[b] at row write_index[b] of ``layer`` in
    ``pool [pages, 2, layers, 128, heads, dim]`` (row r of request b: row r % 128 of page
    lut[b, r // 128]), then out[b] = softmax(q[b] . k^T * scale) v over rows [0, attend_len[b]).
    Returns (out fp64 [B, heads, dim], the pool after the store)."""
    pool = np.array(pool, copy=True)
    B = q.shape[0]
    for b in range(B):
        r = int(write_index[b])
        page, slot = int(lut[b, r // 128]), r % 128
        pool[page, 0, layer, slot] = k_new[b]
        pool[page, 1, layer, slot] = v_new[b]
    out = np.zeros(q.shape, np.float64)
    for b in range(B):
        rows = range(int(attend_len[b]))
        K = np.stack([pool[int(lut[b, r // 128]), 0, layer, r % 128] for r in rows]).astype(np.float64)
        V = np.stack([pool[int(lut[b, r // 128]), 1, layer, r % 128] for r in rows]).astype(np.float64)
        s = np.einsum("hd,rhd->hr", q[b].astype(np.float64), K) * scale
        p = np.exp(s - s.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        out[b] = np.einsum("hr,rhd->hd", p, V)
    return out, pool


def chunk_visible(p, rows, window, prefix):
    """Which of logical rows 0 .. rows - 1 the token at logical row ``p`` sees (bool [rows])."""
    r = np.arange(rows)
    seen = r <= p
    if window:
        seen &= (r > p - window) | (r < prefix)
    return seen


def paged_chunk_attention_ref(q, k_new, v_new, pool, layer, lut, row_offsets, start, scale, window=0, prefix=None,
                              out=None):
    """float64 restatement of the chunk attention: request b's new rows (row_offsets[b] .. row_offsets[b + 1])
    stored from logical row start[b] on, then each attended over the rows it sees, and those alone.
    All arrays fp32 or fp64. Returns (out fp64 [T, heads, dim], the magnitudes that its error scales
    with: sum of p |v| [T, heads, dim] and max over the visible rows of scale * sum |q k| [T, heads], the
    pool after the store). Rows in no request keep ``out``'s."""
    pool = np.array(pool, copy=True)
    T, heads, dim = q.shape
    kv_heads = k_new.shape[1]
    got = np.zeros(q.shape, np.float64) if out is None else np.array(out, np.float64)
    mag, smag = np.zeros(q.shape), np.zeros((T, heads))
    for b in range(len(start)):
        lo, hi, s0 = int(row_offsets[b]), int(row_offsets[b + 1]), int(start[b])
        if hi <= lo:
            continue
        n = s0 + hi - lo
        place = lambda r: (int(lut[b, r // 128]), r % 128)  # noqa: E731
        for i in range(hi - lo):
            page, slot = place(s0 + i)
            pool[page, 0, layer, slot] = k_new[lo + i]
            pool[page, 1, layer, slot] = v_new[lo + i]
        K = np.stack([pool[place(r)[0], 0, layer, place(r)[1]] for r in range(n)]).astype(np.float64)
        V = np.stack([pool[place(r)[0], 1, layer, place(r)[1]] for r in range(n)]).astype(np.float64)
        for i in range(hi - lo):
            seen = chunk_visible(s0 + i, n, window, 0 if prefix is None else int(prefix[b]))
            for h in range(heads):
                hk = h // (heads // kv_heads)
                x, kk, vv = q[lo + i, h].astype(np.float64), K[seen, hk], V[seen, hk]
                s = kk @ x * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                got[lo + i, h] = p @ vv
                mag[lo + i, h] = p @ np.abs(vv)
                smag[lo + i, h] = (np.abs(kk) @ np.abs(x)).max() * abs(scale)
    return got, mag, smag, pool
