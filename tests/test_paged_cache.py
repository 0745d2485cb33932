"""The paged 8-bit KV cache: append, attention, copy, compact (include/infiniop.h).

There is no reference operator; the oracle is the definition evaluated in 64 bits on the CPU.  Codes, scales, tables
and maps must be equal bit for bit; attention is held to a bound derived from its roundings (see `attend_bound`).
"""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest
import torch

from operators_b200 import InfiniopError, ops
from operators_b200.utils import stream_handle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
CODE = torch.float8_e4m3fn
gpu = pytest.mark.gpu


# ---- the cache on the host ------------------------------------------------------------------------------------------

def make_cache(pages, heads, page, dh, seed, layout="head", spare=0, pow2=True, spread=2.0):
    """Random codes and scales (CPU).  layout: storage order of the pool; spare: unused elements behind each row."""
    g = torch.Generator().manual_seed(seed)
    pools = []
    for _ in range(2):
        x = (torch.randn(pages, heads, page, dh, generator=g) * 100).clamp(-448, 448).to(CODE)
        e = torch.randn(pages, heads, generator=g) * spread - 7
        pools.append((strided(x, layout, spare), torch.exp2(e.round() if pow2 else e)))
    (k, ks), (v, vs) = pools
    return k, v, ks, vs


def strided(x, layout, spare):
    """x [N, H, P, D] in storage of the given order with `spare` elements behind each row; the gaps hold NaN codes."""
    order = {"head": (0, 1, 2), "token": (0, 2, 1), "head_first": (1, 0, 2)}[layout]
    shape = [x.shape[i] for i in order]
    store = torch.full((*shape, x.shape[3] + spare), 0x7F, dtype=torch.uint8)
    view = store[..., :x.shape[3]].permute(*[order.index(i) for i in range(3)], 3)
    view.copy_(x.view(torch.uint8))
    return view.view(CODE)


def to_dev(x):
    """The same strides on the GPU (the storage is copied whole)."""
    if x is None:
        return None
    raw = x.view(torch.uint8) if x.dtype == CODE else x
    extent = sum((n - 1) * s for n, s in zip(raw.shape, raw.stride())) + 1 if raw.numel() else 0
    flat = torch.as_strided(raw, (extent,), (1,), raw.storage_offset()).to(DEV)
    y = torch.as_strided(flat, raw.shape, raw.stride())
    return y.view(CODE) if x.dtype == CODE else y


def make_tables(lens, page, num_pages, seed, cols=None):
    """Scattered pages; entries behind a sequence's last page point nowhere."""
    rng = np.random.default_rng(seed)
    ids = rng.permutation(num_pages)
    used = [-(-max(n, 0) // page) for n in lens]
    cols = max(used + [1]) if cols is None else cols
    table, at = torch.full((len(lens), cols), -7, dtype=torch.int32), 0
    for b, n in enumerate(used):
        table[b, :n] = torch.from_numpy(ids[at:at + n].astype(np.int32))
        at += n
    return table


def sequences(counts, lens, rows):
    """(batch index, first row, new tokens, length) as the operators read lengths and offsets."""
    if counts is None:
        return [(b, b, 1, max(n, 0)) for b, n in enumerate(lens)]
    offs = [min(max(o, 0), rows) for o in counts]
    return [(b, offs[b], max(offs[b + 1] - offs[b], 0), max(n, 0)) for b, n in enumerate(lens)]


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def e4m3(x):
    """Nearest e4m3 value (ties to even), saturating; NaN stays NaN.  x: float64 array."""
    a = np.abs(x)
    with np.errstate(all="ignore"):
        step = np.exp2(np.maximum(np.floor(np.log2(np.where((a > 0) & np.isfinite(a), a, 1.0))), -6) - 3)
        return np.where(np.isnan(x), np.nan, np.sign(x) * np.minimum(np.where(np.isfinite(a), np.rint(a / step) * step, 448.0), 448.0))


def append_ref(k, v, kp, vp, ks, vs, table, lens, offs):
    """Codes as float64 values and scales after the append."""
    out, (N, H, P, D) = [], kp.shape
    for x, pool, scale in ((k, kp, ks), (v, vp, vs)):
        x, codes, scale = x.double().numpy(), pool.float().double().numpy().copy(), scale.double().numpy().copy()
        for b, first, n, length in sequences(offs, lens, x.shape[0]):
            lo, hi = max(length - n, 0), min(length, table.shape[1] * P)
            for col in range(lo // P, -(-hi // P) if hi > lo else lo // P):
                page = int(table[b, col])
                if not 0 <= page < N:
                    continue
                p0, p1 = max(lo, col * P), min(hi, col * P + P)
                rows = x[first + p0 - (length - n):first + p1 - (length - n)]
                for h in range(H):
                    new = rows[:, h]
                    a = np.abs(new[np.isfinite(new)]).max(initial=0.0)
                    e = -40 if a == 0 else max(-40, math.ceil(math.log2(a / 448.0)))
                    s, kept = 2.0 ** e, p0 - col * P
                    if kept:
                        s = max(s, scale[page, h])
                        codes[page, h, :kept] = e4m3(codes[page, h, :kept] * (scale[page, h] / s))
                    codes[page, h, kept:kept + p1 - p0] = e4m3(new / s)
                    scale[page, h] = s
        out.append((codes, scale))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def attend_ref(q, kp, vp, ks, vs, table, lens, offs, scale, out):
    """(out, bound): the definition, and for every element how far the operator may be off (see attend_bound)."""
    (N, H, P, D), (T, HQ, _) = kp.shape, q.shape
    G, want, tol = HQ // H, out.double().numpy().copy(), np.zeros((T, HQ, D))
    kf, vf = kp.float().double().numpy(), vp.float().double().numpy()
    ksd, vsd, qd = ks.double().numpy(), vs.double().numpy(), q.double().numpy()
    for b, first, n, length in sequences(offs, lens, T):
        keys = min(length, table.shape[1] * P)
        cols = -(-keys // P)
        ids = table[b, :cols].numpy()
        ok = (ids >= 0) & (ids < N)
        safe = np.where(ok, ids, 0)
        seen = np.repeat(ok, P)[:keys]
        pos = length - n + np.arange(n)
        vis = (np.arange(keys)[None] <= pos[:, None]) & seen[None]                     # [n, keys]
        for h in range(H if n else 0):
            K = (kf[safe, h] * ksd[safe, h][:, None, None]).reshape(-1, D)[:keys]
            V = (vf[safe, h] * vsd[safe, h][:, None, None]).reshape(-1, D)[:keys]
            any_vis = vis.any(0)
            K, V = np.where(any_vis[:, None], K, 0.0), np.where(any_vis[:, None], V, 0.0)
            for j in range(h * G, h * G + G):
                x = qd[first:first + n, j]
                s = np.where(vis, scale * (x @ K.T), -np.inf)
                m = s.max(1, initial=-np.inf, keepdims=True)
                p = np.exp(s - np.where(np.isinf(m), 0.0, m))
                total = p.sum(1, keepdims=True)
                p = p / np.where(total == 0, 1.0, total)
                y = p @ V
                want[first:first + n, j] = y
                mag = abs(scale) * (np.abs(x) @ np.abs(K).T).max(1, initial=0.0)
                tol[first:first + n, j] = attend_bound(y, p @ np.abs(V), np.abs(V).max(initial=0.0), mag[:, None], D, keys, q.dtype)
    return want, tol


def attend_bound(y, mean_abs, v_max, mag, dh, keys, dtype):
    """y = sum_j w_j v_j / sum_j w_j, and the operator's weights carry
      2^-11       their rounding to fp16 before the product with v (half a step of fp16),
      2^-20       2^x by the special-function unit (2 ulp of fp32 and the rounding of its argument's fraction) and the
                  fp32 multiplications around it,
      e           the score's error: each of the dh products and sums of q . k in fp32 is off by at most 2^-23 of the
                  magnitudes summed (2^-24 rounded, 2^-23 truncated), and the scaling by scale * log2(e) and the
                  subtraction of the maximum by a few 2^-23 of the score: (dh + 8) * 2^-23 * max_j |scale| sum|q k|,
    each relative; numerator and denominator count once each: mean |v| times twice their sum.  Sums over the keys are in
    fp32, in parts of at most 2^15 terms that grow by 2^-23 of the running sum: 2 * (2^-8) would be the worst case, but the
    products of a step of 16 keys are summed before they join, so keys / 16 * 2^-23 counts.  Weights are stored times
    2^2 at least relative to a reference that is one row's weight (so at most the largest); below fp16's normal range,
    2^-14, a rounding is off by half a step of 2^-24, that is by 2^-25 / 2^2 = 2^-27 of the reference, and a key's codes
    reach 448 where its page's largest value is at least half of that: keys * 2^-26 * max |v| in all.  One rounding of
    the result at the end."""
    half = torch.finfo(dtype).eps / 2
    e = (dh + 8) * 2.0 ** -23 * mag
    weight = 2.0 ** -11 + 2.0 ** -20 + 2.0 * e + (keys / 16 + 16) * 2.0 ** -23
    return half * np.abs(y) + 2 * weight * mean_abs + keys * 2.0 ** -26 * v_max + float(torch.finfo(dtype).tiny) * half


def close(got, want, tol):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    over = np.abs(got - want) - tol
    assert (over <= 0).all(), "off by %g more than the bound %g at %s" % (
        over.max(), tol[np.unravel_index(over.argmax(), over.shape)], np.unravel_index(over.argmax(), over.shape))


def same_codes(got, want):
    got = got.cpu().float().double().numpy()
    bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), "%d codes differ, first at %s: %r for %r" % (
        bad.sum(), np.argwhere(bad)[0], got[bad][0], want[bad][0])


# ---- host logic (no GPU) ------------------------------------------------------------------------------------------

def test_index_arithmetic(tmp_path):
    """seq_of, written, pages_touched, pages_bound and the scale's exponent, compiled for the host: exhaustive over
    small lengths, and every fp16 and bf16 magnitude."""
    src = tmp_path / "t.cc"
    src.write_text(r'''
#include "paged_index.h"
#include <cstdio>
#include <cstring>
#include <cmath>
#include <climits>
using namespace b200::paged;
static int fails = 0;
#define CHECK(c) do { if (!(c)) { if (fails++ < 5) printf("FAIL line %d\n", __LINE__); } } while (0)
int main() {
    // every value of the offsets is clamped into the rows
    const int32_t lens[] = {5, -3, INT_MIN, INT_MAX}, offs[] = {-9, 3, 2, INT_MAX, 7};
    for (int b = 0; b < 4; ++b) {
        Seq s = seq_of(lens, offs, 6, b);
        CHECK(s.n >= 0 && s.first >= 0 && s.first + s.n <= 6 && s.len >= 0);
    }
    Seq a = seq_of(lens, offs, 6, 0), c = seq_of(lens, offs, 6, 1), d = seq_of(lens, offs, 6, 2);
    CHECK(a.first == 0 && a.n == 3 && a.len == 5);
    CHECK(c.n == 0 && c.len == 0);
    CHECK(d.first == 2 && d.n == 4 && d.len == 0);
    Seq one = seq_of(lens, nullptr, 4, 3);
    CHECK(one.first == 3 && one.n == 1 && one.len == INT_MAX);
    int32_t lo, hi;
    written(one, 640, lo, hi);
    CHECK(hi <= lo);// beyond the table: nothing is written
    for (int len = 0; len < 40; ++len) for (int n = 0; n < 40; ++n) for (int page = 1; page < 12; ++page) for (int cols = 0; cols < 9; ++cols) {
        Seq s{0, n, len};
        written(s, cols * page, lo, hi);
        int touched = 0, last = -1, count = 0;
        for (int i = 0; i < n; ++i) {
            const int pos = len - n + i;
            if (pos < 0 || pos >= cols * page) continue;
            CHECK(pos >= lo && pos < hi);
            ++count;
            if (pos / page != last) ++touched, last = pos / page;
        }
        CHECK(count == (hi > lo ? hi - lo : 0));
        CHECK(pages_touched(lo, hi, [&](int x) { return x / page; }) == touched);
        CHECK(touched <= pages_bound(n, 1, page));
    }
    // 2^x is the smallest power with amax <= 448 * 2^x
    for (int kind = 0; kind < 2; ++kind) for (uint32_t h = 1; h < (kind ? 0x7F80u : 0x7C00u); ++h) {
        float f;
        if (kind) { uint32_t u = h << 16; memcpy(&f, &u, 4); }
        else { const int e = h >> 10, m = h & 1023; f = e ? ldexpf(1024 + m, e - 25) : ldexpf(m, -24); }
        uint32_t u; memcpy(&u, &f, 4);
        const int x = scale_exponent(u);
        CHECK(x >= kMinExp && x <= 120);
        CHECK((double) f <= 448.0 * ldexp(1.0, x));
        if (x > kMinExp) CHECK((double) f > 448.0 * ldexp(1.0, x - 1));
        uint32_t b = pow2_bits(x); float g; memcpy(&g, &b, 4);
        CHECK(g == ldexpf(1.0f, x));
    }
    CHECK(scale_exponent(0) == kMinExp);
    return fails != 0;
}
''')
    exe = tmp_path / "t"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "operators_b200", "csrc"), str(src), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_e4m3_of_the_oracle_is_torch_s():
    codes = torch.arange(256, dtype=torch.uint8).view(CODE).double().numpy()
    fin = codes[np.isfinite(codes)]
    assert (e4m3(fin) == fin).all()
    x = torch.randn(20000, dtype=torch.float64).numpy() * np.exp2(np.random.default_rng(0).uniform(-12, 8, 20000))
    mid = (np.sort(fin)[1:] + np.sort(fin)[:-1]) / 2
    for y in (x, mid):
        assert (e4m3(y) == torch.from_numpy(y).clamp(-448, 448).to(CODE).double().numpy()).all()


@pytest.fixture(scope="module")
def host():
    """(lib, handle) without a GPU: creating these descriptors and refusing calls touches no device."""
    from operators_b200 import build, open_lib
    from operators_b200.liboperators import infiniopHandle_t

    class FakeHandle(ctypes.Structure):
        _fields_ = [("device", ctypes.c_int), ("device_id", ctypes.c_int), ("sm_count", ctypes.c_int), ("smem", ctypes.c_int)]

    build.build()
    lib = open_lib(os.path.join(ROOT, "operators_b200", "lib"))
    ops._declare(lib)
    fake = FakeHandle(1, 0, 148, 232448)
    host.keep = fake
    return lib, ctypes.cast(ctypes.pointer(fake), infiniopHandle_t)


def _small(dtype=torch.float16, rows=3, heads=2, q_heads=4, dh=64, pages=6, page=16, batch=3, cols=2):
    t = {n: torch.zeros(rows, heads, dh, dtype=dtype) for n in ("k", "v")}
    t.update({n: torch.zeros(rows, q_heads, dh, dtype=dtype) for n in ("q", "out")})
    t.update({n: torch.zeros(pages, heads, page, dh, dtype=torch.uint8).view(CODE) for n in ("k_pages", "v_pages")})
    t.update({n: torch.ones(pages, heads) for n in ("k_scales", "v_scales")})
    t["block_table"] = torch.zeros(batch, cols, dtype=torch.int32)
    t["new_table"] = torch.zeros(batch, cols, dtype=torch.int32)
    t["seq_lens"] = torch.zeros(batch, dtype=torch.int32)
    t["q_offsets"] = torch.zeros(batch + 1, dtype=torch.int32)
    t["pairs"] = torch.zeros(5, 2, dtype=torch.int32)
    t["page_map"] = torch.zeros(pages, dtype=torch.int32)
    t["live"] = torch.zeros(1, dtype=torch.int32)
    return t


CACHE = ["k_pages", "v_pages", "k_scales", "v_scales"]
OPS = {
    "append": (ops.PagedCacheAppendOp, ["k", "v"] + CACHE + ["block_table", "seq_lens", "q_offsets"]),
    "attend": (ops.PagedAttentionOp, ["out", "q"] + CACHE + ["block_table", "seq_lens", "q_offsets"]),
    "copy": (ops.PagedCacheCopyOp, CACHE + ["pairs"]),
    "compact": (ops.PagedCacheCompactOp, CACHE + ["new_table", "block_table", "seq_lens", "page_map", "live"]),
}
PARAM, DTYPE, SHAPE, STRIDES, NO_MEMORY, DEVICE = 2, 3, 4, 5, 6, 8
REFUSALS = [
    ("*", "k_pages", lambda x: x[0], SHAPE), ("*", "v_pages", lambda x: x[:, :1], SHAPE),
    ("*", "k_scales", lambda x: x[:4], SHAPE), ("*", "v_scales", lambda x: x[0], SHAPE),
    ("*", "k_pages", lambda x: x.view(torch.uint8), DTYPE), ("*", "v_pages", lambda x: x.view(torch.int8), DTYPE),
    ("*", "k_scales", lambda x: x.half(), DTYPE), ("*", "k_pages", lambda x: x.transpose(2, 3).contiguous().transpose(2, 3), STRIDES),
    ("*", "v_pages", lambda x: x[:1].expand(6, 2, 16, 64), STRIDES),
    ("*", "k_pages", lambda x: torch.as_strided(x, (6, 2, 16, 64), (2048, 32, 64, 1)), STRIDES),
    ("*", "v_scales", lambda x: x[:1].expand(6, 2), STRIDES),
    ("append attend compact", "block_table", lambda x: x[:2], SHAPE), ("append attend compact", "block_table", lambda x: x.long(), DTYPE),
    ("append attend compact", "block_table", lambda x: x.t().contiguous().t(), STRIDES),
    ("append attend compact", "seq_lens", lambda x: x.float(), DTYPE), ("append attend compact", "seq_lens", lambda x: x[:, None], SHAPE),
    ("append attend compact", "seq_lens", lambda x: torch.zeros(6, dtype=torch.int32)[::2], STRIDES),
    ("append attend", "q_offsets", lambda x: x[:3], SHAPE), ("append attend", "q_offsets", lambda x: x.long(), DTYPE),
    ("append", "k", lambda x: x[:, :1], SHAPE), ("append", "v", lambda x: x[:2], SHAPE), ("append", "k", lambda x: x.float(), DTYPE),
    ("append", "v", lambda x: x.bfloat16(), DTYPE), ("append", "k", lambda x: x.transpose(1, 2).contiguous().transpose(1, 2), STRIDES),
    ("append", "k", lambda x: x[:, :, :32], SHAPE),
    ("attend", "q", lambda x: x[:, :3], SHAPE), ("attend", "out", lambda x: x[:, :2], SHAPE), ("attend", "q", lambda x: x.float(), DTYPE),
    ("attend", "out", lambda x: x.bfloat16(), DTYPE), ("attend", "out", lambda x: x[:1].expand(3, 4, 64), STRIDES),
    ("attend", "q", lambda x: x.transpose(1, 2).contiguous().transpose(1, 2), STRIDES),
    ("copy", "pairs", lambda x: x[:, :1], SHAPE), ("copy", "pairs", lambda x: x[0], SHAPE), ("copy", "pairs", lambda x: x.long(), DTYPE),
    ("copy", "pairs", lambda x: torch.zeros(2, 5, dtype=torch.int32).t(), STRIDES),
    ("compact", "new_table", lambda x: x[:2], SHAPE), ("compact", "page_map", lambda x: x[:4], SHAPE),
    ("compact", "live", lambda x: torch.zeros(2, dtype=torch.int32), SHAPE), ("compact", "page_map", lambda x: x.long(), DTYPE),
    ("compact", "new_table", lambda x: x[:1].expand(3, 2), STRIDES),
    ("compact", "page_map", lambda x: torch.zeros(12, dtype=torch.int32)[::2], STRIDES),
]


@pytest.mark.parametrize("case", range(len(REFUSALS)))
def test_refused_descriptors(host, case):
    names, field, change, status = REFUSALS[case]
    for name, (op, fields) in OPS.items():
        if names != "*" and name not in names.split():
            continue
        t = _small()
        t[field] = change(t[field])
        with pytest.raises(InfiniopError) as e:
            op(*host, *[t[f] for f in fields])
        assert e.value.status == status, (name, field)


def test_refused_sizes_and_calls(host):
    lib, handle = host
    # head sizes beyond 256, tables whose tokens pass 31 bits, one-token form with another number of rows
    for name in OPS:
        t = _small(dh=257, page=1)
        with pytest.raises(InfiniopError) as e:
            OPS[name][0](lib, handle, *[t[f] for f in OPS[name][1]])
        assert e.value.status == SHAPE
    for name in ("append", "attend", "compact"):
        t = _small(page=1 << 12, pages=1, dh=1)
        t["block_table"] = t["new_table"] = torch.zeros(3, 1 << 19, dtype=torch.int32)
        with pytest.raises(InfiniopError) as e:
            OPS[name][0](lib, handle, *[t[f] for f in OPS[name][1]])
        assert e.value.status == SHAPE
    for name in ("append", "attend"):
        t = _small(rows=4)
        t["q_offsets"] = None
        with pytest.raises(InfiniopError) as e:
            OPS[name][0](lib, handle, *[t[f] for f in OPS[name][1]])
        assert e.value.status == SHAPE
    t = _small()
    for bad in (math.inf, math.nan):
        with pytest.raises(InfiniopError) as e:
            ops.PagedAttentionOp(lib, handle, *[t[f] for f in OPS["attend"][1]], bad)
        assert e.value.status == PARAM
    # null descriptors and handles
    D, desc = ctypes.c_void_p, ctypes.c_void_p()
    for name, n, extra in (("PagedCacheAppend", 9, []), ("PagedAttention", 9, [1.0]), ("PagedCacheCopy", 5, []), ("PagedCacheCompact", 9, [])):
        create = getattr(lib, "infiniopCreate%sDescriptor" % name)
        assert create(None, ctypes.byref(desc), *([None] * n), *extra) == DEVICE
        assert create(handle, None, *([None] * n), *extra) == NO_MEMORY
        assert create(handle, ctypes.byref(desc), *([None] * n), *extra) == PARAM
        size = ctypes.c_uint64()
        assert getattr(lib, "infiniopGet%sWorkspaceSize" % name)(None, ctypes.byref(size)) == DEVICE
        assert getattr(lib, "infiniopDestroy%sDescriptor" % name)(None) == DEVICE
    # more pairs of a new token and a q head than 31 bits hold, in descriptors alone
    t = _small(dh=1, heads=1, pages=1, page=1)
    t["q"] = t["out"] = torch.empty(1 << 16, 1 << 15, 1, dtype=torch.float16, device="meta")
    with pytest.raises(InfiniopError) as e:
        ops.PagedAttentionOp(lib, handle, *[t[f] for f in OPS["attend"][1]])
    assert e.value.status == SHAPE
    # null pointers, offsets that the descriptor does not know, a short workspace
    t = _small()
    t["long_table"] = torch.zeros(3, 100000, dtype=torch.int32)
    for name, (op, fields) in [*OPS.items(), ("attend", (ops.PagedAttentionOp, [f.replace("block", "long") for f in OPS["attend"][1]]))]:
        with op(lib, handle, *[t[f] for f in fields]) as o:
            assert o.workspace is not None or name != "attend" or "long_table" not in fields
            if o.workspace is not None:
                o.workspace_size -= 1
                with pytest.raises(InfiniopError) as e:
                    o(*[t[f] for f in fields])
                assert e.value.status == NO_MEMORY
                o.workspace_size += 1
            for i, f in enumerate(fields):
                class Null:
                    def data_ptr(self):
                        return None
                with pytest.raises(InfiniopError) as e:
                    o(*[Null() if f == g else t[g] for g in fields])
                assert e.value.status == PARAM, (name, f)
    for name in ("append", "attend"):
        op, fields = OPS[name]
        with op(lib, handle, *[None if f == "q_offsets" else t[f] for f in fields]) as o:
            with pytest.raises(InfiniopError) as e:
                o(*[t[f] for f in fields])
            assert e.value.status == PARAM


def test_misaligned_pointers_are_refused(host):
    """Pointers off their element's size, and a workspace off 16 bytes, which parts are stored to in whole vectors."""
    lib, handle = host
    t = _small()
    t["long_table"] = torch.zeros(3, 100000, dtype=torch.int32)
    long_attend = (ops.PagedAttentionOp, [f.replace("block", "long") for f in OPS["attend"][1]])

    class Off:
        def __init__(self, tensor, by):
            self.tensor, self.by = tensor, by

        def data_ptr(self):
            return self.tensor.data_ptr() + self.by

    for name, (op, fields) in [*OPS.items(), ("attend", long_attend)]:
        with op(lib, handle, *[t[f] for f in fields]) as o:
            for f in fields:
                for by in range(1, t[f].element_size()):
                    with pytest.raises(InfiniopError) as e:
                        o(*[Off(t[g], by) if f == g else t[g] for g in fields])
                    assert e.value.status == PARAM, (name, f, by)
            if o.workspace is not None:
                whole = torch.empty(o.workspace_size + 32, dtype=torch.uint8)
                start = -whole.data_ptr() % 16
                for by in (1, 4, 8):
                    o.workspace = whole[start + by:]
                    with pytest.raises(InfiniopError) as e:
                        o(*[t[f] for f in fields])
                    assert e.value.status == PARAM, (name, by)
    assert name == "attend" and o.workspace is not None


def test_workspace_does_not_depend_on_what_it_holds(host):
    """Nothing is cleared ahead of a call: the wrapper hands out memory as it comes."""
    lib, handle = host
    t = _small()
    with ops.PagedCacheCompactOp(lib, handle, *[t[f] for f in OPS["compact"][1]]) as o:
        assert o.workspace.numel() == o.workspace_size > 0


def test_stream_arguments():
    class Stream:
        cuda_stream = 7

    for stream, handle in ((None, 0), (0, 0), (5, 5), (ctypes.c_void_p(5), 5), (ctypes.c_void_p(None), 0), (Stream(), 7)):
        assert stream_handle(stream) == handle


# ---- append ---------------------------------------------------------------------------------------------------------

def run_append(cuda_lib, k, v, cache, table, lens, offs, stream=None):
    lib, handle = cuda_lib
    d = [to_dev(x) for x in (k, v, *cache, table, lens, offs)]
    torch.cuda.synchronize()
    ops.paged_cache_append(lib, handle, *d, stream=stream)
    torch.cuda.synchronize()
    return d[2:6]


def check_append(cuda_lib, k, v, cache, table, lens, offs):
    got = run_append(cuda_lib, k, v, cache, table, lens, offs)
    want = append_ref(k, v, *cache, table, lens.tolist(), None if offs is None else offs.tolist())
    for g, w in zip(got[:2], want[:2]):
        same_codes(g, w)
    for g, w in zip(got[2:], want[2:]):
        assert (g.cpu().double().numpy() == w).all()
    return got


def new_rows(T, H, D, dtype, seed, spare=0, wide=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D + spare, generator=g) * torch.exp2(wide * torch.randn(T, 1, 1, generator=g))
    return x.to(dtype)[..., :D]


APPEND_CASES = [
    # heads, page, dh, lens, new tokens (None: one each), layout, spare
    (2, 16, 64, [1, 16, 17, 40], None, "head", 0),
    (8, 64, 128, [64, 65, 1000, 63, 128], None, "token", 0),
    (1, 64, 128, [200], [200], "head", 0),
    (3, 20, 80, [5, 20, 21, 100, 0, 333], [5, 20, 20, 7, 0, 333], "token", 16),
    (2, 7, 33, [30, 8, 7], [30, 1, 3], "head", 0),            # codes and elements one at a time
    (2, 256, 256, [700, 256], [700, 3], "head_first", 0),     # blocks beyond what the threads hold
    (4, 1, 96, [9, 4], [9, 2], "head", 0),
    (1, 128, 8, [1000], [600], "head", 8),
    (2, 32, 1, [70], [33], "token", 0),
    (2, 64, 100, [70, 64], [33, 64], "head", 4),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,page,dh,lens,news,layout,spare", APPEND_CASES)
def test_append(cuda_lib, heads, page, dh, lens, news, layout, spare, dtype):
    need = sum(-(-n // page) for n in lens)
    cache = make_cache(need + 3, heads, page, dh, 1, layout, spare)
    table = make_tables(lens, page, need + 3, 2)
    offs = None if news is None else torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32)
    T = len(lens) if news is None else sum(news)
    k, v = (new_rows(T, heads, dh, dtype, s, spare, 3.0) for s in (3, 4))
    check_append(cuda_lib, k, v, cache, table, torch.tensor(lens, dtype=torch.int32), offs)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_special_values(cuda_lib, dtype):
    """Infinities saturate, NaN stays, zeros and tiny rows take the smallest scale, the largest magnitudes their own."""
    H, P, D = 2, 16, 64
    big = float(torch.finfo(dtype).max)
    k = new_rows(16 * 8, H, D, dtype, 5).clone()
    k[3, 0, 5], k[4, 1, 6], k[5, 0, 7] = math.inf, -math.inf, math.nan
    k[16:32] = 0
    k[32:48] = k[32:48] * torch.finfo(dtype).tiny
    k[48:64, 0] = big
    k[64:80] = math.nan
    k[80:96] = math.inf
    k[96:112] = -0.0
    k[112, 0, 0] = 448.0          # the largest code exactly, and the next value above it
    k[112, 1, 0] = 450.0 if dtype == torch.bfloat16 else 448.25
    cache = make_cache(9, H, P, D, 6)
    table = torch.arange(8, dtype=torch.int32)[None].contiguous()
    check_append(cuda_lib, k, -k, cache, table, torch.tensor([128], dtype=torch.int32), torch.tensor([0, 128], dtype=torch.int32))


@gpu
def test_append_token_by_token_keeps_earlier_rows(cuda_lib):
    """A page filled one token at a time, magnitudes growing: kept codes follow the scale; the last state equals the
    oracle's step by step, and the same call again changes nothing."""
    H, P, D = 2, 16, 128
    cache = make_cache(4, H, P, D, 7)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    k = new_rows(20, H, D, torch.float16, 8) * torch.exp2(torch.linspace(-8, 8, 20))[:, None, None]
    k = k.half()
    for n in range(1, 21):
        lens = torch.tensor([n], dtype=torch.int32)
        got = check_append(cuda_lib, k[n - 1:n], k[n - 1:n].neg(), cache, table, lens, None)
        cache = [x.cpu() for x in got]
        again = run_append(cuda_lib, k[n - 1:n], k[n - 1:n].neg(), cache, table, lens, None)
        for a, b in zip(again, got):
            assert torch.equal(a.view(torch.uint8) if a.dtype == CODE else a, b.view(torch.uint8) if b.dtype == CODE else b)


@gpu
def test_append_scale_that_is_no_power_of_two(cuda_lib):
    """A cache filled elsewhere may carry any positive scale: kept if large enough."""
    cache = make_cache(3, 2, 16, 64, 9, pow2=False)
    cache[2][1, 0] = 3.7
    k = new_rows(4, 2, 64, torch.bfloat16, 10)
    check_append(cuda_lib, k, k * 2, cache, torch.tensor([[1, 2]], dtype=torch.int32), torch.tensor([14], dtype=torch.int32),
                 torch.tensor([0, 4], dtype=torch.int32))


@gpu
def test_append_values_that_lead_nowhere(cuda_lib):
    """Page ids outside the pool, offsets outside the rows, lengths below the new tokens, beyond the table and
    negative: those tokens are dropped, everything else is written, nothing else is touched."""
    H, P, D = 2, 16, 64
    cache = make_cache(20, H, P, D, 11)
    lens = [40, 3, 100, -5, 0, 33]
    table = make_tables([40, 16, 64, 16, 16, 33], P, 20, 12, cols=4)
    table[0, 1], table[5, 2] = 20, -2147483648
    offs = torch.tensor([0, 40, 50, 70, 75, 80, 2147483647], dtype=torch.int32)
    k, v = new_rows(113, H, D, torch.float16, 13), new_rows(113, H, D, torch.float16, 14)
    check_append(cuda_lib, k, v, cache, table, torch.tensor(lens, dtype=torch.int32), offs)
    offs = torch.tensor([-7, 40, 30, 70, 200, 80, 90], dtype=torch.int32)
    check_append(cuda_lib, k, v, cache, table, torch.tensor(lens, dtype=torch.int32), offs)


@gpu
def test_append_many_sequences(cuda_lib):
    """More sequences than a block has threads, most without a new token."""
    rng = np.random.default_rng(15)
    lens = rng.integers(0, 50, 700).tolist()
    news = [int(min(n, rng.integers(0, 4) * rng.integers(0, 2))) for n in lens]
    table = make_tables(lens, 16, 2900, 16)
    cache = make_cache(2900, 1, 16, 16, 17)
    offs = torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32)
    k = new_rows(sum(news) + 5, 1, 16, torch.bfloat16, 18)
    check_append(cuda_lib, k, k.neg(), cache, table, torch.tensor(lens, dtype=torch.int32), offs)


# ---- attention ------------------------------------------------------------------------------------------------------

def run_attend(cuda_lib, q, cache, table, lens, offs, scale, out, stream=None):
    lib, handle = cuda_lib
    d = [to_dev(x) for x in (out, q, *cache, table, lens, offs)]
    torch.cuda.synchronize()
    ops.paged_attention(lib, handle, *d, scale=scale, stream=stream)
    torch.cuda.synchronize()
    return d[0]


def wide(table, page):
    """The same sequences in a table with room for 2^20 tokens each: the operator's kernels are chosen by how long a
    sequence may become, so this is how short ones reach those for long ones."""
    room = torch.full((table.shape[0], max(2 ** 20 // page, table.shape[1])), -7, dtype=torch.int32)
    room[:, :table.shape[1]] = table
    return room


def check_attend(cuda_lib, q, cache, table, lens, offs, scale=None, out=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = torch.full_like(q, 3.0) if out is None else out
    lens_t = torch.tensor(lens, dtype=torch.int32)
    offs_t = None if offs is None else torch.tensor(offs, dtype=torch.int32)
    page = cache[0].shape[2]
    for room in (table, wide(table, page)):
        if room is table or max(lens) > table.shape[1] * page:
            want, tol = attend_ref(q, *cache, room, lens, offs, scale, out)
        close(run_attend(cuda_lib, q, cache, room, lens_t, offs_t, scale, out), want, tol)


def poison(cache, table, lens, page):
    """NaN codes behind every sequence's last token (pages belong to one sequence)."""
    k, v = cache[0], cache[1]
    for b, n in enumerate(lens):
        if n > 0 and n % page and n <= table.shape[1] * page:
            for x in (k, v):
                x.view(torch.uint8)[int(table[b, n // page]), :, n % page:] = 0x7F if b % 2 else 0xFF


ATTEND_CASES = [
    # q heads, kv heads, page, dh, lens, new tokens (None: one each), layout, spare
    (1, 1, 16, 64, [1], None, "head", 0),
    (8, 2, 16, 64, [777], None, "token", 0),
    (32, 8, 64, 128, [1, 63, 64, 65, 0, 1000, 2500], None, "head", 0),
    (40, 8, 32, 96, [5, 300, 777], [5, 3, 1], "token", 0),
    (6, 2, 7, 80, [30, 8, 700], None, "head", 16),
    (24, 2, 20, 112, [100, 333], [2, 0], "token", 0),
    (96, 8, 128, 128, [130, 999], None, "head", 0),
    (64, 4, 64, 128, [515], [9], "head_first", 0),
    (4, 4, 1, 64, [37], None, "head", 0),
    (5, 1, 256, 256, [600, 256, 257], [2, 1, 4], "head", 0),
    (3, 3, 16, 33, [50, 17], [3, 17], "head", 0),             # codes one at a time
    (2, 2, 32, 8, [100], [4], "head", 0),
    (4, 2, 16, 1, [40], None, "head", 3),
    (8, 8, 24, 72, [400], [6], "token", 8),
    (4, 2, 64, 128, [33000], None, "head", 0),
    # prompts and chunks
    (8, 2, 64, 128, [300], [300], "head", 0),
    (8, 2, 64, 128, [129, 700, 40, 1], [129, 128, 40, 1], "token", 0),
    (4, 1, 16, 64, [1000], [200], "head", 0),
    (12, 1, 20, 96, [150, 60], [150, 31], "head", 0),
    (6, 2, 128, 80, [900], [333], "head", 0),
    (3, 1, 64, 256, [400, 100], [257, 100], "token", 0),
    (2, 2, 48, 40, [500], [130], "head", 8),
    (5, 1, 33, 17, [200], [90], "head", 0),
    (16, 1, 8, 128, [260], [77], "head", 0),
    (1, 1, 256, 112, [2100], [64], "head", 0),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_heads,kv_heads,page,dh,lens,news,layout,spare", ATTEND_CASES)
def test_attend(cuda_lib, q_heads, kv_heads, page, dh, lens, news, layout, spare, dtype):
    need = sum(-(-n // page) for n in lens)
    cache = make_cache(need + 2, kv_heads, page, dh, 21, layout, spare)
    table = make_tables(lens, page, need + 2, 22)
    poison(cache, table, lens, page)
    T = len(lens) if news is None else sum(news) + 2          # two rows behind the last sequence stay
    offs = None if news is None else [0] + [int(x) for x in np.cumsum(news)]
    q = new_rows(T, q_heads, dh, dtype, 23, spare)
    check_attend(cuda_lib, q, cache, table, lens, offs)


@gpu
@pytest.mark.parametrize("new", [1, 4, 150])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P", [16, 64, 20])
def test_attend_values_that_lead_nowhere(cuda_lib, P, dtype, new):
    """Missing pages are masked (a row that sees none of its keys gets zeros), offsets outside the rows are clamped,
    lengths may be below the new tokens (their first rows see nothing), beyond the table, zero or negative."""
    H, D, G = 2, 64, 3
    lens = [40, 3, 200, -5, 0, 33, 5]
    table = make_tables([40, 16, min(4 * P, 200), 16, 16, 33, 5], P, 20, 32, cols=4)
    if P > 16:
        table[2, 0], table[5, 1] = 20, -3                     # the first keys are missing
    table[0, 1], table[5, 2], table[6, 0] = 20, -2147483648, -1
    cache = make_cache(20, H, P, D, 31)
    if new == 1:
        offs, T = None, 7
    else:
        offs, T = [-4, new, 2 * new, 2 * new + 2, 3 * new, 3 * new + 1, 4 * new, 2147483647], 5 * new
    q = new_rows(T, H * G, D, dtype, 33)
    check_attend(cuda_lib, q, cache, table, lens, offs)


@gpu
@pytest.mark.parametrize("new", [1, 3, 140])
def test_attend_scales_far_apart(cuda_lib, new):
    """Pages whose scales differ by many powers of two, in keys and values, none a power of two: large keys decide
    alone, and a page with huge values and hardly any weight still counts for what it is worth."""
    H, P, D = 2, 16, 128
    cache = make_cache(20, H, P, D, 41, pow2=False, spread=1.0)
    cache[3][::3] *= 2.0 ** 18
    cache[3][1::3] *= 2.0 ** -20
    cache[2][::4] *= 2.0 ** 5
    table = make_tables([300], P, 20, 42)
    q = new_rows(new, 4, D, torch.bfloat16, 43)
    check_attend(cuda_lib, q, cache, table, [300], [0, new])


@gpu
@pytest.mark.parametrize("new", [1, 130])
@pytest.mark.parametrize("dtype,amp", [(torch.float16, 60000.0), (torch.bfloat16, 2.0 ** 100), (torch.bfloat16, 2.0 ** -100),
                                       (torch.float16, 2.0 ** -20)])
def test_attend_queries_at_the_ends_of_their_range(cuda_lib, dtype, amp, new):
    """q as large or as small as its type goes, brought back by the scale; elements of one row far apart."""
    H, P, D = 1, 64, 64
    cache = make_cache(6, H, P, D, 51)
    q = new_rows(new, 2, D, torch.float32, 53).clamp(-1, 1)
    q[:, 1, ::2] *= 2.0 ** -12
    q = (q * amp).to(dtype)
    check_attend(cuda_lib, q, cache, make_tables([330], P, 6, 52), [330], [0, new], scale=0.5 / amp if amp < 2.0 ** 90 else 0.5 * 2.0 ** -100)


@gpu
@pytest.mark.parametrize("new", [1, 200])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
def test_attend_scale_argument(cuda_lib, scale, new):
    """Any finite scale: negative, zero (plain averages), large (hardly more than one key counts)."""
    H, P, D = 2, 32, 64
    cache = make_cache(12, H, P, D, 61)
    cache[3].fill_(2.0 ** -7)
    q = new_rows(new, 4, D, torch.float16, 63)
    check_attend(cuda_lib, q, cache, make_tables([350], P, 12, 62), [350], [0, new], scale=scale)


@gpu
def test_attend_row_with_infinity_stays_alone(cuda_lib):
    """A q row that holds an infinity or NaN spoils its own outputs only."""
    H, P, D = 1, 32, 64
    cache = make_cache(12, H, P, D, 71)
    table = make_tables([350], P, 12, 72)
    for new, table in ((1, table), (1, wide(table, P)), (150, table), (150, wide(table, P))):
        q = new_rows(new, 4, D, torch.float16, 73)
        clean = run_attend(cuda_lib, q, cache, table, torch.tensor([350], dtype=torch.int32), torch.tensor([0, new], dtype=torch.int32), 0.125, torch.zeros_like(q))
        bad = q.clone()
        bad[0, 1, 3], bad[0, 2, 4] = math.inf, math.nan
        got = run_attend(cuda_lib, bad, cache, table, torch.tensor([350], dtype=torch.int32), torch.tensor([0, new], dtype=torch.int32), 0.125, torch.zeros_like(q))
        keep = torch.ones(new, 4, dtype=torch.bool)
        keep[0, 1:3] = False
        assert torch.equal(got.cpu()[keep], clean.cpu()[keep])


def attend_softmax(q, cache, table, lens, offs, scale):
    """softmax(scale q k^T) v of torch in 64 bits over the visible keys, NaN and infinities as they come; rows without a
    visible key are zeros."""
    (N, H, P, D), (T, HQ, _) = cache[0].shape, q.shape
    y, G = torch.zeros(T, HQ, D, dtype=torch.float64), HQ // H
    kf, vf = (cache[i].float().double() * cache[2 + i].double()[:, :, None, None] for i in range(2))
    for b, first, n, length in sequences(offs, lens, T):
        for i in range(n):
            keys = [(int(table[b, j // P]), j % P) for j in range(min(length - n + i + 1, table.shape[1] * P))]
            keys = [(p, s) for p, s in keys if 0 <= p < N]
            if keys:
                p, s = (torch.tensor(x) for x in zip(*keys))
                for h in range(HQ):
                    w = torch.softmax(scale * (kf[p, h // G, s] @ q[first + i, h].double()), 0)
                    y[first + i, h] = w @ vf[p, h // G, s]
    return y


@gpu
@pytest.mark.parametrize("new", [1, 3, 140])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P,dh", [(16, 64), (64, 128), (20, 64), (64, 256)])
def test_attend_rows_of_nan(cuda_lib, P, dh, dtype, new):
    """A row that holds NaN is NaN, and so is one whose scores are all minus infinity (their softmax is 0 / 0); a row
    that sees no key is zeros whatever its query holds.  Every other row is what it is without them."""
    H, G, lens = 2, 2, [300, 0, 40]
    cache = make_cache(25, H, P, dh, 201)
    cache[0][:, :, :, 3] = torch.tensor(1.0).to(CODE)           # all keys agree on the sign of element 3
    table = make_tables(lens, P, 25, 202)
    table[2] = -1                                             # every page of the last sequence is missing
    offs = None if new == 1 else [0, new, new + 2, 2 * new + 2]
    T = 3 if new == 1 else offs[-1]
    q = new_rows(T, H * G, dh, dtype, 203)
    bad = q.clone()
    bad[0, 0, 5], bad[0, 1, 3], bad[0, 2] = math.nan, -math.inf, math.nan
    bad[T - 1, 0, 5], bad[1, 0] = math.nan, math.nan
    bad[new // 2, 3, 0], bad[new // 2, 3, 1] = math.inf, math.nan
    want = torch.isnan(attend_softmax(bad, cache, table, lens, offs, 0.1)).any(-1)
    assert want[0, :3].all() and not want[T - 1].any() and (~want).sum() >= want.numel() // 2
    lens_t, offs_t = torch.tensor(lens, dtype=torch.int32), None if offs is None else torch.tensor(offs, dtype=torch.int32)
    for room in (table, wide(table, P)):
        clean = run_attend(cuda_lib, q, cache, room, lens_t, offs_t, 0.1, torch.full_like(q, 3.0)).cpu()
        got = run_attend(cuda_lib, bad, cache, room, lens_t, offs_t, 0.1, torch.full_like(q, 3.0)).cpu()
        assert got[want].isnan().all()
        assert torch.equal(got[~want], clean[~want])
        assert (got[T - 1] == 0).all()


@gpu
@pytest.mark.parametrize("new", [1, 3, 140])
@pytest.mark.parametrize("P,dh,span", [(16, 64, (32, 64)), (64, 128, (64, 128)), (20, 64, (64, 128)), (64, 256, (0, 200)), (32, 128, (1184, 1216)),
                                       (64, 64, (1280, 1344)), (16, 128, (640, 1500))])
def test_attend_keys_of_nan(cuda_lib, P, dh, span, new):
    """NaN in the keys of one stretch of a sequence, down to a single tile that one warp or one CTA alone looks at: the
    rows that see it are NaN, the earlier tokens' and the other sequence's are not."""
    H, G, lens = 1, 4, [1500, 70]
    need = sum(-(-n // P) for n in lens)
    cache = make_cache(need, H, P, dh, 211)
    table = make_tables(lens, P, need, 212)
    offs = [0, new, 2 * new if new < 70 else new + 70]
    q = new_rows(offs[-1], H * G, dh, torch.float16, 213)
    lens_t, offs_t = torch.tensor(lens, dtype=torch.int32), torch.tensor(offs, dtype=torch.int32)
    hurt = [x.clone() for x in cache]
    for j in range(*span):
        hurt[0].view(torch.uint8)[int(table[0, j // P]), 0, j % P, 7] = 0x7F
    sees = lens[0] - new + torch.arange(new) >= span[0]
    for room in (table, wide(table, P)):
        clean = run_attend(cuda_lib, q, cache, room, lens_t, offs_t, 0.1, torch.full_like(q, 3.0)).cpu()
        got = run_attend(cuda_lib, q, hurt, room, lens_t, offs_t, 0.1, torch.full_like(q, 3.0)).cpu()
        assert got[:new][sees].isnan().all()
        keep = torch.cat([~sees, torch.ones(offs[-1] - new, dtype=torch.bool)])
        assert torch.equal(got[keep], clean[keep])


@gpu
@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("new", [2, 150])
def test_attend_rows_do_not_touch_each_other(cuda_lib, P, new):
    """A row's bits do not depend on what the rows beside it attend to: half of the rows become ones whose running maximum
    keeps rising."""
    H, D, n = 1, 64, 700
    cache = make_cache(-(-n // P), H, P, D, 75)
    table = wide(make_tables([n], P, -(-n // P), 76), P)
    k = cache[0].float()
    for j in range(n):
        k[int(table[0, j // P]), 0, j % P, 0] = j / 8.0
    cache[0].copy_(k.to(CODE))
    cache[2].fill_(1.0 / 16)
    q = new_rows(new, 4, D, torch.bfloat16, 77)
    q[:, :, 0] = 0
    risen = q.clone()
    risen[:, ::2, 0] = 16.0
    args = (table, torch.tensor([n], dtype=torch.int32), torch.tensor([0, new], dtype=torch.int32), 1.0 / 3, torch.zeros_like(q))
    assert torch.equal(run_attend(cuda_lib, q, cache, *args)[:, 1::2], run_attend(cuda_lib, risen, cache, *args)[:, 1::2])


@gpu
@pytest.mark.parametrize("P", [16, 64, 20])
@pytest.mark.parametrize("new", [1, 140])
def test_attend_leap_over_a_page_of_zeros(cuda_lib, P, new):
    """A score leaps by 2^130 at a key whose page holds nothing but zeros (scale 2^-40, as the append writes): its weight is
    small, its share of the sum is not.  A later key of an ordinary page counts for more still."""
    H, D, n = 1, 64, 400
    cache = make_cache(-(-n // P), H, P, D, 221)
    table = make_tables([n], P, -(-n // P), 222)
    k, v = cache[0].float(), cache[1].float()
    k[..., 0] = 0.0
    cache[2].fill_(1.0 / 16)
    cache[3].fill_(2.0 ** -7)
    for j in range(n):
        if 128 // P <= j // P <= 191 // P:
            v[int(table[0, j // P])] = 0.0
            cache[3][int(table[0, j // P])] = 2.0 ** -40
    k[int(table[0, 150 // P]), 0, 150 % P, 0] = 88.0
    k[int(table[0, 245 // P]), 0, 245 % P, 0] = 96.0
    cache[0].copy_(k.to(CODE)), cache[1].copy_(v.to(CODE))
    q = new_rows(new, 4, D, torch.float16, 223) * 0.1
    q[:, :, 0] = 16.0
    # (the leap in powers of two at scale s: 88 s log2(e), 128 to 131 from s = 1.01 on)
    for scale in (1.0, 90 / 88, 1.03):
        check_attend(cuda_lib, q, cache, table, [n], [0, new], scale=scale)


@gpu
@pytest.mark.parametrize("P", [16, 64, 20])
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("step,level", [(30, 0.0), (15, 0.0), (30, 4.0), (-30, 0.0), (75, -8.0)])
def test_attend_scales_in_stairs(cuda_lib, P, new, step, level):
    """The values' scales climb from 2^-40 to 2^110 (or fall) in steps of pages while the scores stay or move a little:
    however far the weights' reference goes, every key keeps its place in the denominator.  300 sequences that are all the
    same, enough for a CTA to walk one from its first key to its last."""
    H, D, B, stair, steps = 1, 64, 300, 192, 150 // abs(step) + 1
    n = stair * steps
    cache = make_cache(-(-n // P), H, P, D, 231)
    table = make_tables([n], P, -(-n // P), 232)
    k = cache[0].float()
    cache[2].fill_(1.0 / 16)
    for j in range(0, n, P):
        p, i = int(table[0, j // P]), j // stair
        k[p, 0, :, 0] = level * i
        cache[3][p] = 2.0 ** ((-40 if step > 0 else 110) + step * i)
    cache[0].copy_(k.to(CODE))
    q = new_rows(new, 4, D, torch.bfloat16, 233) * 0.1
    q[:, :, 0] = 16.0
    want, tol = attend_ref(q, *cache, table, [n], [0, new], 1.0, torch.zeros_like(q))
    lens, offs = torch.full((B,), n, dtype=torch.int32), torch.arange(0, B * new + 1, new, dtype=torch.int32)
    for room in (table, wide(table, P)):
        got = run_attend(cuda_lib, q.repeat(B, 1, 1), cache, room.expand(B, -1).contiguous(), lens, offs, 1.0, torch.zeros(B * new, 4, D, dtype=q.dtype))
        for b in (0, 1, 150, B - 1):
            close(got[b * new:b * new + new], want, tol)


@gpu
@pytest.mark.parametrize("P", [16, 64, 20])
@pytest.mark.parametrize("new", [2, 150])
@pytest.mark.parametrize("start,width", [(200, 300), (200, 1), (690, 5), (511, 2), (64, 64)])
@pytest.mark.parametrize("dh", [64, 256])
def test_attend_rows_beside_leaping_ones(cuda_lib, dh, start, width, new, P):
    """A row's bits do not depend on the rows beside it, where its own weights outgrow fp16 in the very tile in which theirs
    leap beyond 2^100, or where those rows are NaN."""
    H, n = 1, 700
    cache = make_cache(-(-n // P), H, P, dh, 241)
    table = wide(make_tables([n], P, -(-n // P), 242), P)
    k = cache[0].float()
    k[..., 0] = 0.0
    for j in range(start, start + width):
        k[int(table[0, j // P]), 0, j % P, 0] = 14.0 + 0.25 * (j % 8)
    cache[0].copy_(k.to(CODE))
    cache[2].fill_(1.0 / 16)
    q = new_rows(new, 4, dh, torch.bfloat16, 243)
    q[:, :, 0] = 32.0                                         # 28 and more: 40 powers of two
    args = (table, torch.tensor([n], dtype=torch.int32), torch.tensor([0, new], dtype=torch.int32), 1.0 / 0.97, torch.zeros_like(q))
    quiet = run_attend(cuda_lib, q, cache, *args)
    for level in (0.0, 400.0, -400.0, math.nan, math.inf):
        other = q.clone()
        other[:, ::2, 0] = level
        assert torch.equal(run_attend(cuda_lib, other, cache, *args)[:, 1::2], quiet[:, 1::2]), level


@gpu
@pytest.mark.parametrize("new", [1, 6, 70])
def test_attend_strided_rows(cuda_lib, new):
    """q as a slice of a fused projection, out with heads outermost, storage bases off 16 bytes."""
    H, P, D = 2, 32, 64
    cache = make_cache(14, H, P, D, 81)
    table = make_tables([400], P, 14, 82)
    wide = new_rows(new, 8 + 4, D, torch.float16, 83)
    q = wide[:, 2:10]
    out = torch.full((8, new, D), 3.0, dtype=torch.float16).transpose(0, 1)
    check_attend(cuda_lib, q, cache, table, [400], [0, new], out=out)
    odd = torch.zeros(new * 8 * D + 3, dtype=torch.float16)
    odd[3:] = torch.randn(new * 8 * D, generator=torch.Generator().manual_seed(84)).half()
    check_attend(cuda_lib, odd[3:].view(new, 8, D), cache, table, [400], [0, new])


@gpu
@pytest.mark.parametrize("new", [1, 5, 40, 150])
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("course", ["up", "down", "steps", "last"])
def test_attend_scores_that_wander(cuda_lib, course, dh, new):
    """The running maximum rises all the way, never, by leaps, or at the very last key only."""
    H, P, n = 1, 32, 700
    cache = make_cache(24, H, P, dh, 161)
    table = make_tables([n], P, 24, 162)
    pos = np.arange(n)
    level = {"up": pos / 10.0, "down": -pos / 10.0, "steps": 7.0 * (pos // 150), "last": np.where(pos >= n - 2, 60.0, 0.0)}[course]
    k = cache[0].float()
    for j in range(n):                                        # element 0 of a key holds its level, to e4m3's 4 bits
        k[int(table[0, j // P]), 0, j % P, 0] = float(level[j])
    cache[0].copy_(k.to(CODE))
    cache[2].fill_(1.0 / 16)
    q = new_rows(new, 2, dh, torch.float16, 163) * 0.1
    q[:, :, 0] = 16.0
    check_attend(cuda_lib, q, cache, table, [n], [0, new], scale=1.0)


@gpu
@pytest.mark.parametrize("kv_heads,n", [(1, 128), (1, 129), (1, 4096), (2, 300), (40, 1000), (130, 500), (500, 70), (3, 4097)])
def test_attend_one_token_of_every_size_of_call(cuda_lib, kv_heads, n):
    """From one head over a few tokens to more heads than the GPU has places for, with sequences of all lengths up to n."""
    lens = [n, n // 2, 1]
    need = sum(-(-x // 64) for x in lens)
    cache = make_cache(need, kv_heads, 64, 64, 171)
    check_attend(cuda_lib, new_rows(3, kv_heads, 64, torch.bfloat16, 173), cache, make_tables(lens, 64, need, 172), lens, None)


@gpu
@pytest.mark.parametrize("batch", [700, 4100])
def test_attend_many_sequences(cuda_lib, batch):
    rng = np.random.default_rng(181)
    news = [int(x) for x in rng.integers(0, 5, batch)]
    lens = [n + int(x) for n, x in zip(news, rng.integers(0, 40, batch))]
    need = sum(-(-x // 16) for x in lens)
    cache = make_cache(need, 1, 16, 8, 182)
    offs = [0] + [int(x) for x in np.cumsum(news)]
    check_attend(cuda_lib, new_rows(offs[-1], 24, 8, torch.float16, 183), cache, make_tables(lens, 16, need, 184), lens, offs)


@gpu
def test_attend_is_repeatable(cuda_lib):
    """The same call gives the same bits: partial results are joined in a fixed order."""
    cache = make_cache(300, 2, 64, 128, 91)
    table = make_tables([9000, 700], 64, 300, 92)
    for new, table in ((1, table), (100, table), (100, wide(table, 64))):
        q = new_rows(2 * new, 8, 128, torch.bfloat16, 93)
        offs = torch.tensor([0, new, 2 * new], dtype=torch.int32)
        a, b = (run_attend(cuda_lib, q, cache, table, torch.tensor([9000, 700], dtype=torch.int32), offs, 0.09, torch.zeros_like(q)) for _ in range(2))
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("P,D", [(64, 128), (16, 64), (20, 128), (64, 256)])
def test_wait_limit_of_the_prompts_kernel_is_reported(cuda_lib, P, D):
    """Every wait of the prompts kernel is bounded.  With waits that give up after one poll its CTAs stop somewhere on
    their way, let products and copies end and leave; the call returns, and the timeout query reports it.  With the default
    limit restored the same call is complete, on a GPU that is as it was."""
    lib, handle = cuda_lib
    n, new = 3000, 300
    cache = [to_dev(x) for x in make_cache(-(-n // P), 1, P, D, 251)]
    table = wide(make_tables([n], P, -(-n // P), 252), P).to(DEV)
    q = new_rows(new, 8, D, torch.bfloat16, 253).to(DEV)
    lens, offs = torch.tensor([n], dtype=torch.int32, device=DEV), torch.tensor([0, new], dtype=torch.int32, device=DEV)
    out = [torch.zeros_like(q) for _ in range(3)]
    with ops.PagedAttentionOp(lib, handle, q, q, *cache, table, lens, offs) as op:
        op(out[0], q, *cache, table, lens, offs)
        before = ops.device_timeouts(lib, handle)
        try:
            ops.set_wait_limit(lib, handle, 1)
            op(out[1], q, *cache, table, lens, offs)          # returns normally
            torch.cuda.synchronize()
            mid = ops.device_timeouts(lib, handle)
            assert mid > before
        finally:
            ops.set_wait_limit(lib, handle, 0)
        op(out[2], q, *cache, table, lens, offs)
        torch.cuda.synchronize()
    assert ops.device_timeouts(lib, handle) == mid
    assert torch.equal(out[0], out[2])


@gpu
def test_attend_offsets_beyond_32_bits(cuda_lib):
    """Pages whose elements lie beyond 2^32 of the pool's start."""
    lib, handle = cuda_lib
    H, P, D, N = 8, 64, 128, 70000                            # 4.6e9 codes in each pool
    kp, vp = (torch.zeros(N, H, P, D, dtype=torch.uint8, device=DEV).view(CODE) for _ in range(2))
    ids = torch.tensor([[69999, 2, 65537, 66000]], dtype=torch.int32)
    cache = make_cache(4, H, P, D, 101)
    ks, vs = torch.ones(N, H, device=DEV), torch.ones(N, H, device=DEV)
    at = ids[0].long().to(DEV)
    for pool, src in ((kp, cache[0]), (vp, cache[1])):
        pool.view(torch.uint8)[at] = src.view(torch.uint8).to(DEV)
    ks[at], vs[at] = cache[2].to(DEV), cache[3].to(DEV)
    for new, ids in ((1, ids), (1, wide(ids, P)), (100, wide(ids, P)), (100, ids)):
        q = new_rows(new, 16, D, torch.float16, 103)
        want, tol = attend_ref(q, *cache, torch.arange(4, dtype=torch.int32)[None], [250], [0, new], 0.1, torch.zeros_like(q))
        out = torch.zeros_like(q, device=DEV)
        ops.paged_attention(lib, handle, out, q.to(DEV), kp, vp, ks, vs, ids.to(DEV), torch.tensor([250], dtype=torch.int32, device=DEV),
                            torch.tensor([0, new], dtype=torch.int32, device=DEV), scale=0.1)
        torch.cuda.synchronize()
        close(out, want, tol)
    # the same place is appended to, copied from and compacted away
    k = new_rows(3, H, D, torch.float16, 104)
    ops.paged_cache_append(lib, handle, k.to(DEV), k.to(DEV), kp, vp, ks, vs, ids.to(DEV), torch.tensor([253], dtype=torch.int32, device=DEV),
                           torch.tensor([0, 3], dtype=torch.int32, device=DEV))
    want = append_ref(k, k, *cache, torch.arange(4, dtype=torch.int32)[None], [253], [0, 3])
    same_codes(kp[at], want[0])
    same_codes(vp[at], want[1])
    ops.paged_cache_copy(lib, handle, kp, vp, ks, vs, torch.tensor([[69999, 69000]], dtype=torch.int32, device=DEV))
    same_codes(kp[69000], want[0][0])
    table, page_map, live = ids.to(DEV), torch.zeros(N, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.paged_cache_compact(lib, handle, kp, vp, ks, vs, table, table, torch.tensor([253], dtype=torch.int32, device=DEV), page_map, live)
    assert live.item() == 4 and table.cpu().tolist() == [[3, 2, 0, 1]]
    same_codes(vp[table[0].long()], want[1])


# ---- copy and compact -----------------------------------------------------------------------------------------------

MOVE_LAYOUTS = [(2, 16, 64, "head", 0), (8, 64, 128, "token", 0), (3, 20, 80, "token", 16), (2, 7, 33, "head", 0), (1, 5, 12, "head", 0),
                (4, 1, 64, "head_first", 0), (2, 32, 100, "head_first", 4), (1, 1, 1, "head", 0), (5, 1, 3, "token", 1)]


def storage_of(x):
    return torch.as_strided(x.view(torch.uint8), (x.untyped_storage().nbytes(),), (1,), 0)


@gpu
@pytest.mark.parametrize("heads,page,dh,layout,spare", MOVE_LAYOUTS)
def test_copy(cuda_lib, heads, page, dh, layout, spare):
    """Forks (one source, many destinations), padding rows, a page onto itself; all other bytes stay, gaps included."""
    lib, handle = cuda_lib
    N = 40
    cache = make_cache(N, heads, page, dh, 111, layout, spare, pow2=False)
    pairs = [(3, 7), (3, 9), (3, 39), (0, 1), (38, 2), (-1, 5), (5, N), (12, 12), (6, -3), (2147483647, 4)]
    dev = [to_dev(x) for x in cache]
    before = [x.clone() for x in (storage_of(dev[0]), storage_of(dev[1]))]
    ops.paged_cache_copy(lib, handle, *dev, torch.tensor(pairs, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    for x, y in zip(dev, cache):
        want = y.clone() if y.dtype != CODE else y.view(torch.uint8).clone()
        for s, d in pairs:
            if 0 <= s < N and 0 <= d < N:
                want[d] = (y if y.dtype != CODE else y.view(torch.uint8))[s]
        assert torch.equal((x if x.dtype != CODE else x.view(torch.uint8)).cpu(), want)
    # nothing outside the copied pages has changed: undo and compare the whole storage
    for x, y in zip(dev[:2], cache[:2]):
        for s, d in pairs:
            if 0 <= s < N and 0 <= d < N:
                x.view(torch.uint8)[d] = y.view(torch.uint8)[d].to(DEV)
    for x, y in zip(before, (storage_of(dev[0]), storage_of(dev[1]))):
        assert torch.equal(x, y)


def test_copy_of_nothing(host):
    lib, handle = host
    t = _small()
    t["pairs"] = t["pairs"][:0]
    with ops.PagedCacheCopyOp(lib, handle, *[t[f] for f in OPS["copy"][1]]) as o:
        o(*[t[f] for f in OPS["copy"][1]])  # returns before it reaches the device


def compact_ref(table, lens, page, N):
    used = [min(max(n, 0), table.shape[1] * page) for n in lens]
    live = sorted({int(p) for row, n in zip(table, used) for p in row[:-(-n // page)] if 0 <= p < N})
    L = len(live)
    holes = [p for p in range(L) if p not in set(live)]
    to = {p: p for p in live if p < L}
    to.update(zip([p for p in live if p >= L], holes))
    new = table.clone()
    for b, n in enumerate(used):
        for i in range(-(-n // page)):
            new[b, i] = to.get(int(table[b, i]), int(table[b, i]))
    return new, [to.get(p, -1) for p in range(N)], L


COMPACT_CASES = [
    # pages, lens, page size, shared rows (row copied from, row)
    (40, [50, 0, 33, 1, 160], 16, []),
    (40, [0, 0], 16, []),
    (32, [32 * 16], 16, []),                                  # everything lives, the last word of the map is full
    (33, [33 * 16], 16, []),
    (64, [31 * 16, 16, 1], 16, [(0, 1)]),
    (1, [5], 16, []),
    (3000, [20000], 16, []),                                  # one long row
    (100000, [300] * 600, 16, [(3, 5), (3, 7)]),              # many rows, a map longer than one word per thread
    (500, [-3, 1 << 30, 40], 16, []),
]


@gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("N,lens,page,shared", COMPACT_CASES)
def test_compact(cuda_lib, N, lens, page, shared, in_place):
    lib, handle = cuda_lib
    H, D = 2, 16
    table = make_tables([min(n, 320) for n in lens], page, N, 121, cols=max(-(-min(n, 20000) // page) for n in lens) + 1)
    for a, b in shared:
        table[b] = table[a]
    if N == 500:
        table[2, 1] = 500
    cache = make_cache(N, H, page, D, 122, "token" if N % 2 else "head")
    dev, table_d = [to_dev(x) for x in cache], table.to(DEV)
    new = table_d if in_place else torch.zeros_like(table_d)
    page_map, live = torch.full((N,), 99, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.paged_cache_compact(lib, handle, *dev, new, table_d, torch.tensor(lens, dtype=torch.int32, device=DEV), page_map, live)
    torch.cuda.synchronize()
    want, want_map, L = compact_ref(table, lens, page, N)
    assert live.item() == L and page_map.cpu().tolist() == want_map
    assert torch.equal(new.cpu(), want)
    if not in_place:
        assert torch.equal(table_d.cpu(), table)
    for x, y in zip(dev, cache):
        x, y = (z.view(torch.uint8) if z.dtype == CODE else z for z in (x.cpu(), y.clone()))
        moved = [(p, q) for p, q in enumerate(want_map) if q not in (-1, p)]
        if moved:
            y[[q for _, q in moved]] = y[[p for p, _ in moved]]
        assert torch.equal(x, y)


@gpu
def test_compact_empty(cuda_lib):
    """No sequences, no columns, no pages."""
    lib, handle = cuda_lib
    for N, batch, cols in ((5, 0, 3), (5, 3, 0), (0, 2, 2)):
        cache = [to_dev(x) for x in make_cache(N, 1, 4, 16, 1)] if N else [torch.zeros(0, 1, 4, 16, dtype=torch.uint8, device=DEV).view(CODE)] * 2 + [torch.zeros(0, 1, device=DEV)] * 2
        table = torch.full((batch, cols), 1, dtype=torch.int32, device=DEV)
        page_map, live = torch.full((N,), 9, dtype=torch.int32, device=DEV), torch.full((1,), 9, dtype=torch.int32, device=DEV)
        ops.paged_cache_compact(lib, handle, *cache, torch.zeros_like(table), table, torch.full((batch,), 8, dtype=torch.int32, device=DEV), page_map, live)
        torch.cuda.synchronize()
        assert live.item() == 0 and (page_map == -1).all()


# ---- together -------------------------------------------------------------------------------------------------------

@gpu
def test_a_serving_run(cuda_lib):
    """Prompts, decoding, a fork, an ended sequence and a compaction, as a server would do them.  Every attention call
    is checked against the definition on the cache as it stands; the fork and the compaction change no answer."""
    lib, handle = cuda_lib
    H, G, P, D, N, dt = 2, 4, 16, 64, 64, torch.bfloat16
    kp, vp, ks, vs = (to_dev(x) for x in make_cache(N, H, P, D, 131))
    free = list(np.random.default_rng(132).permutation(N))
    table = torch.full((4, 12), -1, dtype=torch.int32)
    lens = [0, 0, 0, 0]

    def grow(b, n):
        while -(-(lens[b] + n) // P) > int((table[b] >= 0).sum()):
            table[b, int((table[b] >= 0).sum())] = int(free.pop())
        lens[b] += n

    def step(news, seed):
        for b, n in enumerate(news):
            grow(b, n)
        offs = [0] + [int(x) for x in np.cumsum(news)]
        T = offs[-1]
        k, v, q = new_rows(T, H, D, dt, seed), new_rows(T, H, D, dt, seed + 1), new_rows(T, H * G, D, dt, seed + 2)
        td, ld, od = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), torch.tensor(offs, dtype=torch.int32, device=DEV)
        ops.paged_cache_append(lib, handle, k.to(DEV), v.to(DEV), kp, vp, ks, vs, td, ld, od)
        return q, attend(q, td, ld, od, offs)

    def attend(q, td, ld, od, offs):
        out = torch.zeros_like(q, device=DEV)
        ops.paged_attention(lib, handle, out, q.to(DEV), kp, vp, ks, vs, td, ld, od)
        torch.cuda.synchronize()
        want, tol = attend_ref(q, *(x.cpu() for x in (kp, vp, ks, vs)), td.cpu(), lens, offs, D ** -0.5, torch.zeros_like(q))
        close(out, want, tol)
        return out

    step([70, 33, 5, 0], 200)                                 # prompts of three requests
    for i in range(20):
        step([1, 1, 1, 0], 300 + 10 * i)
    # request 3 forks from request 0: full pages are shared, the half-filled one is copied
    full = lens[0] // P
    table[3] = table[0]
    table[3, full] = int(free.pop())
    lens[3] = lens[0]
    ops.paged_cache_copy(lib, handle, kp, vp, ks, vs, torch.tensor([[int(table[0, full]), int(table[3, full])]], dtype=torch.int32, device=DEV))
    q, _ = step([1, 1, 1, 1], 600)
    lens[1] = 0                                               # request 1 ends
    offs = [0, 1, 1, 2, 3]
    q = q[[0, 2, 3]]
    od, ld = torch.tensor(offs, dtype=torch.int32, device=DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    before = attend(q, table.to(DEV), ld, od, offs)
    td, page_map, live = table.to(DEV), torch.zeros(N, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.paged_cache_compact(lib, handle, kp, vp, ks, vs, td, td, ld, page_map, live)
    after = attend(q, td, ld, od, offs)
    assert torch.equal(before, after)
    assert live.item() == full + 2 + -(-lens[2] // P) and td[[0, 2, 3]].max().item() < live.item()


@gpu
def test_graph_replays_while_the_sequences_grow(cuda_lib):
    """Append and attention captured once, replayed with new tokens and lengths in the same tensors, next to an eager
    run of the same steps; all on a stream of its own."""
    lib, handle = cuda_lib
    H, G, P, D, B = 2, 4, 16, 128, 3
    start = [30, 1, 47]
    cache = [to_dev(x) for x in make_cache(40, H, P, D, 141)]
    eager = [x.clone() for x in cache]
    table = make_tables([n + 20 for n in start], P, 40, 142).to(DEV)
    lens = torch.tensor(start, dtype=torch.int32, device=DEV)
    k, v = (torch.zeros(B, H, D, dtype=torch.float16, device=DEV) for _ in range(2))
    q, out = (torch.zeros(B, H * G, D, dtype=torch.float16, device=DEV) for _ in range(2))
    s = torch.cuda.Stream()
    with ops.PagedCacheAppendOp(lib, handle, k, v, *cache, table, lens) as app, ops.PagedAttentionOp(lib, handle, out, q, *cache, table, lens) as att:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            app(k, v, *cache, table, lens, stream=s)
            att(out, q, *cache, table, lens, stream=s)
        for i in range(12):
            lens += 1
            for x, seed in ((k, 1), (v, 2), (q, 3)):
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * i + seed)) * (1 + i))
            g.replay()
            other = torch.zeros_like(out)
            ops.paged_cache_append(lib, handle, k, v, *eager, table, lens)
            ops.paged_attention(lib, handle, other, q, *eager, table, lens)
            torch.cuda.synchronize()
            assert torch.equal(out, other)
            for a, b in zip(cache, eager):
                assert torch.equal(a.view(torch.uint8) if a.dtype == CODE else a, b.view(torch.uint8) if b.dtype == CODE else b)
        del g


@gpu
def test_two_streams_at_once(cuda_lib):
    """Two operators with a workspace each on two streams give what they give alone."""
    lib, handle = cuda_lib
    H, P, D = 4, 64, 128
    cache = [to_dev(x) for x in make_cache(400, H, P, D, 151)]
    jobs = []
    for i, (lens, new) in enumerate((([9000, 3000], 1), ([12000], 300))):
        table = make_tables(lens, P, 400, 152 + i).to(DEV)
        T = new * len(lens)
        q = new_rows(T, 16, D, torch.float16, 154 + i).to(DEV)
        offs = torch.arange(0, T + 1, new, dtype=torch.int32, device=DEV)
        jobs.append((torch.zeros_like(q), q, *cache, table, torch.tensor(lens, dtype=torch.int32, device=DEV), offs))
    alone = []
    for j in jobs:
        ops.paged_attention(lib, handle, *j)
        torch.cuda.synchronize()
        alone.append(j[0].clone())
    plans, streams = [ops.PagedAttentionOp(lib, handle, *j) for j in jobs], [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(20):
        for j in jobs:
            j[0].zero_()
        torch.cuda.synchronize()
        for o, s, j in zip(plans, streams, jobs):
            o(*j, stream=s)
        torch.cuda.synchronize()
        for j, a in zip(jobs, alone):
            assert torch.equal(j[0], a)
    for o in plans:
        o.destroy()


@gpu
@pytest.mark.parametrize("how", ["one shot", "made before", "dropped after", "default stream"])
@pytest.mark.parametrize("new", [1, 200])
def test_workspace_memory_and_streams(cuda_lib, new, how):
    """torch hands memory out again while the stream that it was made on still has work queued for it.  A workspace is never
    such memory on another stream: neither ahead of the call (fills of a tensor that is gone are still queued), nor behind
    it (fills of a new tensor start while the call still runs)."""
    lib, handle = cuda_lib
    H, P, D, n = 2, 64, 128, 30000
    cache = [to_dev(x) for x in make_cache(-(-n // P), H, P, D, 261)]
    table = make_tables([n], P, -(-n // P), 262).to(DEV)
    lens, offs = torch.tensor([n], dtype=torch.int32, device=DEV), torch.tensor([0, new], dtype=torch.int32, device=DEV)
    q = new_rows(new, 8 * H, D, torch.bfloat16, 263).to(DEV)
    want, out, side = torch.zeros_like(q), torch.zeros_like(q), torch.cuda.Stream()
    args = (out, q, *cache, table, lens, offs)
    with ops.PagedAttentionOp(lib, handle, want, q, *cache, table, lens, offs) as op:
        op(want, *args[1:])
        size = op.workspace_size
    torch.cuda.synchronize()

    def fills(count):
        x = torch.empty(size, dtype=torch.uint8, device=DEV)
        for _ in range(count):
            x.fill_(255)                                      # (a stretch without an item, sums of NaN)

    if how == "one shot":
        fills(2000)
        ops.paged_attention(lib, handle, *args, stream=side)
    elif how == "made before":
        fills(2000)
        with ops.PagedAttentionOp(lib, handle, *args) as op:
            op(*args, stream=side.cuda_stream)
    elif how == "dropped after":
        op = ops.PagedAttentionOp(lib, handle, *args)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(2000000)
        op(*args, stream=side)
        op.destroy()
        del op
        fills(500)
    else:
        torch.cuda._sleep(2000000)
        with torch.cuda.stream(side):                         # a call without a stream goes to the default one all the same
            ops.paged_attention(lib, handle, *args)
            fills(500)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@gpu
def test_one_shot_calls_in_a_capture(cuda_lib):
    """Calls that make their workspace inside a capture, on the captured stream and on one that forks from it, in every
    form of a stream argument; replayed after the memory of the capture has been asked for again."""
    lib, handle = cuda_lib
    H, P, D, n = 2, 32, 128, 3000
    cache = [to_dev(x) for x in make_cache(-(-n // P), H, P, D, 271)]
    table = wide(make_tables([n], P, -(-n // P), 272), P).to(DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    s, side = torch.cuda.Stream(), torch.cuda.Stream()
    for new in (1, 150):
        offs = torch.tensor([0, new], dtype=torch.int32, device=DEV)
        q = new_rows(new, 4 * H, D, torch.float16, 273).to(DEV)
        outs = [torch.zeros_like(q) for _ in range(5)]
        args = (q, *cache, table, lens, offs)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.paged_attention(lib, handle, outs[0], *args, stream=s)
            ops.paged_attention(lib, handle, outs[1], *args, stream=s.cuda_stream)
            ops.paged_attention(lib, handle, outs[2], *args, stream=ctypes.c_void_p(s.cuda_stream))
            kept = ops.PagedAttentionOp(lib, handle, outs[3], *args)
            kept(outs[3], *args, stream=s)
            side.wait_stream(s)
            kept(outs[4], *args, stream=side)
            s.wait_stream(side)
        for length in (n, 777, 40):
            lens.fill_(max(length, new))
            want = torch.zeros_like(q)
            ops.paged_attention(lib, handle, want, *args)
            for x in outs:
                x.zero_()
            g.replay()
            torch.cuda.synchronize()
            for x in outs:
                assert torch.equal(x, want)
        kept.destroy()
        del g, kept


@gpu
@pytest.mark.parametrize("new,D", [(1, 128), (3, 64), (150, 128), (150, 256)])
def test_captured_attention_over_long_tables(cuda_lib, new, D):
    """The forms that split work over CTAs and join it in a second kernel, captured with a table in a wider tensor and
    replayed twice as often as the lengths change; the outputs written over the queries, on another stream, agree."""
    lib, handle = cuda_lib
    H, G, P = 2, 4, 32
    cache = [to_dev(x) for x in make_cache(120, H, P, D, 191)]
    table = wide(make_tables([1500, 700], P, 120, 192, cols=60), P).to(DEV)
    table = table[:, :table.shape[1] - 5]
    offs = torch.tensor([0, new, 2 * new], dtype=torch.int32, device=DEV)
    lens = torch.tensor([new, new], dtype=torch.int32, device=DEV)
    q = new_rows(2 * new, H * G, D, torch.bfloat16, 193).to(DEV)
    out, s, other = torch.zeros_like(q), torch.cuda.Stream(), torch.cuda.Stream()
    with ops.PagedAttentionOp(lib, handle, out, q, *cache, table, lens, offs) as att:
        assert att.workspace is not None
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            att(out, q, *cache, table, lens, offs, stream=s)
        for l0, l1 in ((new, new), (1500, 700), (151, 0), (1, 650)):
            lens.copy_(torch.tensor([l0, l1], dtype=torch.int32))
            out.fill_(7.0)
            g.replay()
            g.replay()
            torch.cuda.synchronize()
            over = q.clone()
            torch.cuda.synchronize()
            ops.paged_attention(lib, handle, over, over, *cache, table, lens, offs, stream=other)
            torch.cuda.synchronize()
            assert torch.equal(out, over)
            want, tol = attend_ref(q.cpu(), *(x.cpu() for x in cache), table.cpu(), [l0, l1], offs.tolist(), D ** -0.5, torch.zeros_like(q).cpu())
            close(out, want, tol)
        del g
