"""CPU checks of what serves the paged cache: the C entries' refusals before anything
is enqueued, the rotary frequencies, and the definitions of oracle/paged.py."""
import ctypes
import math

import pytest
import torch

from oracle import paged
from tests.test_abi import BIG, call_raw, lib  # noqa: F401
from tests.test_paged_host import BAD_SHAPES, BAD_STRIDES, GOOD, SHAPE, STRIDES, desc

FOUR = dict(page_stride=8 * 16 * 64, head_stride=16 * 64, slot_stride=64, dtype=16, k_scales=16, v_scales=16,
            scale_page_stride=8 * 16 * 4, scale_head_stride=16 * 4, scale_slot_stride=4)


def four(**changed):
    return desc(**{**FOUR, **changed})


def rows(lib, cache=None, into=None, k=16, v=16, q=16, q_out=16, offsets=16, turns=16, count=5,
         strides=(1024, 128, 1024, 128, 4096, 128), heads=32, rotary=128, interleaved=0, amplitude=1.0):
    cache = cache or desc()
    return call_raw(lib, "prismkv_paged_append_rows", cache, into or cache, k, v, q, q_out, offsets, turns, count, *strides,
                    heads, rotary, interleaved, amplitude)


def read(lib, cache=None, offsets=16, k=16, v=16, count=5):
    return call_raw(lib, "prismkv_paged_read", cache or desc(), offsets, k, v, count)


def prompt(lib, cache=None, q=16, offsets=16, lse=16, work=16, out=16, count=5, group=4, scale=0.1, nbytes=BIG):
    return call_raw(lib, "prismkv_paged_prompt", cache or desc(), q, offsets, lse, work, out, count, group, scale, nbytes)


def passes(code):
    """Past every host check: refused by the runtime, as there is no device here."""
    return code not in (0, -1, -2)


@pytest.mark.parametrize("call", [rows, read, prompt])
def test_refused_caches(lib, call):  # noqa: F811
    assert passes(call(lib)) and passes(call(lib, four())) and passes(call(lib, four(dtype=17)))
    for shape in BAD_SHAPES:
        assert call(lib, desc(**dict(zip(SHAPE, shape)))) == -1, shape
    for strides in BAD_STRIDES:
        assert call(lib, desc(**dict(zip(STRIDES, strides)))) == -1, strides
    for dtype in (-1, 3, 15, 18, 32):
        assert call(lib, four(dtype=dtype)) == -2
    for name in ("k", "v", "table", "lengths", "err"):
        assert call(lib, desc(**{name: 0})) == -1, name
    # the scales of pages in 4 bits: rows of 4 bytes here
    for bad in (dict(k_scales=0), dict(v_scales=0), dict(k_scales=18), dict(v_scales=17), dict(scale_page_stride=-4),
                dict(scale_page_stride=6), dict(scale_head_stride=2), dict(scale_slot_stride=0), dict(scale_slot_stride=5),
                dict(scale_page_stride=1 << 40), dict(scale_head_stride=1 << 40), dict(scale_slot_stride=1 << 40),
                dict(slot_stride=48), dict(page_stride=8 * 16 * 64 + 8)):
        assert call(lib, four(**bad)) == -1, bad
    name = f"prismkv_paged_{'append_rows' if call is rows else call.__name__}"
    assert call_raw(lib, name, *[0] * (len(getattr(lib.cdll, name).argtypes) - 1)) == -1  # no cache


def test_four_bits_in_the_earlier_entries(lib):  # noqa: F811
    from tests.test_paged_host import append, attend, evict
    for call in (append, attend, evict):
        assert passes(call(lib, four())) and passes(call(lib, four(dtype=17))), call
        assert call(lib, four(k_scales=0)) == -1 and call(lib, four(scale_slot_stride=2)) == -1
        for name in ("k_scales", "scale_page_stride", "scale_head_stride", "scale_slot_stride"):
            assert call(lib, four(), four(**{name: 2 * FOUR[name]})) == -1, name
    need = lib.query("prismkv_paged_attend_work_bytes", 3, 8, 4, 128, 160, 1, 16)
    assert need > 0 and attend(lib, four(), nbytes=need - 1) == -1


def test_refused_rows(lib):  # noqa: F811
    for bad in (dict(k=0), dict(v=0), dict(k=24), dict(q=0), dict(q_out=0), dict(q=24), dict(q_out=8), dict(heads=0),
                dict(heads=-1), dict(offsets=18), dict(count=-1), dict(count=1 << 31), dict(offsets=0, count=4),
                dict(turns=20), dict(turns=0), dict(rotary=8), dict(rotary=24), dict(rotary=144), dict(interleaved=2),
                dict(amplitude=math.inf), dict(amplitude=math.nan), dict(heads=1 << 30)):
        assert rows(lib, **bad) == -1, bad
    assert passes(rows(lib, q=0, q_out=0, heads=0))  # keys alone
    assert passes(rows(lib, q=0, q_out=0, heads=0, turns=0, rotary=0))  # nothing turned
    assert rows(lib, q=0, q_out=0, heads=0, turns=0, rotary=16) == -1
    for i in range(6):
        for bad in (1028, 1 << 41, -(1 << 41)):
            assert rows(lib, strides=[bad if j == i else 1024 for j in range(6)]) == -1
    for bad in (dict(k=0), dict(v=0), dict(k=8), dict(offsets=2), dict(count=-1), dict(count=1 << 31),
                dict(offsets=0, count=4)):
        assert read(lib, **bad) == -1, bad


def test_refused_prompts(lib):  # noqa: F811
    for bad in (dict(q=0), dict(q=24), dict(out=0), dict(out=8), dict(work=0), dict(work=8), dict(lse=2), dict(offsets=2),
                dict(offsets=0, count=4), dict(count=-1), dict(group=0), dict(group=1025), dict(count=(1 << 28) + 1),
                dict(scale=math.nan), dict(scale=math.inf), dict(scale=3e38)):
        assert prompt(lib, **bad) == -1, bad
    query = lambda *a: lib.query("prismkv_paged_prompt_work_bytes", *a)  # noqa: E731
    need = query(48, 1, 8, 4, 128, 65536, 0)
    # a state is a tile's 128 rows of maxima, sums and products in fp32
    assert need >= 1024 * 128 * 130 * 4 and need % (128 * 130 * 4) == 0
    long = desc(max_pages=4096, sequences=1)
    assert prompt(lib, long, count=48, nbytes=need - 1) == -1 and passes(prompt(lib, long, count=48, nbytes=need))
    assert query(75, 1, 8, 4, 128, 80, 0) == 16  # never cut
    for bad in ((-1, 1, 8, 4, 128, 80, 0), (5, 0, 8, 4, 128, 80, 0), (5, 1, 0, 4, 128, 80, 0), (5, 1, 8, 0, 128, 80, 0),
                (5, 1, 8, 4, 0, 80, 0), (5, 1, 8, 4, 128, 0, 0), (5, 1, 8, 4, 128, 80, 3), (5, 1, 8, 4, 128, 80, 18),
                (1 << 29, 1, 8, 4, 128, 80, 0)):
        assert query(*bad) == 0, bad


def test_prompts_of_more_blocks_than_a_launch_holds(lib):  # noqa: F811
    """Workgroups of 256 threads, of which a launch has fewer than 2^32: 512 for what is cut,
    and one for each KV head, 128 rows of one and sequence that has some."""
    def need(rows, sequences, kv_heads, group):
        return lib.query("prismkv_paged_prompt_work_bytes", rows, sequences, kv_heads, group, 64, 16, 0)

    most = 2 ** 24 - 512
    assert need(65535, 65535, 250, 1) and need(65535, 65535, 257, 1) == 0
    many = desc(sequences=65535, kv_heads=257, max_pages=1)
    assert prompt(lib, many, count=65535, group=1) == -1
    assert passes(prompt(lib, desc(sequences=65535, kv_heads=250, max_pages=1), count=65535, group=1))
    for kv_heads, group in ((8, 4), (16, 1), (3, 7)):
        rows = ((most - 1) // kv_heads - 1) * 128 // group
        assert (rows * group // 128 + 1) * kv_heads < most and need(rows, 1, kv_heads, group)
        rows = (-(-most // kv_heads) - 1) * 128 // group + 128
        assert need(rows, 1, kv_heads, group) == 0
    assert need(5, 65535, 65535, 1)  # (no more tiles than rows)


def test_the_descriptor_mirrors_the_header():
    import re
    from pathlib import Path
    from prismkv_amd._lib import PagedCacheDesc
    text = (Path(__file__).resolve().parents[1] / "include" / "prismkv_hip.h").read_text()
    body = re.search(r"typedef struct prismkv_paged_cache \{(.*?)\} prismkv_paged_cache;", text, re.S).group(1)
    fields = []
    for kind, names in re.findall(r"(uint64_t|int64_t|int32_t)\s+([\w, \n]+);", body):
        fields += [(name.strip(), {"uint64_t": ctypes.c_uint64, "int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32}[kind])
                   for name in names.split(",")]
    assert fields == list(PagedCacheDesc._fields_)
    assert set(GOOD) | set(FOUR) == {name for name, _ in fields}


# ------------------------------------------------------------------ rotary

LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}


@pytest.mark.parametrize("scaling", [None, {"rope_type": "default"}, {"rope_type": "linear", "factor": 4.0}, LLAMA3, YARN,
                                     {**YARN, "beta_fast": 16, "beta_slow": 2}, {**YARN, "attention_factor": 1.25}])
@pytest.mark.parametrize("base,dim", [(10000.0, 64), (5e5, 128), (1e6, 128)])
def test_frequencies_are_transformers(scaling, base, dim):
    """The same numbers as transformers computes from a configuration, in fp32: a power
    of the base and a few products, 2^-18 together."""
    from transformers import Qwen3Config
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    from prismkv_amd import Rotary
    rotary = Rotary(dim, base=base, scaling=scaling, device="cpu")
    kind = (scaling or {}).get("rope_type", "default")
    if kind == "default":
        want, factor = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim), 1.0
    else:
        config = Qwen3Config(hidden_size=2 * dim, num_attention_heads=2, head_dim=dim, rope_theta=base,
                             max_position_embeddings=32768)
        config.rope_parameters = config.rope_scaling = {"rope_theta": base, **scaling}
        want, factor = ROPE_INIT_FUNCTIONS[kind](config, "cpu")
    assert rotary.amplitude == pytest.approx(factor, rel=1e-6)
    assert ((rotary.frequencies - want.double()).abs() <= want.double().abs() * 2.0 ** -18).all()
    # a turn is 2^64: an angle of position p is p * turns, of which the whole turns fall away
    for p in (1, 1000, 3_000_000):
        for f, t in zip(rotary.frequencies.tolist(), rotary.turns.tolist()):
            part = (p * (t % 2 ** 64)) % 2 ** 64 / 2.0 ** 64
            assert abs(math.remainder(part - math.fmod(p * f / (2 * math.pi), 1.0), 1.0)) <= p * 2.0 ** -52


def test_refused_rotaries():
    from prismkv_amd import Rotary
    for bad in (dict(head_dim=128, rotary_dim=8), dict(head_dim=128, rotary_dim=24), dict(head_dim=64, rotary_dim=80),
                dict(head_dim=128, base=0.0), dict(head_dim=128, base=math.inf),
                dict(head_dim=128, scaling={"rope_type": "dynamic"}), dict(head_dim=128, scaling={"rope_type": "linear"}),
                dict(head_dim=128, scaling={"rope_type": "linear", "factor": 0.0}),
                dict(head_dim=128, scaling={**LLAMA3, "high_freq_factor": 1.0}),
                dict(head_dim=128, scaling={**LLAMA3, "beta_fast": 3}),
                dict(head_dim=128, scaling={**YARN, "beta_slow": 64}),
                dict(head_dim=128, scaling={**YARN, "attention_factor": math.inf})):
        with pytest.raises(ValueError):
            Rotary(**bad, device="cpu")
    assert Rotary(128, rotary_dim=48, interleaved=True, device="cpu").turns.shape == (24,)


# ------------------------------------------------------------------ the definitions

def test_what_four_bits_hold():
    sizes = torch.tensor(paged.SIZES, dtype=torch.float64)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(200, 64, generator=gen) * torch.exp(3 * torch.randn(200, 1, generator=gen))
    codes, scales = paged.hold(x)
    got = paged.value(codes, scales)
    # every value is as near as any size of its block can be, and the scale is the smallest
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.double() - 127).repeat_interleave(32, -1)
    best = ((x.double().abs() / unit)[..., None] - sizes).abs().amin(-1) * unit
    assert torch.equal((got - x.double()).abs(), best)
    amax = x.double().unflatten(-1, (-1, 32)).abs().amax(-1)
    unit = unit[:, ::32]
    assert (amax <= 7 * unit).all() and (amax > 3.5 * unit).all()
    assert torch.equal(paged.unpack(paged.pack(codes)), codes)
    ties = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7] * 4])
    assert paged.value(*paged.hold(ties))[0, :8].tolist() == [0, 1, 1, 2, 2, 4, 4, 6]
    assert paged.hold(torch.tensor([[math.nan] + [1.0] * 31]))[1].item() == 255
    assert paged.hold(torch.zeros(1, 32))[1].item() == 2 and paged.hold(torch.zeros(1, 32).half())[1].item() == 104
    assert paged.hold(torch.full((1, 32), 65504.0).half())[1].item() == 140


def test_prompt_is_attend_row_by_row():
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn(2, 9, 16, generator=gen) for _ in range(2))
    q = torch.randn(4, 6, 16, generator=gen)
    (out, lse), _ = paged.prompt(q, k, v, 4)
    for i in range(4):
        n = 9 - 4 + i + 1
        pages = [x[:, :n].permute(1, 0, 2)[:, :, None] for x in (k, v)]
        (want, _, l), _ = paged.attend(q[i:i + 1], *pages, torch.arange(n)[None], [n])[0]
        assert torch.allclose(out[i], want, atol=1e-12) and torch.allclose(lse[i], l, atol=1e-12)


def test_a_turn_keeps_lengths():
    from prismkv_amd import Rotary
    rotary = Rotary(64, rotary_dim=32, device="cpu")
    x = torch.randn(5, 2, 64, dtype=torch.float64).float()
    for interleaved in (False, True):
        y, _ = paged.turn(x, torch.tensor([0, 1, 7, 1000, 10 ** 6]), rotary.frequencies, interleaved=interleaved)
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1)) and torch.equal(y[..., 32:], x[..., 32:].double())
        assert torch.equal(y[0], x[0].double())
