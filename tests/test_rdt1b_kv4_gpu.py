"""GPU tests of the RDT-1B runtime on its 4-bit cross-attention cache
(sfb_rdt1b_set_cache) against the CPU oracle evaluated on exactly the values
that the cache holds, with the model's own bar (max |ours − oracle| < 0.05,
cosine > 0.9999: everything but the cache is the 16-bit model's)."""
import ctypes

import pytest
import torch

from oracle import rdt1b_ref
from servoflow_b200 import _capi
from servoflow_b200.rdt1b import RDT1B, default_config

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def setup(gpu):
    cfg = default_config(num_layers=2, max_lang_len=50, img_len=261, max_sessions=2)
    model = RDT1B(cfg, seed=99)
    g = torch.Generator().manual_seed(43)
    lang = torch.randn(2, cfg.max_lang_len, cfg.lang_dim, generator=g).bfloat16().to(gpu)
    img = torch.randn(2, cfg.img_len, cfg.img_dim, generator=g).bfloat16().to(gpu)
    state = torch.randn(2, cfg.state_dim, generator=g).bfloat16().to(gpu)
    lens = torch.tensor([37, 50], dtype=torch.int32, device=gpu)
    noise = torch.randn(2, cfg.horizon, cfg.action_dim, generator=g).to(gpu)
    ref = rdt1b_ref.RefRDT(rdt1b_ref.load_weights(model, cfg), cfg)
    yield dict(cfg=cfg, model=model, ref=ref, lang=lang, img=img, state=state, lens=lens, noise=noise)
    model.close()


def encode(s, n=2):
    s["model"].encode(s["lang"][:n], s["lens"][:n], s["img"][:n], s["state"][:n])


def held(s):
    """The caches' values as the oracle's kv list."""
    out = []
    for l in range(s["cfg"].num_layers):
        n = s["cfg"].max_lang_len if l % 2 == 0 else s["cfg"].img_len
        k, v = (x[:, :, :n].transpose(1, 2).reshape(2, n, -1).float().cpu() for x in s["model"].kv4_cache(l).dequantize())
        if l % 2 == 0:                                 # slots past a session's length are never written
            for b, n in enumerate(s["lens"].tolist()):
                k[b, n:] = 0
                v[b, n:] = 0
        out.append((k, v))
    return out


def close(ours, ref):
    a, b = ours.float().cpu().reshape(-1).double(), ref.float().reshape(-1).double()
    return (a - b).abs().max().item(), torch.nn.functional.cosine_similarity(a[None], b[None]).item()


def test_network_and_sampling_match_the_oracle_on_the_held_values(setup):
    s, m = setup, setup["model"]
    m.set_cache(4)
    encode(s)
    kv = held(s)
    x = torch.empty_like(s["noise"])
    m.forward(s["noise"], 999.0, x)
    lens, state, noise = s["lens"].cpu(), s["state"].float().cpu(), s["noise"].cpu()
    max_abs, cos = close(x, s["ref"].forward(None, None, lens, state, noise, 999, kv))
    assert max_abs < 0.05 and cos > 0.9999, (max_abs, cos)
    eager, first, replay = (torch.empty_like(s["noise"]) for _ in range(3))
    m.sample(s["noise"], eager, use_graph=False)
    m.sample(s["noise"], first)
    m.sample(s["noise"], replay)
    assert torch.equal(eager, first) and torch.equal(first, replay)
    max_abs, cos = close(replay, s["ref"].sample(None, None, lens, state, noise, kv))
    assert max_abs < 0.05 and cos > 0.9999, (max_abs, cos)


def test_cache_holds_the_conditions_to_half_a_step(setup):
    s, m = setup, setup["model"]
    m.set_cache(4)
    encode(s)
    lang_c, img_c = s["ref"].encode(s["lang"].float().cpu(), s["img"].float().cpu())
    for l, (want_k, want_v) in enumerate(s["ref"].cross_kv_all(lang_c, img_c)):
        cache = m.kv4_cache(l)
        for val, scale, want in zip(cache.dequantize(), (cache.k_scale, cache.v_scale), (want_k, want_v)):
            n = want.shape[1]
            for b in range(2):
                rows = int(s["lens"][b]) if l % 2 == 0 else n
                got = val[b, :, :rows].transpose(0, 1).reshape(rows, -1).cpu()
                step = scale[b, :, :rows].float().repeat_interleave(32, -1).transpose(0, 1).reshape(rows, -1).cpu()
                ref = want[b, :rows]
                # half a step; 0.03 of the largest step's range (7 steps) for the bf16
                # activations, weights' products and norms before the quantisation
                # (a dozen roundings of 2^-9 along the path, the model's bar elsewhere)
                assert ((got - ref).abs() <= 0.5 * step + 0.03 * 7 * step + 0.03).all()


def test_sessions_and_paths(setup):
    s, m = setup, setup["model"]
    m.set_cache(4)
    encode(s)
    both, one = torch.empty_like(s["noise"]), torch.empty_like(s["noise"][:1])
    m.forward(s["noise"], 599.0, both)
    encode(s, 1)
    outs = []
    for path in (0, 1, 2):                             # one session takes the same kernels on every path
        m.set_path(path)
        m.forward(s["noise"][:1], 599.0, one)
        outs.append(one.clone())
    m.set_path(1)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    max_abs, cos = close(outs[0], both[:1].cpu())      # other tile shapes, same values
    assert max_abs < 0.05 and cos > 0.9999, (max_abs, cos)


def test_back_to_16_bits_gives_the_same_bits(setup):
    s, m = setup, setup["model"]
    m.set_cache(16)
    encode(s)
    a, b = torch.empty_like(s["noise"]), torch.empty_like(s["noise"])
    m.sample(s["noise"], a)
    m.set_cache(4)
    encode(s)
    m.sample(s["noise"], b)
    assert not torch.equal(a, b)
    m.set_cache(16)
    encode(s)
    m.sample(s["noise"], b)
    assert torch.equal(a, b)


def test_other_forms_conditions_are_refused(setup):
    s, m = setup, setup["model"]
    x = torch.empty_like(s["noise"])
    m.set_cache(16)
    encode(s)
    m.forward(s["noise"], 1.0, x)
    for bits in (4, 16):
        m.set_cache(bits)
        if bits == 16:
            m.set_cache(4); encode(s); m.set_cache(16)
        with pytest.raises(_capi.SfbError):
            m.forward(s["noise"], 1.0, x)
        with pytest.raises(_capi.SfbError):
            m.sample(s["noise"], x)
        encode(s)
        m.forward(s["noise"], 1.0, x)
    lib = m.lib
    assert lib.sfb_rdt1b_set_cache(m.h, 8) == _capi.SFB_ERR_INVALID
    assert lib.sfb_rdt1b_set_cache(None, 4) == _capi.SFB_ERR_INVALID
    buf = ctypes.create_string_buffer(_capi.KV4_CACHE.size)
    assert lib.sfb_rdt1b_kv4_cache(m.h, 2, buf) == _capi.SFB_ERR_SHAPE
    assert lib.sfb_rdt1b_kv4_cache(m.h, 0, None) == _capi.SFB_ERR_INVALID


def test_tick_re_encodes_after_the_change(setup):
    s, m = setup, setup["model"]
    m.set_cache(16)
    out = [torch.empty_like(s["noise"]) for _ in range(3)]
    kw = dict(lang=s["lang"], lang_len=s["lens"], img=s["img"])
    m.tick(5, s["state"], s["noise"], out[0], **kw)
    _, e0 = m.tick_stats()
    m.set_cache(4)
    m.tick(5, s["state"], s["noise"], out[1], **kw)    # the same frame, the other cache
    m.tick(5, s["state"], s["noise"], out[2])
    _, e1 = m.tick_stats()
    torch.cuda.synchronize()
    assert e1 == e0 + 1 and torch.equal(out[1], out[2]) and not torch.equal(out[0], out[1])


def test_a_change_and_back_without_an_encode_is_refused(setup):
    """What the caches hold after a change of form is not vouched for until an encode."""
    s, m = setup, setup["model"]
    x = torch.empty_like(s["noise"])
    for form, other in ((16, 4), (4, 16)):
        m.set_cache(form)
        encode(s)
        m.sample(s["noise"], x)                        # (captures the graph)
        m.set_cache(other)
        m.set_cache(form)
        with pytest.raises(_capi.SfbError):
            m.forward(s["noise"], 1.0, x)
        for graph in (True, False):
            with pytest.raises(_capi.SfbError):
                m.sample(s["noise"], x, use_graph=graph)
        encode(s)
        m.forward(s["noise"], 1.0, x)
        m.set_cache(form)                              # no change: nothing to encode again
        m.forward(s["noise"], 1.0, x)


def test_a_change_that_finds_no_memory_keeps_none(gpu):
    """The 4-bit caches are allocated all or not at all, and the handle stays as it was."""
    cfg = default_config(num_layers=2, max_lang_len=64, img_len=4374, max_sessions=8)
    model, ballast = RDT1B(cfg, seed=5), None
    try:
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        # of 81 MB for the image block (36 + 36 for its codes) 48 MB are there
        ballast = torch.empty(torch.cuda.mem_get_info()[0] - (48 << 20), dtype=torch.uint8, device=gpu)
        before = torch.cuda.mem_get_info()[0]
        for _ in range(3):
            with pytest.raises(_capi.SfbError):
                model.set_cache(4)
            # (more where the driver gives back a slab that was partly in use)
            assert torch.cuda.mem_get_info()[0] >= before
        ballast = None
        torch.cuda.empty_cache()
        model.set_cache(4)
        assert model.kv4_cache(1).shape == (8, 32, 4384, 64)
    finally:
        del ballast
        model.close()
        torch.cuda.empty_cache()
