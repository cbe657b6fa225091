"""AutoregressiveTransformer.predict_many (a batch of utterances decoding out of paged caches) against predict one utterance at a time:
same number of steps, the same mel and attention maps up to the summation order of the split-bf16 products (the two run different
launch shapes; 2e-4 on mels of order 1, as between the cached and the full decoder in test_gpu_autoregressive.py)."""
import numpy as np
import pytest
import torch

import estts
from estts import configs, ops, weights
from estts.autoregressive_transformer import AutoregressiveTransformer

pytestmark = pytest.mark.gpu


def cfg_of(system_type, dense=1, **kw):
    c = dict(system_type=system_type, encoder_model_dimension=64, decoder_model_dimension=64, encoder_prenet_dimension=64,
             decoder_prenet_dimension=48, encoder_num_heads=[2, 2], decoder_num_heads=[2, 2], encoder_dense_blocks=dense,
             decoder_dense_blocks=dense, encoder_feed_forward_dimension=96, decoder_feed_forward_dimension=96,
             encoder_attention_conv_filters=80, decoder_attention_conv_filters=80, ref_encoder_filters=[8, 8, 16],
             ref_encoder_gru_cell_units=32, gst_style_embed_dim=64, gst_multi_num_heads=2, gst_heads=5, speaker_embed_dim=16,
             mel_channels=80, max_r=3, postnet_conv_filters=32, postnet_conv_layers=3, vocab_size=30,
             encoder_max_position_encoding=64, decoder_max_position_encoding=256)
    c.update(kw)
    return configs.autoregressive_config(**c)


def data_of(cfg, n, seed):
    rng = np.random.default_rng(seed)
    tokens = [rng.integers(1, 30, size=int(k)).astype(np.int32) for k in rng.integers(3, 20, size=n)]
    mels = [rng.normal(size=(int(k), 80)).astype(np.float32) for k in rng.integers(40, 70, size=n)] if 'style' in cfg['system_type'] else None
    spk = [rng.normal(size=(1, 16)).astype(np.float32) for _ in range(n)] if 'speaker' in cfg['system_type'] else None
    return tokens, mels, spk


def one_by_one(model, data, max_length):
    tokens, mels, spk = data
    return [model.predict(t, None if mels is None else mels[i], None if spk is None else spk[i], max_length=max_length, encode=False, verbose=False)
            for i, t in enumerate(tokens)]


def same(a, b, tol):
    assert a['mel'].shape == b['mel'].shape
    assert (a['mel'] - b['mel']).abs().max().item() < tol
    for name in b['decoder_attention']:
        assert a['decoder_attention'][name].shape == b['decoder_attention'][name].shape
        assert (a['decoder_attention'][name] - b['decoder_attention'][name]).abs().max().item() < tol


@pytest.mark.parametrize('system_type,r,dense,n', [('speaker_text', 1, 1, 5), ('speaker_style_text', 3, 2, 4), ('style_text', 2, 0, 3), ('text', 1, 2, 1)])
def test_predict_many_matches_predict(system_type, r, dense, n):
    cfg = cfg_of(system_type, dense)
    model = AutoregressiveTransformer(weights.init_autoregressive_transformer(cfg, seed=5), cfg)
    model.set_constants(reduction_factor=r)
    data = data_of(cfg, n, 7)
    want = one_by_one(model, data, 20 * r)
    for program in (True, False):
        got = model.predict_many(data[0], data[1], data[2], max_length=20 * r, encode=False, program=program)
        assert len(got) == n
        for a, b in zip(got, want):
            same(a, b, 2e-4)


def test_utterances_that_stop_leave_and_the_others_go_on():
    """Stop classes biased so that utterances end at different steps: each has the length it has alone, whatever the group of steps
    between two looks at the stop decisions."""
    cfg = cfg_of('speaker_text', 2)
    w = weights.init_autoregressive_transformer(cfg, seed=11)
    model = AutoregressiveTransformer(w, cfg)
    model.set_constants(reduction_factor=1)
    data = data_of(cfg, 12, 3)
    free_run = one_by_one(model, data, 40)
    # a threshold on the stop logit that the utterances cross at different positions (their logits: a teacher-forced pass over what
    # they produced)
    start = torch.full((1, 1, 80), float(cfg['mel_start_value']), device='cuda')
    logits = [model.call(t[None], torch.cat([start, o['mel'][None, :-1]], 1), x[None])['stop_prob'][0].cpu().numpy()
              for t, o, x in zip(data[0], free_run, data[2])]
    margins = np.concatenate([x[4:, 2] - x[4:, :2].max(1) for x in logits])
    w2 = dict(w)
    b = np.asarray(w['decoder_postnet.stop_linear.bias'])
    w2['decoder_postnet.stop_linear.bias'] = b + np.array([0, 0, -np.quantile(margins, 0.93)], np.float32)
    model = AutoregressiveTransformer(w2, cfg)
    model.set_constants(reduction_factor=1)
    want = one_by_one(model, data, 40)
    lengths = [o['mel'].shape[0] for o in want]
    assert len(set(lengths)) >= 3                    # (at once, in the middle, never)
    for k in (1, 5, 64):
        got = model.predict_many(*data, max_length=40, encode=False, stop_check_every=k)
        assert [o['mel'].shape[0] for o in got] == lengths
        for a, b in zip(got, want):
            same(a, b, 2e-4)


@pytest.mark.parametrize('dtype,tol', [(torch.bfloat16, 3e-2), (torch.float16, 4e-3)])
def test_predict_many_with_16_bit_pages(dtype, tol):
    """Keys and values rounded to half a step of the type (2^-8, 2^-11 relative) stay within a few such steps of the mel."""
    cfg = cfg_of('text', 2)
    model = AutoregressiveTransformer(weights.init_autoregressive_transformer(cfg, seed=2), cfg)
    model.set_constants(reduction_factor=1)
    data = data_of(cfg, 4, 9)
    want = model.predict_many(data[0], max_length=24, encode=False)
    got = model.predict_many(data[0], max_length=24, encode=False, cache_dtype=dtype)
    for a, b in zip(got, want):
        assert a['mel'].shape == b['mel'].shape and (a['mel'] - b['mel']).abs().max().item() < tol


def test_predict_many_at_the_shipped_width():
    """Width 256, 4 heads of 64, 70 utterances, positions past the second page, against a teacher-forced pass over what each utterance
    produced: the frames that come back are decoded from the same frames there, so that the difference is the rounding of two
    passes (3e-4 each against float64, see test_gpu_autoregressive.py).  Against predict() it is not: the loop feeds a rounding back, and
    with random weights of this width 38 steps turn 2e-5 of the first frame into 1e-3."""
    cfg = cfg_of('text', 2, encoder_model_dimension=64, decoder_model_dimension=256, decoder_num_heads=[4, 4], decoder_prenet_dimension=256,
                 decoder_feed_forward_dimension=512)
    model = AutoregressiveTransformer(weights.init_autoregressive_transformer(cfg, seed=4), cfg)
    model.set_constants(reduction_factor=1)
    data = data_of(cfg, 70, 1)
    got = model.predict_many(data[0], max_length=37, encode=False)
    start = torch.full((1, 1, 80), float(cfg['mel_start_value']), device='cuda')
    for m in range(70):
        forced = model.call(data[0][m][None], torch.cat([start, got[m]['mel'][None, :-1]], 1), None)
        assert (forced['final_output'][0] - got[m]['mel']).abs().max().item() < 6e-4
        for name, a in got[m]['decoder_attention'].items():
            assert (forced['decoder_attention'][name] - a).abs().max().item() < 2e-3


def test_predict_many_refuses():
    cfg = cfg_of('speaker_text')
    w = weights.init_autoregressive_transformer(cfg, seed=5)
    model = AutoregressiveTransformer(w, cfg)
    model.set_constants(reduction_factor=1)
    assert model.predict_many([]) == []
    with pytest.raises(ValueError, match='spk_embeds'):
        model.predict_many([[1, 2], [3]], None, [np.zeros((1, 16))], encode=False)
    with pytest.raises(ValueError, match='max_length'):
        model.predict_many([[1, 2]], None, [np.zeros((1, 16))], max_length=300, encode=False)
    silent = dict(cfg, mel_start_value=0.0)
    with pytest.raises(ValueError, match='start vector'):
        AutoregressiveTransformer(w, silent).predict_many([[1, 2]], None, [np.zeros((1, 16))], encode=False)
    odd = cfg_of('text', decoder_num_heads=[4, 4])
    with pytest.raises(ValueError, match='depth'):
        AutoregressiveTransformer(weights.init_autoregressive_transformer(odd, seed=5), odd).predict_many([[1, 2]], encode=False)
