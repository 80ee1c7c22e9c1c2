"""CPU oracle of the self-speculative decode round.  TEST INFRASTRUCTURE -- NOT PART OF THE PRODUCT.

Only ``tests/``, ``__graft_entry__.smoke()`` and ``bench.py``'s CPU-baseline leg (``cpu_baseline`` and
``--impl reference``) may import this package, and only as the checker or as the timed CPU port of the reference
path.  ``gravityocr_b200`` never imports it; the product raises when its CUDA library is missing.

Modules:
  * ``decoder_ref``: torch fp32 CPU restatement of the GLM-OCR decoder, the reference's natcache round, the served
    full-draft round, AR greedy and teacher forcing.
  * ``commit_ref``: numpy restatement of the linear-chain accept, the reference's Triton commit kernel and the host
    commit rules.
  * ``kv8_ref``: the 8-bit K/V cache's rows (quantising, reading back) and the attention over them in 64 bits.

Pins: ``tests/golden/`` holds vectors generated by running the reference itself (natcache + teacher forcing through
transformers' GLM-OCR, the Triton commit kernel under the Triton CPU interpreter, the commit-rules module), by the
committed script ``tests/golden/make_golden.py``.
"""
