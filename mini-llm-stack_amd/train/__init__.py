"""FP8 and INT8 linear training callers of the gfx950 GEMMs.

This package provides ``train.fp8`` and ``train.int8``. Its search path is extended over every
``train`` directory on ``sys.path`` (pkgutil.extend_path), so a reference checkout
placed after this directory still supplies the model, config, training loop and
parallel modules, which then bind this ``train.fp8``.
"""

import pkgutil

__path__ = pkgutil.extend_path(__path__, __name__)
