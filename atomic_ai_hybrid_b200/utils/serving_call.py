"""The serving call that this thread is in (``serving.serving(...)``), for the layers and the diagnostics: a module of
its own, as they may not import ``serving``, which imports them."""
from __future__ import annotations

import contextvars

# a context variable: forwards in other threads are ordinary ones meanwhile
_CALL: contextvars.ContextVar = contextvars.ContextVar("serving_call", default=None)

get_serving = _CALL.get  # the running call, or None
enter, leave = _CALL.set, _CALL.reset
