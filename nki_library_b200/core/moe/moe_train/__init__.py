from .expert_linear import expert_linear  # noqa: F401
from .experts_train import moe_expert_mlp, moe_experts_train  # noqa: F401
from .moe_glu import moe_glu  # noqa: F401
from .sort_tokens import SortedTokens, moe_sort_plan, moe_sort_tokens, moe_unsort_tokens  # noqa: F401
