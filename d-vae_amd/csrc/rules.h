// Token rules on logits: shared pieces of rules.hip and predict.hip.
#pragma once
#include "common.h"

// argument checks of a rules descriptor (DVAE_OK or an error with its text)
int rules_check(const dvae_rules& r, const char* who);
